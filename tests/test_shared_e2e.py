"""The shared-prefix operators together: caches, and generation with drafts."""
import pytest
import torch

from rotatek_b200.cache import SharedPrefixCache, SpanKVCache
from rotatek_b200.llama_e2e import DecoderConfig


def _prefix(P=2, device="cpu", dtype=torch.float32, layers=1, sp=6, sv=20, h=2, d=128, keep=32):
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g).to(device, dtype)  # noqa: E731
    c = SpanKVCache(max_new_tokens=0)
    for i in range(layers):
        c.store_pruned(r(P, h, sv, keep), r(P, h, sp, d), r(P, h, 0, d), r(P, h, sp + sv, d), r(P, h, d, keep),
                       r(P, h, d), i)
    return c


def test_cache_refusals_and_lengths():
    with pytest.raises(ValueError, match="no layers"):
        SharedPrefixCache(SpanKVCache(0), 2, 8)
    with pytest.raises(ValueError, match="must be positive"):
        SharedPrefixCache(_prefix(), 0, 8)
    c = SharedPrefixCache(_prefix(layers=2), 3, 8)
    assert c.batch == 6 and len(c.text) == 2 and c.text[0][0].shape == (6, 2, 8, 128)
    assert c.text[0][0].dtype == torch.uint8 and c.text[0][2].shape == (6, 2, 8)
    c.advance(torch.tensor([5, 1, 2, 3, 4, 0], dtype=torch.int32), 5)
    assert c.lens.tolist() == [5, 1, 2, 3, 4, 0] and c.reach == 5
    with pytest.raises(ValueError, match="full: 5 \\+ 4 tokens > capacity 8"):
        c.append(torch.zeros(6, 2, 4, 128), torch.zeros(6, 2, 4, 128), 0)
    with pytest.raises(ValueError, match="full"):
        c.advance(torch.ones(6, dtype=torch.int32), 4)
    c.lens.fill_(2)
    c.settle()
    assert c.reach == 2


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [True, False])
def test_cache_append_attend_read(fp8):
    from oracle import shared as osh
    c = SharedPrefixCache(_prefix(device="cuda", dtype=torch.bfloat16), 2, 12, fp8=fp8)
    g = torch.Generator(device="cuda").manual_seed(1)
    kv = [torch.randn(4, 2, 5, 128, generator=g, device="cuda").to(torch.bfloat16) for _ in range(4)]
    counts = torch.tensor([5, 3, 1, 4], dtype=torch.int32, device="cuda")
    c.append(kv[0], kv[1], 0, counts=counts)
    c.advance(counts, 5)
    c.append(kv[2], kv[3], 0)
    q = torch.randn(4, 5, 8, 128, generator=g, device="cuda").to(torch.bfloat16)
    lens = c.lens + 5
    got = c.attend(q, 0, lens, 4)
    k, v, ks, vs = c.text[0]
    a = c.prefix.decode_args(0)
    want, mag = osh.shared_decode(q, a["R_partial"], a["delta_mu"], a["k_full"], a["v_full"], None, a["k_sparse"],
                                  a["v_sparse"], k, v, lens, 4, ks, vs)
    # the tolerance of tests/test_shared_gpu.py; logits here reach ~80 (unscaled random R): 2^-16 of them
    tol = 2.0 ** -9 * want.abs() + (2.0 ** -8 + 2.0 ** -8) * mag
    assert ((got.cpu().double() - want).abs() <= tol).all()
    c.advance(torch.full((4,), 5, dtype=torch.int32, device="cuda"), 5)
    rk, rv = c.read(0)
    for b, n in enumerate(counts.tolist()):
        for out, first, then in ((rk, kv[0], kv[2]), (rv, kv[1], kv[3])):
            whole = torch.cat([first[b, :, :n], then[b]], 1).float()
            if fp8:
                val, scale = osh.quantize_rows(whole)
                whole = (val.float() * scale[..., None]).to("cuda")
            assert torch.equal(out[b, :, :n + 5].float(), whole.to(torch.bfloat16).float())
            assert (out[b, :, n + 5:] == 0).all()


def _small(images=2, layers=3):
    from rotatek_b200.llama_e2e import RandomLlamaDecoder
    cfg = DecoderConfig(layers=layers, hidden=256, heads=4, kv_heads=2, ffn=512, vocab=300, prompt=5, vision=70, text=3,
                        max_new_tokens=0, dtype=torch.float32, fused_key_projection=False)
    model = RandomLlamaDecoder(cfg, "cuda", seed=3)
    model.prefill(model.prompt_embeddings(images))
    return model


@pytest.mark.gpu
@pytest.mark.parametrize("draft_layers,drafts", [(2, 3), (1, 1), (3, 4), (0, 3)])
@pytest.mark.parametrize("fp8", [True, False])
def test_drafted_greedy_answers_are_the_undrafted_ones(draft_layers, drafts, fp8):
    """Greedy generation with drafts gives what one token at a time gives (fp32, so
    that no argmax hangs on a rounding), and drafts from all layers are all accepted."""
    from rotatek_b200.shared_e2e import ServingConfig, SharedQuestions
    model = _small()
    counts = torch.tensor([4, 7, 1, 6, 3, 5], dtype=torch.int32, device="cuda")
    asked = torch.randint(0, 300, (6, 7), generator=torch.Generator().manual_seed(5)).cuda()

    def generate(n_layers, t, steps):
        s = SharedQuestions(model, ServingConfig(questions=3, capacity=80, drafts=t, draft_layers=n_layers, fp8=fp8))
        s.ask(asked, counts)
        taken = [s.step()[1] for _ in range(steps)]
        return s.answers(), torch.stack(taken)

    plain, _ = generate(1, 0, 14)
    fast, taken = generate(draft_layers, drafts, 8)
    for a, b in zip(plain, fast):
        n = min(len(a), len(b))
        assert n >= 9 and a[:n] == b[:n]
    if draft_layers == 3:
        assert (taken == drafts).all()


@pytest.mark.gpu
def test_sampled_answers_run_and_stay_in_the_vocabulary():
    from rotatek_b200.shared_e2e import ServingConfig, SharedQuestions
    s = SharedQuestions(_small(1), ServingConfig(questions=4, capacity=60, drafts=2, draft_layers=2, temperature=0.8))
    s.ask(torch.randint(0, 300, (4, 6), device="cuda"), torch.tensor([6, 1, 3, 2], dtype=torch.int32, device="cuda"))
    for _ in range(5):
        tokens, accepted = s.step()
        place = torch.arange(3, device="cuda")
        assert ((tokens >= 0) == (place <= accepted[:, None])).all() and (tokens < 300).all()
    assert all(6 <= len(a) <= 16 for a in s.answers())


def test_a_full_cache_is_refused_before_anything_runs():
    """Neither a step nor a question indexes the RoPE tables or drafts past the capacity."""
    from types import SimpleNamespace

    from rotatek_b200.shared_e2e import ServingConfig, SharedQuestions

    class Untouched:
        cfg = SimpleNamespace(layers=1)

    def never(*args, **kwargs):
        raise AssertionError("ran")

    s = SharedQuestions.__new__(SharedQuestions)
    s.cache, s.model, s.batch = SharedPrefixCache(_prefix(), 3, 8), Untouched(), 6
    s.cfg = ServingConfig(questions=3, capacity=8, drafts=2, draft_layers=1)
    s.last = torch.zeros(6, dtype=torch.int64)
    s.cache.reach = 7
    with pytest.raises(ValueError, match="full: 7 \\+ 2 tokens > capacity 8"):
        s.forward(torch.zeros(6, 2, dtype=torch.int64), s.cache.lens, 1)
    with pytest.raises(ValueError, match="full"):
        s.forward(torch.zeros(6, 1, dtype=torch.int64), s.cache.lens + 1, 1, ahead=1)
    s.forward = never
    s.cache.reach = 6
    with pytest.raises(ValueError, match="full: 6 \\+ 3 tokens > capacity 8"):
        s.step()
    s.cache.reach = 0
    with pytest.raises(ValueError, match="full: 0 \\+ 9 tokens > capacity 8"):
        s.ask(torch.zeros(6, 9, dtype=torch.int64), torch.full((6,), 9, dtype=torch.int32))


def test_rows_ahead_of_the_lengths_need_room():
    c = SharedPrefixCache(_prefix(), 3, 8)
    c.reach = 5
    new = torch.zeros(6, 2, 2, 128)
    with pytest.raises(ValueError, match="full: 5 \\+ 4 tokens > capacity 8"):
        c.append(new, new, 0, at=c.lens + 2, ahead=2)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):       # there is room: on to the kernels
        c.append(new, new, 0, at=c.lens + 1, ahead=1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("draft_layers,drafts,temperature", [(1, 3, 0.0), (0, 5, 0.0), (3, 2, 0.9)])
def test_the_loop_on_the_tensor_cores(draft_layers, drafts, temperature, dtype, monkeypatch):
    """Every attention of questions that go in, are drafted for and checked is within the tolerance of
    tests/test_shared_gpu.py of its 64-bit value, and the emitted tokens are the verification's."""
    from rotatek_b200.llama_e2e import RandomLlamaDecoder
    from rotatek_b200.shared_e2e import ServingConfig, SharedQuestions
    from tests.test_shared_gpu import UNIT, dense

    cfg = DecoderConfig(layers=3, hidden=512, heads=8, kv_heads=2, ffn=512, vocab=400, prompt=40, vision=900, text=3,
                        max_new_tokens=0, dtype=dtype, fused_key_projection=False)
    model = RandomLlamaDecoder(cfg, "cuda", seed=4)
    model.prefill(model.prompt_embeddings(2))
    s = SharedQuestions(model, ServingConfig(questions=4, capacity=80, drafts=drafts, draft_layers=draft_layers,
                                             temperature=temperature))
    attend, seen = s.cache.attend, []

    def checked(q, layer, lens, groups):
        out = attend(q, layer, lens, groups)
        a = s.cache.prefix.decode_args(layer)
        k, v, ks, vs = s.cache.text[layer]
        args = dict(q=q, R_partial=a["R_partial"], delta_mu=a["delta_mu"], k_full=a["k_full"], v_full=a["v_full"],
                    mask_full=a["mask_full"], k_sparse=a["k_sparse"], v_sparse=a["v_sparse"], k_text=k, v_text=v,
                    text_lens=lens, num_kv_groups=groups, k_scale=ks, v_scale=vs)
        want, mag = dense(args)
        off = (out.double() - want).abs()
        assert (off <= UNIT[dtype] * want.abs() + 2.0 ** -11 * mag + 2.0 ** -25).all()
        seen.append(q.shape[1])
        return out

    monkeypatch.setattr(s.cache, "attend", checked)
    counts = torch.tensor([9, 3, 12, 1, 7, 12, 5, 2], dtype=torch.int32, device="cuda")
    s.ask(torch.randint(0, 400, (8, 12), generator=torch.Generator().manual_seed(6)).cuda(), counts)
    emitted = counts + 1
    for _ in range(5):
        tokens, accepted = s.step()
        place = torch.arange(drafts + 1, device="cuda")
        assert ((tokens >= 0) == (place <= accepted[:, None])).all() and (tokens < 400).all()
        emitted = emitted + accepted + 1
    assert torch.equal(s.cache.lens + 1, emitted)
    assert {12, drafts + 1} <= set(seen) and (draft_layers == 0 or 1 in seen)
