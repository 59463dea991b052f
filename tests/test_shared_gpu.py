"""Shared-prefix attention, text caches and draft verification on a B200 against
their float64 definitions (oracle/shared.py).

Attention tolerance, for an output o with A = sum w |v| over its softmax weights:
  16-bit  u |o| + (2 u + 2^-11) A, u = half a unit in the last place (2^-9 bf16,
          2^-12 fp16): the output's rounding; each weight rounded to 16 bits once in
          the numerator (u) and once in the normaliser (u); and logits off by up to
          2^-12 (fp32 sums of 128 products and the rotated query in two 16-bit parts),
          which moves a weight by 2^-12 in each
  fp32    2^-22 |o| + 2^-14 A: logits of size up to about 50 from fp32 sums of up to 256
          products (256 * 2^-24 * 50 / 16 < 2^-15), twice
Quantisation and reading back are exact.  Verification is exact wherever no
decision of the question is closer than 1e-4 (relative) to going the other way.
"""
import math

import pytest
import torch

from oracle import shared as osh

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF_ULP = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -12}


@pytest.fixture(scope="module", autouse=True)
def _library():
    from rotatek_b200 import _lib
    _lib.load()
    yield
    assert _lib.read_status() == 0


def make(P, N, T, hq, hk, sv, sf, cap, dk, dtype=torch.bfloat16, fp8=False, mask=None, bias=True, lens=None, D=128,
         seed=0, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    B = P * N

    def n(*s, scale=1.0):
        return (torch.randn(*s, generator=g, device=DEV) * scale).to(dtype)

    R = torch.linalg.qr(torch.randn(P, hk, D, dk, generator=g, device=DEV))[0].to(dtype)
    spread = torch.exp(-torch.arange(dk, device=DEV) / 10.0)
    spread = torch.sqrt(D * spread / spread.sum())
    a = dict(q=n(B, T, hq, D, scale=std), R_partial=R, delta_mu=n(P, hk, D, scale=0.3) if bias else None,
             k_full=n(P, hk, sf, D), v_full=n(P, hk, sf, D), mask_full=None,
             k_sparse=(torch.randn(P, hk, sv, dk, generator=g, device=DEV) * spread).to(dtype),
             v_sparse=n(P, hk, sv, D), k_text=n(B, hk, cap, D), v_text=n(B, hk, cap, D), num_kv_groups=hq // hk)
    if mask is not None:
        a["mask_full"] = (torch.rand(P, sf, generator=g, device=DEV) < mask).to(torch.uint8)
    if lens is None:
        lens = [cap - (i * max(1, cap // 3)) % (cap + 1) for i in range(B)]
    a["text_lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    if fp8:
        for side in ("k", "v"):
            val, scale = osh.quantize_rows(a[f"{side}_text"])
            a[f"{side}_text"] = val.float().to(torch.float8_e4m3fn).to(DEV).view(torch.uint8)
            a[f"{side}_scale"] = scale.to(DEV)
    return a


def check(a, **kw):
    from rotatek_b200.kernels import rotatek_shared_decode
    got = rotatek_shared_decode(**a, **kw)
    torch.cuda.synchronize()
    compare(got, a)
    return got


def compare(got, a):
    want, mag = osh.shared_decode(**a)
    got64 = got.cpu().double()
    if a["q"].dtype == torch.float32:
        tol = 2.0 ** -22 * want.abs() + 2.0 ** -14 * mag
    else:
        u = HALF_ULP[a["q"].dtype]
        tol = u * want.abs() + (2 * u + 2.0 ** -11) * mag
        if a["q"].dtype == torch.float16:
            tol = tol + 2.0 ** -25          # half a step of the subnormals
    bad = (got64 - want).abs() > tol
    assert torch.isfinite(got64).all()
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {((got64 - want).abs() / tol.clamp_min(1e-30)).max():.2f}"


SHAPES = [
    # P, N, T, H_q, H_kv, S_v, S_f, C, D_keep
    (1, 2, 1, 28, 4, 1000, 64, 64, 32),
    (1, 1, 1, 4, 4, 1, 1, 1, 16),
    (1, 1, 1, 8, 2, 127, 63, 65, 64),
    (1, 3, 2, 8, 2, 129, 65, 33, 32),
    (2, 3, 5, 28, 4, 700, 100, 130, 32),
    (1, 40, 1, 14, 2, 300, 31, 17, 64),         # 280 rows of a head: three row tiles
    (3, 2, 8, 16, 2, 257, 5, 200, 16),
    (1, 2, 3, 32, 2, 140, 70, 96, 32),          # 16 query heads per KV head, 48 rows of a question
    (1, 1, 16, 24, 2, 90, 10, 70, 32),          # 192 rows of one question
    (2, 5, 1, 4, 4, 513, 0, 40, 32),            # no prompt
    (2, 2, 2, 8, 4, 0, 77, 50, 32),             # no visual span
    (1, 4, 2, 8, 2, 200, 20, 0, 32),            # no text
    (1, 2, 4, 8, 2, 0, 0, 90, 32),              # text alone
]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype,fp8", [(torch.bfloat16, False), (torch.float16, False), (torch.bfloat16, True),
                                       (torch.float16, True)])
def test_decode_shapes(shape, dtype, fp8):
    check(make(*shape, dtype=dtype, fp8=fp8, seed=sum(shape)))


@pytest.mark.parametrize("shape,D", [((1, 2, 2, 8, 2, 50, 20, 30, 32), 128), ((2, 2, 3, 6, 2, 33, 9, 12, 24), 64),
                                     ((1, 3, 1, 4, 4, 40, 7, 9, 5), 40), ((1, 1, 2, 4, 2, 20, 4, 6, 200), 256)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fp8", [False, True])
def test_decode_any_width_and_type(shape, D, dtype, fp8):
    check(make(*shape, dtype=dtype, D=D, fp8=fp8, seed=D, mask=0.7))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("T", [1, 4])
def test_decode_lengths(T, fp8):
    """Every kind of length: none, fewer than the queries, one, tile edges, the
    capacity, past it and negative (both clamped)."""
    lens = [0, 1, 2, 3, 4, 15, 16, 17, 31, 32, 33, 63, 64, 65, 95, 96, 99, 100, 250, -3]
    check(make(1, len(lens), T, 8, 2, 150, 40, 100, 32, fp8=fp8, lens=lens, seed=5))


@pytest.mark.parametrize("mask", [0.0, 0.05, 0.8, 1.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_decode_prompt_mask(mask, dtype):
    check(make(2, 3, 2, 8, 2, 100, 333, 20, 32, dtype=dtype, mask=mask, seed=7))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fp8", [False, True])
def test_decode_rows_that_see_nothing_are_zero(dtype, fp8):
    """All prompt tokens masked, no visual span, and a length below the drafts'."""
    a = make(1, 4, 3, 8, 2, 0, 50, 20, 32, dtype=dtype, fp8=fp8, mask=0.0, lens=[0, 1, 2, 3])
    got = check(a)
    for b, n in enumerate([0, 1, 2, 3]):
        for t in range(3):
            assert (got[b, t] == 0).all().item() == (n - (2 - t) <= 0)
    none = make(1, 2, 1, 4, 2, 0, 0, 0, 16, dtype=dtype)
    assert (check(none) == 0).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fp8", [False, True])
def test_decode_ignores_what_is_not_seen(bad, dtype, fp8):
    """Masked prompt tokens and text rows past the length hold NaN / infinity in
    Keys, Values and scales: outputs are those without them, to the bit."""
    a = make(2, 3, 2, 8, 2, 140, 200, 80, 32, dtype=dtype, fp8=fp8, mask=0.7, lens=[0, 3, 17, 64, 79, 80], seed=9)
    from rotatek_b200.kernels import rotatek_shared_decode
    clean = rotatek_shared_decode(**a)
    hidden = (a["mask_full"] == 0)[:, None, :, None]
    past = (torch.arange(80, device=DEV) >= a["text_lens"][:, None])[:, None, :, None]
    for name in ("k_full", "v_full"):
        a[name] = torch.where(hidden, torch.tensor(bad, device=DEV, dtype=dtype), a[name])
    for name in ("k_text", "v_text"):
        fill = torch.tensor(0x7F, device=DEV, dtype=torch.uint8) if fp8 else torch.tensor(bad, device=DEV, dtype=dtype)
        a[name] = torch.where(past, fill, a[name])
    if fp8:
        for name in ("k_scale", "v_scale"):
            a[name] = torch.where(past[..., 0], torch.tensor(bad, device=DEV), a[name])
    dirty = check(a)
    assert torch.equal(clean, dirty)


def test_decode_extreme_logits():
    """Logits of hundreds, of both signs: one token takes all the weight."""
    for dtype in (torch.bfloat16, torch.float16):
        a = make(1, 2, 2, 8, 2, 300, 70, 90, 32, dtype=dtype, std=1.0, seed=3)
        a["q"] = a["q"] * 16
        a["k_full"] = a["k_full"] * 4
        from rotatek_b200.kernels import rotatek_shared_decode
        got = rotatek_shared_decode(**a).cpu().double()
        want, mag = osh.shared_decode(**a)
        # logits reach ~700 with 2^-16 relative error from the rotated query's two parts:
        # weights move by up to 2 * 700 * 2^-16 log2(e)
        tol = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -5) * mag
        assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("fp8", [False, True])
def test_decode_text_scales_of_any_size(fp8):
    """Value rows whose sizes differ by 2^40 within a question (and rows of zeros)."""
    a = make(1, 2, 2, 8, 2, 64, 10, 150, 32, dtype=torch.bfloat16, lens=[150, 131], seed=11)
    size = torch.exp2(torch.randint(-30, 11, (2, 2, 150, 1), device=DEV).float())
    size[:, :, 7] = 0
    a["v_text"] = (a["v_text"].float() * size).to(torch.bfloat16)
    if fp8:
        for side in ("k", "v"):
            val, scale = osh.quantize_rows(a[f"{side}_text"])
            a[f"{side}_text"] = val.float().to(torch.float8_e4m3fn).to(DEV).view(torch.uint8)
            a[f"{side}_scale"] = scale.to(DEV)
    check(a)


def test_decode_strided_and_unaligned_views():
    a = make(2, 2, 3, 8, 2, 150, 60, 40, 32, seed=13)
    qkv = torch.randn(4, 3, 12, 128, device=DEV).to(torch.bfloat16)
    check({**a, "q": qkv[:, :, :8]})                                        # fused projection slice
    wide = torch.randn(4, 3, 8, 130, device=DEV).to(torch.bfloat16)
    check({**a, "q": wide[..., 1:129]})                                     # 2-byte aligned queries
    cache = torch.randn(2, 2, 300, 128, device=DEV).to(torch.bfloat16)
    check({**a, "v_sparse": cache[:, :, 60:210], "v_full": cache[:, :, :60]})
    bshd = torch.randn(4, 40, 2, 128, device=DEV).to(torch.bfloat16)
    check({**a, "k_text": bshd.transpose(1, 2)})                            # tokens before heads
    odd = torch.randn(4, 2, 40, 129, device=DEV).to(torch.bfloat16)
    check({**a, "v_text": odd[..., 1:]})                                    # rows no 16-byte copy can take
    oddk = torch.randn(2, 2, 150, 33, device=DEV).to(torch.bfloat16)
    check({**a, "k_sparse": oddk[..., :32]})
    one = a["k_full"][:1].expand(2, -1, -1, -1)                             # both prefixes are one tensor
    check({**a, "k_full": one})
    lens = torch.tensor([40, 0, 9, 0, 33, 0, 2, 0], dtype=torch.int32, device=DEV)
    check({**a, "text_lens": lens[::2]})
    mask = (torch.rand(60, 2, device=DEV) < 0.6).to(torch.uint8)
    check({**a, "mask_full": mask.t()})


def test_decode_into_a_given_tensor():
    a = make(1, 3, 2, 8, 2, 100, 30, 20, 32, seed=15)
    from rotatek_b200.kernels import rotatek_shared_decode
    buf = torch.zeros(3, 8, 2, 128, device=DEV, dtype=torch.bfloat16)
    got = check(a, out=buf.transpose(1, 2))
    assert got.data_ptr() == buf.data_ptr()
    odd = torch.zeros(3, 2, 8, 131, device=DEV, dtype=torch.bfloat16)
    compare(rotatek_shared_decode(**a, out=odd[..., 1:129]), a)
    assert (odd[..., 0] == 0).all() and (odd[..., 129:] == 0).all()


def test_decode_is_the_same_each_time_and_on_other_streams():
    from rotatek_b200.kernels import rotatek_shared_decode
    a = make(2, 9, 2, 28, 4, 2000, 100, 150, 32, fp8=True, seed=17)
    b = make(1, 5, 1, 28, 4, 1500, 64, 90, 32, seed=18)
    first, other = rotatek_shared_decode(**a), rotatek_shared_decode(**b)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for i in range(10):
        for s, args in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                outs.append(rotatek_shared_decode(**args))
    torch.cuda.synchronize()
    for i in range(0, 20, 2):
        assert torch.equal(outs[i], first) and torch.equal(outs[i + 1], other)


def test_decode_captured_and_replayed_while_lengths_grow():
    from rotatek_b200.kernels import rotatek_shared_decode
    a = make(1, 4, 1, 8, 2, 500, 30, 64, 32, fp8=True, lens=[1, 2, 3, 4], seed=19)
    rotatek_shared_decode(**a)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = rotatek_shared_decode(**a)
    for step in (0, 1, 30, 60):
        a["text_lens"].copy_(torch.tensor([1, 2, 3, 4]) + step)
        g.replay()
        torch.cuda.synchronize()
        compare(out, a)


def test_decode_equals_the_decode_of_each_question_alone():
    """A question's attention does not depend on who shares its prefix, and is the
    framework's rotatek_decode of its own copy of everything."""
    from rotatek_b200.kernels import rotatek_decode, rotatek_shared_decode
    a = make(1, 3, 1, 28, 4, 600, 40, 24, 32, lens=[24, 10, 1], seed=21)
    got = rotatek_shared_decode(**a)
    for b, n in enumerate([24, 10, 1]):
        ref, _, _ = rotatek_decode(
            a["q"][b:b + 1, 0], a["R_partial"], a["delta_mu"],
            torch.cat([a["k_full"], a["k_text"][b:b + 1, :, :n]], 2),
            torch.cat([a["v_full"], a["v_text"][b:b + 1, :, :n]], 2), None, a["k_sparse"], a["v_sparse"], 7)
        # each is within its tolerance of the same float64 value
        assert (got[b:b + 1].float() - ref.float()).abs().max() < 2.0 ** -6


# ------------------------------------------------------------------ text caches
def filled_caches(B, H, C, D, dtype, fp8, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if not fp8:
        return [torch.randn(B, H, C, D, generator=g, device=DEV).to(dtype) for _ in range(2)], [None, None]
    return ([torch.randint(0, 120, (B, H, C, D), generator=g, device=DEV, dtype=torch.uint8) for _ in range(2)],
            [torch.rand(B, H, C, generator=g, device=DEV) for _ in range(2)])


@pytest.mark.parametrize("B,H,T,C,D", [(1, 1, 1, 1, 128), (3, 4, 1, 50, 128), (2, 8, 77, 200, 128), (5, 3, 7, 9, 128),
                                       (2, 2, 5, 16, 64), (2, 3, 4, 8, 33), (40, 8, 33, 64, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("fp8", [True, False])
def test_append(B, H, T, C, D, dtype, fp8):
    """Written rows are exact, all others keep their bits; rows past the capacity
    are dropped, counts bound each question's rows."""
    from rotatek_b200.kernels import append_text
    g = torch.Generator(device=DEV).manual_seed(B * T + D)
    kv = torch.randn(B, T, 2 * H, D, generator=g, device=DEV).mul_(
        torch.exp2(torch.randint(-12, 9, (B, T, 2 * H, 1), generator=g, device=DEV).float())).to(dtype)
    kv[0, 0, 0] = 0
    new = [kv[:, :, :H].transpose(1, 2), kv[:, :, H:].transpose(1, 2)]
    for counted in (False, True):
        caches, scales = filled_caches(B, H, C, D, dtype, fp8, 3)
        lens = [(7 * i) % (C + 2) - 1 if B > 1 else 0 for i in range(B)]
        counts = [(i * 3) % (T + 1) for i in range(B)] if counted else [T] * B
        want = [c.clone() for c in caches]
        want_s = [None if s is None else s.clone() for s in scales]
        quant = [osh.quantize_rows(n) for n in new]
        for i in range(B):
            for t in range(counts[i]):
                at = lens[i] + t
                if 0 <= at < C:
                    for side in range(2):
                        if fp8:
                            want[side][i, :, at] = quant[side][0][i, :, t].float().to(torch.float8_e4m3fn).view(
                                torch.uint8).to(DEV)
                            want_s[side][i, :, at] = quant[side][1][i, :, t].to(DEV)
                        else:
                            want[side][i, :, at] = new[side][i, :, t]
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
        append_text(new[0], new[1], i32(lens), caches[0], caches[1], k_scale=scales[0], v_scale=scales[1],
                    counts=i32(counts) if counted else None)
        for side in range(2):
            assert torch.equal(caches[side], want[side])
            if fp8:
                assert torch.equal(scales[side], want_s[side])


def test_append_special_values():
    """Rows of zeros, subnormals, values at the rounding ties, infinities and NaN."""
    from rotatek_b200.kernels import append_text
    x = torch.zeros(1, 1, 8, 128, device=DEV, dtype=torch.float32)
    x[0, 0, 1] = 1e-41
    x[0, 0, 2, :5] = torch.tensor([448.0, 17.0, 19.0, 2.0 ** -10, -(2.0 ** -9) * 1.5])
    x[0, 0, 3, :3] = torch.tensor([math.inf, 3.0, -1.0])
    x[0, 0, 4, :3] = torch.tensor([math.nan, 3.0, -1.0])
    x[0, 0, 5] = -math.inf
    x[0, 0, 6] = torch.linspace(-3.3e38, 3.3e38, 128)
    x[0, 0, 7] = 2.0 ** -120 * torch.linspace(-1, 1, 128)
    for dtype in (torch.float32, torch.bfloat16):
        y = x.to(dtype)
        caches, scales = filled_caches(1, 1, 8, 128, dtype, True, 1)
        append_text(y, y, torch.zeros(1, dtype=torch.int32, device=DEV), *caches, k_scale=scales[0], v_scale=scales[1])
        val, scale = osh.quantize_rows(y)
        got = osh.e4m3_values(caches[0].cpu())
        assert torch.equal(scales[0].cpu(), scale)
        assert torch.equal(torch.isnan(got), torch.isnan(val))
        assert torch.equal(torch.nan_to_num(got, nan=0.0), torch.nan_to_num(val, nan=0.0))


@pytest.mark.parametrize("B,H,C,D", [(1, 1, 1, 128), (3, 4, 50, 128), (2, 8, 333, 128), (2, 3, 20, 64), (2, 2, 9, 33)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_read(B, H, C, D, dtype):
    from rotatek_b200.kernels import read_text
    caches, scales = filled_caches(B, H, C, D, dtype, True, 5)
    lens = torch.tensor([(C - 5 * i) if i % 3 < 2 else 0 for i in range(B)], dtype=torch.int32, device=DEV)
    past = (torch.arange(C, device=DEV) >= lens[:, None])[:, None]
    for s in scales:
        s.masked_fill_(past, math.nan)             # never read
    got = read_text(*caches, lens, k_scale=scales[0], v_scale=scales[1], dtype=dtype)
    for out, cache, scale in zip(got, caches, scales):
        want = torch.where(past[..., None], 0.0, cache.view(torch.float8_e4m3fn).float() * scale[..., None]).to(dtype)
        assert torch.equal(out, want)


def test_append_then_read_strided():
    """Caches with tokens before heads, and as views of one buffer."""
    from rotatek_b200.kernels import append_text, read_text
    g = torch.Generator(device=DEV).manual_seed(2)
    both = torch.zeros(3, 40, 2, 4, 128, device=DEV, dtype=torch.uint8)
    k8, v8 = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    sc = torch.zeros(3, 4, 2, 40, device=DEV)
    new = torch.randn(3, 4, 11, 128, generator=g, device=DEV).to(torch.bfloat16)
    lens = torch.tensor([0, 5, 29], dtype=torch.int32, device=DEV)
    append_text(new, new * 2, lens, k8, v8, k_scale=sc[:, :, 0], v_scale=sc[:, :, 1])
    k, v = read_text(k8, v8, lens + 11, k_scale=sc[:, :, 0], v_scale=sc[:, :, 1], dtype=torch.float32)
    val, scale = osh.quantize_rows(new)
    for i, n in enumerate([0, 5, 29]):
        want = (val[i].float() * scale[i][..., None]).to(DEV)
        assert torch.equal(k[i, :, n:n + 11], want)
        assert torch.equal(v[i, :, n:n + 11], want * 2)
        assert (k[i, :, :n] == 0).all() and (k[i, :, n + 11:] == 0).all()


# ------------------------------------------------------------------ verification
def make_verify(B, T, V, dtype, logits, seed, spread=2.5, near=0.7):
    g = torch.Generator(device=DEV).manual_seed(seed)
    target = torch.randn(B, T + 1, V, generator=g, device=DEV) * spread
    draft = target[:, :T] + near * torch.randn(B, T, V, generator=g, device=DEV)
    temperature = 0.5 + torch.rand(B, generator=g, device=DEV)
    temperature[::3] = 0.0
    soft = torch.softmax(draft / temperature.clamp_min(0.2)[:, None, None], -1)
    drafts = torch.where(temperature[:, None] > 0, torch.multinomial(soft.view(-1, V), 1, generator=g).view(B, T)
                         if T else torch.zeros(B, 0, dtype=torch.int64, device=DEV), draft.argmax(-1))
    lens = torch.tensor([(T - i) % (T + 1) for i in range(B)], dtype=torch.int32, device=DEV)
    return dict(target_logits=target.to(dtype), draft_tokens=drafts, draft_logits=draft.to(dtype) if logits else None,
                uniforms=torch.rand(B, T, generator=g, device=DEV),
                noise=torch.empty(B, V, device=DEV).exponential_(generator=g).clamp_min_(1e-9),
                temperature=temperature, draft_lens=lens)


def check_verify(a):
    from rotatek_b200.kernels import verify_drafts
    tokens, accepted = verify_drafts(**a)
    want_t, want_a, margin = osh.verify(a["target_logits"], a["draft_tokens"], a["draft_logits"], a["uniforms"],
                                        a["noise"], a["temperature"], a.get("draft_lens"))
    sure = margin > 1e-4
    assert sure.float().mean() > 0.9
    assert torch.equal(tokens.cpu()[sure], want_t[sure]) and torch.equal(accepted.cpu()[sure], want_a[sure])
    return tokens, accepted


@pytest.mark.parametrize("B,T,V", [(1, 1, 7), (2, 0, 100), (7, 3, 1000), (33, 5, 4097), (4, 8, 32000), (3, 64, 513),
                                   (2, 2, 131071), (5, 4, 8192), (3, 2, 1)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("logits", [True, False])
def test_verify(B, T, V, dtype, logits):
    check_verify(make_verify(B, T, V, dtype, logits, seed=B + T + V))


def test_verify_without_lengths_and_strided():
    a = make_verify(6, 4, 3001, torch.bfloat16, True, 1)
    del a["draft_lens"]
    check_verify(a)
    wide = torch.randn(6, 5, 3100, device=DEV).to(torch.bfloat16)
    wide[:, :, 50:3051] = a["target_logits"]
    check_verify({**a, "target_logits": wide[:, :, 50:3051], "uniforms": a["uniforms"].t().contiguous().t()})


def test_verify_masked_and_tied_logits():
    """-inf logits (tokens that may not follow), whole rows of them, equal logits."""
    from rotatek_b200.kernels import verify_drafts
    a = make_verify(9, 3, 700, torch.float16, True, 4)
    ban = torch.rand(9, 4, 700, device=DEV) < 0.9
    a["target_logits"] = a["target_logits"].masked_fill(ban, -math.inf)
    check_verify(a)
    a["target_logits"] = torch.zeros_like(a["target_logits"])            # ties: the lowest index
    a["temperature"] = torch.zeros_like(a["temperature"])
    tokens, accepted = check_verify(a)
    assert set(tokens[torch.arange(9), accepted.long()].tolist()) == {0}
    a["noise"] = torch.ones_like(a["noise"])
    a["temperature"] = torch.ones_like(a["temperature"])
    a["draft_lens"] = torch.zeros_like(a["draft_lens"])
    tokens, accepted = verify_drafts(**a)                                 # a race with equal runners
    assert (tokens[:, 0] == 0).all() and (tokens[:, 1:] == -1).all() and (accepted == 0).all()
    a["target_logits"] = torch.full_like(a["target_logits"], -math.inf)   # nothing may follow
    tokens, accepted = verify_drafts(**a)
    assert (tokens[:, 0] == 0).all() and (accepted == 0).all()


def test_verify_equal_models_accept_all_and_bad_ids_are_rejected():
    from rotatek_b200.kernels import verify_drafts
    a = make_verify(8, 4, 2000, torch.float32, True, 6)
    a["draft_logits"] = a["target_logits"][:, :4].contiguous()
    a["temperature"] = torch.full_like(a["temperature"], 0.8)
    del a["draft_lens"]
    _, accepted = verify_drafts(**a)
    assert (accepted == 4).all()
    # rejected where nothing is left of the difference: the target's own race
    a["draft_tokens"][:, 1] = -1
    a["draft_tokens"][1, 1] = 2000
    tokens, accepted = verify_drafts(**a)
    assert (accepted == 1).all()
    p = torch.softmax(a["target_logits"][:, 1].double() / 0.8, -1) / a["noise"].double()
    assert torch.equal(tokens[:, 1], p.argmax(-1)) and (tokens[:, 2:] == -1).all()


def test_verify_draws_the_targets_distribution():
    """Over many questions the first token follows p, whatever the draft model is:
    each of 6 tokens within 5 standard deviations."""
    from rotatek_b200.kernels import verify_drafts
    B, V = 60000, 6
    g = torch.Generator(device=DEV).manual_seed(8)
    tl, dl = torch.randn(V, generator=g, device=DEV), torch.randn(V, generator=g, device=DEV)
    drafts = torch.multinomial(torch.softmax(dl, 0), B, replacement=True, generator=g)[:, None]
    tokens, accepted = verify_drafts(
        torch.stack([tl, tl]).expand(B, 2, V), drafts, dl.expand(B, 1, V), torch.rand(B, 1, generator=g, device=DEV),
        torch.empty(B, V, device=DEV).exponential_(generator=g), torch.ones(B, device=DEV))
    p = torch.softmax(tl.double(), 0).cpu()
    freq = torch.bincount(tokens[:, 0].cpu(), minlength=V).double() / B
    assert ((freq - p).abs() < 5 * torch.sqrt(p * (1 - p) / B)).all()
    assert 0.05 < accepted.float().mean() < 0.999


def test_verify_captured():
    from rotatek_b200.kernels import verify_drafts
    a = make_verify(4, 3, 5000, torch.bfloat16, True, 10)
    want = verify_drafts(**a)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = verify_drafts(**a)
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("up", [True, False])
def test_decode_maximum_that_keeps_moving(dtype, up):
    """Logits that climb (or fall) by hundreds along the prefix, in every block anew, for
    more than one tile of rows: the accumulators are rescaled again and again."""
    a = make(1, 40, 1, 14, 2, 2000, 200, 30, 32, dtype=dtype, seed=23, bias=False)
    ramp = torch.linspace(-1, 1, 2000, device=DEV) * (1 if up else -1)
    row = torch.zeros(32, device=DEV)
    row[0] = 1.0
    direction = a["R_partial"][0, :, :, 0].float()                       # q . R column 0 = 20 for every query
    q = a["q"].float() * 0.05
    q = q + 20.0 * direction.repeat_interleave(7, 0)
    a["q"] = q.to(dtype)
    a["k_sparse"] = (a["k_sparse"].float() * 0.05 + 60.0 * ramp[:, None] * row).to(dtype)
    a["k_full"] = (a["k_full"].float() * 0.1).to(dtype)
    from rotatek_b200.kernels import rotatek_shared_decode
    got = rotatek_shared_decode(**a).cpu().double()
    want, mag = osh.shared_decode(**a)
    # logits reach 106 with the rotated query in two 16-bit parts (2^-16): weights move by
    # up to 2 * 106 * 2^-16 * log2(e) < 2^-7.7
    u = HALF_ULP[dtype]
    assert ((got - want).abs() <= u * want.abs() + (2 * u + 2.0 ** -7) * mag + 2.0 ** -25).all()


def test_decode_many_units_and_short_ranges():
    """Grids where a CTA's share is a block, less than a block's weight apart, or several
    units; more units than SMs."""
    for shape in [(3, 1, 1, 8, 8, 1, 1, 2, 16), (40, 1, 1, 8, 8, 130, 3, 2, 16), (5, 30, 2, 40, 8, 129, 0, 3, 32)]:
        check(make(*shape, seed=shape[0]))


def test_verify_large_noise_and_tiny_temperature():
    """Temperatures near zero pick the argmax; enormous and tiny noise stay finite."""
    from rotatek_b200.kernels import verify_drafts
    a = make_verify(6, 2, 3000, torch.float32, False, 12)
    a["temperature"] = torch.full((6,), 1e-4, device=DEV)
    a["draft_lens"] = torch.zeros(6, dtype=torch.int32, device=DEV)
    a["noise"][::2] *= 1e30
    a["noise"][1::2] *= 1e-25
    tokens, _ = verify_drafts(**a)
    best = a["target_logits"][:, 0].argmax(-1)
    top = a["target_logits"][:, 0].topk(2).values
    clear = (top[:, 0] - top[:, 1]) > 0.01          # e^100 outweighs any noise ratio here
    assert clear.any() and torch.equal(tokens[clear, 0], best[clear])


@pytest.mark.parametrize("where", ["q", "k_full", "k_sparse", "k_text", "k_scale", "text alone", "q infinite"])
@pytest.mark.parametrize("dtype,fp8,T,hq", [(torch.bfloat16, False, 1, 8), (torch.bfloat16, True, 1, 8), (torch.bfloat16, True, 5, 8),
                                            (torch.float16, False, 5, 8), (torch.float32, False, 2, 8), (torch.bfloat16, False, 1, 80)])
def test_decode_nan_that_is_seen_comes_out(where, dtype, fp8, T, hq):
    """A NaN query row or Key makes NaN of every output that it reaches, also where it is all
    that a row's partial result holds, and of no other."""
    if where == "k_scale" and not fp8:
        pytest.skip("no scales")
    N, hk = 3, 2
    shape = (1, N, T, hq, hk, 0, 0, 40, 32) if where == "text alone" else (1, N, T, hq, hk, 1500, 70, 40, 32)
    a = make(*shape, dtype=dtype, fp8=fp8, seed=3, lens=[40, 33, 40])
    G = hq // hk
    hit = torch.zeros(N, T, hq, dtype=torch.bool)
    if where in ("q", "text alone"):
        a["q"][1, 0, 1, 5] = math.nan
        hit[1, 0, 1] = True
    elif where == "q infinite":
        a["q"][1, 0, 1] = math.inf
        hit[1, 0, 1] = True
    elif where in ("k_full", "k_sparse"):
        a[where][0, 1, 0, 3] = math.nan
        hit[:, :, G:] = True
    elif where == "k_scale":
        a["k_scale"][2, 1, 0] = math.nan
        hit[2, :, G:] = True
    else:
        if fp8:
            a["k_text"][2, 1, 0, 3] = 0x7f           # e4m3's NaN
        else:
            a["k_text"][2, 1, 0, 3] = math.nan
        hit[2, :, G:] = True
    from rotatek_b200.kernels import rotatek_shared_decode
    got = rotatek_shared_decode(**a).cpu().double()
    assert torch.isnan(got[hit]).all()
    assert torch.isfinite(got[~hit]).all()
    want, mag = osh.shared_decode(**a)
    tol = 1e-4 if dtype == torch.float32 else 2.0 ** -6
    assert ((got - want).abs()[~hit] <= tol * (1 + mag)[~hit]).all()


def test_tensors_of_every_kind_are_taken():
    """Parameters, tensors that require a gradient and dimensions of one entry with odd strides."""
    from rotatek_b200.kernels import append_text, rotatek_shared_decode
    a = make(1, 1, 1, 8, 1, 140, 20, 30, 32, seed=31)
    want = rotatek_shared_decode(**a)
    b = dict(a, q=torch.nn.Parameter(a["q"]), k_sparse=a["k_sparse"].clone().requires_grad_(),
             v_full=a["v_full"].as_strided(a["v_full"].shape, (7, 3, *a["v_full"].stride()[2:])))
    assert torch.equal(rotatek_shared_decode(**b), want)
    k, v = torch.zeros(1, 2, 9, 128, device=DEV, dtype=torch.bfloat16), torch.zeros(1, 2, 9, 128, device=DEV, dtype=torch.bfloat16)
    new = torch.nn.Parameter(torch.ones(1, 2, 3, 128, device=DEV, dtype=torch.bfloat16))
    append_text(new, new, torch.tensor([4], dtype=torch.int32, device=DEV), k, v)
    assert (k[:, :, 4:7] == 1).all() and (v[:, :, :4] == 0).all() and (v[:, :, 7:] == 0).all()
    with pytest.raises(RuntimeError, match="CUDA"):
        append_text(new.cpu(), new, torch.tensor([4], dtype=torch.int32, device=DEV), k, v)


def far(x, stride):
    """x with its dimension 1 moved `stride` elements apart (one allocation of that reach)."""
    shape = x.shape
    inner = torch.empty(shape[0:1] + shape[2:]).stride()
    buf = torch.empty((shape[1] - 1) * stride + x[:, 0].numel(), dtype=x.dtype, device=x.device)
    y = buf.as_strided(shape, (inner[0], stride, *inner[1:]))
    y.copy_(x)
    return y


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("T", [1, 9])
def test_decode_offsets_past_32_bits(fp8, T):
    """Heads of the spans and of the text 2^31 elements and more apart."""
    a = make(1, 3, T, 8, 2, 140, 70, 50, 32, fp8=fp8, seed=41)
    for name in ("k_full", "v_full", "k_sparse", "v_sparse", "k_text", "v_text"):
        b = dict(a, **{name: far(a[name], 2 ** 31 + 1024)})
        check(b)
        del b


def test_text_offsets_past_32_bits():
    from rotatek_b200.kernels import append_text, read_text
    B, H, C, T = 2, 2, 40, 7
    g = torch.Generator(device=DEV).manual_seed(42)
    new = torch.randn(2, B, H, T, 128, generator=g, device=DEV).to(torch.bfloat16)
    lens = torch.tensor([3, 30], dtype=torch.int32, device=DEV)
    near = [torch.zeros(B, H, C, 128, dtype=torch.uint8, device=DEV) for _ in range(2)]
    scales = [torch.zeros(B, H, C, device=DEV) for _ in range(2)]
    append_text(new[0], new[1], lens, *near, k_scale=scales[0], v_scale=scales[1])
    away = [far(torch.zeros_like(near[0]), 2 ** 31 + 4096) for _ in range(2)]
    far_scales = [far(torch.zeros_like(scales[0]), 2 ** 31 + 4096) for _ in range(2)]
    append_text(far(new[0], 2 ** 31 + 4096), new[1], lens, *away, k_scale=far_scales[0], v_scale=far_scales[1])
    for i in range(2):
        assert torch.equal(away[i], near[i]) and torch.equal(far_scales[i], scales[i])
    want = read_text(*near, lens + T, k_scale=scales[0], v_scale=scales[1])
    got = read_text(*away, lens + T, k_scale=far_scales[0], v_scale=far_scales[1])
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


def test_verify_offsets_past_32_bits():
    a = make_verify(3, 2, 1000, torch.float16, True, 43)
    a["target_logits"] = far(a["target_logits"], 2 ** 31 + 8)
    a["draft_logits"] = far(a["draft_logits"], 2 ** 31 + 8)
    check_verify(a)


UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}       # a rounding to 16 bits, relative


def alternating(a, name):
    """a's Values `name` become v, -v, v, -v, ...: outputs are what the weights leave of v."""
    v = a[name]
    sign = 1 - 2 * (torch.arange(v.shape[2], device=DEV) % 2)
    a[name] = (v[:, :, :1].float() * sign[:, None]).to(v.dtype).expand_as(v).contiguous()


def check_weights(a):
    """Weights to 16 bits and more.  The logits here are below 2 in size: products exact in fp32,
    sums off by 128 * 2^-24 * 2, the rotated query in two 16-bit parts (2^-16 in bf16) by 2 * 2^-16;
    the weights in two parts by 2^-16 or less.  Numerator and normaliser: 2 * (2^-15 + 2^-16) < 2^-13.
    One 16-bit part would move a weight by up to 2^-9 (bf16) or 2^-12 (fp16)."""
    from rotatek_b200.kernels import rotatek_shared_decode
    got = rotatek_shared_decode(**a).cpu().double()
    want, mag = osh.shared_decode(**a)
    tol = UNIT[a["q"].dtype] * want.abs() + 2.0 ** -13 * mag + 2.0 ** -25
    off = (got - want).abs()
    assert (off <= tol).all(), f"{int((off > tol).sum())} of {off.numel()}, worst {(off / tol).max():.2f}"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("name,sv,sf", [("v_full", 0, 4), ("v_full", 0, 64), ("v_sparse", 4, 0), ("v_sparse", 128, 0),
                                        ("v_sparse", 99, 0)])
def test_decode_prefix_weights_hold_their_bits(name, sv, sf, dtype):
    """Values that cancel leave the errors of the softmax weights in the output."""
    a = make(1, 40, 1, 14, 2, sv, sf, 0, 32, dtype=dtype, seed=51, std=0.3, bias=False)
    alternating(a, name)
    check_weights(a)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,cap", [(1, 4), (1, 32), (6, 9), (6, 300)])
def test_decode_text_weights_hold_their_bits(T, cap, dtype):
    """16-bit text, as the prefix above."""
    a = make(1, 20, T, 16, 2, 0, 0, cap, 32, dtype=dtype, lens=[cap] * 20, seed=52, std=0.3)
    alternating(a, "v_text")
    check_weights(a)


def quantise_text(a):
    for side in ("k", "v"):
        val, scale = osh.quantize_rows(a[f"{side}_text"])
        a[f"{side}_text"] = val.float().to(torch.float8_e4m3fn).to(DEV).view(torch.uint8)
        a[f"{side}_scale"] = scale.to(DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,cap", [(1, 4), (1, 32), (6, 9), (6, 300)])
def test_decode_text8_weights_hold_their_bits(T, cap, dtype):
    """8-bit text, as the prefix above, for either text kernel."""
    a = make(1, 20, T, 16, 2, 0, 0, cap, 32, dtype=dtype, lens=[cap] * 20, seed=53, std=0.3)
    alternating(a, "v_text")
    quantise_text(a)
    check_weights(a)


@pytest.mark.parametrize("T", [2, 9])
@pytest.mark.parametrize("size", [1e-3, 1e-5, 1e-9])
@pytest.mark.parametrize("beside", ["zeros", "weightless", "unseen"])
def test_decode_text8_small_values_hold_the_weight(beside, size, T):
    """Value rows of `size` that hold all the weight, beside a row of zeros (its scale is 1), a row
    1e9 times larger whose weight is 0, or one that the earlier queries may not see."""
    a = make(1, 2, T, 8, 2, 0, 0, 150, 32, dtype=torch.bfloat16, lens=[150, 131], seed=54)
    a["q"][..., 0] = 4.0
    v = a["v_text"].float() * size
    if beside == "zeros":
        v[:, :, [5, 40, 130]] = 0
    elif beside == "weightless":
        a["k_text"][:, :, 40, 0] = -1000.0            # logits near -350
        v[:, :, 40] *= 1e9
    else:
        v[0, :, 149] *= 1e9
        v[1, :, 130] *= 1e9
    a["v_text"] = v.to(torch.bfloat16)
    quantise_text(a)
    check(a)


@pytest.mark.parametrize("T", [1, 9])
def test_decode_text8_queries_of_any_range(T):
    """bf16 queries with one channel 2^18 times the others, where the Keys are 0: the other
    channels alone make the logits, and keep their bits."""
    a = make(1, 3, T, 8, 2, 0, 0, 60, 32, dtype=torch.bfloat16, lens=[60, 33, 20], seed=55, std=0.5)
    a["q"][..., 7] = 2.0 ** 18
    a["k_text"][..., 7] = 0
    quantise_text(a)
    check_weights(a)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype,fp8", [(torch.bfloat16, False), (torch.float16, False), (torch.bfloat16, True),
                                       (torch.float16, True), (torch.float32, True)])
@pytest.mark.parametrize("T,lens", [(4, [33, 64, 7, 4]), (9, [33, 64, 40, 9]), (40, [45, 64, 40, 70])])
@pytest.mark.parametrize("back", [1, 3])
def test_decode_later_drafts_do_not_reach_earlier_queries(back, T, lens, dtype, fp8, bad):
    """The row of the last draft but `back - 1` holds NaN or infinity in its Key, its Value and their
    scales: the queries before it stay the same to the bit, it and those after it show it."""
    from rotatek_b200.kernels import rotatek_shared_decode
    a = make(1, 4, T, 8, 2, 140, 20, 70, 32, dtype=dtype, fp8=fp8, lens=lens, seed=61)
    clean = rotatek_shared_decode(**a)
    at = a["text_lens"].long() - back
    rows = torch.arange(4, device=DEV)
    variants = [("v_text", True)] + ([("v_scale", True), ("k_scale", True)] if fp8 else [("k_text", bad != bad)])
    for name, shows in variants:
        b = dict(a, **{name: a[name].clone()})
        if b[name].dtype == torch.uint8:
            b[name][rows, :, at, 64:] = 0x7F               # e4m3's NaN; the other channels stay numbers
        elif name == "v_text":
            b[name][rows, :, at, 64:] = bad
        else:
            b[name][rows, :, at] = bad
        got = rotatek_shared_decode(**b)
        assert torch.equal(got[:, :T - back], clean[:, :T - back])
        if name == "v_text":
            assert torch.isfinite(got[..., :64]).all() and not torch.isfinite(got[:, T - back:, :, 64:]).any()
        elif shows and bad != bad:
            assert torch.isnan(got[:, T - back:]).all()


def test_threads_on_one_stream():
    """Threads that share the default stream, with calls of several launches each: every result is
    that of the call alone, to the bit."""
    import threading
    from rotatek_b200.kernels import rotatek_shared_decode, verify_drafts
    args = [make(2, 3, 2, 8, 2, 700, 90, 150, 32, fp8=bool(i % 2), seed=70 + i) for i in range(4)]
    logits = [make_verify(6, 3, 9000, torch.bfloat16, True, 80 + i) for i in range(4)]
    want = [(rotatek_shared_decode(**a), *verify_drafts(**v)) for a, v in zip(args, logits)]
    torch.cuda.synchronize()
    out = [[] for _ in range(4)]

    def call(i):
        for _ in range(60):
            out[i].append((rotatek_shared_decode(**args[i]), *verify_drafts(**logits[i])))

    threads = [threading.Thread(target=call, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(4):
        assert len(out[i]) == 60
        for got in out[i]:
            assert all(torch.equal(g, w) for g, w in zip(got, want[i]))


FIRST_CALL = """
import torch
from rotatek_b200 import _lib, synthetic
from rotatek_b200.kernels import rotatek_decode
from tests.test_shared_gpu import compare, make
from rotatek_b200.kernels import rotatek_shared_decode
a = make(1, 4, 2, 8, 2, 500, 30, 64, 32, fp8=True, seed=19)
d = synthetic.make_decode(2, 28, 4, 3000, 100, keep=32, seed=1, device="cuda:0", dtype=torch.bfloat16).as_kwargs()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = rotatek_shared_decode(**a)
assert not _lib._workspaces
h = torch.cuda.CUDAGraph()
with torch.cuda.graph(h):
    held, _, _ = rotatek_decode(**d)
assert not _lib._workspaces
eager, _, _ = rotatek_decode(**d)
torch.cuda.synchronize()
for _ in range(2):
    g.replay()
    h.replay()
    torch.cuda.synchronize()
    compare(out, a)
    assert torch.equal(held, eager) and torch.equal(rotatek_decode(**d)[0], eager) and eager.abs().sum() > 0
assert torch.equal(rotatek_shared_decode(**a), out) and _lib.read_status() == 0
"""


def test_first_call_of_a_process_may_be_captured():
    import os
    import subprocess
    import sys
    repo = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", FIRST_CALL], cwd=repo, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_text_of_one_question_takes_the_wide_kernel_whatever_its_strides():
    """The stride of a dimension with one entry is never used and may be anything."""
    from torch.profiler import ProfilerActivity, profile

    from rotatek_b200.kernels import append_text, read_text
    lens = torch.tensor([3], dtype=torch.int32, device=DEV)
    caches = [torch.zeros(1, 1, 40, 128, dtype=torch.uint8, device=DEV).as_strided((1, 1, 40, 128), (7, 5, 128, 1))
              for _ in range(2)]
    scales = [torch.zeros(1, 1, 40, device=DEV) for _ in range(2)]
    new = torch.randn(1, 1, 6, 128, device=DEV).to(torch.bfloat16).as_strided((1, 1, 6, 128), (3, 1, 128, 1))
    with profile(activities=[ProfilerActivity.CUDA]) as seen:
        append_text(new, new, lens, *caches, k_scale=scales[0], v_scale=scales[1])
        k, v = read_text(*caches, lens + 6, k_scale=scales[0], v_scale=scales[1])
        torch.cuda.synchronize()
    names = " ".join(e.name for e in seen.events())
    assert "append_rows_kernel" in names and "read_rows_kernel" in names
    val, scale = osh.quantize_rows(new)
    assert torch.equal(k[:, :, 3:9].cpu().float(), (val.float() * scale[..., None]).to(torch.bfloat16).float())
    assert torch.equal(k, v) and (k[:, :, :3] == 0).all()


@pytest.mark.parametrize("heat", [1e-6, 1e-8, 1e-9, 1e-12, 1e-30, 1e-38])
@pytest.mark.parametrize("dtype,logits", [(torch.bfloat16, True), (torch.float32, True), (torch.float32, False)])
def test_verify_temperatures_next_to_nothing(heat, dtype, logits):
    """All of p is at the largest logits, whatever the temperature's size: the products of logits and
    1 / temperature are far beyond what their difference of a bit could bear."""
    a = make_verify(12, 3, 5000, dtype, logits, 44, near=0.2)
    a["target_logits"] = a["target_logits"] + 30
    a["temperature"] = torch.full((12,), heat, device=DEV)
    if not logits:                                   # some proposals are the likeliest token
        best = a["target_logits"][:, :3].argmax(-1)
        a["draft_tokens"] = torch.where(torch.rand(12, 3, device=DEV) < 0.7, best, a["draft_tokens"])
    _, accepted = check_verify(a)
    assert accepted.sum() > 0


# ------------------------------------------------------------------ long ranges, several chunks, whole questions
def dense(a):
    """``osh.shared_decode`` (out, A) in float64 on the GPU, a KV head of a question at a time."""
    q = a["q"].double()
    B, T, hq, D = q.shape
    G, P, hk, cap = a["num_kv_groups"], a["R_partial"].shape[0], a["R_partial"].shape[1], a["k_text"].shape[2]
    out, mag = torch.zeros_like(q), torch.zeros_like(q)
    lens = a["text_lens"].clamp(0, cap).tolist()

    def text(side, b, h, n):
        x = a[f"{side}_text"][b, h, :n]
        if a.get(f"{side}_scale") is None:
            return x.double()
        return x.view(torch.float8_e4m3fn).double() * a[f"{side}_scale"][b, h, :n, None].double()

    for h in range(hk):
        for p in range(P):
            keys = a["k_sparse"][p, h].double() @ a["R_partial"][p, h].double().T
            if a["delta_mu"] is not None:
                keys = keys + a["delta_mu"][p, h].double()
            there = slice(None) if a["mask_full"] is None else a["mask_full"][p].bool()
            keys = torch.cat([a["k_full"][p, h].double()[there], keys])
            values = torch.cat([a["v_full"][p, h].double()[there], a["v_sparse"][p, h].double()])
            for b in range(p * (B // P), (p + 1) * (B // P)):
                n = lens[b]
                k, v = torch.cat([keys, text("k", b, h, n)]), torch.cat([values, text("v", b, h, n)])
                if k.shape[0] == 0:
                    continue
                s = q[b, :, h * G:(h + 1) * G].reshape(T * G, D) @ k.T / math.sqrt(D)
                seen = n - (T - 1) + torch.arange(T, device=DEV).repeat_interleave(G)
                s[:, keys.shape[0]:].masked_fill_(torch.arange(n, device=DEV) >= seen[:, None], -math.inf)
                w = torch.softmax(s, 1).nan_to_num(0.0)              # a row that sees nothing
                out[b, :, h * G:(h + 1) * G] = (w @ v).view(T, G, D)
                mag[b, :, h * G:(h + 1) * G] = (w @ v.abs()).view(T, G, D)
    return out, mag


def check_dense(a, logits=0.0):
    """The tolerance of ``compare`` where logits stay below 50, more for larger ones: they are off by 2^-16
    of their size (the rotated query's two parts), which moves a weight by as much, twice."""
    from rotatek_b200.kernels import rotatek_shared_decode
    got = rotatek_shared_decode(**a).double()
    want, mag = dense(a)
    tol = UNIT[a["q"].dtype] * want.abs() + (2.0 ** -11 + 2 * logits * 2.0 ** -16) * mag + 2.0 ** -25
    off = (got - want).abs()
    assert (off <= tol).all(), f"{int((off > tol).sum())} of {off.numel()}, worst {(off / tol).max():.2f}"


def test_dense_is_the_oracle():
    a = make(2, 2, 3, 8, 2, 40, 20, 30, 32, fp8=True, mask=0.6, seed=90, lens=[30, 0, 2, 17])
    for x, y in zip(dense(a), osh.shared_decode(**a)):
        assert (x.cpu() - y).abs().max() < 1e-12


LONG = [
    # P, N, T, H_q, H_kv, S_v, S_f, C, D_keep: a CTA takes a dozen blocks and more of a unit, several units
    (2, 2, 1, 64, 64, 2900, 300, 20, 32),
    (1, 3, 1, 160, 160, 2000, 1000, 10, 16),
    (3, 2, 1, 128, 64, 1700, 700, 0, 64),
    (1, 32, 1, 128, 32, 7000, 200, 30, 32),          # full tiles of 128 rows
    (1, 21, 3, 80, 16, 9000, 64, 40, 64),            # 315 rows: two full tiles and a part
    (1, 2, 1, 320, 160, 0, 3000, 5, 32),             # prompt alone
]


@pytest.mark.parametrize("shape", LONG)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("mask", [None, 0.7])
def test_decode_long_ranges(shape, dtype, mask):
    """Every stage and buffer of the prefix kernel is used again and again within a unit."""
    check_dense(make(*shape, dtype=dtype, mask=mask, seed=91))


@pytest.mark.parametrize("shape", [LONG[0], LONG[3]])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("way", ["up", "down", "there and back"])
def test_decode_long_ranges_with_a_moving_maximum(shape, dtype, way):
    """Logits that climb by more than 2^8 from block to block of a long range: the lazy maximum moves
    a dozen times within a unit."""
    a = make(*shape, dtype=dtype, seed=92, bias=False)
    sv, groups = shape[5], a["num_kv_groups"]
    t = torch.linspace(0, 1, sv, device=DEV)
    t = {"up": t, "down": 1 - t, "there and back": 1 - (2 * t - 1).abs()}[way]
    direction = a["R_partial"][0, :, :, 0].float()                       # q . R column 0 = 20 for every query
    a["R_partial"] = a["R_partial"][:1].expand_as(a["R_partial"]).contiguous()
    a["q"] = (a["q"].float() * 0.05 + 20.0 * direction.repeat_interleave(groups, 0)).to(dtype)
    ramp = torch.zeros(sv, a["k_sparse"].shape[-1], device=DEV)
    ramp[:, 0] = 250.0 * t                                                # logits up to 442
    a["k_sparse"] = (a["k_sparse"].float() * 0.05 + ramp).to(dtype)
    a["k_full"] = (a["k_full"].float() * 0.1).to(dtype)
    check_dense(a, logits=442)


@pytest.mark.parametrize("dtype,fp8", [(torch.bfloat16, False), (torch.float16, False), (torch.bfloat16, True),
                                       (torch.float16, True)])
@pytest.mark.parametrize("T", [1, 3, 7])
def test_decode_several_text_chunks(T, dtype, fp8):
    """Lengths around the edges of chunks of 256, for rows of either text kernel."""
    lens = [0, 1, 255, 256, 257, 258, 511, 512, 513, 700, 768, 769, 800, 1023, 1024, 1025, 1099, 1100]
    check_dense(make(1, len(lens), T, 8, 2, 200, 30, 1100, 32, dtype=dtype, fp8=fp8, lens=lens, seed=93))
    check_dense(make(1, len(lens), T, 8, 2, 0, 0, 1100, 32, dtype=dtype, fp8=fp8, lens=lens, seed=94))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("T", [1, 6])
@pytest.mark.parametrize("questions,cap", [(40, 1100), (75, 2100)])
def test_decode_longer_chunks(questions, cap, T, fp8):
    """Enough questions for chunks of 512 and of 1024 tokens, and more than one of them each."""
    lens = [(i * 211) % (cap + 1) for i in range(questions - 4)] + [512, 1024, 1025, cap]
    check_dense(make(1, questions, T, 32, 8, 130, 10, cap, 32, fp8=fp8, lens=lens, seed=95))


@pytest.mark.parametrize("dtype,fp8", [(torch.bfloat16, False), (torch.float16, True), (torch.bfloat16, True)])
@pytest.mark.parametrize("N,T,hq,hk,cap,lens", [(3, 33, 8, 2, 40, [33, 40, 34]), (2, 100, 28, 4, 300, [300, 120]),
                                                (2, 577, 16, 2, 700, [577, 690]), (2, 70, 4, 4, 100, [20, 100])])
def test_decode_whole_questions(N, T, hq, hk, cap, lens, dtype, fp8):
    """The questions themselves: T up to 577, causal among them, and one shorter than T."""
    check_dense(make(1, N, T, hq, hk, 500, 40, cap, 32, dtype=dtype, fp8=fp8, lens=lens, seed=96))


@pytest.mark.parametrize("where", ["v_full", "v_sparse", "v_text"])
@pytest.mark.parametrize("dtype,fp8,N,T", [(torch.bfloat16, False, 2, 1), (torch.float16, False, 2, 1), (torch.bfloat16, True, 2, 1),
                                           (torch.bfloat16, True, 2, 9), (torch.float32, False, 2, 1), (torch.bfloat16, False, 100, 4)])
def test_decode_nan_values_with_next_to_no_weight_come_out(where, dtype, fp8, N, T):
    """A NaN Value that is seen makes NaN of its channel however small its weight, wherever the weight
    is: the other tokens' logits are hundreds larger in another partial result."""
    from rotatek_b200.kernels import rotatek_shared_decode
    a = make(1, N, T, 8, 2, 300, 70, 600, 32, dtype=dtype, lens=[600] * N, seed=97, bias=False)
    a["q"][..., 0] = 40.0
    big = 300 if where != "v_text" else 590
    a["k_text"][:, :, :, 0] = 0
    a["k_text"][:, :, big, 0] = 200.0                                     # a logit of 700
    a["R_partial"] = torch.zeros_like(a["R_partial"])
    a["R_partial"][:, :, torch.arange(32) + 1, torch.arange(32)] = 1      # channel 0 is not rotated
    a["k_full"][..., 0] = 0
    if fp8:
        quantise_text(a)
    if where == "v_text" and fp8:
        a["v_text"][:, :, 3, 5] = 0x7F
    else:
        a[where][:, :, 3, 5] = math.nan
    got = rotatek_shared_decode(**a)
    assert torch.isnan(got[..., 5]).all()
    rest = torch.arange(128, device=DEV) != 5
    assert torch.isfinite(got[..., rest]).all()
