"""Timed cases of the operators that serve many questions on shared images.

One image (or video) is prefilled once: its prompt and its rotated, truncated
visual Keys are a *prefix* that every question on it shares.  Each question
keeps only its own text tokens.  Four operators make a decoding step of it:

    attend   ``kernels.rotatek_shared_decode``: attention of T new tokens per
             question over the shared prefix and the question's own text
    append   ``kernels.append_text``: the new tokens' Keys and Values quantised
             to e4m3 as they are written into the question's text cache
    read     ``kernels.read_text``: such a cache back in a 16-bit type
    verify   ``kernels.verify_drafts``: which drafted tokens the target model
             accepts, and the token that follows them

Cases are dicts of plain values; ``run`` computes them in elementary torch
operations in 32 bits, or, where ``own`` is set, by the calls above.
"""
import math

import torch

own = False

D = 128                     # head width of every attention case
E4M3_MAX = 448.0
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _attend(name, prefixes, questions, tokens, q_heads, kv_heads, vision, full, cap, keep, dtype, fp8, mask, bias,
            text_min=1):
    return dict(name=name, op="attend", prefixes=prefixes, questions=questions, tokens=tokens, q_heads=q_heads,
                kv_heads=kv_heads, vision=vision, full=full, cap=cap, keep=keep, dtype=dtype, fp8=fp8, mask=mask,
                bias=bias, text_min=text_min)


def _append(name, batch, kv_heads, tokens, cap, dtype, ragged):
    return dict(name=name, op="append", batch=batch, kv_heads=kv_heads, tokens=tokens, cap=cap, dtype=dtype,
                ragged=ragged)


def _read(name, batch, kv_heads, cap, dtype, text_min):
    return dict(name=name, op="read", batch=batch, kv_heads=kv_heads, cap=cap, dtype=dtype, text_min=text_min)


def _verify(name, batch, drafts, vocab, dtype, logits, greedy, ragged):
    return dict(name=name, op="verify", batch=batch, drafts=drafts, vocab=vocab, dtype=dtype, logits=logits,
                greedy=greedy, ragged=ragged)


def listed():
    return [
        # two questions just asked about one small image: a step where latency is all
        _attend("attend-two-questions", 1, 2, 1, 28, 4, 1000, 64, 64, 32, "bf16", False, False, True),
        # eight conversations on one image at the decode benchmark's context length
        _attend("attend-conversations", 1, 8, 1, 28, 4, 15360, 640, 640, 32, "bf16", False, False, True),
        # four images, sixteen questions each, a target model checking four drafted tokens; padded prompts, 8-bit text
        _attend("attend-drafted", 4, 16, 5, 28, 4, 15360, 640, 512, 32, "bf16", True, True, True),
        # a model without shared heads, two images of one long-context decoder; text cache in 16 bits
        _attend("attend-every-head", 2, 12, 1, 32, 32, 16384, 32, 160, 32, "f16", False, False, True),
        # one long video, sixty-four questions with eight tokens checked per step
        _attend("attend-video-drafted", 1, 64, 8, 64, 8, 31744, 1024, 1001, 32, "bf16", True, False, True),
        # one decoded token of eight questions
        _append("append-token", 8, 4, 1, 512, "bf16", False),
        # the questions themselves, prefilled together: lengths differ
        _append("append-questions", 64, 8, 577, 1024, "bf16", True),
        # one question's cache handed to code that wants 16-bit tensors
        _read("read-one", 1, 4, 200, "bf16", 150),
        # every question's cache of one layer
        _read("read-batch", 64, 8, 1024, "f16", 300),
        # one conversation, three drafted tokens
        _verify("verify-one", 1, 3, 32000, "f16", True, False, False),
        # a batch; some rows greedy, drafts of different lengths
        _verify("verify-batch", 64, 5, 32000, "f16", True, True, True),
        # a large vocabulary and drafts that a table lookup proposes, without draft probabilities
        _verify("verify-lookup", 128, 8, 131071, "bf16", False, True, True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "read", "verify"])
    if op == "attend":
        while True:
            q_heads, kv_heads = rng.choice([(28, 4), (32, 32), (32, 8), (64, 8), (12, 4)])
            c = _attend("", rng.randint(1, 4), _log_int(rng, 1, 64), rng.choice([1, 1, 2, 3, 5, 8]), q_heads, kv_heads,
                        _log_int(rng, 1, 32000), _log_int(rng, 1, 1024), _log_int(rng, 8, 1024),
                        rng.choice([16, 32, 32, 64]), rng.choice(["bf16", "f16"]), rng.random() < 0.5,
                        rng.random() < 0.5, rng.random() < 0.7, 8)
            if work(c)["flops"] < 1.5e11 and work(c)["bytes"] < 2e9:
                break
    elif op == "append":
        tokens = _log_int(rng, 1, 600)
        c = _append("", _log_int(rng, 1, 64), rng.choice([1, 4, 8]), tokens, tokens + _log_int(rng, 1, 400),
                    rng.choice(["bf16", "f16", "f32"]), rng.random() < 0.5)
    elif op == "read":
        cap = _log_int(rng, 1, 1024)
        c = _read("", _log_int(rng, 1, 64), rng.choice([1, 4, 8]), cap, rng.choice(["bf16", "f16"]), rng.randint(0, cap))
    else:
        c = _verify("", _log_int(rng, 1, 128), rng.randint(1, 8), _log_int(rng, 1000, 131072),
                    rng.choice(["bf16", "f16", "f32"]), rng.random() < 0.6, rng.random() < 0.5, rng.random() < 0.5)
        while c["batch"] * c["drafts"] * c["vocab"] > 64 * 1024 * 1024:
            c["batch"] = max(1, c["batch"] // 2)
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs
def _spread(lo, hi, n, g):
    """n whole numbers from lo to hi, evenly spread, in an order that g gives."""
    steps = torch.arange(n, device=DEV, dtype=torch.int64)
    vals = hi - steps * (hi - lo) // max(1, n - 1) if n > 1 else torch.full((1,), hi, device=DEV)
    return vals[torch.randperm(n, generator=g, device=DEV)].to(torch.int32)


def _lens_sum(lo, hi, n):
    return sum(hi - i * (hi - lo) // max(1, n - 1) for i in range(n)) if n > 1 else hi


def _e4m3_cache(shape, g):
    """A cache's bytes as quantised N(0, 1) rows leave them, and the rows' scales."""
    x = torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)
    scale = x.abs().amax(-1) / E4M3_MAX
    return (x / scale[..., None]).to(torch.float8_e4m3fn).view(torch.uint8), scale


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = TYPES[case["dtype"]]

    def normal(*shape, dtype=dt, scale=1.0):
        return (torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32) * scale).to(dtype)

    s = dict(case=case, op=case["op"])
    if case["op"] == "attend":
        p, n, t, hq, hk = (case[k] for k in ("prefixes", "questions", "tokens", "q_heads", "kv_heads"))
        b, sv, sf, cap, keep = p * n, case["vision"], case["full"], case["cap"], case["keep"]
        # queries as a fused projection leaves them: a slice of [B, T, (H_q + 2 H_kv) D]
        qkv = normal(b, t, hq + 2 * hk, D)
        s["q"] = qkv[:, :, :hq]
        basis = torch.linalg.qr(torch.randn(p, hk, D, keep, generator=g, device=DEV, dtype=torch.float32))[0]
        s["R"] = basis.to(dt)
        s["delta_mu"] = normal(p, hk, D, scale=0.3) if case["bias"] else None
        s["k_full"], s["v_full"] = normal(p, hk, sf, D), normal(p, hk, sf, D)
        s["mask"] = None
        if case["mask"]:   # padded prompts: about a fifth of the tokens are not there
            s["mask"] = (torch.rand(p, sf, generator=g, device=DEV) < 0.8).to(torch.uint8)
        # rotated Keys: the first channels carry most of the spread
        spread = torch.exp(-torch.arange(keep, device=DEV, dtype=torch.float32) / 10)
        spread = torch.sqrt(100 * spread / spread.sum())
        s["k_sparse"] = (torch.randn(p, hk, sv, keep, generator=g, device=DEV) * spread).to(dt)
        s["v_sparse"] = normal(p, hk, sv, D)
        s["lens"] = _spread(max(case["text_min"], t), cap, b, g) if cap >= t else torch.full(
            (b,), cap, device=DEV, dtype=torch.int32)
        if case["fp8"]:
            s["k_text"], s["k_scale"] = _e4m3_cache((b, hk, cap, D), g)
            s["v_text"], s["v_scale"] = _e4m3_cache((b, hk, cap, D), g)
        else:
            s["k_text"], s["v_text"] = normal(b, hk, cap, D), normal(b, hk, cap, D)
            s["k_scale"] = s["v_scale"] = None
    elif case["op"] == "append":
        b, h, t, cap = case["batch"], case["kv_heads"], case["tokens"], case["cap"]
        kv = normal(b, t, 2 * h, D)           # the Key and Value part of a fused projection
        s["k_new"], s["v_new"] = kv[:, :, :h].transpose(1, 2), kv[:, :, h:].transpose(1, 2)
        s["lens"] = _spread(0, cap - t, b, g)
        s["counts"] = _spread(t // 3, t, b, g) if case["ragged"] else None
        s["k_text"], s["k_scale"] = _e4m3_cache((b, h, cap, D), g)
        s["v_text"], s["v_scale"] = _e4m3_cache((b, h, cap, D), g)
    elif case["op"] == "read":
        b, h, cap = case["batch"], case["kv_heads"], case["cap"]
        s["lens"] = _spread(case["text_min"], cap, b, g)
        s["k_text"], s["k_scale"] = _e4m3_cache((b, h, cap, D), g)
        s["v_text"], s["v_scale"] = _e4m3_cache((b, h, cap, D), g)
        s["dtype"] = dt
    else:
        b, t, v = case["batch"], case["drafts"], case["vocab"]
        target = torch.randn(b, t + 1, v, generator=g, device=DEV, dtype=torch.float32) * 2.5
        temperature = 0.6 + 0.6 * torch.rand(b, generator=g, device=DEV)
        if case["greedy"]:
            temperature[torch.rand(b, generator=g, device=DEV) < 0.3] = 0.0
        race = torch.empty(b, t, v, device=DEV).exponential_(generator=g).clamp_min_(1e-10)
        if case["logits"]:                    # a smaller model's logits, and tokens drawn from them
            draft = (target[:, :t] + torch.randn(b, t, v, generator=g, device=DEV)).to(dt)
            soft = torch.softmax(draft.float() / temperature.clamp_min(0.05)[:, None, None], -1)
            s["drafts"] = torch.where(temperature[:, None] > 0, (soft / race).argmax(-1), draft.float().argmax(-1))
            s["draft_logits"] = draft
            del soft
        else:                                 # proposals without probabilities: about three of four are the likeliest
            wild = torch.randint(0, v, (b, t), generator=g, device=DEV)
            s["drafts"] = torch.where(torch.rand(b, t, generator=g, device=DEV) < 0.75, target[:, :t].argmax(-1), wild)
            target[:, :t].scatter_add_(2, s["drafts"][..., None], torch.full((b, t, 1), 9.0, device=DEV))
            s["draft_logits"] = None
        s["target"] = target.to(dt)
        s["temperature"] = temperature
        s["uniforms"] = torch.rand(b, t, generator=g, device=DEV)
        s["noise"] = torch.empty(b, v, device=DEV).exponential_(generator=g).clamp_min_(1e-10)
        s["draft_lens"] = _spread(0, t, b, g) if case["ragged"] else None
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from rotatek_b200 import kernels

    if s["op"] == "attend":
        return kernels.rotatek_shared_decode(
            s["q"], s["R"], s["delta_mu"], s["k_full"], s["v_full"], s["mask"], s["k_sparse"], s["v_sparse"],
            s["k_text"], s["v_text"], s["lens"], s["case"]["q_heads"] // s["case"]["kv_heads"],
            k_scale=s["k_scale"], v_scale=s["v_scale"])
    if s["op"] == "append":
        kernels.append_text(s["k_new"], s["v_new"], s["lens"], s["k_text"], s["v_text"], k_scale=s["k_scale"],
                            v_scale=s["v_scale"], counts=s["counts"])
        return _cache_values(s)
    if s["op"] == "read":
        return kernels.read_text(s["k_text"], s["v_text"], s["lens"], k_scale=s["k_scale"], v_scale=s["v_scale"],
                                 dtype=s["dtype"])
    return kernels.verify_drafts(s["target"], s["drafts"], s["draft_logits"], s["uniforms"], s["noise"],
                                 s["temperature"], draft_lens=s["draft_lens"])


def _run_plain(s):
    return {"attend": _plain_attend, "append": _plain_append, "read": _plain_read, "verify": _plain_verify}[s["op"]](s)


def _cache_values(s):
    """An 8-bit cache as the values it stands for, with its scales."""
    return (s["k_text"].view(torch.float8_e4m3fn), s["k_scale"], s["v_text"].view(torch.float8_e4m3fn), s["v_scale"])


def _plain_attend(s):
    c = s["case"]
    p, n, t, hq, hk = (c[k] for k in ("prefixes", "questions", "tokens", "q_heads", "kv_heads"))
    b, groups, cap = p * n, hq // hk, c["cap"]
    q = s["q"].float() * (1.0 / math.sqrt(D))
    shared = q.view(p, n, t, hk, groups, D).permute(0, 3, 1, 2, 4, 5).reshape(p, hk, n * t * groups, D)
    alone = q.view(b, t, hk, groups, D).permute(0, 2, 1, 3, 4).reshape(b, hk, t * groups, D)

    s_vis = (shared @ s["R"].float()) @ s["k_sparse"].float().transpose(-1, -2)
    if s["delta_mu"] is not None:
        s_vis += shared @ s["delta_mu"].float()[..., None]
    s_full = shared @ s["k_full"].float().transpose(-1, -2)
    v_full = s["v_full"].float()
    if s["mask"] is not None:
        there = s["mask"].bool()[:, None]
        s_full = s_full.masked_fill(~there[:, :, None], -math.inf)
        v_full = torch.where(there[..., None], v_full, 0.0)

    k_text, v_text = s["k_text"], s["v_text"]
    if s["k_scale"] is not None:
        k_text = k_text.view(torch.float8_e4m3fn).float() * s["k_scale"][..., None]
        v_text = v_text.view(torch.float8_e4m3fn).float() * s["v_scale"][..., None]
    place = torch.arange(cap, device=DEV)
    v_text = torch.where((place < s["lens"][:, None])[:, None, :, None], v_text.float(), 0.0)
    last = s["lens"][:, None] - (t - 1) + torch.arange(t, device=DEV)          # tokens that query t sees
    seen = place < last.repeat_interleave(groups, 1)[..., None]                 # [B, T G, cap]
    s_text = (alone @ k_text.float().transpose(-1, -2)).masked_fill(~seen[:, None], -math.inf)

    def rows(x):         # [B, H, T G, ..] -> [P, H, N T G, ..]
        return x.view(p, n, hk, t * groups, -1).transpose(1, 2).reshape(p, hk, n * t * groups, -1)

    top = torch.maximum(s_vis.amax(-1, keepdim=True), torch.maximum(
        s_full.amax(-1, keepdim=True), rows(s_text.amax(-1, keepdim=True))))
    top = torch.where(top == -math.inf, 0.0, top)
    top_alone = top.view(p, hk, n, t * groups, 1).transpose(1, 2).reshape(b, hk, t * groups, 1)
    e_vis, e_full = s_vis.sub_(top).exp_(), (s_full - top).exp_()
    e_text = (s_text - top_alone).exp_()
    total = e_vis.sum(-1, keepdim=True) + e_full.sum(-1, keepdim=True) + rows(e_text.sum(-1, keepdim=True))
    out = e_vis @ s["v_sparse"].float() + e_full @ v_full + rows(e_text @ v_text)
    out = torch.where(total > 0, out / total, 0.0)
    out = out.view(p, hk, n, t, groups, D).permute(0, 2, 3, 1, 4, 5).reshape(b, t, hq, D)
    return out.to(s["q"].dtype)


def _plain_append(s):
    c = s["case"]
    b, h, t, cap = c["batch"], c["kv_heads"], c["tokens"], c["cap"]
    count = s["counts"] if s["counts"] is not None else torch.full_like(s["lens"], t)
    step = torch.minimum(torch.arange(t, device=DEV), (count[:, None] - 1).clamp_min(0))   # past the last: it again
    place = (s["lens"][:, None] + step).clamp_max(cap - 1).long()[:, None].expand(b, h, t)
    fresh = (count > 0)[:, None, None]
    for new, cache, scales in ((s["k_new"], s["k_text"], s["k_scale"]), (s["v_new"], s["v_text"], s["v_scale"])):
        x = new.float().gather(2, step.long()[:, None, :, None].expand(b, h, t, D))
        amax = x.abs().amax(-1)
        scale = torch.where(amax > 0, (amax / E4M3_MAX).clamp_min(2.0 ** -126), 1.0)
        bits = (x / scale[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
        wide = place[..., None].expand(b, h, t, D)
        bits = torch.where(fresh[..., None], bits, cache.gather(2, wide))
        scale = torch.where(fresh, scale, scales.gather(2, place))
        cache.scatter_(2, wide, bits)
        scales.scatter_(2, place, scale)
    return _cache_values(s)


def _plain_read(s):
    there = (torch.arange(s["case"]["cap"], device=DEV) < s["lens"][:, None])[:, None, :, None]
    return tuple(torch.where(there, x.view(torch.float8_e4m3fn).float() * scale[..., None], 0.0).to(s["dtype"])
                 for x, scale in ((s["k_text"], s["k_scale"]), (s["v_text"], s["v_scale"])))


def _plain_verify(s):
    b, t, v = s["case"]["batch"], s["case"]["drafts"], s["case"]["vocab"]
    greedy = s["temperature"] <= 0
    heat = torch.where(greedy, 1.0, s["temperature"])[:, None, None]

    def soft(x):
        x = x.float() / heat
        e = (x - x.amax(-1, keepdim=True)).exp_()
        return e / e.sum(-1, keepdim=True)

    target = s["target"].float()
    best = target.argmax(-1)                                                     # [B, T + 1]
    p = soft(s["target"])
    if s["draft_logits"] is not None:
        q = soft(s["draft_logits"])
    else:
        q = torch.zeros(b, t, v, device=DEV).scatter_(2, s["drafts"][..., None], 1.0)
    at = s["drafts"][..., None]
    chance = s["uniforms"] * q.gather(2, at)[..., 0] < p[:, :t].gather(2, at)[..., 0]
    ok = torch.where(greedy[:, None], s["drafts"] == best[:, :t], chance)
    lens = s["draft_lens"].long() if s["draft_lens"] is not None else torch.full((b,), t, device=DEV)
    ok &= torch.arange(t, device=DEV) < lens[:, None]
    accepted = ok.long().cumprod(1).sum(1)
    row = torch.arange(b, device=DEV)
    p_row = p[row, accepted]
    q_row = torch.where((accepted < lens)[:, None], q[row, accepted.clamp_max(t - 1)], 0.0)
    rest = (p_row - q_row).clamp_min(0.0)
    weight = torch.where((rest > 0).any(-1, keepdim=True), rest, p_row)
    nxt = torch.where(greedy, best[row, accepted], (weight / s["noise"]).argmax(-1))
    place = torch.arange(t + 1, device=DEV)
    padded = torch.cat([s["drafts"], s["drafts"][:, :1]], 1)
    tokens = torch.where(place < accepted[:, None], padded, -1)
    tokens = torch.where(place == accepted[:, None], nxt[:, None], tokens)
    return tokens, accepted.to(torch.int32)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "attend":
        p, n, t, hq, hk = (case[k] for k in ("prefixes", "questions", "tokens", "q_heads", "kv_heads"))
        b, sv, sf, cap, keep = p * n, case["vision"], case["full"], case["cap"], case["keep"]
        e = 2
        text = _lens_sum(max(case["text_min"], t), cap, b) if cap >= t else b * cap
        byts = 2 * b * t * hq * D * e + p * hk * e * (D * keep + D * case["bias"] + sv * (keep + D) + 2 * sf * D)
        byts += p * sf * case["mask"] + 4 * b + text * hk * 2 * (D + 4 if case["fp8"] else D * e)
        rows = b * t * hq
        flops = 2 * rows * (D * keep + D * case["bias"] + sv * (keep + D) + sf * 2 * D) + 4 * t * hq * text * D
        return {"bytes": byts, "flops": flops}
    if case["op"] == "append":
        b, h, t = case["batch"], case["kv_heads"], case["tokens"]
        rows = h * (_lens_sum(t // 3, t, b) if case["ragged"] else b * t)
        return {"bytes": 2 * rows * (D * TYPES[case["dtype"]].itemsize + D + 4) + 8 * b, "flops": 4 * rows * D}
    if case["op"] == "read":
        b, h, cap = case["batch"], case["kv_heads"], case["cap"]
        rows = h * _lens_sum(case["text_min"], cap, b)
        return {"bytes": 2 * rows * (D + 4) + 2 * b * h * cap * D * TYPES[case["dtype"]].itemsize, "flops": 2 * rows * D}
    b, t, v = case["batch"], case["drafts"], case["vocab"]
    lens = _lens_sum(0, t, b) if case["ragged"] else b * t
    rows = lens + b + (lens if case["logits"] else 0)
    return {"bytes": rows * v * TYPES[case["dtype"]].itemsize + 4 * b * v, "flops": 4 * rows * v + 4 * b * v}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "append": _exact_append, "read": _exact_read, "verify": _exact_verify}[s["op"]](s)


def _exact_attend(s):
    c = s["case"]
    p, n, t, hq, hk = (c[k] for k in ("prefixes", "questions", "tokens", "q_heads", "kv_heads"))
    groups = hq // hk
    q = s["q"].double()
    out = torch.zeros(p * n, t, hq, D, dtype=torch.float64, device=DEV)
    lens = s["lens"].tolist()
    for i in range(p):
        for h in range(hk):
            # the visual Keys at full width: R k + delta_mu has the same product with a query
            vis = s["k_sparse"][i, h].double() @ s["R"][i, h].double().T
            if s["delta_mu"] is not None:
                vis = vis + s["delta_mu"][i, h].double()
            keys, values = torch.cat([s["k_full"][i, h].double(), vis]), torch.cat(
                [s["v_full"][i, h].double(), s["v_sparse"][i, h].double()])
            if s["mask"] is not None:
                take = torch.cat([s["mask"][i].bool(), torch.ones(c["vision"], dtype=torch.bool, device=DEV)])
                keys, values = keys[take], values[take]
            for j in range(i * n, (i + 1) * n):
                kt, vt = s["k_text"][j, h, :lens[j]], s["v_text"][j, h, :lens[j]]
                if s["k_scale"] is not None:
                    kt = kt.view(torch.float8_e4m3fn).double() * s["k_scale"][j, h, :lens[j], None].double()
                    vt = vt.view(torch.float8_e4m3fn).double() * s["v_scale"][j, h, :lens[j], None].double()
                kt, vt = kt.double(), vt.double()
                x = q[j, :, h * groups:(h + 1) * groups].reshape(t * groups, D)
                left = x @ keys.T / math.sqrt(D)
                right = x @ kt.T / math.sqrt(D)
                newest = torch.arange(t, device=DEV).repeat_interleave(groups)[:, None] - (t - 1) + lens[j]
                right = right.masked_fill(torch.arange(lens[j], device=DEV) >= newest, -math.inf)
                w = torch.softmax(torch.cat([left, right], 1), 1)
                o = w[:, :keys.shape[0]] @ values + w[:, keys.shape[0]:] @ vt
                out[j, :, h * groups:(h + 1) * groups] = o.view(t, groups, D)
    return out


def _nearest_e4m3(x):
    """The e4m3 value nearest to x (ties to even; steps of 2^-9 below 2^-6; at most 448), in 64 bits."""
    a = x.abs().clamp_max(E4M3_MAX)
    step = torch.exp2(torch.floor(torch.log2(a.clamp_min(2.0 ** -6))) - 3)
    return torch.copysign((torch.round(a / step) * step).clamp_max(E4M3_MAX), x)


def _exact_append(s):
    out = []
    lens = s["lens"].tolist()
    t = s["case"]["tokens"]
    counts = s["counts"].tolist() if s["counts"] is not None else [t] * len(lens)
    for new, cache, scales in ((s["k_new"], s["k_text"], s["k_scale"]), (s["v_new"], s["v_text"], s["v_scale"])):
        values, scales = cache.view(torch.float8_e4m3fn).double(), scales.double()
        for j, (at, k) in enumerate(zip(lens, counts)):
            x = new[j, :, :k].double()
            scale = x.abs().amax(-1) / E4M3_MAX if k else x.new_zeros(x.shape[:2])
            scale = torch.where(scale > 0, scale, 1.0)
            values[j, :, at:at + k] = _nearest_e4m3(x / scale[..., None])
            scales[j, :, at:at + k] = scale
        out += [values, scales]
    return tuple(out)


def _exact_read(s):
    out = []
    for x, scale in ((s["k_text"], s["k_scale"]), (s["v_text"], s["v_scale"])):
        y = x.view(torch.float8_e4m3fn).double() * scale.double()[..., None]
        for j, n in enumerate(s["lens"].tolist()):
            y[j, :, n:] = 0
        out.append(y)
    return tuple(out)


def _exact_verify(s):
    b, t = s["drafts"].shape
    tokens = torch.full((b, t + 1), -1, dtype=torch.int64)
    accepted = torch.zeros(b, dtype=torch.int32)
    lens = s["draft_lens"].tolist() if s["draft_lens"] is not None else [t] * b
    heat, drafts, chance = s["temperature"].tolist(), s["drafts"].tolist(), s["uniforms"].tolist()
    for j in range(b):
        for i in range(lens[j] + 1):
            x = s["target"][j, i].double()
            p = torch.softmax(x / heat[j], 0) if heat[j] > 0 else None
            rest = p
            if i < lens[j]:
                d = drafts[j][i]
                if p is None:
                    ok = d == int(x.argmax())
                else:
                    if s["draft_logits"] is not None:
                        q = torch.softmax(s["draft_logits"][j, i].double() / heat[j], 0)
                    else:
                        q = torch.zeros_like(p)
                        q[d] = 1
                    ok = chance[j][i] * float(q[d]) < float(p[d])
                    rest = (p - q).clamp_min(0)
                    if not bool((rest > 0).any()):
                        rest = p
                if ok:
                    tokens[j, i] = d
                    continue
            accepted[j] = i
            tokens[j, i] = int(x.argmax()) if p is None else int((rest / s["noise"][j].double()).argmax())
            break
    return tokens, accepted
