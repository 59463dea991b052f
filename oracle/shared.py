"""Float64 definitions of the shared-prefix operators (test infrastructure).

``shared_decode`` also returns A = sum_i w_i |v_i| for every output, w the
softmax weights: what a relative error of the weights can move an output by.
"""
from __future__ import annotations

import math

import torch

from oracle.fp8 import round_e4m3


def e4m3_values(t: torch.Tensor) -> torch.Tensor:
    t = t if t.dtype == torch.float8_e4m3fn else t.view(torch.float8_e4m3fn)
    return t.float().double()


def shared_decode(q, R_partial, delta_mu, k_full, v_full, mask_full, k_sparse, v_sparse, k_text, v_text, text_lens,
                  num_kv_groups, k_scale=None, v_scale=None):
    """(out, A), both [B, T, H_q, D] float64, on the CPU."""
    cpu = lambda t: None if t is None else t.detach().cpu()  # noqa: E731
    q, R, dm, kf, vf, mask, ks, vs, kt, vt, lens, ksc, vsc = map(cpu, (
        q, R_partial, delta_mu, k_full, v_full, mask_full, k_sparse, v_sparse, k_text, v_text, text_lens, k_scale,
        v_scale))
    b, t, hq, d = q.shape
    p, cap, g = R.shape[0], kt.shape[2], num_kv_groups
    out = torch.zeros(b, t, hq, d, dtype=torch.float64)
    mag = torch.zeros_like(out)
    for j in range(b):
        i = j // (b // p)
        n = min(max(int(lens[j]), 0), cap)
        there = torch.ones(kf.shape[2], dtype=torch.bool) if mask is None else mask[i] != 0
        for x in range(t):
            seen = max(0, n - (t - 1 - x))
            for h in range(hq):
                kv = h // g
                qq = q[j, x, h].double()
                text_k = kt[j, kv, :seen]
                text_v = vt[j, kv, :seen]
                if ksc is not None:
                    text_k = e4m3_values(text_k) * ksc[j, kv, :seen, None].double()
                    text_v = e4m3_values(text_v) * vsc[j, kv, :seen, None].double()
                logits = [kf[i, kv].double()[there] @ qq,
                          ks[i, kv].double() @ (R[i, kv].double().T @ qq) + (0.0 if dm is None else dm[i, kv].double() @ qq),
                          text_k.double() @ qq]
                s = torch.cat(logits) / math.sqrt(d)
                v = torch.cat([vf[i, kv].double()[there], vs[i, kv].double(), text_v.double()])
                if s.numel() == 0:
                    continue
                w = torch.softmax(s, 0)
                out[j, x, h], mag[j, x, h] = w @ v, w @ v.abs()
    return out, mag


def quantize_rows(x: torch.Tensor):
    """(e4m3 values float64, scale float32) of rows x[..., D]: fp32 scale and
    division as the device does them, then the nearest e4m3 value."""
    x = x.detach().cpu().float()
    fin = torch.where(torch.isfinite(x), x.abs(), 0.0)
    amax = fin.amax(-1)
    scale = torch.where(amax > 0, (amax / 448.0).clamp_min(2.0 ** -126), 1.0)
    y = (x / scale[..., None]).clamp(-448.0, 448.0)
    val = torch.from_numpy(round_e4m3(torch.nan_to_num(y, nan=0.0).numpy()))
    return torch.where(torch.isnan(y), math.nan, val), scale


def verify(target, drafts, draft_logits, uniforms, noise, temperature, draft_lens=None):
    """(tokens, accepted, margin): margin[b] is the smallest relative distance of
    any decision of question b from going the other way."""
    cpu = lambda t: None if t is None else t.detach().cpu()  # noqa: E731
    target, drafts, draft_logits, uniforms, noise, temperature, draft_lens = map(cpu, (
        target, drafts, draft_logits, uniforms, noise, temperature, draft_lens))
    b, t1, v = target.shape
    t = t1 - 1
    tokens = torch.full((b, t1), -1, dtype=torch.int64)
    accepted = torch.zeros(b, dtype=torch.int32)
    margin = torch.full((b,), math.inf, dtype=torch.float64)

    def soft(x, heat):
        x = x.double()
        if not bool((x > -math.inf).any()):
            return torch.zeros_like(x)
        return torch.softmax(x / heat, 0)

    for j in range(b):
        heat = float(temperature[j])
        n = t if draft_lens is None else min(max(int(draft_lens[j]), 0), t)
        for k in range(n + 1):
            x = target[j, k]
            first = int(torch.nonzero(x == x.max())[0]) if bool((x > -math.inf).any()) else 0
            p = soft(x, heat) if heat > 0 else None
            weight = p
            if k < n:
                d = int(drafts[j, k])
                valid = 0 <= d < v
                if p is None:
                    ok = valid and d == first
                else:
                    if draft_logits is not None:
                        qq = soft(draft_logits[j, k], heat)
                    else:
                        qq = torch.zeros_like(p)
                        if valid:
                            qq[d] = 1.0
                    ok = False
                    if valid:
                        a, c = float(uniforms[j, k]) * float(qq[d]), float(p[d])
                        ok = a < c
                        if a or c:
                            margin[j] = min(margin[j], abs(a - c) / max(a, c))
                    weight = (p - qq).clamp_min(0)
                    if not bool((weight > 0).any()):
                        weight = p
                if ok:
                    tokens[j, k] = d
                    continue
            accepted[j] = k
            if p is None:
                tokens[j, k] = first
            else:
                race = weight / noise[j].double()
                top = torch.topk(race, min(2, v)).values
                if float(top[0]) > 0 and v > 1:
                    margin[j] = min(margin[j], float((top[0] - top[1]) / top[0]))
                tokens[j, k] = int(torch.nonzero(race == race.max())[0])
            break
    return tokens, accepted, margin
