"""Many questions on shared images, with drafted tokens: the shared-prefix operators
run together.

A random-init decoder (``llama_e2e.RandomLlamaDecoder``) prefills P images once.  Every
image then serves N questions at the same time: a question owns only its text cache
(e4m3 by default), and every step

    appends   the new tokens' Keys and Values to the text caches  (append_text)
    attends   over the shared prefix and the question's own text  (rotatek_shared_decode)
    verifies  the drafted tokens and draws the next one           (verify_drafts)

The questions themselves go in as one ragged step (their tokens attend causally, as
drafts do).  Drafts come from the decoder's own first ``draft_layers`` layers -- they
share its caches, which the checking step overwrites with the same rows -- or, with
``draft_layers = 0``, repeat what followed the last token earlier in the question
(proposals without probabilities).

    python -m rotatek_b200.shared_e2e [--images P] [--questions N] [--drafts T] ...
"""
from __future__ import annotations

import argparse
import time
from dataclasses import dataclass
from typing import List, Optional

import torch
import torch.nn.functional as F

from rotatek_b200.cache import SharedPrefixCache
from rotatek_b200.kernels import verify_drafts
from rotatek_b200.llama_e2e import DecoderConfig, RandomLlamaDecoder


@dataclass
class ServingConfig:
    questions: int = 8           # per image
    capacity: int = 256          # text tokens of a question
    drafts: int = 4              # tokens drafted per step
    draft_layers: int = 2        # layers that draft; 0: propose by lookup
    temperature: float = 0.0     # 0: greedy
    fp8: bool = True             # text caches in e4m3


class SharedQuestions:
    """Greedy or sampled generation for the questions of prefilled images."""

    def __init__(self, model: RandomLlamaDecoder, cfg: ServingConfig, seed: int = 0):
        """``model`` has been prefilled: row p of its batch is image p."""
        if model.cache is None:
            raise ValueError("prefill the model first")
        if not 0 <= cfg.draft_layers <= model.cfg.layers:
            raise ValueError(f"draft_layers must be in [0, {model.cfg.layers}]")
        self.model, self.cfg = model, cfg
        self.cache = SharedPrefixCache(model.cache, cfg.questions, cfg.capacity, cfg.fp8)
        self.batch, self.device = self.cache.batch, model.device
        self.gen = torch.Generator(device=self.device).manual_seed(seed)
        self.temperature = torch.full((self.batch,), cfg.temperature, device=self.device)
        # RoPE of every position a question can reach
        c, last = model.cfg, model.seq_len + cfg.capacity
        inv = 1.0 / (c.rope_theta ** (torch.arange(0, c.head_dim, 2, device=self.device, dtype=torch.float32) / c.head_dim))
        ang = torch.arange(last, device=self.device, dtype=torch.float32)[:, None] * inv
        ang = torch.cat([ang, ang], -1)
        self.cos, self.sin = ang.cos().to(c.dtype), ang.sin().to(c.dtype)
        self.last: Optional[torch.Tensor] = None       # [B] the token that the next step starts from
        self.history: List[torch.Tensor] = []           # emitted [B, T + 1] tokens, -1 padded

    # ------------------------------------------------------------------ model
    @torch.no_grad()
    def forward(self, tokens: torch.Tensor, start: torch.Tensor, layers: int, counts=None, ahead: int = 0) -> torch.Tensor:
        """Logits [B, T, V] of T new tokens per question that follow ``start`` [B]
        int32 stored ones, through the first ``layers`` layers; their Keys and Values
        are stored behind ``start``, which is at most ``ahead`` past the lengths.
        ``counts``: tokens[b, :counts[b]] are real, the lengths end at start + counts,
        and the logits of real tokens alone mean anything."""
        m, c = self.model, self.model.cfg
        b, t = tokens.shape
        self.cache.need_room(ahead + t)          # the RoPE tables end where the caches do
        lens = start + (t if counts is None else counts)
        # query i of the T attends to rows < lens - (T - 1 - i): with ragged counts the real
        # tokens are moved to the end, so that the last one is the last query
        shift = torch.zeros_like(start) if counts is None else t - counts
        order = (torch.arange(t, device=self.device) - shift[:, None]).clamp_min(0)
        pos = m.seq_len + start[:, None] + order
        x = m.embed[tokens.gather(1, order.long())]
        cos, sin = self.cos[pos.long()][:, None], self.sin[pos.long()][:, None]
        groups = c.heads // c.kv_heads
        for li in range(layers):
            L = m.layers[li]
            q, k, v = m._qkv(L, x)
            q, k = m._rope(q, cos, sin), m._rope(k, cos, sin)
            if counts is None:
                self.cache.append(k, v, li, at=start, ahead=ahead)
            else:                     # real tokens first, as they are stored
                back = (torch.arange(t, device=self.device) + shift[:, None]).clamp_max(t - 1)
                back = back[:, None, :, None].expand(b, c.kv_heads, t, c.head_dim).long()
                self.cache.append(k.gather(2, back), v.gather(2, back), li, counts=counts, at=start, ahead=ahead)
            o = self.cache.attend(q.transpose(1, 2), li, lens, groups)
            x = x + F.linear(o.reshape(b, t, -1), L["wo"])
            x = x + m._mlp(L, x)
        return F.linear(m._rms(x, m.norm), m.lm_head)

    # ------------------------------------------------------------------ steps
    def _noise(self, *shape) -> torch.Tensor:
        return torch.empty(*shape, device=self.device).exponential_(generator=self.gen).clamp_min_(1e-20)

    def _draw(self, logits: torch.Tensor) -> torch.Tensor:
        """The next token of each question from logits [B, V]: a verification of no drafts."""
        b = logits.shape[0]
        none = torch.empty(b, 0, dtype=torch.int64, device=self.device)
        tokens, _ = verify_drafts(logits[:, None], none, None, none.float(), self._noise(b, logits.shape[-1]),
                                  self.temperature)
        return tokens[:, 0]

    def ask(self, tokens: torch.Tensor, counts: torch.Tensor) -> torch.Tensor:
        """Put the questions in: tokens [B, T], the first counts[b] (int32, at least 1) of
        row b; returns the first answer token of each."""
        self.cache.need_room(tokens.shape[1])
        logits = self.forward(tokens, self.cache.lens, self.model.cfg.layers, counts)
        self.cache.advance(counts, tokens.shape[1])
        self.last = self._draw(logits[:, -1].contiguous())
        self.seen = torch.cat([tokens.masked_fill(torch.arange(tokens.shape[1], device=self.device) >= counts[:, None], -1),
                               self.last[:, None]], 1)
        self.history = [self.last[:, None]]
        return self.last

    def _propose(self):
        """(drafts [B, T], their logits [B, T, V] or None) from the state before the step."""
        cfg, t = self.cfg, self.cfg.drafts
        if t == 0:
            return torch.empty(self.batch, 0, dtype=torch.int64, device=self.device), None
        if cfg.draft_layers == 0:
            # what followed the latest earlier occurrence of the last token (itself if none)
            s = self.seen
            place = torch.arange(s.shape[1], device=self.device)
            newest = torch.where(s >= 0, place, -1).amax(1)
            hit = (s == self.last[:, None]) & (place < newest[:, None])
            found = torch.where(hit, place, -1).amax(1)
            at = (found[:, None] + 1 + torch.arange(t, device=self.device)).clamp_max(s.shape[1] - 1)
            drafts = torch.where(found[:, None] >= 0, s.gather(1, at), self.last[:, None])
            return torch.where(drafts >= 0, drafts, self.last[:, None]), None
        token, drafts, logits = self.last, [], []
        for i in range(t):
            out = self.forward(token[:, None], self.cache.lens + i, cfg.draft_layers, ahead=i)[:, 0]
            token = self._draw(out.contiguous())
            drafts.append(token)
            logits.append(out)
        return torch.stack(drafts, 1), torch.stack(logits, 1)

    @torch.no_grad()
    def step(self):
        """Draft, check and advance once: (tokens [B, T + 1] -- the new answer tokens, -1 past
        them -- and accepted [B])."""
        t = self.cfg.drafts
        self.cache.need_room(t + 1)
        drafts, draft_logits = self._propose()
        logits = self.forward(torch.cat([self.last[:, None], drafts], 1), self.cache.lens, self.model.cfg.layers)
        tokens, accepted = verify_drafts(logits, drafts, draft_logits,
                                         torch.rand(self.batch, t, device=self.device, generator=self.gen),
                                         self._noise(self.batch, logits.shape[-1]), self.temperature)
        self.cache.advance(accepted + 1, t + 1)
        self.last = tokens.gather(1, accepted.long()[:, None])[:, 0]
        self.seen = torch.cat([self.seen, tokens], 1)
        self.history.append(tokens)
        return tokens, accepted

    def answers(self) -> List[List[int]]:
        """The answer tokens of every question so far (one synchronisation)."""
        return [[int(x) for x in row if x >= 0] for row in torch.cat(self.history, 1).tolist()]


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--images", type=int, default=2)
    ap.add_argument("--questions", type=int, default=8, help="questions per image")
    ap.add_argument("--vision", type=int, default=4096, help="visual tokens of an image")
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--drafts", type=int, default=4)
    ap.add_argument("--draft-layers", type=int, default=2)
    ap.add_argument("--steps", type=int, default=16)
    ap.add_argument("--temperature", type=float, default=0.0)
    ap.add_argument("--text16", action="store_true", help="text caches in 16 bits")
    a = ap.parse_args(argv)
    cfg = DecoderConfig(layers=a.layers, hidden=3584, heads=28, kv_heads=4, ffn=4096, vision=a.vision, text=16,
                        max_new_tokens=0)
    model = RandomLlamaDecoder(cfg, "cuda")
    model.prefill(model.prompt_embeddings(a.images))
    s = SharedQuestions(model, ServingConfig(questions=a.questions, capacity=64 + (a.drafts + 1) * (a.steps + 1),
                                             drafts=a.drafts, draft_layers=a.draft_layers, temperature=a.temperature,
                                             fp8=not a.text16))
    counts = 8 + torch.arange(s.batch, device="cuda", dtype=torch.int32) % 25
    s.ask(torch.randint(0, cfg.vocab, (s.batch, 32), device="cuda"), counts)
    s.step()
    torch.cuda.synchronize()
    begun, taken = time.perf_counter(), []
    for _ in range(a.steps):
        taken.append(s.step()[1])
    torch.cuda.synchronize()
    took = time.perf_counter() - begun
    accepted = torch.stack(taken).float().mean().item()
    print(f"{s.batch} questions on {a.images} images of {a.vision} visual tokens: {accepted:.2f} of {a.drafts} drafts "
          f"accepted, {(accepted + 1) * s.batch * a.steps / took:.0f} tokens/s, {took / a.steps * 1e3:.2f} ms per step")


if __name__ == "__main__":
    main()
