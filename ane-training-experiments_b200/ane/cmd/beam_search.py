"""Beam search over a paged cache of the caller (ane.paged), on a small random attention model.

    python -m ane.cmd.beam_search -beams 8 -prompt 100 -steps 40

The prompt runs once.  Every step attends over the beams' shared prompt once for all of them
(PrefixPlan), picks the best continuations on the device, forks their parents' slots into a second
bank (shared pages counted, partly filled ones copied) and frees the first, without waiting for
the device: parents never come to the host.  At the end the live pages are gathered at the pool's
start (compact) and the best beam's are copied into a cache of their own, from which it could
continue.  The model is a stand-in (weights drawn from the seed); the reference has no beam search.
"""
from __future__ import annotations

import argparse
import math
from dataclasses import dataclass

import torch

from ..paged import PAGE, PagedCache, PrefixPlan


@dataclass
class Model:
    """Attention layers x += Wo attend(Wq x, Wk x, Wv x) on RMS-normalised rows, tied embedding."""

    embed: torch.Tensor   # [vocab, dim] f32
    layers: list          # of (wq [dim, heads, hd], wk, wv [dim, kv, hd], wo [heads * hd, dim])
    heads: int
    kv_heads: int
    head_dim: int
    dtype: str


VOCAB = 500


def random_model(seed: int, vocab=VOCAB, dim=128, heads=4, kv_heads=2, head_dim=64, layers=2, dtype="bf16") -> Model:
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = lambda *s: torch.randn(s, generator=g, device="cuda") / math.sqrt(dim)  # noqa: E731
    return Model(3 * w(vocab, dim), [(2 * w(dim, heads, head_dim), 2 * w(dim, kv_heads, head_dim), w(dim, kv_heads, head_dim),
                                      w(heads * head_dim, dim)) for _ in range(layers)], heads, kv_heads, head_dim, dtype)


def rms(x):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5)


def rows(m: Model, tokens, attend):
    """Log-probabilities after each of `tokens`' rows; attend(layer, q, k, v) -> [rows, heads, hd]."""
    x = m.embed[tokens]
    for i, (wq, wk, wv, wo) in enumerate(m.layers):
        h = rms(x)
        q, k, v = (torch.einsum("rd,dhe->rhe", h, w) for w in (wq, wk, wv))
        x = x + attend(i, q, k, v).float().flatten(1) @ wo
    return torch.log_softmax(rms(x) @ m.embed.T, -1)


class Search:
    def __init__(self, m: Model, beams: int, prompt, steps: int):
        self.m, self.beams, self.steps, self.prompt = m, beams, steps, prompt
        n, self.total = len(prompt), len(prompt) + steps
        each = -(-self.total // PAGE)
        # the prompt's slot and two banks of beams; a bank's beams share at least the prompt's pages
        self.cache = PagedCache(m.dtype, len(m.layers), each + 2 * beams * (each - n // PAGE + 1), m.kv_heads, m.head_dim,
                                1 + 2 * beams, each)
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        self.banks = [ints(list(range(1 + b * beams, 1 + (b + 1) * beams))) for b in (0, 1)]
        self.where = self.cache.element_index()
        shared = n // PAGE * PAGE
        plan = lambda slots, r, sizes, prefix: PrefixPlan(self.cache, m.heads, slots, r, sizes, prefix, max_ctx=each * PAGE)  # noqa: E731
        self.first = plan([0], [n], [1], [0])
        self.plans = [plan(b.tolist(), [1] * beams, [beams], [shared]) for b in self.banks]
        self.cache.fork(ints([-1]), ints([0]), ints([0]), ints([n]))

    def write(self, layer, slots, positions, k, v):
        """K and V rows [n, kv, hd] of positions [n] of slots [n] into their pages."""
        page = self.cache.table[slots.long(), (positions // PAGE).long()].long()
        at = self.where[(positions % PAGE).long()]  # [n, hd]
        for b, x in enumerate((k, v)):
            self.cache.pool[layer, page[:, None, None], torch.arange(self.m.kv_heads, device="cuda")[None, :, None], b,
                            at[:, None]] = x.to(self.cache.torch_dtype)

    def run_rows(self, plan, slots, positions, tokens, ctx):
        def attend(layer, q, k, v):
            self.write(layer, slots, positions, k, v)
            return plan.attend(layer, q.to(self.cache.torch_dtype), ctx)
        return rows(self.m, tokens, attend)

    def run(self):
        """(tokens [beams, steps], log-probabilities [beams]), best first."""
        n, B, V = len(self.prompt), self.beams, self.m.embed.shape[0]
        full = lambda x, k=B: torch.full((k,), x, dtype=torch.int32, device="cuda")  # noqa: E731
        at = torch.arange(n, dtype=torch.int32, device="cuda")
        lp = self.run_rows(self.first, torch.zeros_like(at), at, torch.tensor(self.prompt, device="cuda"), full(n, 1))[-1]
        score, token = lp.topk(B)
        out = token[:, None]
        self.cache.fork(full(0), self.banks[0], full(n), full(n + 1))
        bank = 0
        for pos in range(n, self.total - 1):
            slots = self.banks[bank]
            lp = self.run_rows(self.plans[bank], slots, full(pos), token, full(pos + 1))
            score, best = (score[:, None] + lp).flatten().topk(B)
            parent, token = best // V, best % V
            out = torch.cat([out[parent], token[:, None]], 1)
            self.cache.fork(slots[parent], self.banks[1 - bank], full(pos + 1), full(pos + 2))
            self.cache.free(slots)
            bank = 1 - bank
        self.bank = bank
        return out, score

    def keep_best(self) -> PagedCache:
        """The best beam's pages, gathered from the compacted pool into a cache of their own."""
        self.cache.compact()
        slot = self.banks[self.bank][:1]
        room = torch.full((1,), self.total, dtype=torch.int32, device="cuda")
        each = -(-self.total // PAGE)
        kept = PagedCache(self.m.dtype, len(self.m.layers), each, self.m.kv_heads, self.m.head_dim, 1, each)
        zero = torch.zeros_like(slot)
        kept.fork(zero - 1, zero, zero, room)
        self.cache.copy(self.cache.table[slot.long()][0].contiguous(), kept.table[0], to=kept)
        kept.check()
        self.cache.check()
        return kept


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(prog="beam_search", description=__doc__.split("\n", 1)[0])
    ap.add_argument("-beams", type=int, default=8)
    ap.add_argument("-prompt", type=int, default=100, help="prompt length (random tokens)")
    ap.add_argument("-steps", type=int, default=40)
    ap.add_argument("-seed", type=int, default=1)
    ap.add_argument("-dtype", choices=("fp16", "bf16"), default="bf16")
    a = ap.parse_args(argv)
    if min(a.beams, a.prompt, a.steps) <= 0:
        ap.error("-beams, -prompt and -steps must be positive")
    if a.beams > VOCAB:
        ap.error(f"-beams: the first step has {VOCAB} continuations")
    m = random_model(a.seed, dtype=a.dtype)
    g = torch.Generator().manual_seed(a.seed)
    s = Search(m, a.beams, torch.randint(0, m.embed.shape[0], (a.prompt,), generator=g).tolist(), a.steps)
    tokens, score = s.run()
    kept = s.keep_best()
    live = s.cache.n_pages - int(s.cache.n_free.item())
    print(f"beams={a.beams} prompt={a.prompt} steps={a.steps} logprob={float(score[0]):.4f}")
    print("tokens=" + " ".join(str(t) for t in tokens[0].tolist()))
    print(f"pages live={live} separate={(a.beams + 1) * -(-s.total // PAGE)} kept={kept.n_pages - int(kept.n_free.item())}")
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
