"""Attention over shared prefixes (ane.paged.PrefixPlan) against the definition in 64 bits.

Tolerance, from the arithmetic and fixed before the first run.  With u the unit roundoff of the
cache's type, A = sum_t p_t |v_t| the row's weighted mean of |v|: the output is rounded once
(u |o|) and a softmax weight may be carried in the type (u A).  A score is a 32-bit dot product
of head_dim exact products and two more 32-bit roundings, so it is off by at most
ds = head_dim 2^-24 scale sum_i |q_i k_i| + 2^-22 |score| (natural units); the row sum adds at
most ctx 2^-24 and the exponential 2^-21.  So |lse| is off by at most
e = max_t ds + ctx 2^-24 + 2^-21 + 2^-23 |lse|, and the output by u |o| + u A + 2 e A + the type's
smallest step."""
import math

import numpy as np
import pytest

from ane import _abi

pytestmark = pytest.mark.gpu

U = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"fp16": 2.0 ** -24, "bf16": 2.0 ** -133}


class Batch:
    """A pool whose unused values are NaN, with sequences in groups at scattered pages."""

    def __init__(self, dtype, kv, hd, sizes, prefixes, ctx, rows, heads, layers=2, seed=0, spare=7, extra_pages=2, spread=1.0):
        import torch
        from ane.paged import PagedCache, PrefixPlan
        rng = np.random.default_rng(seed)
        n = len(ctx)
        assert sum(sizes) == n == len(rows)
        self.group = np.repeat(np.arange(len(sizes)), sizes)
        prefix = np.repeat(prefixes, sizes)
        need = [max(0, -(-int(c) // 16) - int(p) // 16) for c, p in zip(ctx, prefix)]
        pages = sum(need) + sum(p // 16 for p in prefixes) + spare
        most = max(max(int(p) // 16 + k for p, k in zip(prefix, need)), 1) + extra_pages
        slots = rng.permutation(n + 3)[:n]
        self.cache = PagedCache(dtype, layers, pages, kv, hd, n + 3, most)
        ids = rng.permutation(pages)
        table = np.full((n + 3, most), -1, np.int32)
        at = 0
        first = {}
        for s in range(n):
            g = int(self.group[s])
            if g not in first:
                first[g] = ids[at:at + prefixes[g] // 16]
                at += prefixes[g] // 16
            table[slots[s], : prefixes[g] // 16] = first[g]
            table[slots[s], prefixes[g] // 16: prefixes[g] // 16 + need[s]] = ids[at:at + need[s]]
            at += need[s]
        self.cache.table.copy_(torch.from_numpy(table))
        self.dtype, self.kv, self.hd, self.heads, self.layer = dtype, kv, hd, heads, layers - 1
        self.ctx, self.rows, self.slots, self.table, self.prefix = list(ctx), list(rows), slots, table, prefix
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.cache.pool.fill_(float("nan"))
        where = self.cache.element_index()
        self.k, self.v = [], []
        shared = {}
        for s in range(n):
            c, gi = int(ctx[s]), int(self.group[s])
            k = torch.randn((max(c, int(prefix[s])), kv, hd), generator=g, device="cuda").mul_(spread).to(self.cache.torch_dtype)
            v = torch.randn((max(c, int(prefix[s])), kv, hd), generator=g, device="cuda").to(self.cache.torch_dtype)
            if gi in shared:
                k[: prefix[s]], v[: prefix[s]] = shared[gi]
            else:
                shared[gi] = (k[: prefix[s]].clone(), v[: prefix[s]].clone())
            for t0 in range(0, k.shape[0], 16):
                page = int(table[slots[s], t0 // 16]) if t0 // 16 < most else -1
                if page < 0:
                    continue
                m = min(16, k.shape[0] - t0)
                for h in range(kv):
                    for b, x in ((0, k), (1, v)):
                        self.cache.pool[self.layer, page, h, b][where[:m].reshape(-1)] = x[t0:t0 + m, h].reshape(-1)
            self.k.append(k)
            self.v.append(v)
        self.q = torch.randn((int(sum(rows)), heads, hd), generator=g, device="cuda").to(self.cache.torch_dtype)
        self.d_ctx = torch.tensor(list(ctx), dtype=torch.int32, device="cuda")
        self.plan = PrefixPlan(self.cache, heads, slots, rows, sizes, prefixes, max_ctx=most * 16)

    def run(self, **kw):
        import torch
        lse = torch.full((self.q.shape[0], self.heads), 7.0, device="cuda")
        out = self.plan.attend(self.layer, kw.pop("q", self.q), kw.pop("ctx", self.d_ctx), lse=lse, **kw)
        self.cache.check()
        return out, lse

    def want(self, scale=None):
        """(o, lse, tolerance of o, tolerance of lse) in 64 bits."""
        import torch
        scale = self.hd ** -0.5 if scale is None else scale
        gq, at = self.heads // self.kv, 0
        got = [[], [], [], []]
        u = U[self.dtype]
        for s, (c, r) in enumerate(zip(self.ctx, self.rows)):
            q = self.q[at:at + r].double()
            at += r
            k = self.k[s][:c].double().repeat_interleave(gq, 1)
            v = self.v[s][:c].double().repeat_interleave(gq, 1)
            x = torch.einsum("rhd,thd->rht", q, k) * scale
            ds = self.hd * 2.0 ** -24 * scale * torch.einsum("rhd,thd->rht", q.abs(), k.abs()) + 2.0 ** -22 * x.abs()
            t = torch.arange(c, device="cuda")
            seen = t[None] <= (c - r + torch.arange(r, device="cuda"))[:, None]
            x = x.masked_fill(~seen[:, None], -math.inf)
            ds = ds.masked_fill(~seen[:, None], 0.0)
            none = ~seen.any(1) if c else torch.ones(r, dtype=torch.bool, device="cuda")
            lse = torch.logsumexp(x, -1) if c else torch.full((r, self.heads), -math.inf, dtype=torch.float64, device="cuda")
            p = torch.where(none[:, None, None], 0.0, torch.exp(x - torch.where(none[:, None], 0.0, lse)[..., None]))
            o, mean = torch.einsum("rht,thd->rhd", p, v), torch.einsum("rht,thd->rhd", p, v.abs())
            e = (ds.amax(-1) if c else torch.zeros_like(lse)) + c * 2.0 ** -24 + 2.0 ** -21
            e = e + torch.where(none[:, None], 0.0, 2.0 ** -23 * lse.abs())
            got[0].append(o)
            got[1].append(lse)
            got[2].append(u * o.abs() + u * mean + 2 * e[..., None] * mean + TINY[self.dtype])
            got[3].append(e)
        return [torch.cat(g) for g in got]

    def check(self, out, lse, scale=None):
        import torch
        o, l, to, tl = self.want(scale)
        d = (out.double() - o).abs()
        assert bool((d <= to).all()), f"out is {float((d / to).max()):.3g} of its tolerance off"
        assert torch.equal(torch.isinf(lse), torch.isinf(l)) and bool((lse[torch.isinf(l)] < 0).all())
        d = (lse.double() - l).abs()[~torch.isinf(l)]
        assert bool((d <= tl[~torch.isinf(l)]).all()), f"lse is off by {float(d.max()):.3g}"


def lengths(rng, prefixes, sizes, suffix, rows=1):
    return [int(p + max(rows, rng.integers(1, suffix + 1))) for p, k in zip(prefixes, sizes) for _ in range(k)]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("heads,kv,hd", [(12, 12, 64), (16, 8, 128), (6, 2, 128), (7, 1, 64), (8, 1, 128), (16, 1, 64), (12, 1, 128)])
def test_one_token_each(dtype, heads, kv, hd):
    rng = np.random.default_rng(heads + hd)
    sizes, prefixes = [5, 1, 9], [160, 48, 16]
    b = Batch(dtype, kv, hd, sizes, prefixes, lengths(rng, prefixes, sizes, 70), [1] * 15, heads, seed=heads)
    b.check(*b.run())


@pytest.mark.parametrize("size", [1, 2, 3, 4, 8, 17, 64, 65, 130])
def test_group_sizes_around_a_tile(size):
    rng = np.random.default_rng(size)
    b = Batch("bf16", 2, 128, [size], [208], lengths(rng, [208], [size], 40), [1] * size, 4, layers=1, seed=size)
    b.check(*b.run())


@pytest.mark.parametrize("prefix", [0, 16, 48, 64, 80, 1024, 2000, 4112])
@pytest.mark.parametrize("hd,heads,kv", [(64, 4, 2), (128, 8, 2)])
def test_prefix_lengths(prefix, hd, heads, kv):
    rng = np.random.default_rng(prefix)
    b = Batch("fp16", kv, hd, [6], [prefix], lengths(rng, [prefix], [6], 33), [1] * 6, heads, layers=1, seed=prefix)
    b.check(*b.run())


@pytest.mark.parametrize("suffix", [1, 15, 16, 17, 64, 65, 511, 513, 1500])
def test_own_positions(suffix):
    ctx = [96 + suffix, 96 + max(1, suffix // 2), 97, 96 + suffix]
    b = Batch("bf16", 2, 64, [4], [96], ctx, [1] * 4, 6, layers=1, seed=suffix)
    b.check(*b.run())


@pytest.mark.parametrize("dtype,heads,kv,hd", [("bf16", 16, 8, 128), ("fp16", 3, 3, 64), ("bf16", 7, 1, 128), ("fp16", 6, 2, 64)])
@pytest.mark.parametrize("rows", [2, 5, 17, 64, 129, 200])
def test_several_rows_each(dtype, heads, kv, hd, rows):
    rng = np.random.default_rng(rows)
    sizes, prefixes = [3, 2], [112, 64]
    each = [rows, 1, max(1, rows // 3), rows, 0]
    ctx = [int(p + r + rng.integers(0, 30)) for p, r in zip([112] * 3 + [64] * 2, each)]
    b = Batch(dtype, kv, hd, sizes, prefixes, ctx, each, heads, layers=1, seed=rows)
    b.check(*b.run())


@pytest.mark.parametrize("dtype,heads,kv,hd", [("bf16", 8, 4, 128), ("fp16", 8, 4, 64)])
def test_long_ranges_of_many_rows(dtype, heads, kv, hd):
    # enough work an item that two row tiles share a CTA: more than 128 score rows a kv head, 28 steps
    rng = np.random.default_rng(hd)
    rows = [int(r) for r in rng.integers(65, 129, 38)]
    b = Batch(dtype, kv, hd, [1] * 38, [0] * 38, [int(c) for c in rng.integers(1700, 1800, 38)], rows, heads, layers=1, seed=hd)
    b.check(*b.run())


@pytest.mark.parametrize("prefix", [1040, 6160])
def test_many_rows_on_one_long_prefix(prefix):
    rng = np.random.default_rng(prefix)
    b = Batch("bf16", 8, 64, [20], [prefix], lengths(rng, [prefix], [20], 90, 40), [40] * 20, 16, layers=1, seed=prefix)
    b.check(*b.run())


@pytest.mark.parametrize("rows", [1, 40])
def test_rows_that_see_nothing_or_little(rows):
    # idle places, a context shorter than the rows, one inside the prefix, one of a single position
    ctx = [0, 112 + rows, max(0, rows - 3), 100, 1, 0, 16]
    b = Batch("bf16", 2, 128, [5, 2], [112, 0], ctx, [rows] * 7, 4, seed=5)
    out, lse = b.run()
    b.check(out, lse)
    assert bool((out[:rows] == 0).all()) and bool((lse[:rows] == -math.inf).all())


def test_no_prefix_anywhere_and_all_idle():
    b = Batch("fp16", 1, 64, [1] * 4, [0] * 4, [3, 700, 1, 20], [1] * 4, 8, seed=2)
    b.check(*b.run())
    b = Batch("fp16", 1, 64, [4], [32], [0] * 4, [1] * 4, 2, seed=3)
    out, lse = b.run()
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


def test_large_scores_and_scale():
    # scores of some hundreds: one position takes all the weight; then an explicit small scale
    b = Batch("bf16", 2, 128, [9], [176], [200] * 9, [1] * 9, 4, seed=4, spread=30.0)
    b.check(*b.run())
    b.check(*b.run(scale=0.01), scale=0.01)


@pytest.mark.parametrize("rows", [1, 33])
def test_strided_queries_and_outputs(rows):
    import torch
    b = Batch("bf16", 2, 64, [3], [64], [64 + rows + i for i in range(3)], [rows] * 3, 4, seed=6)
    n = 3 * rows
    wide = torch.full((4, n, 3 * 64), float("nan"), dtype=torch.bfloat16, device="cuda")  # head-major, in a wider row
    wide[:, :, 64:128] = b.q.transpose(0, 1)
    out = torch.full((n, 5, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    got, lse = b.run(q=wide.transpose(0, 1)[:, :, 64:128], out=out[:, :4])
    b.check(got, lse)
    assert bool((out[:, 4] == 3.0).all())


def test_same_bits_again_on_another_stream_and_in_a_graph():
    import torch
    rng = np.random.default_rng(9)
    b = Batch("bf16", 2, 128, [20, 3], [512, 64], lengths(rng, [512, 64], [20, 3], 300), [1] * 23, 8, layers=1, seed=9)
    a, la = b.run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c, lc = b.run()
    s.synchronize()
    assert torch.equal(a, c) and torch.equal(la, lc)
    out = torch.zeros_like(a)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        b.plan.attend(b.layer, b.q, b.d_ctx, out=out)
    for _ in range(2):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, a)


def test_contexts_grow_under_one_plan():
    # the plan's bound is the table's width: the same plan serves the steps of a decode loop
    import torch
    b = Batch("fp16", 2, 64, [6], [64], [64 + 90 + i for i in range(6)], [1] * 6, 6, seed=11)
    full = list(b.ctx)
    for c in ([65, 66, 80, 81, 64 + 64, 64 + 65], [64] * 6, full):
        b.ctx = c
        b.check(*b.run(ctx=torch.tensor(c, dtype=torch.int32, device="cuda")))


def test_a_plan_serves_every_layer_and_pools_past_32_bit_offsets():
    import torch
    from ane.paged import PagedCache, PrefixPlan
    n = 36_000  # x 64 KiB x 2 layers = 4.7 GB
    c = PagedCache("bf16", 2, n, 8, 128, 2, 4)
    ids = [n - 1, 5, n - 2, n - 3]
    c.table[0] = torch.tensor(ids, dtype=torch.int32)
    c.table[1] = torch.tensor([n - 1, 5, 9, 0], dtype=torch.int32)
    small = PagedCache("bf16", 2, 8, 8, 128, 2, 4)
    small.table[0] = torch.tensor([0, 1, 2, 3], dtype=torch.int32)
    small.table[1] = torch.tensor([0, 1, 4, 5], dtype=torch.int32)
    small.pool.normal_()
    for i, p in enumerate(ids + [9, 0]):
        c.pool[:, p] = small.pool[:, i]
    q = torch.randn(2, 16, 128, device="cuda").bfloat16()
    ctx = torch.tensor([60, 50], dtype=torch.int32, device="cuda")
    for layer in (0, 1):
        got = [PrefixPlan(x, 16, [0, 1], [1, 1], [2], [32], 64).attend(layer, q, ctx) for x in (c, small)]
        c.check()
        assert torch.equal(*got)


def test_bad_pages_and_contexts_are_reported():
    import torch
    b = Batch("bf16", 1, 64, [3], [32], [40, 50, 60], [1] * 3, 2, seed=12)
    table = b.cache.table.clone()
    for slot, entry in ((b.slots[1], 2), (b.slots[0], 0)):
        for bad in (-1, b.cache.n_pages):
            b.cache.table.copy_(table)
            b.cache.table[:, 0] = bad if entry == 0 else b.cache.table[:, 0]
            b.cache.table[int(slot), entry] = bad
            with pytest.raises(_abi.LLMError) as e:
                b.run()
            assert e.value.code == _abi.LLM_ERR_DEVICE and "bad page" in str(e.value)
    b.cache.table.copy_(table)
    with pytest.raises(_abi.LLMError) as e:
        b.run(ctx=torch.tensor([40, 10_000, 60], dtype=torch.int32, device="cuda"))
    assert e.value.code == _abi.LLM_ERR_INVALID
    b.check(*b.run())


def test_refused_arguments():
    import torch
    from ane.paged import PrefixPlan
    b = Batch("bf16", 2, 64, [2], [32], [40, 50], [1, 1], 4, seed=13)
    c = b.cache

    def refused(f, code=_abi.LLM_ERR_INVALID):
        with pytest.raises(_abi.LLMError) as e:
            f()
        assert e.value.code == code
    for args in [(3, [0, 1], [1, 1], [2], [32], 64), (4, [0, 1], [1, 1], [2], [31], 64), (4, [0, 1], [1, 1], [2], [80], 64),
                 (4, [0, 1], [1, 1], [1], [32], 64), (4, [0, -1], [1, 1], [2], [32], 64), (4, [0, 1], [1, -1], [2], [32], 64),
                 (4, [0, 1], [1, 1], [2], [32], 0), (4, [0, 1], [1], [2], [32], 64), (4, [], [], [], [], 64), (0, [0], [1], [1], [0], 64)]:
        refused(lambda: PrefixPlan(c, *args))
    refused(lambda: PrefixPlan(c, 4, [0, 99], [1, 1], [2], [32], 64).attend(0, b.q, b.d_ctx))
    for q in (b.q.float(), b.q[:1], b.q[:, :3], b.q.cpu(), b.q.transpose(1, 2).contiguous().transpose(1, 2)):
        refused(lambda: b.plan.attend(0, q, b.d_ctx))
    refused(lambda: b.plan.attend(2, b.q, b.d_ctx))
    refused(lambda: b.plan.attend(-1, b.q, b.d_ctx))
    refused(lambda: b.plan.attend(0, b.q, b.d_ctx.long()))
    refused(lambda: b.plan.attend(0, b.q, b.d_ctx[:1]))
    refused(lambda: b.plan.attend(0, b.q, b.d_ctx, scale=math.inf))
    refused(lambda: b.plan.attend(0, b.q, b.d_ctx, lse=torch.empty(2, 3, device="cuda")))
    odd = torch.zeros(2 * 4 * 64 + 8, dtype=torch.bfloat16, device="cuda")[4:-4].view(2, 4, 64)
    refused(lambda: b.plan.attend(0, odd, b.d_ctx))
    thin = torch.zeros(2, 4, 68, dtype=torch.bfloat16, device="cuda")[:, :, :64]
    refused(lambda: b.plan.attend(0, thin, b.d_ctx))
    b.check(*b.run())
