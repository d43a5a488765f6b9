"""NaN and infinity in the values that attention over shared prefixes sees: a row with a NaN score or a
score of +inf is NaN, as a softmax in torch gives it, whatever kernel its item went to and however
many states it was joined from; a score of -inf has weight 0; only a row without any weight gives
zeros and lse -inf.  A NaN in V stays in its column.  Rows and columns that do not see the value keep
their tolerance (test_gpu_prefix's, over the finite scores)."""
import math

import numpy as np
import pytest

from test_gpu_prefix import TINY, U, Batch

pytestmark = pytest.mark.gpu


class Poked(Batch):
    """A batch in which single values of K and V can be replaced after it was made."""

    def poke(self, s, t, h, which, dim, value):
        """Value at position t of kv head h: dimension `dim` of K (which 0) or V (1), for sequence s and,
        inside the shared prefix, for its whole group."""
        for o in range(len(self.ctx)) if t < self.prefix[s] else [s]:
            if self.group[o] != self.group[s]:
                continue
            x = (self.k, self.v)[which][o]
            if t < x.shape[0]:
                x[t, h, dim] = value
        page = int(self.table[self.slots[s], t // 16])
        at = self.cache.element_index()[t % 16]
        self.cache.pool[self.layer, page, h, which][at[dim]] = value

    def compare(self, out, lse):
        """Against 64 bits (V finite); returns the truth of (row, head) being NaN."""
        import torch
        gq, at, scale = self.heads // self.kv, 0, self.hd ** -0.5
        nans = []
        for s, (c, r) in enumerate(zip(self.ctx, self.rows)):
            q, o, l = (x[at:at + r].double() for x in (self.q, out, lse))
            at += r
            if c == 0:
                continue
            k, v = (x[s][:c].double().repeat_interleave(gq, 1) for x in (self.k, self.v))
            seen = torch.arange(c, device="cuda")[None] <= (c - r + torch.arange(r, device="cuda"))[:, None]
            x = torch.einsum("rhd,thd->rht", q, k) * scale
            x = torch.where(seen[:, None], x, -math.inf)
            ds = self.hd * 2.0 ** -24 * scale * torch.einsum("rhd,thd->rht", q.abs(), k.abs()) + 2.0 ** -22 * x.abs()
            ds = torch.where(torch.isfinite(x) & torch.isfinite(ds), ds, 0.0).amax(-1)
            nan = (x.isnan() | (x == math.inf)).any(-1)          # [r, heads]
            none = (x == -math.inf).all(-1)
            want_l = torch.logsumexp(x, -1)
            p = torch.exp(x - torch.where(none, 0.0, want_l)[..., None])
            want, mean = torch.einsum("rht,thd->rhd", p, v), torch.einsum("rht,thd->rhd", p, v.abs())
            e = ds + c * 2.0 ** -24 + 2.0 ** -21 + torch.where(none, 0.0, 2.0 ** -23 * want_l.abs())
            tol = U[self.dtype] * (want.abs() + mean) + 2 * e[..., None] * mean + TINY[self.dtype]
            assert bool(o[nan].isnan().all()), "a row with a NaN or infinite score is not NaN"
            assert bool(l[nan].isnan().all())
            assert bool((o[none] == 0).all()) and bool((l[none] == -math.inf).all())
            rest = ~nan & ~none
            assert bool(((o - want).abs() <= tol)[rest].all())
            assert bool(((l - want_l).abs() <= e)[rest].all())
            nans.append(nan)
        return torch.cat(nans)


# a call that goes to the column kernel, its states joined in the same launch; columns joined by a
# launch of their own; tiles of one stream and of two, states joined and output written at once
SHAPES = {
    "columns": dict(sizes=[2], prefixes=[32], rows=[1] * 2, heads=4, kv=2),
    "columns, many": dict(sizes=[3] * 12, prefixes=[48] * 12, rows=[1] * 36, heads=4, kv=2),
    "tile and columns": dict(sizes=[30], prefixes=[1040], rows=[1] * 30, heads=4, kv=2),
    "tile without states": dict(sizes=[1, 1], prefixes=[0, 0], rows=[40, 70], heads=4, kv=2),
    "tiles": dict(sizes=[6], prefixes=[208], rows=[33] * 6, heads=4, kv=2),
    "tile pairs": dict(sizes=[1] * 38, prefixes=[0] * 38, rows=[128] * 38, heads=8, kv=4, more=1790),
    "one stream": dict(sizes=[1] * 60, prefixes=[0] * 60, rows=[9] * 60, heads=16, kv=8),
}


def batch(shape, dtype, hd, seed):
    s = dict(SHAPES[shape])
    rng = np.random.default_rng(seed)
    more = s.pop("more", 90)
    ctx = [int(p + max(r, rng.integers(more - 89, more + 1))) for p, r in zip(np.repeat(s["prefixes"], s["sizes"]), s["rows"])]
    return Poked(dtype, s["kv"], hd, s["sizes"], s["prefixes"], ctx, s["rows"], s["heads"], layers=1, seed=seed)


@pytest.mark.parametrize("dtype,hd", [("bf16", 128), ("fp16", 64)])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_nan_scores(shape, dtype, hd):
    b = batch(shape, dtype, hd, 1)
    b.poke(1, b.ctx[1] - 1, 0, 0, 5, math.nan)       # the last position of sequence 1, kv head 0
    nan = b.compare(*b.run())
    assert int(nan.sum()) == b.heads // b.kv         # its last row's heads and nobody else's
    b.poke(0, 3, 1, 0, 0, math.nan)                  # an early position, shared where there is a prefix
    nan = b.compare(*b.run())
    assert bool(nan[: b.rows[0]].any())


@pytest.mark.parametrize("dtype,hd", [("bf16", 64), ("fp16", 128)])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_nan_queries(shape, dtype, hd):
    b = batch(shape, dtype, hd, 2)
    b.q[1, b.heads - 1, hd - 1] = math.nan
    nan = b.compare(*b.run())
    assert int(nan.sum()) == 1 and bool(nan[1, b.heads - 1])


@pytest.mark.parametrize("dtype,hd", [("bf16", 128), ("fp16", 64)])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_infinite_scores(shape, dtype, hd):
    # the sign of q's dimension decides: +inf makes the row NaN, -inf takes the position out
    b = batch(shape, dtype, hd, 3)
    b.poke(1, b.ctx[1] - 1, 1, 0, 7, math.inf)
    nan = b.compare(*b.run())
    gq = b.heads // b.kv
    row = b.rows[0] + b.rows[1] - 1
    q = b.q[row, gq:2 * gq, 7]
    assert nan[row, gq:2 * gq].tolist() == (q > 0).tolist()


@pytest.mark.parametrize("dtype,hd", [("bf16", 64), ("fp16", 128)])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_rows_whose_scores_are_all_minus_infinity(shape, dtype, hd):
    import torch
    b = batch(shape, dtype, hd, 4)
    keys = b.cache.pool[b.layer, :, :, 0]
    where = b.cache.element_index()[:, 9]
    keys[..., where] = math.inf
    for k in b.k:
        k[..., 9] = math.inf
    b.q[..., 9] = -1.0
    b.q[0, 0, 9] = 1.0
    nan = b.compare(*b.run())
    assert int(nan.sum()) == 1
    out, lse = b.run()
    rest = torch.ones_like(lse, dtype=torch.bool)
    rest[0, 0] = False
    assert bool((out[rest] == 0).all()) and bool((lse[rest] == -math.inf).all())


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_non_finite_values_stay_in_their_column(shape, value):
    # position 0 of each group: every row sees it
    b = batch(shape, "bf16", 128, 5)
    b.poke(0, 0, 0, 1, 17, value)
    out, lse = b.run()
    mine = np.repeat(b.group == b.group[0], b.rows)
    gq = b.heads // b.kv
    import torch
    off = ~torch.isfinite(out)
    want = torch.zeros_like(off)
    want[torch.from_numpy(mine).cuda(), :gq, 17] = True
    assert torch.equal(off, want) and bool(torch.isfinite(lse).all())
