"""Page requests on device-resident tables (ane.paged.PagedCache: copy, fork, free, compact)
against a host model of the same rules, kept in Python lists: every table word and every pool
value is compared after each request.  No tolerance: pages are moved, not computed."""
import numpy as np
import pytest

from ane import _abi

pytestmark = pytest.mark.gpu


class HostPages:
    """The rules of the page requests on Python lists; pool values are numpy rows per page."""

    def __init__(self, cache):
        self.c = cache
        self.n_free = int(cache.n_free.item())
        self.npages = cache.npages.tolist()
        self.refs = cache.refs.tolist()
        self.free = cache.free_pages.tolist()
        self.table = cache.table.cpu().numpy().astype(np.int64)
        self.pool = self.bits(cache)

    @staticmethod
    def bits(cache):
        import torch
        return cache.pool.view(torch.int16).cpu().numpy().copy()

    def fork(self, parents, children, lens, rooms):
        was = list(self.npages)
        for p, c, length, room in zip(parents, children, lens, rooms):
            keep = was[c] if p == c else length // 16
            if p != c:
                for j in range(keep):
                    self.table[c, j] = self.table[p, j]
                    self.refs[self.table[p, j]] += 1
            held = keep
            while held * 16 < room:
                self.n_free -= 1
                self.table[c, held] = self.free[self.n_free]
                self.refs[self.free[self.n_free]] = 1
                held += 1
            if p != c and length % 16:
                self.pool[:, self.table[c, keep]] = self.pool[:, self.table[p, keep]]
            self.npages[c] = held

    def release(self, slots):
        empty = []
        for s in slots:
            for j in range(self.npages[s]):
                e = self.table[s, j]
                self.refs[e] -= 1
                if self.refs[e] == 0:
                    empty.append(int(e))
            self.npages[s] = 0
            self.table[s] = -1
        for e in sorted(empty):
            self.free[self.n_free] = e
            self.n_free += 1

    def compact(self):
        live = [p for p, r in enumerate(self.refs) if r > 0]
        holes = [p for p in range(len(live)) if self.refs[p] == 0]
        to = dict(zip([p for p in live if p >= len(live)], holes))
        for a, b in to.items():
            self.pool[:, b] = self.pool[:, a]
            self.refs[b], self.refs[a] = self.refs[a], 0
        for s in range(self.table.shape[0]):
            for j in range(self.npages[s]):
                self.table[s, j] = to.get(int(self.table[s, j]), self.table[s, j])
        n = len(self.refs)
        for k in range(n - len(live)):
            self.free[k] = n - 1 - k
        self.n_free = n - len(live)

    def same(self):
        c = self.c
        c.check()
        assert int(c.n_free.item()) == self.n_free
        assert c.npages.tolist() == self.npages
        assert c.refs.tolist() == self.refs
        assert c.free_pages.tolist() == self.free
        np.testing.assert_array_equal(c.table.cpu().numpy(), self.table)
        np.testing.assert_array_equal(self.bits(c), self.pool)


def make(dtype="bf16", layers=2, pages=64, kv=2, hd=64, seqs=12, most=9, seed=0):
    import torch
    from ane.paged import PagedCache
    c = PagedCache(dtype, layers, pages, kv, hd, seqs, most)
    g = torch.Generator(device="cuda").manual_seed(seed)
    c.pool.normal_(generator=g)
    return c


def ints(*a):
    import torch
    return torch.tensor(a, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype,layers,kv,hd", [("bf16", 2, 2, 64), ("fp16", 1, 1, 64), ("fp16", 3, 3, 128), ("bf16", 1, 8, 128)])
@pytest.mark.parametrize("length", [1, 15, 16, 17, 48, 63])
def test_fork_shares_full_pages_and_copies_the_partial_one(dtype, layers, kv, hd, length):
    c = make(dtype, layers, 40, kv, hd)
    h = HostPages(c)
    for request in [((-1,), (3,), (0,), (64,)),                                    # a new sequence
                    ((3, 3, 3), (0, 7, 11), (length,) * 3, (length, length + 1, length + 40)),
                    ((7, -1, 0), (7, 2, 5), (0, 0, min(length, 16)), (length + 33, 0, 16))]:  # grow, empty, fork again
        c.fork(*(ints(*x) for x in request))
        h.fork(*request)
        h.same()


def test_fork_with_parent_growing_in_the_same_request():
    c, request = make(), ((4, 4, 4), (4, 6, 8), (0, 20, 32), (100, 21, 32))
    h = HostPages(c)
    for r in [((-1,), (4,), (0,), (33,)), request]:
        c.fork(*(ints(*x) for x in r))
        h.fork(*r)
    h.same()


def test_free_counts_references_and_pushes_ascending():
    c = make(pages=50)
    h = HostPages(c)
    for r in [((-1, -1), (0, 1), (0, 0), (70, 16)), ((0, 0, 1), (2, 3, 4), (40, 64, 16), (90, 64, 17))]:
        c.fork(*(ints(*x) for x in r))
        h.fork(*r)
    for slots in [(0,), (9,), (3, 2), (4, 1), (0, 1, 2, 3)]:  # 9 and the last list: empty slots
        c.free(ints(*slots))
        h.release(slots)
        h.same()
    assert h.n_free == 50


def test_free_of_a_slot_listed_twice_counts_once():
    c = make()
    h = HostPages(c)
    r = ((-1,), (0,), (0,), (40,))
    c.fork(*(ints(*x) for x in r))
    h.fork(*r)
    c.free(ints(0, 0, 0))
    h.release([0])
    h.same()


@pytest.mark.parametrize("pages,rooms", [(31, (0, 0, 0)), (32, (16, 16, 16)), (33, (140, 140, 140)), (97, (130, 1, 77)), (2100, (144, 144, 144))])
def test_compact_moves_the_fewest_pages(pages, rooms):
    c = make(pages=pages, seqs=40, most=9)
    h = HostPages(c)
    for i in range(12):  # leave holes: sequences come, every other one goes
        if h.n_free * 16 < sum(rooms) + 48:
            break
        r = ((-1,) * 3, (3 * i, 3 * i + 1, 3 * i + 2), (0,) * 3, rooms)
        c.fork(*(ints(*x) for x in r))
        h.fork(*r)
        c.free(ints(3 * i, 3 * i + 2)), h.release((3 * i, 3 * i + 2))
        if i % 2:
            c.free(ints(3 * i + 1)), h.release((3 * i + 1,))
    before = HostPages.bits(c)
    c.compact()
    h.compact()
    h.same()
    moved = int((HostPages.bits(c) != before).any(axis=(0, 2, 3, 4)).sum())
    assert moved <= sum(1 for r in h.refs if r > 0)
    c.compact()  # again: nothing left to move
    h.compact()
    h.same()


def test_random_life_of_a_pool():
    rng = np.random.default_rng(7)
    c = make("fp16", 1, 300, 1, 64, seqs=64, most=12, seed=3)
    h = HostPages(c)
    length = {}
    for step in range(60):
        empty = [s for s in range(64) if h.npages[s] == 0]
        if rng.random() < 0.25 and length:
            gone = rng.choice(list(length), size=min(len(length), 7), replace=False).tolist()
            c.free(ints(*gone))
            h.release(gone)
            for s in gone:
                del length[s]
        elif rng.random() < 0.15:
            c.compact()
            h.compact()
        elif len(empty) > 6:
            kids = rng.choice(empty, size=5, replace=False).tolist()
            par = [int(rng.choice(list(length))) if length and rng.random() < 0.7 else -1 for _ in kids]
            lens = [int(rng.integers(0, length[p] + 1)) if p >= 0 else 0 for p in par]
            rooms = [min(192, n + int(rng.integers(1, 50))) for n in lens]
            if length and rng.random() < 0.5:  # one of the others grows
                s = int(rng.choice(list(length)))
                par, kids, lens, rooms = par + [s], kids + [s], lens + [0], rooms + [min(192, length[s] + 20)]
            if sum(-(-r // 16) + 1 for r in rooms) > h.n_free:
                continue
            c.fork(ints(*par), ints(*kids), ints(*lens), ints(*rooms))
            h.fork(par, kids, lens, rooms)
            for s, r in zip(kids, rooms):
                length[s] = max(length.get(s, 0), r)
        h.same()


def test_copy_between_pools_and_within_one():
    import torch
    a, b = make(pages=40, seed=1), make(pages=23, seed=2)
    wa, wb = HostPages.bits(a), HostPages.bits(b)
    src, dst = [5, 0, 39, 7], [22, 1, 0, 9]
    a.copy(ints(*src), ints(*dst), to=b)
    a.copy(ints(1, 2), ints(30, 31))
    a.copy(ints(), ints())
    a.check()
    for s, d in zip(src, dst):
        wb[:, d] = wa[:, s]
    wa[:, [30, 31]] = wa[:, [1, 2]]
    np.testing.assert_array_equal(HostPages.bits(a), wa)
    np.testing.assert_array_equal(HostPages.bits(b), wb)
    # on another stream, after work queued there
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a.pool[:, 3] += 1
        a.copy(ints(3), ints(4))
    s.synchronize()
    assert torch.equal(a.pool[:, 3], a.pool[:, 4])


@pytest.mark.parametrize("request_,code", [
    (((-1,), (0,), (0,), (16 * 9 + 1,)), _abi.LLM_ERR_INVALID),           # more pages than a row holds
    (((-1,), (12,), (0,), (16,)), _abi.LLM_ERR_INVALID),                  # no such slot
    (((12,), (0,), (0,), (16,)), _abi.LLM_ERR_INVALID),
    (((-2,), (0,), (0,), (16,)), _abi.LLM_ERR_INVALID),
    (((-1,), (0,), (5,), (16,)), _abi.LLM_ERR_INVALID),                   # a new sequence has no positions
    (((1,), (0,), (49,), (49,)), _abi.LLM_ERR_INVALID),                   # longer than the parent's pages
    (((1,), (0,), (-1,), (16,)), _abi.LLM_ERR_INVALID),
    (((1,), (0,), (30,), (29,)), _abi.LLM_ERR_INVALID),                   # no room for its own positions
    (((-1,), (1,), (0,), (16,)), _abi.LLM_ERR_INVALID),                   # the child is not empty
    (((-1, 1), (0, 0), (0, 16), (16, 16)), _abi.LLM_ERR_INVALID),         # a child twice
    (((1, -1, -1), (0, 2, 3), (17, 0, 0), (40, 144, 144)), _abi.LLM_ERR_OOM),
])
def test_refused_forks_change_nothing(request_, code):
    c = make(pages=16)
    h = HostPages(c)
    r = ((-1,), (1,), (0,), (40,))
    c.fork(*(ints(*x) for x in r))
    h.fork(*r)
    c.fork(*(ints(*x) for x in request_))
    with pytest.raises(_abi.LLMError) as e:
        c.check()
    assert e.value.code == code
    h.same()  # the status was cleared and every table is as it was
    good = ((1,), (0,), (20,), (20,))
    c.fork(*(ints(*x) for x in good))
    h.fork(*good)
    h.same()


def test_bad_slots_and_pages_are_reported():
    c = make(pages=16)
    h = HostPages(c)
    c.free(ints(-1, 12))
    with pytest.raises(_abi.LLMError) as e:
        c.check()
    assert e.value.code == _abi.LLM_ERR_INVALID
    c.copy(ints(0, 16, -1), ints(1, 2, 3))  # the pairs that are in range are copied
    h.pool[:, 1] = h.pool[:, 0]
    with pytest.raises(_abi.LLMError):
        c.check()
    h.same()


def test_pages_requests_in_a_cuda_graph():
    import torch
    c = make(pages=64)
    par, kids, lens, rooms, gone = ints(-1, -1), ints(0, 1), ints(0, 0), ints(30, 50), ints(0, 1)
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        c.fork(par, kids, lens, rooms)
        c.free(gone)
        c.compact()
    h = HostPages(c)
    for _ in range(3):
        g.replay()
        h.fork((-1, -1), (0, 1), (0, 0), (30, 50))
        h.release((0, 1))
        h.compact()
        torch.cuda.synchronize()
        h.same()


def test_offsets_past_32_bits():
    """Pages whose byte offset in the pool passes 2^32 (and whose element offset passes 2^31)."""
    import torch
    from ane.paged import PagedCache
    n = 70_000  # x 64 KiB pages of one layer = 4.6 GB
    c = PagedCache("bf16", 1, n, 8, 128, 4, 4)
    c.pool[0, 0].normal_()
    c.copy(ints(0), ints(n - 1))
    c.copy(ints(n - 1), ints(n - 2))
    c.check()
    assert torch.equal(c.pool[0, n - 2], c.pool[0, 0])
    c.free_pages[n - 1] = n - 3  # handed out next
    c.free_pages[2] = 0          # (in its place on the stack)
    c.fork(ints(-1), ints(0), ints(0), ints(5))
    c.pool[0, n - 3].normal_()
    keep = c.pool[0, n - 3].clone()
    c.compact()
    c.check()
    assert c.table[0].tolist() == [0, -1, -1, -1] and int(c.n_free.item()) == n - 1
    assert torch.equal(c.pool[0, 0], keep)
