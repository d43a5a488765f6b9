"""Page requests at sizes that take their other launches: forks of many requests or many bytes (a
checking kernel of one CTA, then rows and copies on all SMs), frees of more slots than CTAs, and
compactions whose CTAs copy several runs.  Same host model as test_gpu_pages; no tolerance."""
import numpy as np
import pytest

from ane import _abi
from test_gpu_pages import HostPages, ints, make

pytestmark = pytest.mark.gpu


def fork(c, h, *request):
    c.fork(*(ints(*x) for x in request))
    h.fork(*request)


def refuse(c, h, code, *request):
    c.fork(*(ints(*x) for x in request))
    with pytest.raises(_abi.LLMError) as e:
        c.check()
    assert e.value.code == code
    h.same()


def sequences(n, room, first=0):
    """Requests for n new sequences of `room` positions."""
    return [-1] * n, list(range(first, first + n)), [0] * n, [room] * n


def test_forks_of_more_requests_than_a_cta_has_threads():
    rng = np.random.default_rng(1)
    c = make("bf16", 2, 9000, 1, 64, seqs=2400, most=6)
    h = HostPages(c)
    refuse(c, h, _abi.LLM_ERR_OOM, *sequences(2400, 96))  # the pool is full before the last thousand
    fork(c, h, *sequences(300, 70))  # 5 pages each
    h.same()
    # 1500 children with and without partly filled pages, 200 new ones and 100 that grow, in any order
    req = [(int(rng.integers(0, 300)), 300 + i, int(rng.integers(0, 81))) for i in range(1500)]
    req = [(p, k, n, int(min(96, n + rng.integers(0, 30)))) for p, k, n in req]
    req += [(-1, 1800 + i, 0, int(rng.integers(0, 97))) for i in range(200)]
    req += [(p, p, 7, int(rng.integers(0, 97))) for p in rng.permutation(300)[:100].tolist()]
    order = rng.permutation(len(req))
    parents, children, lens, rooms = (list(x) for x in zip(*(req[i] for i in order)))
    free = h.n_free
    # refused whole, wherever the fault stands: a child twice a thousand requests apart, a slot out of
    # range, a length that its parent does not have, and more pages than are free
    for at, change in ((1750, (1, children[3])), (0, (1, 2400)), (1799, (0, -2)), (1030, (3, 97)), (1024, (2, 97))):
        bad = [list(x) for x in (parents, children, lens, rooms)]
        bad[change[0]][at] = change[1]
        if change[0] == 2:
            bad[0][at], bad[1][at], bad[3][at] = 0, 2399, 96
        refuse(c, h, _abi.LLM_ERR_INVALID, *bad)
    fork(c, h, parents, children, lens, rooms)
    h.same()
    assert 0 < h.n_free < free
    # every slot to its widest: more than there are; then as many of them as there is room for
    grow = [list(range(2400)), list(range(2400)), [0] * 2400, [96] * 2400]
    need = np.cumsum([6 - held for held in h.npages])
    assert need[-1] > h.n_free
    refuse(c, h, _abi.LLM_ERR_OOM, *grow)
    most = int((need <= h.n_free).sum())
    assert most > 1024
    refuse(c, h, _abi.LLM_ERR_OOM, *(x[:most + 1] for x in grow))
    fork(c, h, *(x[:most] for x in grow))
    h.same()
    c.free(ints(*range(2400)))
    h.release(range(2400))
    h.same()
    assert h.n_free == 9000


def test_a_fork_that_needs_every_free_page():
    c = make("fp16", 1, 1200, 1, 64, seqs=700, most=4)
    h = HostPages(c)
    fork(c, h, *sequences(300, 64))
    h.same()
    assert h.n_free == 0
    refuse(c, h, _abi.LLM_ERR_OOM, *sequences(300, 16, 300))
    fork(c, h, list(range(300)), list(range(300, 600)), [32] * 300, [32] * 300)  # shares only
    h.same()


@pytest.mark.parametrize("n", [100, 200, 256])
def test_forks_of_many_bytes(n):
    rng = np.random.default_rng(n)
    c = make("bf16", 3, 1100, 4, 128, seqs=300, most=6)
    h = HostPages(c)
    fork(c, h, *sequences(20, 90))
    lens = [int(x) for x in rng.integers(1, 91, n)]
    parents = [int(x) for x in rng.integers(0, 20, n)]
    fork(c, h, parents, list(range(20, 20 + n)), lens, [min(96, x + 3) for x in lens])
    h.same()
    free = rng.permutation(20 + n)[: n // 2].tolist()
    c.free(ints(*free))
    h.release(free)
    h.same()


def test_free_of_more_slots_than_ctas():
    c = make("fp16", 1, 4000, 1, 64, seqs=1500, most=4)
    h = HostPages(c)
    fork(c, h, *sequences(900, 60))
    fork(c, h, list(range(400)), list(range(900, 1300)), [32] * 400, [32] * 400)
    gone = np.random.default_rng(2).permutation(1500)[:1100].tolist()  # empty slots among them
    c.free(ints(*gone, *gone[:50]))                                    # and some listed twice
    h.release(gone)
    h.same()
    c.free(ints(*([-1, 1500] * 400), *range(1500)))                    # bad ones are skipped and reported
    with pytest.raises(_abi.LLMError) as e:
        c.check()
    assert e.value.code == _abi.LLM_ERR_INVALID
    h.release(range(1500))
    h.same()
    assert h.n_free == 4000


# one launch with two and with eight runs a CTA; two launches with one run and with four
@pytest.mark.parametrize("pages,layers,kv,hd", [(1000, 2, 2, 128), (2048, 3, 5, 64), (2500, 1, 1, 64), (2100, 3, 2, 128)])
def test_compactions_of_many_moves(pages, layers, kv, hd):
    rng = np.random.default_rng(pages)
    c = make("bf16", layers, pages, kv, hd, seqs=600, most=8)
    h = HostPages(c)
    rooms = [int(x) for x in rng.integers(1, 129, 250)]
    n = 0
    while n < 250 and sum(-(-r // 16) for r in rooms[:n + 1]) < pages - 60:
        n += 1
    fork(c, h, [-1] * n, list(range(n)), [0] * n, rooms[:n])
    kids = [s for s in range(n) if rooms[s] >= 32][:60]
    fork(c, h, kids, list(range(300, 300 + len(kids))), [16] * len(kids), [16] * len(kids))
    gone = [s for s in range(n) if s % 2 == 0]
    c.free(ints(*gone))
    h.release(gone)
    before = list(h.refs)
    live = sum(r > 0 for r in before)
    moves = sum(r > 0 for r in before[live:])
    assert moves > 100
    c.compact()
    h.compact()
    h.same()
