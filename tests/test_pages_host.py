"""Argument checks of the page requests that need no GPU: the C entries refuse before any launch."""
import ctypes as C

import pytest

from ane import _abi

INVALID, UNSUPPORTED = _abi.LLM_ERR_INVALID, _abi.LLM_ERR_UNSUPPORTED


def cache(**kw):
    """A cache struct of plausible sizes over host addresses that no entry may touch."""
    v = dict(dtype=_abi.LLM_DTYPE_BF16, n_layers=1, n_pages=8, n_kv_heads=1, head_dim=64, max_seqs=4, max_pages=4, pool=1 << 20)
    v |= {k: 1 << 20 for k in ("n_free", "status", "npages", "refs", "free_pages", "table", "work")}
    return _abi.llm_page_cache(**(v | kw))


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=3), INVALID, "dtype"), (dict(head_dim=96), UNSUPPORTED, "head_dim"), (dict(n_layers=0), INVALID, "positive"),
    (dict(n_pages=-1), INVALID, "positive"), (dict(max_pages=0), INVALID, "positive"), (dict(n_kv_heads=2000), INVALID, "range"),
    (dict(pool=None), INVALID, "pool"), (dict(pool=(1 << 20) + 8), INVALID, "pool"),
])
def test_bad_caches_are_refused(kw, code, text):
    L, bad = _abi.lib(), cache(**kw)
    p, x = C.addressof(bad), 1 << 20
    for rc in (L.llm_pages_copy(0, p, p, x, x, 1, None), L.llm_pages_fork(0, p, x, x, x, x, 1, None),
               L.llm_pages_free(0, p, x, 1, None), L.llm_pages_compact(0, p, None), L.llm_pages_status(0, p, None)):
        assert rc == code and text in _abi.last_error()


@pytest.mark.parametrize("field", ["n_free", "status", "npages", "refs", "free_pages", "table", "work"])
def test_missing_tables_are_refused(field):
    L, x = _abi.lib(), 1 << 20
    for value in (None, (1 << 20) + 2):
        bad = cache(**{field: value})
        p = C.addressof(bad)
        for rc in (L.llm_pages_fork(0, p, x, x, x, x, 1, None), L.llm_pages_free(0, p, x, 1, None), L.llm_pages_compact(0, p, None)):
            assert rc == INVALID and "table" in _abi.last_error()


def test_bad_requests_are_refused_and_empty_ones_are_not():
    L, good, other, x = _abi.lib(), cache(), cache(n_kv_heads=2), 1 << 20
    p, o = C.addressof(good), C.addressof(other)
    assert L.llm_pages_copy(0, p, o, x, x, 1, None) == INVALID and "different" in _abi.last_error()
    assert L.llm_pages_copy(0, None, p, x, x, 1, None) == INVALID
    assert L.llm_pages_copy(0, p, p, None, x, 1, None) == INVALID
    assert L.llm_pages_copy(0, p, p, x, x, -1, None) == INVALID
    assert L.llm_pages_fork(0, p, x, x, x, x, 5, None) == INVALID and "5 requests for 4 slots" in _abi.last_error()
    assert L.llm_pages_fork(0, p, x, None, x, x, 1, None) == INVALID
    assert L.llm_pages_free(0, p, None, 1, None) == INVALID
    # nothing asked: nothing enqueued
    assert L.llm_pages_copy(0, p, p, None, None, 0, None) == 0
    assert L.llm_pages_fork(0, p, None, None, None, None, 0, None) == 0
    assert L.llm_pages_free(0, p, None, 0, None) == 0


def test_work_words():
    L = _abi.lib()
    assert L.llm_pages_work_words(0, 4) == 0 and L.llm_pages_work_words(4, 0) == 0 and L.llm_pages_work_words(1 << 29, 4) == 0
    assert L.llm_pages_work_words(64, 4) == 16 + 2 * 4 + 2 + 2 * 64


def plan_args(**kw):
    """Arguments of llm_prefix_plan_create for two sequences, with some of them replaced."""
    i32 = lambda *a: (C.c_int32 * len(a))(*a)  # noqa: E731
    v = dict(device=0, dtype=_abi.LLM_DTYPE_F16, n_heads=4, n_kv_heads=2, head_dim=64, slots=i32(0, 1), rows=i32(1, 1), n_seqs=2,
             sizes=i32(2), prefixes=i32(32), n_groups=1, max_ctx=64)
    v |= {k: i32(*x) if isinstance(x, tuple) else x for k, x in kw.items()}
    return list(v.values())


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=_abi.LLM_DTYPE_W8A8_BF16), INVALID, "dtype"), (dict(head_dim=80), UNSUPPORTED, "head_dim"),
    (dict(n_heads=5), INVALID, "multiple"), (dict(n_kv_heads=0), INVALID, "multiple"), (dict(n_seqs=0), INVALID, "positive"),
    (dict(n_groups=0), INVALID, "positive"), (dict(max_ctx=-1), INVALID, "positive"), (dict(slots=None), INVALID, "nil"),
    (dict(rows=None), INVALID, "nil"), (dict(sizes=(0,)), INVALID, "group 0"), (dict(sizes=(3,)), INVALID, "in all"),
    (dict(prefixes=(8,)), INVALID, "multiple of 16"), (dict(prefixes=(-16,)), INVALID, "multiple of 16"),
    (dict(prefixes=(80,)), INVALID, "max_ctx"), (dict(slots=(0, -1)), INVALID, "out of range"), (dict(rows=(1, -1)), INVALID, "rows"),
])
def test_bad_plans_are_refused(kw, code, text):
    L, h = _abi.lib(), C.c_void_p()
    assert L.llm_prefix_plan_create(*plan_args(**kw), C.byref(h)) == code
    assert text in _abi.last_error() and not h.value
    assert L.llm_prefix_plan_create(*plan_args(), None) == INVALID
    assert L.llm_prefix_plan_destroy(None) == INVALID
