"""Argument checks of the paged caches that need no GPU: what would fault on the device, or race there,
is refused on the host before any launch.  Addresses are host numbers that no entry may touch."""
import ctypes as C

import pytest

from ane import _abi
from test_pages_host import cache

INVALID = _abi.LLM_ERR_INVALID
X = 1 << 20


@pytest.mark.parametrize("odd", [X + 1, X + 2, X + 3])
def test_misaligned_lists_are_refused(odd):
    L, good = _abi.lib(), cache()
    p = C.addressof(good)
    calls = [lambda a, b, c, d: L.llm_pages_copy(0, p, p, a, b, 1, None), lambda a, b, c, d: L.llm_pages_fork(0, p, a, b, c, d, 1, None),
             lambda a, b, c, d: L.llm_pages_free(0, p, a, 1, None)]
    for call, n in zip(calls, (2, 4, 1)):
        for i in range(n):
            args = [X] * 4
            args[i] = odd
            assert call(*args) == INVALID and "misaligned" in _abi.last_error()


def test_a_copy_with_a_misaligned_status_word_is_refused():
    L, good = _abi.lib(), cache()
    for odd in (None, X + 1, X + 2):
        bad = cache(status=odd)
        assert L.llm_pages_copy(0, C.addressof(bad), C.addressof(good), X, X, 1, None) == INVALID and "table" in _abi.last_error()


def test_a_copy_into_a_cache_on_another_gpu_is_refused():
    # two caches as their constructor leaves them, on GPUs that need not exist
    import torch
    from ane.paged import PagedCache
    a, b = (object.__new__(PagedCache) for _ in range(2))
    for c, gpu in ((a, 0), (b, 1)):
        c._lib, c.device, c.c_struct = _abi.lib(), torch.device("cuda", gpu), cache()
        c._ref = C.addressof(c.c_struct)
        c._stream = lambda: 0
    lists = torch.zeros(0, dtype=torch.int32), torch.zeros(0, dtype=torch.int32)
    with pytest.raises(_abi.LLMError) as e:
        a.copy(*lists, to=b)
    assert e.value.code == INVALID and "cuda:1" in str(e.value)
    with pytest.raises(_abi.LLMError) as e:
        a.copy(*lists, to="elsewhere")
    assert e.value.code == INVALID


def test_lists_that_are_not_tensors_are_refused_like_other_arguments():
    import torch
    from ane.paged import PagedCache
    c = object.__new__(PagedCache)
    c._lib, c.device, c.c_struct = _abi.lib(), torch.device("cuda", 0), cache()
    c._ref, c._stream = C.addressof(c.c_struct), lambda: 0
    for call in (lambda: c.copy([1], [2]), lambda: c.fork([-1], [0], [0], [16]), lambda: c.free([0]), lambda: c.free(None)):
        with pytest.raises(_abi.LLMError) as e:
            call()
        assert e.value.code == INVALID


def test_more_beams_than_tokens_are_refused():
    from ane.cmd import beam_search
    for n in ("501", "100000"):
        with pytest.raises(SystemExit):
            beam_search.main(["-beams", n])
