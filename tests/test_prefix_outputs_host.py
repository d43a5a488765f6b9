"""Strides of llm_prefix_attend, without a GPU: the library runs in a child process over stand-ins of
the runtime calls that a plan makes (test_plan_upload_host), and what passes the checks ends in a
launch, which the stand-in refuses.  An output whose (row, head) vectors overlap would be
written by several CTAs at once; it is refused.  A stride that no address is formed with (of a
single row or head) is not looked at."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

from ane import _abi
from test_plan_upload_host import STAND_IN

CHILD = r"""
import ctypes as C, sys
sys.path.insert(0, sys.argv[2])
from ane import _abi
fake, L, X = C.CDLL(sys.argv[1]), _abi.lib(), 1 << 20
i32 = lambda *a: (C.c_int32 * len(a))(*a)


def attend(rows, heads, kv, q_row, q_head, o_row, o_head):
    h, n = C.c_void_p(), len(rows)
    rc = L.llm_prefix_plan_create(0, _abi.LLM_DTYPE_BF16, heads, kv, 64, i32(*range(n)), i32(*rows), n, i32(n), i32(0), 1, 64, C.byref(h))
    assert rc == 0
    c = _abi.llm_page_cache(_abi.LLM_DTYPE_BF16, 1, 8, kv, 64, n, 4, *[X] * 8)
    rc = L.llm_prefix_attend(h, C.addressof(c), 0, X, X, q_row, q_head, 0.0, X, o_row, o_head, None, None)
    text = _abi.last_error()
    assert L.llm_prefix_plan_destroy(h) == 0
    return rc, text


def overlap(rows, heads, row, head):
    "by the definition: every element of every vector once"
    seen = set()
    for r in range(rows):
        for h in range(heads):
            for d in range(0, 64, 8):
                at = r * row + h * head + d
                if at in seen:
                    return True
                seen.add(at)
    return False


bad = 0
for rows, heads in (((1, 1), 4), ((3,), 2), ((2, 1, 2), 6), ((1,), 4), ((5,), 1), ((1,), 1)):
    n = sum(rows)
    for row in (0, 8, 56, 64, 72, 128, 136, 192, 256, 264, 384, 512):
        for head in (0, 32, 64, 88, 128, 320, 328):
            rc, text = attend(rows, heads, 1, heads * 64, 64, row, head)
            want = overlap(n, heads, row, head)
            assert (rc == _abi.LLM_ERR_INVALID) == want and ("overlap" in text) == want, (rows, heads, row, head, rc, text)
            assert want or rc == _abi.LLM_ERR_CUDA, (rc, text)
            bad += want
            # rows of q may be one row, or lie in one another
            rc, text = attend(rows, heads, 1, row, head, heads * 64, 64)
            assert rc == _abi.LLM_ERR_CUDA, (rc, text)
assert bad > 50
for q_row, q_head, rows, heads in ((260, 64, (1,), 4), (-4, 64, (1,), 4), (64, 3, (2, 1), 1), (7, 9, (1,), 1)):
    for args in ((q_row, q_head, 4096, 64), (4096, 64, q_row, q_head)):
        assert attend(rows, heads, 1, *args)[0] == _abi.LLM_ERR_CUDA, args
for args in ((260, 64, 256, 64), (256, 60, 256, 64), (256, 64, 260, 64), (256, 64, 256, 68), (-256, 64, 256, 64), (256, 64, 256, -64)):
    rc, text = attend((2, 1), 4, 1, *args)
    assert rc == _abi.LLM_ERR_INVALID and "stride" in text, args
print("complete")
"""


def test_strides(tmp_path):
    src, so, child = tmp_path / "runtime.c", tmp_path / "runtime.so", tmp_path / "child.py"
    src.write_text(STAND_IN)
    child.write_text(CHILD)
    subprocess.run(["cc", "-shared", "-fPIC", "-w", "-o", str(so), str(src)], check=True)
    package = Path(_abi.LIB_PATH).parent.parent
    r = subprocess.run([sys.executable, str(child), str(so), str(package)], capture_output=True, text=True, timeout=300,
                       env={**os.environ, "LD_PRELOAD": str(so), "CUDA_VISIBLE_DEVICES": ""})
    assert r.returncode == 0 and "complete" in r.stdout, r.stdout + r.stderr
