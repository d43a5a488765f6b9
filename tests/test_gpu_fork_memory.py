"""Device memory and attention over shared prefixes in a context: a batch whose plan finds none runs per
sequence (the default), and what a plan holds is counted.  The shortage is made on the host: the child
process's allocations of more than 256 KiB are refused while a switch is on."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

from ane import _abi
from test_gpu_fork import CFG, engine

pytestmark = pytest.mark.gpu

REFUSE = r"""
#define _GNU_SOURCE
#include <dlfcn.h>
#include <stddef.h>
static int on, refused;
void shortage(int v) { on = v; }
int refusals(void) { return refused; }
int cudaMalloc(void** p, size_t n) {
  static int (*real)(void**, size_t);
  if (on && n > (256 << 10)) return ++refused, 2; /* cudaErrorMemoryAllocation */
  if (!real) real = (int (*)(void**, size_t))dlsym(dlopen("libcudart.so.12", RTLD_LAZY | RTLD_NOLOAD), "cudaMalloc");
  return real(p, n);
}
"""

CHILD = r"""
import ctypes as C, sys
sys.path[:0] = sys.argv[2:]
import numpy as np
from ane import _abi
from test_gpu_fork import CFG, engine

short = C.CDLL(sys.argv[1])
N, LEN = 240, 400  # just past the default's threshold (test_gpu_fork_more)
rng = np.random.default_rng(1)
prompt, tok = rng.integers(3, CFG.vocab, LEN).tolist(), rng.integers(3, CFG.vocab, (4, N))


def run(mode, shortage):
    eng = engine(CFG, "bf16", slots=N, max_pos=448)
    eng.set_option(_abi.LLM_OPT_SHARED_PREFIX, 0)
    eng.prefill([0], [prompt])
    eng.fork(0, list(range(1, N)), LEN)
    eng.decode_step(list(range(N)), tok[0], [LEN] * N, want_logits=True)  # a step's buffers are there
    eng.set_option(_abi.LLM_OPT_SHARED_PREFIX, mode)
    short.shortage(shortage)
    out, tries = [], []
    for i in range(1, 4):
        before = short.refusals()
        out.append(eng.decode_step(list(range(N)), tok[i], [LEN + i] * N, want_logits=True)[1])
        tries.append(short.refusals() - before)
    gen = eng.generate(list(range(N)), tok[0], [LEN + 4] * N, 3) if mode != 2 else None
    short.shortage(0)
    eng.close()
    return out, tries, gen


plain, _, plain_gen = run(0, 0)
got, tries, gen = run(1, 1)
assert tries == [1, 0, 0], tries  # looked for memory once, not in every step
for a, b in zip(plain, got):
    np.testing.assert_array_equal(a, b)
np.testing.assert_array_equal(plain_gen, gen)
shared, tries, _ = run(1, 0)
assert any((a != b).any() for a, b in zip(plain, shared))  # with memory, the default does share here
try:
    run(2, 1)
except _abi.LLMError as e:
    assert e.code == _abi.LLM_ERR_OOM
else:
    raise AssertionError("option 2 must not run per sequence")
print("complete")
"""


def test_a_batch_whose_plan_finds_no_memory_runs_per_sequence(tmp_path):
    src, so, child = tmp_path / "short.c", tmp_path / "short.so", tmp_path / "child.py"
    src.write_text(REFUSE)
    child.write_text(CHILD)
    subprocess.run(["cc", "-shared", "-fPIC", "-w", "-o", str(so), str(src), "-ldl"], check=True)
    here = Path(__file__).resolve().parent
    paths = [str(here), str(here.parent / "oracle"), str(Path(_abi.LIB_PATH).parent.parent)]
    r = subprocess.run([sys.executable, str(child), str(so), *paths], capture_output=True, text=True, timeout=300,
                       env={**os.environ, "LD_PRELOAD": str(so)})
    assert r.returncode == 0 and "complete" in r.stdout, r.stdout + r.stderr


def test_the_memory_of_a_plan_is_counted():
    eng = engine(CFG, "bf16")
    eng.set_option(_abi.LLM_OPT_SHARED_PREFIX, 2)
    eng.prefill([0], [list(range(3, 103))])
    eng.fork(0, [1, 2, 3, 4], 100)
    eng.decode_step([5], [4], [0])
    before = eng.memory()["other"]
    eng.decode_step(list(range(5)), [4] * 5, [100] * 5)
    held = eng.memory()["other"] - before
    # two or more states of 128 f32 sums and two more for each of 5 rows and 4 heads
    assert held >= 2 * 5 * 4 * (128 + 2) * 4
    eng.generate(list(range(5)), [4] * 5, [101] * 5, 2)
    assert eng.memory()["other"] - before >= 2 * held  # a plan of its own
    eng.close()
