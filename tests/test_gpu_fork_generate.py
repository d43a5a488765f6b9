"""Forks and releases between the steps of a generate batch.  A shared page is read-only, so steps that
would write into one are refused before anything is enqueued, and a batch whose sharing changed
attends to what its slots hold now.  A batch of one slot runs per sequence whatever the option, so
its tokens are compared bit for bit; K and V behind attention over shared prefixes within
parity.REF_ORDER_TOL, the bound of two orders of operations."""
import numpy as np
import pytest

from ane import _abi
from parity import REF_ORDER_TOL
from test_gpu_fork import CFG, engine

pytestmark = pytest.mark.gpu


def refused(f):
    with pytest.raises(_abi.LLMError) as e:
        f()
    assert e.value.code == _abi.LLM_ERR_STATE and "shared" in str(e.value)


def rows(eng, seq, n):
    """K and V of layer 0 and the last of the first n positions of a slot."""
    return np.stack([np.concatenate(eng.read_kv(layer, seq, t)) for layer in (0, eng.cfg.n_layers - 1) for t in range(n)])


@pytest.mark.parametrize("mode", [0, 2])
def test_steps_into_pages_that_a_fork_shared_are_refused(mode):
    prompt = list(range(3, 13))
    eng = engine(CFG, "bf16", slots=4, max_pos=96)
    eng.set_option(_abi.LLM_OPT_SHARED_PREFIX, mode)
    first = int(eng.prefill([0], [prompt])[0])
    want = eng.generate([0], [first], [10], 40)
    eng.release(0)
    eng.prefill([0], [prompt])
    eng.generate_begin([0], [first], [10], 40)
    eng.generate_steps(5)                      # positions 10..14; 15 is next
    eng.fork(0, [1], 32)                       # pages 0 and 1, of which 15 positions are written
    eng.synchronize()
    before = rows(eng, 1, 32)
    refused(lambda: eng.generate_steps(1))
    refused(lambda: eng.generate_steps(20))
    eng.generate_steps(0)
    refused(lambda: eng.profile_step(1))       # writes the next step's K and V too
    refused(lambda: eng.trace_step())
    np.testing.assert_array_equal(rows(eng, 1, 32), before)
    eng.release(1)                             # nothing shared: the batch goes on where it was
    eng.generate_steps(2)                      # 15 and 16
    eng.fork(0, [1, 2], 16)                    # a complete page behind the batch
    eng.generate_steps(3)                      # 17..19
    eng.fork(0, [3], 48)                       # page 1, where the next step is, and page 2
    refused(lambda: eng.generate_steps(1))
    eng.release(3)
    eng.fork(0, [3], 35)                       # pages 0 and 1 are shared, 32..34 a copy
    refused(lambda: eng.generate_steps(13))    # 20..31 lie in page 1
    eng.release(3)
    eng.generate_steps(30)
    np.testing.assert_array_equal(eng.generate_end(), want)
    eng.close()


def test_sharing_behind_or_elsewhere_does_not_stop_a_batch():
    prompt = list(range(3, 13))
    eng = engine(CFG, "bf16", slots=3, max_pos=96)
    eng.set_option(_abi.LLM_OPT_SHARED_PREFIX, 0)
    first = int(eng.prefill([0], [prompt])[0])
    want = eng.generate([0], [first], [10], 20)
    eng.release(0)
    eng.prefill([0], [prompt])
    eng.fork(0, [1], 10)                       # a copy: nothing shared
    eng.release(0)
    eng.fork(1, [0], 10)
    eng.generate_begin([0], [first], [10], 40)
    eng.fork(1, [2], 10)                       # sharing changed elsewhere: nothing to refuse
    eng.generate_steps(3)
    eng.release(2)
    eng.fork(0, [2], 32)
    refused(lambda: eng.generate_steps(1))
    eng.release(2)
    eng.generate_steps(17)
    np.testing.assert_array_equal(eng.generate_end(), want)
    eng.close()

def test_a_slot_that_changed_between_steps_is_read_as_it_is_now():
    """Slot 3 leaves a group over prompt A between two steps and comes back as a copy of prompt B."""
    rng = np.random.default_rng(5)
    a, b = (rng.integers(3, CFG.vocab, 72).tolist() for _ in range(2))
    seqs, pos = [0, 1, 2, 3], [72] * 4
    got = []
    for mode in (0, 2):
        eng = engine(CFG, "fp16", slots=6, max_pos=128)
        eng.set_option(_abi.LLM_OPT_SHARED_PREFIX, mode)
        eng.prefill([0, 5], [a, b])
        eng.fork(0, [1, 2, 3], 72)
        eng.generate_begin(seqs, [7, 8, 9, 10], pos, 8)
        eng.generate_steps(0)
        eng.release(3)
        eng.fork(5, [3], 72)
        eng.generate_steps(1)
        eng.synchronize()
        got.append([np.stack(eng.read_kv(CFG.n_layers - 1, s, 72)) for s in seqs])
        eng.close()
    for x, y in zip(*got):
        assert float(np.abs(x - y).max()) <= REF_ORDER_TOL["fp16"]
