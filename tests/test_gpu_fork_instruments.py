"""What a context says of a decode step over shared prefixes: the launches it counts, the timeline it
records, the attention it times and the bytes that it gives for it."""
import numpy as np
import pytest

from ane import _abi
from test_gpu_fork import CFG, MHA, engine

pytestmark = pytest.mark.gpu

ACT = 2  # bytes of a K or V value


def batch(cfg, dtype, mode):
    """Two groups (70 positions of 5 slots, 33 of 2) and a lone slot (20), begun."""
    rng = np.random.default_rng(1)
    eng = engine(cfg, dtype)
    eng.set_option(_abi.LLM_OPT_SHARED_PREFIX, mode)
    eng.prefill([0, 1, 8], [rng.integers(3, cfg.vocab, n).tolist() for n in (70, 33, 20)])
    eng.fork(0, [2, 3, 4, 5], 70)
    eng.fork(1, [6], 33)
    seqs = [0, 6, 2, 3, 8, 4, 1, 5]
    pos = [{6: 33, 1: 33, 8: 20}.get(s, 70) for s in seqs]
    eng.generate_begin(seqs, rng.integers(3, cfg.vocab, len(seqs)), pos, 6)
    return eng, seqs, pos


@pytest.mark.parametrize("mode", [0, 2])
def test_counts_follow_the_step_that_is_asked_about(mode):
    eng, seqs, _ = batch(CFG, "bf16", mode)
    shared = eng.kernel_count(len(seqs))       # of the batch that was begun, before its first step
    eng.generate_steps(1)
    assert eng.kernel_count(len(seqs)) == shared
    eng.generate_end()
    alone = engine(CFG, "bf16")
    alone.prefill([0], [[5, 6, 7]])
    alone.decode_step([0], [5], [3])
    plain = alone.kernel_count(len(seqs))
    alone.close()
    # shared: tile, column and join launches where one was
    assert shared == plain + (2 * CFG.n_layers if mode == 2 else 0)
    for s in seqs:
        eng.release(s)
    eng.prefill([0], [[5, 6, 7]])              # nothing shared any more
    eng.decode_step([0], [5], [3])
    assert eng.kernel_count(len(seqs)) == plain and eng.step_parts(len(seqs)) == 1
    eng.close()


def launches(table):
    return [line for line in table.splitlines()[1:] if line.strip()]


@pytest.mark.parametrize("cfg,dtype", [(CFG, "bf16"), (MHA, "fp16"), (CFG, "w8a8_bf16")])
@pytest.mark.parametrize("mode", [0, 2])
def test_the_timeline_has_every_launch_that_is_counted(cfg, dtype, mode):
    eng, seqs, _ = batch(cfg, dtype, mode)
    counted = eng.kernel_count(len(seqs))
    table, us = eng.trace_step()
    assert us > 0
    # the finish kernel keeps no record
    assert len(launches(table)) == counted - 1, table
    for layer in range(cfg.n_layers):
        assert any("attention" in line and f" L{layer} " in line for line in launches(table)), table
    eng.close()


@pytest.mark.parametrize("cfg,dtype", [(CFG, "bf16"), (MHA, "fp16"), (CFG, "w8a8_bf16")])
def test_the_timed_attention_is_the_step_s(cfg, dtype):
    n = 8
    per = 2 * cfg.n_kv_heads * cfg.head_dim * ACT
    rows = n * cfg.n_heads * cfg.head_dim * (ACT + (4 if dtype.startswith("w8a8") else ACT))
    out = []
    for mode in (0, 2):
        eng, seqs, pos = batch(cfg, dtype, mode)
        eng.generate_steps(2)
        us, nbytes = eng.time_attention(2)
        assert us > 0
        # 64 positions of the five and 32 of the two are read once
        saved = 0 if mode == 0 else 4 * 64 + 32
        assert nbytes == per * (sum(pos) + 2 * n - saved) + rows
        eng.generate_steps(4)                  # the state is as it was
        out.append(eng.generate_end())
        eng.close()
    plain, _, _ = batch(cfg, dtype, 2)
    plain.generate_steps(6)
    np.testing.assert_array_equal(out[1], plain.generate_end())
    plain.close()
