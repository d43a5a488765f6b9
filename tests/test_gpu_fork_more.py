"""Forked slots in the rest of the token loop: prefill of a suffix, sampling, the default choice of
attention, and refusals that leave everything as it was."""
import numpy as np
import pytest

import oracle as O
from ane import _abi
from parity import REF_ORDER_TOL
from test_gpu_fork import CFG, MHA, engine

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cfg,dtype", [(CFG, "bf16"), (MHA, "fp16"), (CFG, "w8a8_bf16")])
@pytest.mark.parametrize("length", [48, 133])
def test_prefill_of_forked_slots(cfg, dtype, length):
    # a common system prompt, then each slot's own suffix: as if each had prefilled both in turn
    rng = np.random.default_rng(length)
    prompt = rng.integers(3, cfg.vocab, length).tolist()
    slots = [0, 3, 1, 5]
    suffixes = [rng.integers(3, cfg.vocab, n).tolist() for n in (1, 40, 17, 90)]
    tok = rng.integers(3, cfg.vocab, (6, 4))
    got = []
    for mode in (None, 0, 2):
        eng = engine(cfg, dtype)
        if mode is None:
            eng.prefill(slots, [prompt] * 4)
        else:
            eng.set_option(_abi.LLM_OPT_SHARED_PREFIX, mode)
            eng.prefill([0], [prompt])
            eng.fork(0, slots[1:], length)
        _, first = eng.prefill(slots, suffixes, start_pos=[length] * 4, want_logits=True)
        pos = np.array([length + len(s) for s in suffixes])
        got.append([first] + [eng.decode_step(slots, tok[i], pos + i, want_logits=True)[1] for i in range(6)])
        eng.close()
    for a, b, c in zip(*got):
        np.testing.assert_array_equal(a, b)
        assert float(np.abs(a - c).max()) <= REF_ORDER_TOL[dtype]
    np.testing.assert_array_equal(got[0][0], got[2][0])  # prefill attention is per sequence either way


def test_sampling_over_shared_prefixes():
    rng = np.random.default_rng(4)
    T, seed = 0.8, 99
    eng = engine(CFG, "bf16")
    eng.set_option(_abi.LLM_OPT_SHARED_PREFIX, 2)
    first = eng.prefill([0], [rng.integers(3, CFG.vocab, 70).tolist()])
    slots = [4, 0, 7, 2, 9]
    eng.fork(0, [s for s in slots if s], 70)
    start = np.full(5, first[0])
    eng.set_sampling(T, seed, True)
    cur, toks, off = start, [], 0
    for k in range(12):
        cur, logits = eng.decode_step(slots, cur, [70 + k] * 5, want_logits=True)
        for s, t, row in zip(slots, cur, logits):
            assert t == O.sample_from_logits(row, T, O.uniform(seed, s, k))
            off += t != np.argmax(row)
        toks.append(cur)
    assert off > 0 and any(len(set(t.tolist())) > 1 for t in toks)  # the samples part
    eng.set_sampling(T, seed, True)
    np.testing.assert_array_equal(eng.generate(slots, start, [70] * 5, 12), np.array(toks))
    eng.close()


def test_the_default_goes_by_the_bytes_it_saves():
    # 15 us at 6.5e6 bytes a us: 97.5 MB of K and V a layer, 1024 bytes a position here.  400 common
    # positions: 239 rows save 238 * 400 of them (97.48 MB), 240 rows 97.89 MB
    rng = np.random.default_rng(6)
    logits = []
    for mode in (None, 0):
        eng = engine(CFG, "bf16", slots=240, max_pos=448)
        eng.set_option(_abi.LLM_OPT_OVERLAP, 0)
        if mode is not None:
            eng.set_option(_abi.LLM_OPT_SHARED_PREFIX, mode)
        eng.prefill([0], [np.random.default_rng(7).integers(3, CFG.vocab, 400).tolist()])
        eng.fork(0, list(range(1, 240)), 400)
        tok = np.random.default_rng(8).integers(3, CFG.vocab, 240)
        per_step = []
        for n in (239, 240):
            out = eng.decode_step(list(range(n)), tok[:n], [400] * n, want_logits=True)[1]
            per_step.append(eng.kernel_count(n))
            logits.append(out)
        assert per_step[1] - per_step[0] == (2 * CFG.n_layers if mode is None else 0)
        eng.close()
    np.testing.assert_array_equal(logits[0], logits[2])
    d = float(np.abs(logits[1] - logits[3]).max())
    assert 0 < d <= REF_ORDER_TOL["bf16"]


def test_refused_forks_leave_slots_and_pages_as_they_were():
    eng = engine(CFG, "bf16", slots=4, max_pos=64)
    prompts = [list(range(3, 43)), list(range(50, 85))]
    eng.prefill([0, 2], prompts)
    eng.fork(0, [3], 20)

    def state():
        return [np.concatenate(eng.read_kv(layer, s, t)) for layer in range(CFG.n_layers)
                for s, n in ((0, 40), (2, 35), (3, 20)) for t in range(n)]
    before = state()
    for parent, children, n, code in ((0, [1, 1], 8, _abi.LLM_ERR_INVALID), (0, [1, 4], 8, _abi.LLM_ERR_INVALID),
                                      (0, [1, 2], 20, _abi.LLM_ERR_STATE), (0, [1], 49, _abi.LLM_ERR_POS_RANGE),
                                      (1, [1], 1, _abi.LLM_ERR_POS_RANGE), (0, [0], 8, _abi.LLM_ERR_STATE)):
        with pytest.raises(_abi.LLMError) as e:
            eng.fork(parent, children, n)
        assert e.value.code == code
    np.testing.assert_array_equal(np.stack(state()), np.stack(before))
    with pytest.raises(_abi.LLMError):
        eng.read_kv(0, 1, 0)                             # still empty
    # every page that they do not hold can be had: 4 x 4 pages, 3 + 3 + 1 held (one shared)
    eng.prefill([1], [list(range(3, 67))])
    eng.fork(1, [], 64)
    eng.prefill([2, 3], [[5] * 29, [6] * 32], start_pos=[35, 32])
    eng.prefill([0], [[7] * 24], start_pos=[40])
    for s in range(4):
        eng.release(s)
    eng.prefill(list(range(4)), [list(range(3, 67))] * 4)  # all of them again
    eng.close()
