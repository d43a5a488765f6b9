"""llm_seq_fork and decode steps over shared prefixes (LLM_OPT_SHARED_PREFIX), against slots that
were prefilled one by one.  The forked pages hold the same values, so per-sequence attention must
give the same bits; over shared prefixes attention sums in another order, which moves logits by
rounding only: the bounds are those of two orders of operations at one precision
(parity.REF_ORDER_TOL)."""
import numpy as np
import pytest

from ane import _abi
from ane.stories import Engine, ModelConfig, SyntheticWeights
from parity import REF_ORDER_TOL

pytestmark = pytest.mark.gpu

CFG = ModelConfig(dim=256, hidden=512, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=128, vocab=2048, max_seq=512, qk_norm=True,
                  tied_embed=True, norm_eps=1e-6, rope_theta=1e6, name="fork")
MHA = ModelConfig(dim=256, hidden=512, n_layers=2, n_heads=4, n_kv_heads=4, head_dim=64, vocab=1024, max_seq=512, name="fork-mha")
WEIGHTS = {}


def engine(cfg, dtype, slots=12, max_pos=400):
    if cfg.name not in WEIGHTS:
        WEIGHTS[cfg.name] = SyntheticWeights(cfg, 77, 1.0, stddev=0.04)
    return Engine(cfg, dtype, 0).load(WEIGHTS[cfg.name]).kv_alloc(slots, max_pos)


def steps(eng, seqs, prompt_len, first, n, seed):
    """n decode steps with given tokens; logits of each."""
    rng = np.random.default_rng(seed)
    toks = rng.integers(3, eng.cfg.vocab, (n, len(seqs)))
    toks[0] = first
    return [eng.decode_step(seqs, toks[i], [prompt_len + i] * len(seqs), want_logits=True)[1] for i in range(n)]


@pytest.mark.parametrize("cfg,dtype", [(CFG, "bf16"), (MHA, "fp16"), (CFG, "w8a8_bf16")])
@pytest.mark.parametrize("length", [7, 48, 133])
def test_forks_equal_separate_prefills(cfg, dtype, length):
    rng = np.random.default_rng(length)
    prompt = rng.integers(3, cfg.vocab, length).tolist()
    seqs = [4, 0, 9, 2, 7, 11]
    a = engine(cfg, dtype)
    a.prefill(seqs, [prompt] * len(seqs))
    first = rng.integers(3, cfg.vocab, len(seqs))
    want = steps(a, seqs, length, first, 20, 1)
    for mode in (0, 2):
        b = engine(cfg, dtype)
        b.set_option(_abi.LLM_OPT_SHARED_PREFIX, mode)
        b.prefill([4], [prompt])
        b.fork(4, [s for s in seqs if s != 4], length)
        got = steps(b, seqs, length, first, 20, 1)
        for layer in range(cfg.n_layers):
            for s in seqs:
                for x, y in zip(a.read_kv(layer, s, length - 1), b.read_kv(layer, s, length - 1)):
                    np.testing.assert_array_equal(x, y)
        for x, y in zip(want, got):
            if mode == 0:
                np.testing.assert_array_equal(x, y)
            else:
                assert float(np.abs(x - y).max()) <= REF_ORDER_TOL[dtype]
        b.close()
    a.close()


@pytest.mark.parametrize("cfg,dtype", [(MHA, "w8a8_fp16"), (CFG, "w8a8_bf16"), (MHA, "fp16")])
def test_groups_and_lone_sequences_in_one_step(cfg, dtype):
    # a group of four, a group of two and two sequences that share with nobody
    rng = np.random.default_rng(8)
    prompts = {s: rng.integers(3, cfg.vocab, n).tolist() for s, n in ((0, 100), (1, 64), (2, 45), (3, 5))}
    seqs = [6, 2, 0, 8, 1, 7, 3, 5]
    owner = {6: 0, 7: 0, 8: 0, 5: 1}
    runs = []
    for mode in (0, 2):
        eng = engine(cfg, dtype)
        eng.set_option(_abi.LLM_OPT_SHARED_PREFIX, mode)
        eng.prefill(list(prompts), list(prompts.values()))
        eng.fork(0, [6, 7, 8], 100)
        eng.fork(1, [5], 64)
        pos = np.array([len(prompts[owner.get(s, s)]) for s in seqs], np.int32)
        tok = np.random.default_rng(9).integers(3, cfg.vocab, (20, len(seqs)))
        runs.append([eng.decode_step(seqs, tok[i], pos + i, want_logits=True)[1] for i in range(20)])
        eng.close()
    for x, y in zip(*runs):
        assert float(np.abs(x - y).max()) <= REF_ORDER_TOL[dtype]


def test_generate_over_shared_prefixes_follows_the_step_loop():
    rng = np.random.default_rng(3)
    prompts = [rng.integers(3, CFG.vocab, n).tolist() for n in (70, 33)]
    eng = engine(CFG, "bf16")
    eng.set_option(_abi.LLM_OPT_SHARED_PREFIX, 2)
    eng.prefill([0, 1], prompts)
    eng.fork(0, [2, 3, 4, 5], 70)
    eng.fork(1, [6, 7], 33)
    seqs = [5, 6, 0, 2, 7, 3, 1, 4]  # groups interleaved in the batch
    pos = [33 if s in (1, 6, 7) else 70 for s in seqs]
    tok = rng.integers(3, CFG.vocab, len(seqs))
    out = eng.generate(seqs, tok, pos, 24)
    for s in range(2, 8):
        eng.release(s)
    # the same batch again by steps, with graphs and without
    for graphs in (1, 0):
        eng.set_option(_abi.LLM_OPT_CUDA_GRAPHS, graphs)
        eng.fork(0, [2, 3, 4, 5], 70)
        eng.fork(1, [6, 7], 33)
        cur, p = tok, np.array(pos)
        for i in range(24):
            cur = eng.decode_step(seqs, cur, p)
            np.testing.assert_array_equal(cur, out[i])
            p = p + 1
        for s in range(2, 8):
            eng.release(s)
    eng.close()


def test_pages_return_when_the_last_holder_leaves():
    eng = engine(CFG, "bf16", slots=3, max_pos=64)  # 12 pages
    prompt = list(range(3, 43))
    eng.prefill([0], [prompt])                       # 3 pages
    eng.fork(0, [1], 40)                             # 2 shared, 1 copied
    first = eng.read_kv(0, 0, 5)
    eng.release(0)
    for x, y in zip(first, eng.read_kv(0, 1, 5)):
        np.testing.assert_array_equal(x, y)          # slot 1 still holds them
    eng.prefill([0, 2], [list(range(3, 67))] * 2)    # 8 more: 11 of 12
    for x, y in zip(first, eng.read_kv(0, 1, 5)):
        np.testing.assert_array_equal(x, y)
    eng.release(1)
    eng.release(0)
    eng.prefill([0, 1], [list(range(3, 67))] * 2)    # every page is free again
    eng.close()


def test_shared_pages_are_read_only_and_bad_forks_are_refused():
    eng = engine(CFG, "bf16", slots=4, max_pos=64)
    eng.prefill([0], [list(range(3, 43))])
    eng.fork(0, [1], 40)

    def refused(code, f):
        with pytest.raises(_abi.LLMError) as e:
            f()
        assert e.value.code == code
    # positions below 32 lie in shared pages, 32..39 in each slot's own copy
    refused(_abi.LLM_ERR_STATE, lambda: eng.decode_step([1], [5], [31]))
    refused(_abi.LLM_ERR_STATE, lambda: eng.prefill([0], [[5, 6]]))
    refused(_abi.LLM_ERR_STATE, lambda: eng.prefill([1], [[5] * 4], start_pos=[30]))
    refused(_abi.LLM_ERR_STATE, lambda: eng.generate_begin([0], [5], [16], 2))
    eng.decode_step([0, 1], [5, 6], [32, 40])
    refused(_abi.LLM_ERR_STATE, lambda: eng.fork(0, [1], 8))            # not empty
    refused(_abi.LLM_ERR_INVALID, lambda: eng.fork(0, [2, 2], 8))
    refused(_abi.LLM_ERR_INVALID, lambda: eng.fork(0, [4], 8))
    refused(_abi.LLM_ERR_INVALID, lambda: eng.fork(-1, [2], 8))
    refused(_abi.LLM_ERR_POS_RANGE, lambda: eng.fork(0, [2], 0))
    refused(_abi.LLM_ERR_POS_RANGE, lambda: eng.fork(0, [2], 49))
    refused(_abi.LLM_ERR_POS_RANGE, lambda: eng.fork(2, [3], 1))        # an empty parent
    refused(_abi.LLM_ERR_INVALID, lambda: eng.set_option(_abi.LLM_OPT_SHARED_PREFIX, 3))
    eng.release(1)
    eng.prefill([0], [[5, 6]])  # nothing shared any more
    eng.close()


def test_a_fork_that_finds_no_free_page_changes_nothing():
    eng = engine(CFG, "bf16", slots=3, max_pos=32)   # 6 pages
    eng.prefill([0], [list(range(3, 35))])           # 2
    eng.fork(0, [1, 2], 32)                          # shared
    eng.release(1)
    eng.release(2)
    eng.prefill([1], [list(range(3, 35))])           # 4
    eng.fork(1, [2], 17)                             # 5
    eng.release(0)                                   # 3
    eng.prefill([0], [list(range(3, 35))])           # 5
    eng.release(2)                                   # 4
    eng.prefill([2], [[7]])                          # 5
    eng.release(2)
    eng.fork(0, [2], 20)                             # 5
    eng.release(2)
    with pytest.raises(_abi.LLMError) as e:
        eng.fork(0, [2], 33)
    assert e.value.code == _abi.LLM_ERR_POS_RANGE
    eng.close()
    eng = engine(CFG, "bf16", slots=4, max_pos=16)   # 4 pages, one a slot
    eng.prefill([0, 1], [[5, 6, 7]] * 2)
    eng.prefill([2], [[5]])
    eng.release(2)
    eng.fork(0, [2, 3], 3)                           # the last two
    eng.release(3)
    eng.prefill([3], [[9]])
    eng.release(2)
    eng.fork(3, [2], 1)
    with pytest.raises(_abi.LLMError) as e:
        eng.fork(0, [2], 3)
    assert e.value.code == _abi.LLM_ERR_STATE
    eng.close()
