"""The beam search example: page requests and attention over shared prefixes together.  Every beam's
log-probability is recomputed from its whole token sequence with dense attention in 64 bits (q, k, v
and the attention output rounded to the cache's type, as the search holds them).

Tolerance: attention outputs differ by their rounding (2^-8 of bf16, 2^-11 of fp16, relative), which
the 64-to-128-wide sums after it average: a log-probability of a step moves by a few 2^-8 at most, so
steps * 2^-6 (bf16) and steps * 2^-9 (fp16) bound a sum over the steps, fixed before the first run."""
import pytest

pytestmark = pytest.mark.gpu


def dense(m, tokens, dtype):
    """Log-probabilities after every token, without a cache."""
    import torch
    from ane.cmd.beam_search import rows

    def attend(layer, q, k, v):
        q, k, v = (x.to(dtype).double() for x in (q, k, v))
        g = q.shape[1] // k.shape[1]
        k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
        s = torch.einsum("rhd,thd->hrt", q, k) * q.shape[2] ** -0.5
        n = s.shape[1]
        s = s.masked_fill(torch.triu(torch.ones(n, n, dtype=torch.bool, device="cuda"), 1), float("-inf"))
        return torch.einsum("hrt,thd->rhd", torch.softmax(s, -1), v).to(dtype)
    return rows(m, tokens, attend)


@pytest.mark.parametrize("dtype,beams,prompt,steps", [("bf16", 5, 37, 30), ("fp16", 8, 64, 20), ("bf16", 1, 15, 25), ("fp16", 33, 200, 12)])
def test_scores_equal_the_dense_model(dtype, beams, prompt, steps):
    import torch
    from ane.cmd.beam_search import Search, random_model
    m = random_model(beams, dtype=dtype)
    g = torch.Generator().manual_seed(prompt)
    p = torch.randint(0, m.embed.shape[0], (prompt,), generator=g).tolist()
    s = Search(m, beams, p, steps)
    tokens, score = s.run()
    s.cache.check()
    assert tokens.shape == (beams, steps) and bool((score[:-1] >= score[1:]).all())
    tol = steps * (2.0 ** -6 if dtype == "bf16" else 2.0 ** -9)
    for b in sorted({0, beams // 2, beams - 1}):
        lp = dense(m, torch.cat([torch.tensor(p, device="cuda"), tokens[b]])[:-1], s.cache.torch_dtype)[prompt - 1:]
        assert abs(float(lp.gather(1, tokens[b][:, None]).sum()) - float(score[b])) <= tol
    # counts: one reference per held page, the prompt's complete pages held by every beam
    held = s.cache.table[s.cache.table >= 0]
    assert torch.equal(torch.bincount(held.long(), minlength=s.cache.n_pages).int(), s.cache.refs)
    shared = s.cache.table[0, : prompt // 16]
    assert bool((s.cache.refs[shared.long()] == beams + 1).all())
    live = int((s.cache.refs > 0).sum())
    before = [s.cache.pool[:, s.cache.table[int(x)][: -(-(prompt + steps - 1) // 16)].long()].clone() for x in s.banks[s.bank]]
    kept = s.keep_best()
    assert bool((s.cache.refs[:live] > 0).all()) and int(s.cache.n_free.item()) == s.cache.n_pages - live
    for x, pages in zip(s.banks[s.bank], before):
        assert torch.equal(s.cache.pool[:, s.cache.table[int(x)][: pages.shape[1]].long()], pages)
    assert torch.equal(kept.pool[:, kept.table[0][: before[0].shape[1]].long()], before[0])


def test_command_line():
    from ane.cmd import beam_search
    assert beam_search.main(["-beams", "3", "-prompt", "20", "-steps", "5"]) == 0
    with pytest.raises(SystemExit):
        beam_search.main(["-beams", "0"])
