"""Scoring continuations over the cached prompt, on a B200, against the FP32 golden run on every prefix."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", params=["tiny-hd96", "tiny-hd128"])
def model(request):
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from minicpm5_mk import mk_weights
    from minicpm5_mk.mk_config import PRESETS
    from minicpm5_mk.mk_init import random_state_dict, synthetic_ids
    from oracle import golden
    cfg = PRESETS[request.param]
    sd = random_state_dict(cfg, seed=1234)
    return cfg, mk_weights.prepare_mk_weights(sd, cfg), golden.golden_weights(sd, cfg), \
        synthetic_ids(1, 400, seed=11, vocab=cfg.vocab)[0]


def _want(ids, at, W, cfg):
    """(log-probability of ids[at], bound): the repository's accuracy target for logits, 2e-2 of their range, for
    the token's logit and for the normaliser."""
    from oracle import golden
    lg = golden.forward_logits(ids[:at], W, cfg).double()
    return float(torch.log_softmax(lg, 0)[int(ids[at])]), 2 * 2e-2 * float(lg.max() - lg.min())


@pytest.mark.parametrize("n,page", [(1, 16), (130, 32), (257, 64)])
def test_prompt_and_candidates_against_the_golden(model, n, page):
    from minicpm5_mk.continuations import ContinuationScorer
    cfg, pw, W, ids = model
    s = ContinuationScorer(cfg, pw, pages=60, page_size=page)
    prompt = s.prefill(ids[:n].tolist()).cpu()
    assert prompt.shape == (n - 1,)
    for i in sorted({1, n // 2, n - 1} - {0} if n > 1 else set()):
        w, tol = _want(ids, i, W, cfg)
        assert abs(float(prompt[i - 1]) - w) <= tol, (i, float(prompt[i - 1]), w, tol)
    cands = [ids[300:305].tolist(), ids[310:311].tolist(), [], ids[320:340].tolist()]
    got = [t.cpu() for t in s.score(cands)]
    assert [len(t) for t in got] == [5, 1, 0, 20]
    for c, t in zip(cands, got):
        for j in sorted({0, len(c) // 2, len(c) - 1} if c else set()):
            full = torch.cat([ids[:n], torch.tensor(c)])
            w, tol = _want(full, n + j, W, cfg)
            assert abs(float(t[j]) - w) <= tol, (j, float(t[j]), w, tol)
    # nothing of the prompt has changed: the same calls give the same bits, after compaction too
    again = s.score(cands)
    assert all(torch.equal(a, b.cpu()) for a, b in zip(got, again))
    assert s.compact() == -(-n // page)
    assert all(torch.equal(a, b.cpu()) for a, b in zip(got, s.score(cands)))
    top, lps = s.alternatives(4)
    from oracle import golden
    lg = golden.forward_logits(ids[:n], W, cfg).double()
    assert int(top[0]) == int(lg.argmax()) or float(lg.max() - lg[int(top[0])]) <= 2 * 2e-2 * float(lg.max() - lg.min())
    assert bool((lps[:-1] >= lps[1:]).all())


def test_running_out_of_pages_and_bad_lengths(model):
    from minicpm5_mk import _lib
    from minicpm5_mk.continuations import ContinuationScorer
    cfg, pw, _, ids = model
    s = ContinuationScorer(cfg, pw, pages=6, page_size=16)
    with pytest.raises(ValueError):
        s.score([[1]])
    with pytest.raises(ValueError):
        s.prefill([])
    with pytest.raises(ValueError):
        s.prefill([1] * (cfg.max_seq + 1))
    with pytest.raises(_lib.MkError):
        s.prefill(ids[:200].tolist())
    s.prefill(ids[:50].tolist())  # 4 pages
    with pytest.raises(_lib.MkError):
        s.score([[1, 2], [3], [4]])
    s.prefill(ids[:50].tolist())
    assert len(s.score([[1, 2]])[0]) == 2
