"""The operators on paged caches together, as beam search uses them (examples/beam_search.py): prompts in pieces, beams that share pages, pages that
change hands, ended beams -- against a search in 64 bits that keeps no cache and reorders nothing.

Where two continuations' scores in 64 bits are nearer than TOL, which of them is kept is open; from there on the searches differ, so the test
follows the library's choice and asks that it is a choice within TOL of the best."""
import importlib.util
import math
import os

import pytest
import torch

import helpers

pytestmark = pytest.mark.gpu
TOL = {torch.float32: 2e-3, torch.bfloat16: 0.15}         # an fp32 forward pass of two layers; keys and values in bf16, 2^-8 each


@pytest.fixture(scope="module")
def ex():
    spec = importlib.util.spec_from_file_location("beam_search", os.path.join(helpers.ROOT, "examples", "beam_search.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def log_probs(ex, w, ids):
    """[rows][T] -> log probabilities after every token, float64 [rows][T][VOCAB]"""
    d = lambda t: t.double()
    rms = lambda x: x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    B, T = ids.shape
    x = d(w.emb)[ids]
    f = 10000.0 ** (-torch.arange(ex.HD // 2, device="cuda", dtype=torch.float64) * 2 / ex.HD)
    a = torch.arange(T, device="cuda", dtype=torch.float64)[:, None] * f
    c, s = a.cos()[:, None], a.sin()[:, None]
    half = ex.HD // 2
    turn = lambda y: torch.cat([y[..., :half] * c - y[..., half:] * s, y[..., half:] * c + y[..., :half] * s], -1)
    mask = torch.ones(T, T, dtype=torch.bool, device="cuda").tril()
    for l in w.layers:
        qkv = (rms(x) @ d(l["qkv"]).t()).view(B, T, ex.H + 2 * ex.NKV, ex.HD)
        q, k, v = turn(qkv[:, :, :ex.H]), turn(qkv[:, :, ex.H:ex.H + ex.NKV]), qkv[:, :, ex.H + ex.NKV:]
        k, v = (t.repeat_interleave(ex.H // ex.NKV, 2) for t in (k, v))
        p = torch.einsum("bthd,bshd->bhts", q, k) / math.sqrt(ex.HD)
        p = torch.softmax(p.masked_fill(~mask, float("-inf")), -1)
        x = x + torch.einsum("bhts,bshd->bthd", p, v).reshape(B, T, -1) @ d(l["o"]).t()
        h = rms(x) @ d(l["up"]).t()
        x = x + (h * torch.sigmoid(h)) @ d(l["down"]).t()
    return torch.log_softmax(rms(x) @ d(w.head).t(), -1)


def scored(ex, w, prompt, text):
    """Scores of texts [beams][n] in 64 bits, and whether they have ended: nothing counts after EOS."""
    ids = torch.cat([prompt.expand(text.shape[0], -1), text.long()], 1)
    lp = log_probs(ex, w, ids)[:, prompt.shape[0] - 1:-1].gather(2, text.long()[:, :, None])[:, :, 0]
    ended = (text == ex.EOS).cumsum(1) - (text == ex.EOS).int() > 0            # an EOS stands before
    return lp.masked_fill(ended, 0.0).sum(1), ended


@pytest.mark.parametrize("cache", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("groups,beams,length,new", [(3, 4, 200, 24), (1, 1, 16, 20), (2, 7, 129, 40), (5, 3, 31, 17)])
def test_search(ex, cache, groups, beams, length, new):
    w = ex.Weights(3)
    w.head[ex.EOS] *= 3.0                                     # so that beams end
    g = torch.Generator().manual_seed(groups * 10 + beams)
    prompts = torch.randint(0, ex.VOCAB, (groups, length), generator=g)
    text, scores, done = ex.search(w, prompts.tolist(), beams, new, cache)
    tol = TOL[cache]
    for i in range(groups):
        prompt = prompts[i].cuda()
        want, ended = scored(ex, w, prompt, text[i])
        assert ((want - scores[i].double()).abs() <= tol).all(), (want - scores[i]).abs().max()
        assert (scores[i, :-1] >= scores[i, 1:]).all()
        assert len({tuple(t) for t in text[i].tolist()}) == beams
        assert torch.equal(done[i] != 0, (text[i] == ex.EOS).any(1))
        assert (text[i][ended] == ex.EOS).all()
        # no continuation of what the last step had to choose from is better than the worst that it kept
        last, old = text[i][:, :-1], scored(ex, w, prompt, text[i][:, :-1])[0]
        nxt = log_probs(ex, w, torch.cat([prompt.expand(beams, -1), last.long()], 1))[:, -1]
        kept = {tuple(t) for t in text[i].tolist()}
        over = (last == ex.EOS).any(1)
        for k in range(beams):
            if over[k]:
                continue
            best = old[k] + nxt[k]
            for t in best.topk(beams + 1).indices.tolist():
                if tuple(last[k].tolist() + [t]) not in kept:
                    assert best[t] <= scores[i, -1].double() + 2 * tol


def test_one_beam_is_greedy(ex):
    w = ex.Weights(5)
    prompt = torch.randint(0, ex.VOCAB, (1, 50), generator=torch.Generator().manual_seed(2))
    text, scores, _ = ex.search(w, prompt.tolist(), 1, 30, torch.float32)
    ids = torch.cat([prompt.cuda(), text[0].long()], 1)
    lp = log_probs(ex, w, ids)[0, 49:-1]
    for t in range(30):
        if ex.EOS in text[0, 0, :t].tolist():
            break
        assert lp[t, text[0, 0, t]] >= lp[t].max() - 1e-3


def test_the_same_again(ex):
    w = ex.Weights(6)
    prompts = torch.randint(0, ex.VOCAB, (2, 70), generator=torch.Generator().manual_seed(3)).tolist()
    a, b = (ex.search(w, prompts, 5, 33) for _ in range(2))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
