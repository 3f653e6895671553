"""moe_router with a selection bias on rows that hold NaN or infinities, against the formula in 64 bits.

A logit of NaN or -inf is no candidate; the scores to which the bias is added are the candidates' own: softmax over the candidates, where logits of +inf share
the whole of it among them (the limit).  Weights do not change with a bias: over the selected logits with renormalize, else over all logits, where what is not finite
shows.  Tolerances: test_gpu_router."""
import math

import pytest
import torch

import catccos_amd as cc
from test_gpu_router import RTOL

pytestmark = pytest.mark.gpu
K = 4


def candidates_scores(row, scoring):
    """Scores in 64 bits by which candidates are compared; None: no candidate."""
    there = [e for e, v in enumerate(row) if v == v and v > -math.inf]
    top = max((row[e] for e in there), default=0.0)
    if scoring == "sigmoid":
        return [1 / (1 + math.exp(-v)) if e in there else None for e, v in enumerate(row)]
    raw = {e: (1.0 if row[e] == top else 0.0) if top == math.inf else math.exp(row[e] - top) for e in there}
    total = sum(raw.values())
    return [raw[e] / total if e in raw else None for e in range(len(row))]


def selected(row, bias, scoring):
    keys = [(s + b, -e) for e, (s, b) in enumerate(zip(candidates_scores(row, scoring), bias)) if s is not None and s + b > -math.inf]
    keys.sort(reverse=True)
    assert all(a[0] - b[0] > 1e-6 for a, b in zip(keys[:K], keys[1:K + 1])), "the case's keys are too near one another for fp32"
    return [-e for _, e in keys[:K]] + [-1] * (K - len(keys[:K]))


def rows(e):
    gen = torch.Generator().manual_seed(e)
    l = torch.randn(12, e, generator=gen)
    bias = torch.randperm(e, generator=gen).float() * 0.0371              # (no multiple of it is near a share of 1/2 or 1)
    l[0, 3] = math.nan                                   # an expert that the bias dislikes or likes
    l[1, int(bias.argmax())] = math.nan                  # the one that it likes best
    l[2, 1::2] = math.nan
    l[3, 1:] = math.nan                                  # one candidate
    l[4] = math.nan                                      # none
    l[5, 5] = math.inf
    l[6, 2], l[6, 7] = math.inf, math.inf
    l[7, 4], l[7, 9] = math.inf, math.nan
    l[8, 6:] = -math.inf
    l[8, 0] = math.nan
    l[9, 3] = math.nan                                   # of a masked token
    l[10, int(bias.argmax())] = math.inf                 # selected for certain
    return l, bias


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("e", [16, 72, 200, 500, 1000])
def test_candidates_are_selected_by_their_own_scores(e, renorm, scoring, dtype):
    l, bias = rows(e)
    l = l.to(dtype)
    mask = torch.ones(12, dtype=torch.bool)
    mask[9] = False
    probs, idx = cc.moe_router(l.cuda(), K, scoring=scoring, renormalize=renorm, bias=bias.cuda(), token_mask=mask.cuda())
    probs, idx = probs.cpu().double(), idx.cpu()
    for t in range(12):
        row = [float(v) for v in l[t]]
        want = selected(row, [float(b) for b in bias], scoring) if mask[t] else [-1] * K
        assert idx[t].tolist() == want, t
        got = probs[t][idx[t] >= 0]
        assert (probs[t][idx[t] < 0] == 0).all()
        if not len(got):
            continue
        chosen = l[t][idx[t][idx[t] >= 0].long()].double()
        if scoring == "sigmoid":
            w = torch.sigmoid(chosen)
        elif renorm:
            w = torch.softmax(chosen, 0)                 # NaN where a chosen logit is +inf
        else:
            w = torch.softmax(l[t].double(), 0)[idx[t][idx[t] >= 0].long()]      # NaN where any logit is not a number below +inf
        w = w / w.sum() if renorm else w
        assert torch.equal(got.isnan(), w.isnan()), t
        ok = ~w.isnan()
        assert ((got - w).abs()[ok] <= RTOL * w[ok]).all(), t


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_an_expert_that_the_bias_takes_out_of_service(scoring):
    l, bias = rows(64)
    bias[5] = -math.inf                                  # row 5's infinite logit among them
    bias[int(bias.argmax())] = math.nan
    _, idx = cc.moe_router(l.cuda(), K, scoring=scoring, bias=bias.cuda())
    assert not (idx == 5).any()
    usable = [float(b) if b == b else -math.inf for b in bias]
    for t in range(12):
        assert idx[t].tolist() == selected([float(v) for v in l[t]], usable, scoring), t
