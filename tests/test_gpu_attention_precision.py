"""GPU: what fragment attention (ai2bmd_amd/attention.py) may lose to the rows' type: one rounding of each result, nothing
on the way to it.  The cases and the bounds of float32 arithmetic are those of test_gpu_attention.py."""
import math

import numpy as np
import pytest
import torch

from test_gpu_attention import CLIP, E, TYPES, Case, unit

pytestmark = pytest.mark.gpu


def one_against_many(T, n, queries, power, dim=32, heads=2):
    """the first key's score is 0, all others' -power (in units of log 2); values 0 and 1"""
    case = Case([n], T, heads=heads, dim=dim, slope=False, lut=CLIP, queries=[queries])
    case.q.zero_()
    case.v.fill_(1.0)
    case.v[0] = 0.0
    case.terms["residue"].fill_(9)
    case.terms["residue"][0] = 0
    case.terms["query_residue"].zero_()
    case.terms["table"].zero_()
    case.terms["table"][:, 8] = -power * math.log(2.0)
    return case


@pytest.mark.parametrize("T", TYPES, ids=str)
@pytest.mark.parametrize("n,queries", [(40001, 1), (40001, 40), (9001, 9001), (32, 32), (64, 60)])
def test_many_small_terms_under_one_large_one(T, n, queries):
    """Terms of 2^-25.5 of the largest, which a float16 product at 1 takes for 0: n of them are n 2^-25.5 of the result.
    Bound: P to T and the result to T (u each; the weights are equal, so their roundings add up), the score's own error
    (26 + |table| and the exponent's step: 100 E) and the sums; under 2^-14 a float16 result is a multiple of 2^-24."""
    case = one_against_many(T, n, queries, 25.5)
    out = case.plan().forward(case.q, case.k, case.v, **case.terms)
    weight = math.exp(float(case.terms["table"][0, 8].double()))
    want = (n - 1) * weight / (1 + (n - 1) * weight)
    limit = (2 * unit(T) + E * (100 + n / 8)) * want + (2.0 ** -25 if T == torch.float16 else 0.0)
    assert (out.double() - want).abs().max() <= limit


@pytest.mark.parametrize("sizes,queries", [([20], None), ([60], None), ([300], None), ([1700], [1])])
@pytest.mark.parametrize("height", [2.0 ** 19.9, 1.162e7, -1.162e7, 1.163e7, -1.163e7, 2.3e7, -2.33e7, 1e8, 1.5e8, 3e9, -1e8, -1.5e8])
def test_float16_scores_of_any_height(sizes, queries, height):
    """equal scores, up to a height at which float32 no longer tells 14 from 16 (2^24 in units of log 2 is 1.1629e7): the mean
    over the keys (P to float16, the result to float16), and gradients that are finite"""
    case = Case(sizes, torch.float16, heads=2, dim=16, slope=False, lut=[0], queries=queries)
    case.q.zero_()
    case.terms["table"][:] = height
    got = case.results()
    mean = case.v[:sizes[0]].double().mean(0)
    assert ((got["out"].double() - mean).abs() <= 2 * unit(torch.float16) * case.v.double().abs().mean(0) + 2.0 ** -25).all()
    assert all(torch.isfinite(x).all() for x in got.values())


KINDS = {"one tile": dict(sizes=[22, 12, 32, 1] * 3), "one tile, shared heads": dict(sizes=[19, 3, 32] * 3, kv=2, heads=4),
         "many of one tile": dict(sizes=[1 + (7 * i) % 32 for i in range(520)], heads=2, dim=16), "two tiles": dict(sizes=[44, 33, 64, 50]),
         "two tiles, dim 64": dict(sizes=[44, 64], dim=64), "a wave each": dict(sizes=[70, 300, 97], kv=4), "shared tiles": dict(sizes=[150, 130, 65, 260] * 4),
         "pieces": dict(sizes=[1700, 513, 700], queries=[1, 2, 35], kv=2, dim=64), "wide": dict(sizes=[20, 75, 200], heads=4, kv=1, dim=128)}


@pytest.mark.parametrize("T", TYPES[1:], ids=str)
@pytest.mark.parametrize("kind", KINDS)
def test_results_are_rounded_once(T, kind):
    """P and dS reach the products in two parts of T each: hi is off by u of a term, lo by u of that.
    Bound: u |result|, u^2 of the sums' terms (u times what one rounding of P and dS would have been) and the bound of the
    float32 arithmetic alone.  float16: the parts' absolute step is 2^-39 of P and of the largest dS, at most 2 D max|do|
    max|v|, for each of n terms; a result under 2^-14 is a multiple of 2^-24."""
    case = Case(T=T, lut=CLIP, **KINDS[kind])
    got, once = case.results(), case.reference()
    case.T = torch.float32
    bare = case.reference()
    u, extra = unit(T), 0.0
    if T == torch.float16:
        top = lambda x: float(x.double().abs().max())
        n = int(max(np.max(case.end - case.start), np.max(case.q_end - case.q_start))) * case.heads // case.kv
        extra = 2.0 ** -25 + 2.0 ** -38 * n * max(top(case.q), top(case.k), top(case.dout), 1.0) * (1 + 2 * case.dim ** 0.5 * top(case.dout) * top(case.v))
    for name, (value, bound) in bare.items():
        own = got[name].dtype == T
        limit = 1.1 * (1 + u) * bound + (u * value.abs() + 1.1 * u * (once[name][1] - bound) + extra if own else 1e-30)
        off = (got[name].double() - value).abs()
        assert (off <= limit).all(), (name, int((off > limit).sum()), float((off / limit).max()))
