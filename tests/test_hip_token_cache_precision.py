"""Attention over a cache and masked attention where precision is decided: rows whose mass is one key and a long tail, weights of 16 bits,
distances far from the keys.  Plain forms: test_hip_token_cache.py.

Bounds, of |got - want|, with u half a step of the output's type (bf16 2^-8, fp16 2^-11) and w_j the weights over their sum:
  * u |want|: the output's own rounding;
  * sum_j r_j |v_j|, r_j what the rounding of a weight takes from it: u w_j where weights are one operand of the output's type, for fp16 not
    below half its smallest step, 2^-25, relative to the largest weight that an operand holds, 2^11 (the kernels scale
    fp16 weights by that, so that the largest of a row, up to 2^4 over the running maximum, is still finite): 2^-36 of the row's largest
    weight; 2^-16 w_j where weights are two bf16 operands (half a step of a half step, 2^-8 2^-8);
  * scores: with n elements of q that are not zero the fp32 score is off by at most (n + 8) 2^-24 times the sum of its terms' sizes, the
    exponent's products and sums by a few 2^-24 of the score: 2 (n + 8) 2^-24 score, relative to every weight;
  * sums of N keys in fp32, 32 keys to a product, 8 roundings at most within one: (N / 4 + 64) 2^-24 of sum_j w_j |v_j|;
  * 2^-24 for outputs that are subnormal in fp16."""
import math

import pytest
import torch

from test_hip_token_cache import DEV, cache_reference, encode, masked_reference, ops, run_cache, run_masked  # noqa: F401

pytestmark = pytest.mark.gpu


def within(got, want, top, score, kind, weights, nonzero, keys, tail=0.0):
    """`weights`: relative rounding of a weight; `tail`: what the smallest weights may lose, sum_j |v_j| 2^-36 at most"""
    u = torch.finfo(kind).eps / 2
    assert bool(torch.isfinite(want).all())
    bound = u * want.abs() + (weights + 2 * (nonzero + 8) * 2.0 ** -24 * score.unsqueeze(-1) + (keys / 4 + 64) * 2.0 ** -24) * top + tail + 2.0 ** -24
    off = (got.double().cpu() - want).abs() / bound
    assert float(off.nan_to_num(math.inf).max()) <= 1.0, float(off.nan_to_num(math.inf).max())


# ---- one key far above all others, whose value is zero: the row's result is the tail's -----------------------------------------------

def sink(g, q_lead, k_lead, axis, N, D, at, gap):
    """Queries along the first axis; keys of score 0 to 1, one of `gap` with a value of zero; values from 20 to 60."""
    q = torch.zeros(*q_lead, D)
    q[..., 0] = 1
    k, v = torch.zeros(*k_lead, D), 20 + 40 * torch.rand(*k_lead, D, generator=g)
    k[..., 0] = torch.rand(*k_lead, generator=g)
    k.select(axis, at)[..., 0] = gap
    v.select(axis, at)[...] = 0
    return q.half(), k.half(), v.half()


GAPS = [11.0, 15.0, 17.5, 19.0]


@pytest.mark.parametrize("gap", GAPS)
@pytest.mark.parametrize("D,Lq,Lk,at,mode", [(64, 40, 900, 5, "plain"), (128, 300, 3001, 0, "plain"), (256, 33, 500, 2, "plain"), (32, 500, 500, 0, "causal"), (96, 130, 700, 9, "cap"),
                                             (64, 70, 2000, 1, "bias"), (128, 600, 600, 300, "doc"), (64, 4, 9000, 0, "plain")])
def test_a_tail_far_below_one_key_of_a_prompt(ops, D, Lq, Lk, at, mode, gap):  # noqa: F811
    g = torch.Generator().manual_seed(D + Lk)
    q, k, v = sink(g, (1, Lq, 2), (1, Lk, 1), 1, Lk, D, at, gap)
    slopes = torch.tensor([2.0 ** -14, 2.0 ** -13]) if mode == "bias" else None
    doc = (torch.arange(Lk) // 300).int().unsqueeze(0) if mode == "doc" else None
    cap = 200.0 if mode == "cap" else 0.0
    args = (1.0, mode == "causal", cap, slopes, None, None, None, doc)
    want, top, score = masked_reference(q, k, v, *args)
    within(run_masked(ops, q, k, v, *args), want, top, score + (cap and 4 * cap / 10), torch.float16, 2.0 ** -11, 1, Lk, Lk * 60 * 2.0 ** -36)


TAILS = [  # B, T, Hq, Hkv, D, C, P, where the far key lies: own tokens, the prefix
    (1, 1, 2, 1, 64, 400, 0, "own"),                  # a workgroup a stream
    (2, 1, 4, 2, 128, 3000, 0, "own"),                # shares
    (2, 5, 8, 2, 32, 3000, 0, "own"),                 # waves on different rows
    (2, 1, 4, 2, 256, 900, 0, "own"),
    (2, 1, 4, 2, 96, 60, 500, "prefix"),
    (2, 1, 4, 2, 64, 500, 60, "own"),
    (64, 1, 16, 2, 64, 33, 9000, "prefix"),           # the product over the prefix is large: the kernel of whole prompts
    (64, 1, 16, 2, 64, 33, 9000, "own"),
    (40, 2, 8, 1, 256, 20, 7600, "prefix"),
]


@pytest.mark.parametrize("gap", GAPS)
@pytest.mark.parametrize("case", TAILS, ids=lambda c: "x".join(map(str, c)))
def test_a_tail_far_below_one_key_of_a_cache(ops, case, gap):  # noqa: F811
    B, T, Hq, Hkv, D, C, P, where = case
    g = torch.Generator().manual_seed(D + C)
    q, k, v = sink(g, (B, T, Hq), (B, Hkv, C), 2, C, D, 2, gap if where == "own" else 0.5)
    _, pk, pv = sink(g, (1,), (Hkv, P), 1, P, D, 2, gap if where == "prefix" else 0.5) if P else (None, torch.zeros(Hkv, 0, D).half(), torch.zeros(Hkv, 0, D).half())
    x = {"q": q, "k": k, "v": v, "pk": pk, "pv": pv, "ks": None, "vs": None, "pks": None, "pvs": None}
    lens = torch.full((B,), C, dtype=torch.int32)
    got = run_cache(ops, x, lens, "plain", 1.0, 0.0, None, P)
    few = {**x, **{n: x[n][:2] for n in ("q", "k", "v")}}
    want, top, score = cache_reference(few, lens[:2], "plain", 1.0, 0.0, None, P)
    within(got[:2], want, top, score, torch.float16, 2.0 ** -11, 1, C + P, (C + P) * 60 * 2.0 ** -36)


# ---- caches whose weights are two bf16 operands: their rounding is below the output's, whichever kernel takes the keys -----------------

def peaked(g, *shape):
    """Four elements of a query, scores of about +-5: a few keys have nearly all of the weight"""
    q = torch.zeros(*shape)
    q[..., :4] = 3 * torch.randn(*shape[:-1], 4, generator=g)
    return q


WIDE = [  # B, T, Hq, Hkv, D, C, P, cap, slopes, formats
    (2, 1, 4, 2, 64, 500, 0, 0.0, False, "plain mxfp8 mxfp4"),
    (2, 5, 8, 2, 128, 2000, 0, 0.0, False, "plain mxfp8 mxfp4"),
    (3, 1, 8, 2, 256, 100, 333, 0.0, True, "plain mxfp8"),
    (24, 1, 16, 2, 96, 40, 700, 30.0, False, "plain mxfp4"),
    (32, 1, 16, 1, 32, 20, 9000, 0.0, False, "mxfp8"),
    (128, 4, 32, 2, 32, 9, 3500, 0.0, False, "plain"),                 # the product over the prefix is large: the kernel of whole prompts
    (128, 4, 32, 2, 64, 33, 1800, 0.0, False, "plain"),
    (128, 4, 32, 2, 64, 33, 1800, 25.0, True, "plain"),
    (128, 4, 32, 2, 64, 300, 1800, 0.0, True, "plain"),
    (128, 4, 32, 2, 96, 33, 2000, 0.0, True, "plain"),
    (128, 4, 32, 2, 128, 33, 1500, 25.0, False, "plain"),
    (128, 4, 32, 2, 128, 33, 1500, 0.0, True, "plain"),
    (128, 4, 32, 2, 256, 9, 800, 0.0, False, "plain"),
    (128, 4, 32, 2, 256, 9, 800, 40.0, True, "plain"),
    (1, 512, 32, 2, 64, 512, 1800, 0.0, False, "plain"),
]


@pytest.mark.parametrize("case,form", [(c, f) for c in WIDE for f in c[9].split()], ids=lambda c: c if isinstance(c, str) else "x".join(map(str, c[:9])))
def test_weights_over_a_cache_of_bf16_have_16_bits(ops, case, form):  # noqa: F811
    B, T, Hq, Hkv, D, C, P, cap, alibi, _ = case
    g = torch.Generator().manual_seed(sum(case[:7]))
    rows = lambda *lead: torch.randn(*lead, D, generator=g)  # noqa: E731
    x = {"q": peaked(g, B, T, Hq, D).to(torch.bfloat16)}
    for n, lead in (("k", (B, Hkv, C)), ("v", (B, Hkv, C)), ("pk", (Hkv, P)), ("pv", (Hkv, P))):
        x[n], x[n + "s"] = (rows(*lead).to(torch.bfloat16), None) if form == "plain" else encode(rows(*lead), form)
    lens = torch.tensor([max(T, C - 7 * b) for b in range(B)], dtype=torch.int32)
    slopes = torch.exp2(-torch.arange(1, Hq + 1).float() * 8 / Hq) if alibi else None
    got = run_cache(ops, x, lens, form, 1.0, cap, slopes, P)
    few = {**x, **{n: None if x[n] is None else x[n][:6] for n in ("q", "k", "v", "ks", "vs")}}
    want, top, _ = cache_reference(few, lens[:6], form, 1.0, cap, slopes, P)
    # sizes of scores that have weight: their products, 30 of bias at most below the row's largest, 8 roundings of the cap
    score = cache_reference(few, lens[:6], form, 1.0, 0.0, None, P)[2] + (30.0 if alibi else 0.0) + cap / 3
    within(got[:6], want, top, score, torch.bfloat16, 2.0 ** -16, 4, C + P)


# ---- positions far from the keys: what all keys of a row have in common is no part of a softmax -------------------------------------

@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("start,causal", [([10 ** 6, -10 ** 6], False), ([2 ** 30, 12345678], True), ([2 ** 31 - 1, -2 ** 31], False), ([700, -300], False)])
@pytest.mark.parametrize("D,Lq,Lk", [(64, 50, 400), (128, 200, 300), (256, 7, 2000)])
def test_queries_far_from_the_keys(ops, D, Lq, Lk, start, causal, cap, kind):  # noqa: F811
    """The distance of key j is that of the nearest key and what j adds to it, and the first part is the same for all keys of a row."""
    g = torch.Generator().manual_seed(D)
    q, k, v = (torch.randn(2, n, h, D, generator=g).to(kind) for n, h in ((Lq, 4), (Lk, 2), (Lk, 2)))
    slopes = torch.tensor([0.5, 0.1, -0.03, 2.0 ** -8])
    lens = torch.tensor([Lk, Lk - 90], dtype=torch.int32)
    at = torch.tensor(start, dtype=torch.int64).clamp(-2 ** 30, 2 ** 30)
    args = (D ** -0.5, causal, cap, slopes, lens)
    want, top, _ = masked_reference(q, k, v, *args, at, None, None)
    score = torch.full(want.shape[:-1], 30.0 + 0.5 * 60 + 0.03 * (Lk + Lq))    # sizes that carry weight: products, bias from the nearest key on
    got = ops.attention_masked(q.to(DEV), k.to(DEV), v.to(DEV), D ** -0.5, causal, cap, slopes.to(DEV), lens.to(DEV),
                               torch.tensor(start, dtype=torch.int32, device=DEV), None, None, None)
    within(got, want, top, score, kind, torch.finfo(kind).eps / 2, D, Lk, Lk * float(v.abs().max()) * 2.0 ** -36)


# ---- scores so large that fp32 holds no fraction of them --------------------------------------------------------------------------

@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", [2.0 ** 8, 2.0 ** 11, 2.0 ** 12.5])
@pytest.mark.parametrize("D,mode", [(64, "plain"), (128, "plain"), (256, "plain"), (64, "bias"), (128, "bias"), (64, "negative")])
def test_scores_without_a_fraction(ops, D, mode, size, kind):  # noqa: F811
    """Scores of up to 2^26: neighbouring fp32 numbers are up to 8 apart, and so are products and references.  The largest score is alone by far
    more than that, and its value is the answer: its weight is a power of 2 with any fraction, rounded for the product, not in the sum."""
    g = torch.Generator().manual_seed(D)
    Lq, Lk = 70, 500
    q, k = torch.zeros(2, Lq, 2, D), torch.zeros(2, Lk, 1, D)
    q[..., 0] = size * (1 + torch.arange(Lq).view(1, Lq, 1) / 128)                   # (8 bits)
    k[..., 0] = size * (1 + torch.stack([torch.randperm(Lk, generator=g) for _ in range(2)]).view(2, Lk, 1) % 128 / 128)
    best = k[:, :, 0, 0].argmax(1)
    for b in range(2):                                                               # one largest key, the others at most half of it
        k[b, :, 0, 0] /= 2
        k[b, best[b], 0, 0] *= 2
    q, k, v = q.to(kind), k.to(kind), torch.randn(2, Lk, 1, D, generator=g).to(kind)
    scale = -1.0 if mode == "negative" else 1.0
    k = -k if mode == "negative" else k
    want = v[torch.arange(2), best, 0].view(2, 1, 1, D).expand(2, Lq, 2, D)
    slopes = torch.tensor([0.25, 2.0 ** -6], device=DEV) if mode == "bias" else None
    d = [t.to(DEV) for t in (q, k, v)]
    got = ops.attention_masked(*d, scale, False, 0.0, slopes, None, None, None, None, None)
    u, none = torch.finfo(kind).eps / 2, torch.zeros(want.shape[:-1], dtype=torch.float64)
    within(got, want.double(), want.double().abs(), none, kind, u, 1, Lk)
    if mode != "negative" and D != 128:
        lens = torch.full((2,), Lk, dtype=torch.int32, device=DEV)
        head_major = [t.transpose(1, 2).contiguous() for t in d[1:]]
        got = ops.cache_attention(d[0][:, -1:], *head_major, None, None, lens, None, None, None, None, "plain", scale, 0.0, slopes)
        within(got, want[:, -1:].double(), want[:, -1:].double().abs(), none[:, -1:], kind, u, 1, Lk)
