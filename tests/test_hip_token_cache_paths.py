"""Token cache and attention: both sides of every rule by which the work is split, score forms that have a kernel of their own, offsets
beyond 32 bits, graphs and the methods of HipOps.  Plain forms and tolerances: test_hip_token_cache.py."""
import math

import pytest
import torch

from test_hip_token_cache import DEV, attend, cache_case, cache_reference, decode, encode, masked_inputs, masked_reference, near, ops, run_cache, run_masked, values  # noqa: F401

pytestmark = pytest.mark.gpu


def lengths(B, C, T=1):
    return [max(0, C - (b * b * 37) % (C + 1)) if b else C for b in range(B)]


SPLITS = [  # B, T, Hq, Hkv, D, C, P, cap, slopes, formats
    (1, 1, 4, 1, 64, 512, 0, 0.0, False, "plain mxfp4"),                # four units: a workgroup a stream
    (1, 1, 4, 1, 64, 513, 0, 0.0, True, "plain mxfp4"),                 # one token more: shares
    (20, 1, 8, 8, 32, 640, 0, 0.0, False, "mxfp8"),                     # 160 streams of five units: a workgroup a stream
    (20, 1, 8, 8, 32, 641, 0, 0.0, False, "mxfp8"),                     # ... and six
    (1, 2, 2, 1, 32, 20000, 0, 0.0, True, "plain mxfp8"),               # over 64 parts a row
    (1, 1, 8, 2, 128, 1500, 0, 20.0, False, "plain mxfp4"),             # over eight parts a row
    (70, 1, 2, 1, 64, 700, 0, 0.0, False, "mxfp8"),                     # more than 64 sequences, shares
    (2, 1, 4, 2, 64, 600, 33, 0.0, False, "plain mxfp8"),               # shares and a prefix
    (3, 2, 16, 2, 256, 30, 31, 0.0, True, "mxfp8 mxfp4"),               # prefix chunks of 32 keys and their ends
    (3, 2, 16, 2, 256, 30, 32, 15.0, False, "mxfp8"),
    (3, 2, 16, 2, 96, 30, 33, 0.0, False, "mxfp8 mxfp4"),
    (6, 1, 8, 1, 128, 30, 127, 0.0, False, "plain mxfp8"),              # 48 rows
    (16, 1, 16, 2, 128, 40, 300, 0.0, False, "plain"),                  # 128 rows of the prefix
    (16, 1, 16, 2, 96, 600, 65, 0.0, True, "plain"),                    # ... with a bias, and shares
    (9, 2, 16, 2, 64, 20, 70, 25.0, True, "plain"),                     # ... cap and bias, two tokens, some before the first
    (33, 2, 2, 1, 256, 5, 100, 0.0, False, "plain"),
    (130, 1, 2, 1, 32, 3, 1, 0.0, False, "plain"),                      # a prefix of one token
    (3, 1, 4, 2, 64, 0, 40, 0.0, False, "plain mxfp8"),                 # no room for a token
    (2, 3, 16, 2, 128, 700, 0, 0.0, True, "plain mxfp8 mxfp4"),         # 24 rows: over the same keys, or 16 and 8
    (2, 8, 16, 2, 64, 300, 50, 9.0, False, "plain mxfp8 mxfp4"),        # 64 rows
    (1, 17, 8, 2, 32, 900, 0, 0.0, False, "mxfp8 mxfp4"),               # 68 rows
    (16, 1, 16, 1, 64, 20, 9000, 0.0, True, "plain mxfp4"),             # 256 rows of a prefix, waves over the same keys
    (33, 1, 16, 1, 32, 20, 9000, 0.0, False, "mxfp8"),                  # 528 rows, 8 bits
]


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case,form", [(c, f) for c in SPLITS for f in c[9].split()], ids=lambda c: c if isinstance(c, str) else "x".join(map(str, c[:7])))
def test_cache_attention_on_both_sides_of_its_rules(ops, case, form, kind):  # noqa: F811
    B, T, Hq, Hkv, D, C, P, cap, alibi, _ = case
    g = torch.Generator().manual_seed(sum(case[:7]))
    x = cache_case(g, B, T, Hq, Hkv, D, C, P, form, kind)
    lens = torch.tensor(lengths(B, C), dtype=torch.int32)
    slopes = torch.exp2(-torch.arange(1, Hq + 1).float() * 8 / Hq) if alibi else None
    want, top, score = cache_reference(x, lens, form, D ** -0.5, cap, slopes, P)
    near(run_cache(ops, x, lens, form, D ** -0.5, cap, slopes, P), want, top, score, kind)


LARGE = [  # B, T, Hq, Hkv, D, C, P, cap, slopes: products over a prefix that go to the kernel of whole prompts
    (8, 16, 16, 2, 64, 40, 13800, 0.0, False),
    (8, 16, 16, 2, 64, 700, 13800, 0.0, True),
    (16, 8, 16, 2, 96, 9, 15300, 25.0, False),
    (8, 16, 16, 2, 128, 17, 11500, 20.0, True),
    (9, 16, 16, 1, 256, 30, 3200, 0.0, True),
    (9, 16, 16, 1, 256, 30, 5100, 0.0, True),
    (700, 1, 3, 1, 32, 3, 26800, 0.0, False),
]


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", LARGE, ids=lambda c: "x".join(map(str, c[:7])))
def test_a_large_product_over_a_prefix(ops, case, kind):  # noqa: F811
    B, T, Hq, Hkv, D, C, P, cap, alibi = case
    g = torch.Generator().manual_seed(sum(case[:7]))
    x = cache_case(g, B, T, Hq, Hkv, D, C, P, "plain", kind)
    lens = torch.tensor(lengths(B, C), dtype=torch.int32)
    slopes = torch.exp2(-torch.arange(1, Hq + 1).float() * 8 / Hq) if alibi else None
    got = run_cache(ops, x, lens, "plain", D ** -0.5, cap, slopes, P)
    some = torch.arange(0, B, max(1, B // 8))                               # (the reference of some sequences)
    few = {**x, **{n: x[n][some] for n in ("q", "k", "v")}}
    want, top, score = cache_reference(few, lens[some], "plain", D ** -0.5, cap, slopes, P)
    near(got[some.to(DEV)], want, top, score, kind)
    if D == 256:                                                            # the same prefix, its tokens 2 MB apart
        y = {**x, "pk": far(x["pk"], (1 << 20) - 8, 1), "pv": far(x["pv"], (1 << 20) - 64, 1)}
        assert torch.equal(run_cache(ops, y, lens, "plain", D ** -0.5, cap, slopes, P), got)


@pytest.mark.parametrize("form,D", [("plain", 64), ("plain", 256), ("mxfp8", 128)])
@pytest.mark.parametrize("scale,cap,slope", [(-0.1, 0.0, 0.0), (0.0, 0.0, 0.0), (-0.1, 0.0, 0.02), (0.0, 0.0, -0.01), (1e-30, 0.0, 0.5), (0.1, 9.0, 0.3), (-0.1, 9.0, -0.02), (0.1, 0.0, 1e6)])
def test_scales_caps_and_slopes_of_every_sign(ops, form, D, scale, cap, slope):  # noqa: F811
    g = torch.Generator().manual_seed(D)
    x = cache_case(g, 17, 1, 8, 2, D, 50, 90, form, torch.float16)
    lens = torch.tensor(lengths(17, 50), dtype=torch.int32)
    slopes = torch.full((8,), slope) * (1 + torch.arange(8)) / 8 if slope else None
    want, top, score = cache_reference(x, lens, form, scale, cap, slopes, 90)
    near(run_cache(ops, x, lens, form, scale, cap, slopes, 90), want, top, score, torch.float16)
    if form == "plain":
        case = (2, 70, 300, 4, 2, D, True, cap, False, [300, 111], [230, 60], [80, 0], None)
        q, k, v, _, *rest = masked_inputs(case, torch.bfloat16)
        slopes = None if slopes is None else slopes[:4].contiguous()
        for causal in (True, False):
            args = (scale, causal, cap, slopes, rest[0], rest[1], rest[2] if causal else None, None)
            want, top, score = masked_reference(q, k, v, *args)
            near(run_masked(ops, q, k, v, *args), want, top, score, torch.bfloat16)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cap,scale", [(256.0, 0.125), (257.0, 0.125), (257.0, 12.0), (1e4, 0.125), (1e4, 300.0), (3e7, 0.125), (1e30, -0.125)])
def test_wide_caps(ops, cap, scale, kind):  # noqa: F811
    """A cap far above the scores changes them little, not at random; scores on both sides of a quarter of it."""
    g = torch.Generator().manual_seed(4)
    for form in ("plain", "mxfp8"):
        x = cache_case(g, 3, 2, 4, 2, 64, 60, 40, form, kind)
        lens = torch.tensor([60, 17, 3], dtype=torch.int32)
        want, top, score = cache_reference(x, lens, form, scale, cap, None, 40)
        near(run_cache(ops, x, lens, form, scale, cap, None, 40), want, top, score, kind)
    q, k, v, *_ = masked_inputs((2, 80, 90, 4, 2, 64, True, cap, False, None, None, None, None), kind)
    for slopes in (None, torch.tensor([0.5, 0.1, 0.02, 0.0])):
        args = (scale, True, cap, slopes, None, torch.tensor([10, 0], dtype=torch.int32), None, None)
        want, top, score = masked_reference(q, k, v, *args)
        near(run_masked(ops, q, k, v, *args), want, top, score, kind)


PROMPTS = [  # B, Lq, Lk, Hq, Hkv, D, causal, cap, slopes, lens, start, prefix, docs
    (1, 512, 512, 4, 4, 64, True, 0.0, True, None, None, None, None),               # keys in parts, a bias on both sides of the rows
    (1, 300, 300, 2, 2, 128, True, 0.0, False, None, None, None, "sorted"),
    (2, 400, 400, 4, 2, 64, True, 0.0, True, None, None, None, "sorted"),
    (1, 700, 700, 2, 1, 256, False, 0.0, True, None, None, None, "sorted"),
    (1, 900, 900, 2, 1, 96, True, 30.0, True, [850], None, None, "sorted"),
    (1, 64, 2500, 2, 1, 128, True, 0.0, True, [2400], [2436], [100], None),
    (2, 9, 1500, 8, 8, 40, False, 0.0, False, [1500, 700], None, None, None),
    (1, 1200, 100, 1, 1, 64, True, 0.0, True, None, [-500], None, None),            # many rows before the first key
    (1, 5100, 5100, 1, 1, 64, True, 0.0, False, None, None, None, "sorted"),        # documents in parts
    (1, 4100, 4100, 1, 1, 128, False, 0.0, True, [4000], None, None, "mixed"),
    (1, 2100, 33, 8, 1, 32, False, 0.0, True, None, [7], None, None),
    (5, 1, 70, 16, 4, 64, True, 0.0, False, [70, 1, 0, 33, 64], [69, 0, 3, 40, 63], None, None),
]


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", PROMPTS, ids=lambda c: "x".join(map(str, c[:6])))
def test_attention_masked_on_both_sides_of_its_rules(ops, case, kind):  # noqa: F811
    q, k, v, *rest = masked_inputs(case, kind, 3)
    args = (case[5] ** -0.5, case[6], case[7], *rest)
    want, top, score = masked_reference(q, k, v, *args)
    near(run_masked(ops, q, k, v, *args), want, top, score, kind)


@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_values_of_other_documents_may_be_anything(ops, D):  # noqa: F811
    case = (1, 600, 600, 2, 1, D, True, 0.0, D == 64, None, None, None, None)
    q, k, v, slopes, *_ = masked_inputs(case, torch.bfloat16)
    doc = (torch.arange(600) // 100).int().unsqueeze(0)
    k[:, 200:300], v[:, 200:300] = math.nan, math.inf
    args = (D ** -0.5, True, 0.0, slopes, None, None, None, doc)
    got = run_masked(ops, q, k, v, *args)
    clean = torch.ones(600, dtype=torch.bool)
    clean[200:300] = False
    want, top, score = masked_reference(q, k.nan_to_num(0.0, 0.0, 0.0), v.nan_to_num(0.0, 0.0, 0.0), *args)
    near(got[:, clean.to(DEV)], want[:, clean], top[:, clean], score[:, clean], torch.bfloat16)
    assert bool(got[:, 200:300].isnan().all())


# ---- offsets beyond 32 bits: few tokens, far apart ------------------------------------------------------------------------------

def far(x, stride, lead):
    """x [..., N, D] on the device with `stride` elements from a token to the next (axis `lead`)."""
    shape = list(x.shape)
    strides, at = [0] * len(shape), stride * shape[lead]
    for i in range(len(shape) - 1):
        if i != lead:
            strides[i], at = at, at * shape[i]
    strides[lead], strides[-1] = stride, 1
    size = sum((n - 1) * s for n, s in zip(shape, strides)) + 1
    y = torch.empty(size, dtype=x.dtype, device=DEV).as_strided(shape, strides)
    y.copy_(x.to(DEV))
    assert size * x.element_size() > 1 << 32
    return y


def test_offsets_of_a_cache_beyond_32_bits(ops):  # noqa: F811
    g = torch.Generator().manual_seed(1)
    x = cache_case(g, 1, 1, 4, 1, 64, 150, 140, "plain", torch.bfloat16)
    lens = torch.tensor([149], dtype=torch.int32)
    want = run_cache(ops, x, lens, "plain", 0.125, 0.0, None, 140)
    y = {**x, "k": far(x["k"], (1 << 24) - 8, 2), "v": far(x["v"], (1 << 24) - 64, 2)}
    assert torch.equal(run_cache(ops, y, lens, "plain", 0.125, 0.0, None, 140), want)
    y = {**x, "pk": far(x["pk"], (1 << 24) - 16, 1), "pv": far(x["pv"], (1 << 24) - 8, 1)}
    assert torch.equal(run_cache(ops, y, lens, "plain", 0.125, 0.0, None, 140), want)
    q = torch.randn(70, 1, 4, 64, generator=g).to(torch.bfloat16)           # 280 rows of the prefix
    x = {**x, "q": q, "k": x["k"].expand(70, 1, 150, 64), "v": x["v"].expand(70, 1, 150, 64)}
    lens = torch.full((70,), 149, dtype=torch.int32)
    want = run_cache(ops, x, lens, "plain", 0.125, 0.0, None, 140)
    y = {**x, "pk": y["pk"], "pv": y["pv"]}
    assert torch.equal(run_cache(ops, y, lens, "plain", 0.125, 0.0, None, 140), want)


def test_offsets_of_a_quantised_cache_beyond_32_bits(ops):  # noqa: F811
    g = torch.Generator().manual_seed(2)
    new = values(g, 1, 150, 1, 64)
    codes, scales = encode(new.transpose(1, 2), "mxfp8")
    held, held_s = far(torch.zeros_like(codes), (1 << 25) - 16, 2), torch.zeros_like(scales, device=DEV)
    ops.cache_write(new.to(DEV), None, torch.zeros(1, dtype=torch.int32, device=DEV), None, held, held_s, None, None, "mxfp8")
    assert torch.equal(held.cpu(), codes) and torch.equal(held_s.cpu(), scales)
    got = ops.cache_read(held, held_s, None, "mxfp8", torch.float32)
    assert torch.equal(got.cpu().double(), decode(codes, scales, "mxfp8"))
    q, lens = torch.randn(1, 1, 2, 64, generator=g).half().to(DEV), torch.tensor([150], dtype=torch.int32, device=DEV)
    near_codes = codes.to(DEV)
    call = lambda k: ops.cache_attention(q, k, k, held_s, held_s, lens, None, None, None, None, "mxfp8", 0.125, 0.0, None)  # noqa: E731
    assert torch.equal(call(held), call(near_codes))


def test_offsets_of_a_prompt_beyond_32_bits(ops):  # noqa: F811
    case = (1, 300, 300, 2, 1, 64, True, 0.0, False, None, None, None, None)
    q, k, v, *rest = masked_inputs(case, torch.float16)
    args = (0.125, True, 0.0, *rest)
    want = run_masked(ops, q, k, v, *args)
    step = (1 << 23) - 8
    assert torch.equal(run_masked(ops, far(q, step, 1), far(k, step, 1), far(v, step, 1), *args), want)


# ---- graphs, calls at once, entry points ----------------------------------------------------------------------------------------

def test_two_graphs_replayed_at_once_and_between_eager_calls(ops):  # noqa: F811
    g = torch.Generator().manual_seed(5)
    x = cache_case(g, 4, 1, 8, 2, 128, 3000, 200, "mxfp4", torch.bfloat16)
    d = {k: v.to(DEV) for k, v in x.items()}
    doc = (torch.arange(700) // 90).int().unsqueeze(0).to(DEV)
    m = torch.randn(1, 700, 2, 64, generator=g).half().to(DEV)
    lens = [torch.tensor(l, dtype=torch.int32, device=DEV) for l in ([3000, 7, 555, 2000], [1, 2999, 0, 1234])]

    def call(n):
        a = ops.cache_attention(d["q"], d["k"], d["v"], d["ks"], d["vs"], n, d["pk"], d["pv"], d["pks"], d["pvs"], "mxfp4", 0.09, 0.0, None)
        return a, ops.attention_masked(m, m, m, 0.125, True, 0.0, None, None, None, None, doc, doc)

    want = [call(n) for n in lens]
    streams, graphs, outs = [torch.cuda.Stream() for _ in lens], [], []
    torch.cuda.synchronize()
    for s, n in zip(streams, lens):
        with torch.cuda.stream(s):
            call(n)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(call(n))
        graphs.append(graph)
    for _ in range(3):
        for got in outs:
            for o in got:
                o.fill_(3.0)
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        eager = call(lens[0])
        torch.cuda.synchronize()
        for got, ref in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(got, ref))
        assert all(torch.equal(a, b) for a, b in zip(eager, want[0]))


def test_methods_of_hip_ops_answer_like_the_ops(ops):  # noqa: F811
    from det_sam2_amd.hip_model import HipOps
    hip = HipOps(DEV)
    g = torch.Generator().manual_seed(6)
    new = [values(g, 2, 30, 2, 64, kind=torch.bfloat16).to(DEV) for _ in range(2)]
    pos = torch.tensor([0, 5], dtype=torch.int32, device=DEV)
    kc, ks, vc, vs = hip.cache_alloc(2, 2, 40, 64, "mxfp4")
    for t in (kc, ks, vc, vs):
        t.zero_()
    other = [t.clone() for t in (kc, ks, vc, vs)]
    hip.cache_write(new[0], pos, kc, ks, "mxfp4", v=new[1], v_codes=vc, v_scales=vs)
    ops.cache_write(new[0], new[1], pos, None, *other, "mxfp4")
    assert all(torch.equal(a, b) for a, b in zip((kc, ks, vc, vs), other))
    assert torch.equal(hip.cache_read(kc, ks, "mxfp4", lens=pos), ops.cache_read(kc, ks, pos, "mxfp4", torch.bfloat16))
    q = torch.randn(2, 3, 4, 64, generator=g).to(torch.bfloat16).to(DEV)
    lens = pos + 30
    got = hip.cache_attention(q, kc, vc, lens, scale=0.125, format="mxfp4", k_scales=ks, v_scales=vs, cap=20.0)
    assert torch.equal(got, ops.cache_attention(q, kc, vc, ks, vs, lens, None, None, None, None, "mxfp4", 0.125, 20.0, None))
    got = hip.attention_masked(q, *new, scale=0.125, causal=True, q_start=pos)
    assert torch.equal(got, ops.attention_masked(q, *new, 0.125, True, 0.0, None, None, pos, None, None, None))


def test_the_same_call_gives_the_same_bits(ops):  # noqa: F811
    """No atomics, no order that depends on the run: ragged shares, parts and joins, ten times."""
    g = torch.Generator().manual_seed(9)
    x = cache_case(g, 5, 2, 8, 2, 64, 4000, 0, "plain", torch.float16)
    lens = torch.tensor([4000, 1, 0, 3001, 129], dtype=torch.int32)
    first = run_cache(ops, x, lens, "plain", 0.125, 0.0, None, 0)
    assert all(torch.equal(run_cache(ops, x, lens, "plain", 0.125, 0.0, None, 0), first) for _ in range(9))
