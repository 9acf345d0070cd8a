"""Token cache (quantised write / read), attention over it and masked attention (`torch.ops.det_sam2.cache_write`, `cache_read`,
`cache_attention`, `attention_masked`) against plain 64-bit implementations.

Tolerances.  A cache holds exactly defined codes: write and read are compared bit for bit.  Attention is compared with
|got - want| <= u (|want| + top), u half a step of the output's type (bf16 2^-8, fp16 2^-11) and top = sum_j w_j |v_j| / sum_j w_j, the
size of the terms that the output is the sum of:
  * the output's own rounding is at most u |want|;
  * where the weights are rounded to the type before the product (masked attention; 16-bit caches of fp16 values) each term w_j v_j is
    off by at most u of itself, u top in all; everywhere else the weights carry 16 bits or more;
  * scores, exponentials and sums are fp32: the fp32 score of D products is off by at most (D + 8) 2^-24 sum_d |q_d k_d| scale,
    which enters the weight as a relative error; with the inputs used here (|q.k| scale sums below 60, D <= 256) that is below
    264 * 2^-24 * 60 < 2^-10 at the very worst sign pattern.  The `score` term below counts it from the inputs themselves.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

MAXIMUM = {"mxfp8": 448.0, "mxfp4": 6.0}
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from det_sam2_amd import _capi
    return _capi.load_torch_ops()


# ---- plain implementations in 64 bits -----------------------------------------------------------------------------------------

def grid_of(form):
    if form == "mxfp4":
        return torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
    low = [m / 8 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)]
    return torch.tensor(low[:127], dtype=torch.float64)


def encode(x, form):
    """[..., D] -> (codes as the cache holds them, scale bytes)"""
    x = x.double().cpu()
    g = x.unflatten(-1, (-1, 32))
    most = g.abs().amax(-1)
    fine = torch.isfinite(g).all(-1)
    e = torch.full(most.shape, -126, dtype=torch.int64)
    for _ in range(300):                                               # the smallest power of two that is large enough
        grow = fine & (most > MAXIMUM[form] * 2.0 ** e.double())
        if not grow.any():
            break
        e = torch.where(grow, e + 1, e)
    y = torch.where(fine.unsqueeze(-1), g, torch.zeros((), dtype=torch.float64)) / 2.0 ** e.double().unsqueeze(-1)
    grid = grid_of(form)
    up = torch.searchsorted(grid, y.abs().contiguous()).clamp(1, grid.numel() - 1)
    below, above = y.abs() - grid[up - 1], grid[up] - y.abs()
    code = torch.where((above < below) | ((above == below) & (up % 2 == 0)), up, up - 1)
    sign = torch.signbit(y).long()
    code = code | sign << (7 if form == "mxfp8" else 3)
    code = code.flatten(-2)
    if form == "mxfp4":
        code = code[..., 0::2] | code[..., 1::2] << 4
    return code.to(torch.uint8), torch.where(fine, e + 127, torch.full_like(e, 255)).to(torch.uint8)


def decode(codes, scales, form):
    codes, s = codes.cpu().long(), scales.cpu().double()
    if form == "mxfp4":
        codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    n = 8 if form == "mxfp4" else 128
    half = torch.full((n,), math.nan, dtype=torch.float64)
    grid = grid_of(form)
    half[:grid.numel()] = grid
    v = torch.cat((half, -half))[codes]
    f = torch.where(s == 255, torch.full_like(s, math.nan), 2.0 ** (s - 127))
    return v * f.repeat_interleave(32, -1)


def attend(q, k, v, seen, bias, scale, cap):
    """One head: q [R,D], k, v [N,D], seen [R,N], bias [R,N] -> (o, top, score): the output, sum w |v| and the score sums' size"""
    x = (q @ k.T) * scale
    size = (q.abs() @ torch.nan_to_num(k, 0.0, 0.0, 0.0).abs().T) * abs(scale)
    if cap:
        x = cap * torch.tanh(x / cap)
    x = torch.where(seen, x - bias, torch.full_like(x, -math.inf))
    m = x.amax(-1, keepdim=True)
    w = torch.exp(x - torch.where(m == -math.inf, torch.zeros_like(m), m))
    w = torch.where(seen, w, torch.zeros_like(w))
    total = w.sum(-1, keepdim=True)
    w = torch.where(total == 0, w, w / total)
    clean = torch.nan_to_num(v, 0.0, 0.0, 0.0)
    o = w @ clean
    for j in torch.nonzero(~torch.isfinite(v).all(-1)).flatten().tolist():   # 0 * inf of a hidden key is no term
        bad = torch.where(torch.isfinite(v[j]), torch.zeros_like(v[j]), v[j])
        row = torch.where(~torch.isfinite(v[j]).unsqueeze(0), w[:, j:j + 1] * bad.unsqueeze(0), torch.zeros_like(o))
        o = o + torch.where(seen[:, j:j + 1], row, torch.zeros_like(o))
    return o, torch.nan_to_num(w, 0.0) @ clean.abs(), (torch.where(seen, size, torch.zeros_like(size)) + bias.abs() * seen).amax(-1)


def near(got, want, top, score, kind):
    u = torch.finfo(kind).eps / 2
    got, d = got.double().cpu(), got.shape[-1]
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want))
    fine = torch.isfinite(want)
    bound = u * (want.abs() + top) + 2 * (d + 8) * 2.0 ** -24 * score.unsqueeze(-1) * top + 2.0 ** -24
    off = ((got - want).abs() / bound)[fine]
    assert not off.numel() or float(off.max()) <= 1.0, float(off.max())


def values(g, *shape, kind=torch.float32):
    x = torch.randn(*shape, generator=g) * torch.exp(0.6 * torch.randn(shape[-1], generator=g))
    return x.to(kind)


# ---- write and read -----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("form", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,T,H,D,C", [(1, 1, 1, 32, 1), (3, 5, 2, 64, 11), (2, 67, 3, 96, 100), (4, 1, 8, 128, 9), (1, 300, 1, 256, 301), (2, 9, 1, 4096, 12)])
def test_write_and_read_hold_exactly_the_defined_codes(ops, form, kind, B, T, H, D, C):
    g = torch.Generator().manual_seed(B * 1000 + T + D)
    k, v = values(g, B, T, H, D, kind=kind), values(g, B, T, H, D, kind=kind)
    pos = torch.tensor([(C - T) * b // max(1, B - 1) for b in range(B)], dtype=torch.int32)
    count = torch.tensor([T - b if T > b else 0 for b in range(B)], dtype=torch.int32)
    W = D // 2 if form == "mxfp4" else D
    bufs = [torch.randint(0, 255, (B, H, C, n), dtype=torch.uint8, generator=g) for n in (W, D // 32, W, D // 32)]
    want = [x.clone() for x in bufs]
    for x, c, s in ((k, want[0], want[1]), (v, want[2], want[3])):
        codes, scales = encode(x, form)
        for b in range(B):
            p, n = int(pos[b]), int(count[b])
            c[b, :, p:p + n], s[b, :, p:p + n] = codes[b, :n].transpose(0, 1), scales[b, :n].transpose(0, 1)
    dev = [x.to(DEV) for x in bufs]
    ops.cache_write(k.to(DEV), v.to(DEV), pos.to(DEV), count.to(DEV), *dev, form)
    for a, b in zip(dev, want):
        assert torch.equal(a.cpu(), b)
    lens = (pos + count).to(DEV)
    for i in (0, 2):
        for out in (torch.float32, torch.bfloat16, torch.float16):
            got = ops.cache_read(dev[i], dev[i + 1], lens, form, out).cpu()
            ref = decode(want[i], want[i + 1], form).to(out)
            ref = torch.where((torch.arange(C) < (pos + count).unsqueeze(1))[:, None, :, None], ref, torch.zeros((), dtype=out))
            assert got.dtype == out and torch.equal(got.isnan(), ref.isnan()) and torch.equal(got.nan_to_num(7.0), ref.nan_to_num(7.0))


@pytest.mark.parametrize("form", ["mxfp8", "mxfp4"])
def test_write_at_the_borders_of_the_format(ops, form):
    """Ties, the largest code, powers of two around the scale's step, subnormal and zero groups, and groups with infinities and NaN."""
    top = MAXIMUM[form]
    grid = grid_of(form)
    rows = [torch.zeros(32), torch.full((32,), 2.0 ** -149), torch.full((32,), -0.0)]
    for e in (-126, -30, 0, 5, 100):
        for m in (top, top * (1 + 2.0 ** -20), top * (1 - 2.0 ** -20), top / 2 * (1 + 2.0 ** -20)):
            mid = (grid[:-1] + grid[1:]) / 2
            pick = mid[torch.linspace(0, mid.numel() - 1, 31).long()]
            signs = torch.tensor([1.0, -1.0]).repeat(16)[:31]
            rows.append(torch.cat((torch.tensor([m]).double(), pick * signs)).double() * 2.0 ** e)
    for bad in (math.inf, -math.inf, math.nan):
        r = torch.linspace(-1, 1, 32).double()
        r[13] = bad
        rows.append(r)
    rows.append(torch.full((32,), torch.finfo(torch.float32).max))
    x = torch.stack([r.double() for r in rows]).float().view(1, len(rows), 1, 32)
    codes, scales = encode(x, form)
    c = torch.zeros(1, 1, len(rows), 16 if form == "mxfp4" else 32, dtype=torch.uint8, device=DEV)
    s = torch.zeros(1, 1, len(rows), 1, dtype=torch.uint8, device=DEV)
    ops.cache_write(x.to(DEV), None, torch.zeros(1, dtype=torch.int32, device=DEV), None, c, s, None, None, form)
    assert torch.equal(s.cpu()[0, 0, :, 0], scales[0, :, 0, 0])
    assert torch.equal(c.cpu()[0, 0], codes[0, :, 0])
    got, ref = ops.cache_read(c, s, None, form, torch.float32).cpu(), decode(codes, scales, form).float().transpose(1, 2)
    assert torch.equal(got.isnan(), ref.isnan()) and torch.equal(got.nan_to_num(7.0), ref.nan_to_num(7.0))


def test_write_drops_rows_outside_the_cache_and_takes_strided_views(ops):
    g = torch.Generator().manual_seed(3)
    B, T, H, D, C = 4, 6, 2, 64, 8
    x = values(g, T, B, H, 2 * D).to(DEV)[..., D:].transpose(0, 1)                     # [B,T,H,D], strides of another order
    store = torch.full((B, C, H, D), 99, dtype=torch.uint8, device=DEV)
    scale = torch.full((B, C, H, 2), 98, dtype=torch.uint8, device=DEV)
    pos = torch.tensor([-3, 0, 5, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    count = torch.tensor([6, -1, 100, 6], dtype=torch.int32, device=DEV)
    ops.cache_write(x, None, pos, count, store.transpose(1, 2), scale.transpose(1, 2), None, None, "mxfp8")
    codes, scales = encode(x, "mxfp8")
    want, ws = torch.full((B, C, H, D), 99, dtype=torch.uint8), torch.full((B, C, H, 2), 98, dtype=torch.uint8)
    want[0, 0:3], ws[0, 0:3] = codes[0, 3:], scales[0, 3:]                             # rows -3 .. -1 are dropped
    want[2, 5:8], ws[2, 5:8] = codes[2, :3], scales[2, :3]                             # rows behind the capacity too
    assert torch.equal(store.cpu(), want) and torch.equal(scale.cpu(), ws)
    # sizes of zero write nothing
    ops.cache_write(x[:, :0], None, pos, None, store.transpose(1, 2), scale.transpose(1, 2), None, None, "mxfp8")
    assert torch.equal(store.cpu(), want)
    assert ops.cache_read(store.transpose(1, 2)[:, :, :0], scale.transpose(1, 2)[:, :, :0], None, "mxfp8", torch.float16).shape == (B, H, 0, D)


# ---- attention over a cache ---------------------------------------------------------------------------------------------------

def cache_case(g, B, T, Hq, Hkv, D, C, P, form, kind):
    held = lambda *lead: values(g, *lead, D)  # noqa: E731
    out = {"q": torch.randn(B, T, Hq, D, generator=g).to(kind)}
    for name, lead in (("k", (B, Hkv, C)), ("v", (B, Hkv, C)), ("pk", (Hkv, P)), ("pv", (Hkv, P))):
        x = held(*lead)
        if form == "plain":
            out[name], out[name + "s"] = x.to(kind), None
        else:
            out[name], out[name + "s"] = encode(x, form)
    return out


def cache_reference(x, lens, form, scale, cap, slopes, P):
    val = lambda n: x[n].double() if form == "plain" else decode(x[n], x[n + "s"], form)  # noqa: E731
    q, k, v, pk, pv = x["q"].double(), val("k"), val("v"), val("pk"), val("pv")
    B, T, Hq, D = q.shape
    G = Hq // k.shape[1]
    o, top, score = torch.zeros(B, T, Hq, D, dtype=torch.float64), torch.zeros(B, T, Hq, D, dtype=torch.float64), torch.zeros(B, T, Hq, dtype=torch.float64)
    for b in range(B):
        n = max(0, min(int(lens[b]), k.shape[2]))
        at = P + n - T + torch.arange(T)
        key = torch.arange(P + n)
        seen = (key[None] <= at[:, None]) & (at >= P)[:, None]
        dist = (at[:, None] - key[None]).double()
        for h in range(Hq):
            kk, vv = torch.cat((pk[h // G], k[b, h // G, :n])), torch.cat((pv[h // G], v[b, h // G, :n]))
            if not len(kk):
                continue
            bias = dist * float(slopes[h]) if slopes is not None else torch.zeros_like(dist)
            o[b, :, h], top[b, :, h], score[b, :, h] = attend(q[b, :, h], kk, vv, seen, bias * seen, scale, cap)
    return o, top, score


def run_cache(ops, x, lens, form, scale, cap, slopes, P):
    d = {k: None if v is None else v.to(DEV) for k, v in x.items()}
    pre = [d["pk"], d["pv"], d["pks"], d["pvs"]] if P else [None] * 4
    return ops.cache_attention(d["q"], d["k"], d["v"], d["ks"], d["vs"], lens.to(DEV), *pre, form, scale, cap, None if slopes is None else slopes.to(DEV))


CACHE = [  # B, T, Hq, Hkv, D, C, P, lens, cap, slopes
    (1, 1, 1, 1, 32, 1, 0, [1], 0.0, False),
    (3, 1, 4, 2, 64, 40, 0, [0, 33, 40], 0.0, False),                   # an empty sequence among others
    (2, 1, 8, 1, 128, 700, 0, [699, 64], 30.0, True),                   # several parts, one of them of one sequence only
    (2, 5, 12, 3, 96, 70, 0, [5, 70], 0.0, True),                       # 20 rows a key head: two tiles
    (2, 3, 8, 4, 256, 90, 0, [2, 90], 15.0, False),                     # fewer tokens than the new ones: the first sees nothing
    (4, 2, 6, 2, 64, 33, 50, [2, 1, 33, 0], 0.0, True),                 # a short prefix, sequences without anything
    (9, 1, 16, 2, 128, 20, 333, [1, 20, 7, 3, 9, 11, 2, 5, 8], 0.0, False),   # rows of the prefix over several waves
    (5, 2, 16, 1, 256, 9, 130, [9, 2, 3, 4, 5], 20.0, False),
    (2, 1, 32, 8, 128, 2300, 0, [2300, 131], 0.0, False),
    (1, 40, 2, 1, 32, 64, 31, [64], 0.0, False),                        # 80 rows: several row groups
]


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("form", ["plain", "mxfp8", "mxfp4"])
@pytest.mark.parametrize("case", CACHE, ids=lambda c: "x".join(map(str, c[:7])))
def test_cache_attention(ops, case, form, kind):
    B, T, Hq, Hkv, D, C, P, lens, cap, alibi = case
    g = torch.Generator().manual_seed(sum(case[:7]))
    x = cache_case(g, B, T, Hq, Hkv, D, C, P, form, kind)
    lens = torch.tensor(lens, dtype=torch.int32)
    slopes = torch.exp2(-torch.arange(1, Hq + 1).float() * 8 / Hq) if alibi else None
    want, top, score = cache_reference(x, lens, form, D ** -0.5, cap, slopes, P)
    near(run_cache(ops, x, lens, form, D ** -0.5, cap, slopes, P), want, top, score, kind)


@pytest.mark.parametrize("form", ["plain", "mxfp8"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_cache_attention_ignores_what_lies_in_hidden_places(ops, form, D):
    """NaN and infinities behind a sequence's last token, and in a new token that earlier new tokens do not see."""
    g = torch.Generator().manual_seed(D)
    x = cache_case(g, 2, 3, 4, 2, D, 50, 0, form, torch.bfloat16)
    lens = torch.tensor([40, 7], dtype=torch.int32)
    for b in range(2):
        n = int(lens[b])
        if form == "plain":
            x["k"][b, :, n:], x["v"][b, :, n:] = math.nan, math.inf
            x["v"][b, 0, n - 1, 5], x["v"][b, 1, n - 2, 6] = math.inf, math.nan       # seen by the last token / the last two
        else:
            x["ks"][b, :, n:], x["vs"][b, :, n:] = 255, 255
            x["vs"][b, 0, n - 1, 0] = 255
    want, top, score = cache_reference(x, lens, form, D ** -0.5, 0.0, None, 0)
    assert want.isfinite().any() and not want.isfinite().all()
    near(run_cache(ops, x, lens, form, D ** -0.5, 0.0, None, 0), want, top, score, torch.bfloat16)


def test_cache_attention_takes_views_in_other_orders(ops):
    g = torch.Generator().manual_seed(8)
    x = cache_case(g, 2, 2, 4, 2, 64, 70, 40, "mxfp8", torch.float16)
    lens = torch.tensor([70, 33], dtype=torch.int32)
    want = run_cache(ops, x, lens, "mxfp8", 0.125, 0.0, None, 40)
    y = dict(x)
    y["q"] = torch.cat((x["q"], x["q"]), -1).to(DEV)[..., :64]
    for n in ("k", "v", "ks", "vs"):
        y[n] = x[n].transpose(1, 2).contiguous().to(DEV).transpose(1, 2)               # token-major caches
    for n in ("pk", "pv", "pks", "pvs"):
        y[n] = x[n].transpose(0, 1).contiguous().to(DEV).transpose(0, 1)
    assert torch.equal(run_cache(ops, y, lens, "mxfp8", 0.125, 0.0, None, 40), want)


# ---- masked attention ---------------------------------------------------------------------------------------------------------

MASKED = [  # B, Lq, Lk, Hq, Hkv, D, causal, cap, slopes, lens, start, prefix, docs
    (1, 1, 1, 1, 1, 8, False, 0.0, False, None, None, None, None),
    (2, 33, 65, 2, 1, 64, False, 0.0, False, [0, 65], None, None, None),             # a sequence of no keys
    (2, 100, 100, 4, 2, 72, True, 0.0, False, None, None, None, None),
    (1, 70, 200, 6, 2, 128, True, 20.0, True, [190], [130], None, None),
    (2, 64, 128, 2, 2, 96, True, 0.0, True, None, [64, 10], [100, 0], None),          # prefix mask
    (1, 257, 257, 8, 1, 32, True, 0.0, False, None, None, None, "sorted"),
    (2, 190, 190, 2, 2, 64, False, 0.0, True, None, None, None, "mixed"),            # documents in any order, rows of none
    (1, 5, 900, 4, 1, 256, False, 50.0, False, None, None, None, None),              # few rows: keys split over workgroups
    (1, 3, 700, 2, 2, 40, True, 0.0, False, None, [-2], None, None),                 # a first token before the first key
    (1, 600, 64, 2, 1, 128, False, 0.0, True, None, None, None, None),               # several row tiles, one key tile
]


def masked_inputs(case, kind, seed=0):
    B, Lq, Lk, Hq, Hkv, D, causal, cap, alibi, lens, start, prefix, docs = case
    g = torch.Generator().manual_seed(seed + Lq * 7 + Lk + D)
    q = torch.randn(B, Lq, Hq, D, generator=g).to(kind)
    k, v = values(g, B, Lk, Hkv, D, kind=kind), values(g, B, Lk, Hkv, D, kind=kind)
    ints = lambda z: None if z is None else torch.tensor(z, dtype=torch.int32)  # noqa: E731
    doc = None
    if docs == "sorted":
        doc = torch.sort(torch.randint(0, 6, (B, Lk), generator=g), -1).values.int()
        doc[:, -9:] = -1
    elif docs == "mixed":
        doc = torch.randint(-1, 4, (B, Lk), generator=g).int()
    slopes = torch.exp2(-torch.arange(1, Hq + 1).float() * 8 / Hq) if alibi else None
    return q, k, v, slopes, ints(lens), ints(start), ints(prefix), doc


def masked_reference(q, k, v, scale, causal, cap, slopes, lens, start, prefix, doc):
    q, k, v = q.double(), k.double(), v.double()
    B, Lq, Hq, D = q.shape
    Lk, G = k.shape[1], Hq // k.shape[2]
    o, top, score = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(B, Lq, Hq, dtype=torch.float64)
    key = torch.arange(Lk)
    for b in range(B):
        at = torch.arange(Lq) + (int(start[b]) if start is not None else 0)
        seen = torch.ones(Lq, Lk, dtype=torch.bool)
        if causal:
            seen = key[None] <= at[:, None]
            if prefix is not None:
                seen |= key[None] < int(prefix[b])
        if lens is not None:
            seen &= key[None] < int(lens[b])
        if doc is not None:
            seen &= (doc[b][:Lq, None] == doc[b][None]) & (doc[b] >= 0)[None]
        dist = (at[:, None] - key[None]).abs().double()
        for h in range(Hq):
            bias = dist * float(slopes[h]) if slopes is not None else torch.zeros_like(dist)
            o[b, :, h], top[b, :, h], score[b, :, h] = attend(q[b, :, h], k[b, :, h // G], v[b, :, h // G], seen, bias * seen, scale, cap)
    return o, top, score


def run_masked(ops, q, k, v, scale, causal, cap, slopes, lens, start, prefix, doc):
    d = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    return ops.attention_masked(d(q), d(k), d(v), scale, causal, cap, d(slopes), d(lens), d(start), d(prefix), d(doc), d(doc))


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", MASKED, ids=lambda c: "x".join(map(str, c[:6])))
def test_attention_masked(ops, case, kind):
    q, k, v, *rest = masked_inputs(case, kind)
    args = (case[5] ** -0.5, case[6], case[7], *rest)
    want, top, score = masked_reference(q, k, v, *args)
    near(run_masked(ops, q, k, v, *args), want, top, score, kind)


@pytest.mark.parametrize("case", [MASKED[2], MASKED[4], MASKED[5], MASKED[6]], ids=lambda c: "x".join(map(str, c[:6])))
def test_attention_masked_ignores_what_lies_in_hidden_places(ops, case):
    """NaN and infinities in single keys and values: rows that do not see them are untouched."""
    q, k, v, *rest = masked_inputs(case, torch.float16)
    Lk = case[2]
    for j, bad in ((Lk // 2, math.nan), (Lk - 3, math.inf), (Lk // 3, -math.inf)):
        v[:, j, :, 1::3] = bad
    k[:, Lk // 2 + 1] = math.nan
    args = (case[5] ** -0.5, case[6], case[7], *rest)
    want, top, score = masked_reference(q, k, v, *args)
    assert want.isfinite().any() and not want.isfinite().all()
    near(run_masked(ops, q, k, v, *args), want, top, score, torch.float16)


def test_attention_masked_takes_views_in_other_orders(ops):
    q, k, v, *rest = masked_inputs(MASKED[3], torch.bfloat16)
    args = (0.1, True, 20.0, *rest)
    want = run_masked(ops, q, k, v, *args)
    head_major = lambda t: t.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)  # noqa: E731
    wide = torch.cat((v, v), -1).to(DEV)[..., v.shape[-1]:]
    assert torch.equal(run_masked(ops, head_major(q), head_major(k), wide, *args), want)


# ---- together, as they are used -----------------------------------------------------------------------------------------------

def test_a_stream_is_answered_token_by_token_from_the_cache_that_it_writes(ops):
    """A prompt is read with masked attention, its keys and values enter an 8-bit cache behind a shared prefix, then tokens are
    answered one at a time, the step captured in a graph and replayed between eager work: every answer equals the 64-bit one over
    the values that the cache holds."""
    g = torch.Generator().manual_seed(11)
    B, Hq, Hkv, D, C, P, n, steps = 3, 8, 2, 64, 64, 45, 20, 6
    kind, form, scale = torch.bfloat16, "mxfp8", 0.125
    new = [(torch.randn(B, 1, Hq, D, generator=g).to(kind), values(g, B, 1, Hkv, D, kind=kind), values(g, B, 1, Hkv, D, kind=kind)) for _ in range(steps)]
    pk, pv = (encode(values(g, Hkv, P, D), form) for _ in range(2))
    k0, v0 = values(g, B, n, Hkv, D, kind=kind), values(g, B, n, Hkv, D, kind=kind)
    x = {"pk": pk[0], "pks": pk[1], "pv": pv[0], "pvs": pv[1]}
    cache = {m + s: torch.full((B, Hkv, C, w), 255, dtype=torch.uint8, device=DEV) for m in "kv" for s, w in (("", D), ("s", D // 32))}
    pos = torch.zeros(B, dtype=torch.int32, device=DEV)
    count = torch.tensor([n, 3, 0], dtype=torch.int32, device=DEV)
    q0 = torch.randn(B, n, Hq, D, generator=g).to(kind)
    args = (scale, True, 0.0, None, count.cpu(), None, None, None)
    want, top, score = masked_reference(q0, k0, v0, *args)
    near(run_masked(ops, q0, k0, v0, *args), want, top, score, kind)
    ops.cache_write(k0.to(DEV), v0.to(DEV), pos, count, cache["k"], cache["ks"], cache["v"], cache["vs"], form)
    pos += count
    q, k, v = (t.to(DEV) for t in new[0])
    dp = {a: b.to(DEV) for a, b in x.items()}

    def step():
        ops.cache_write(k, v, pos, None, cache["k"], cache["ks"], cache["v"], cache["vs"], form)
        return ops.cache_attention(q, cache["k"], cache["v"], cache["ks"], cache["vs"], pos + 1, dp["pk"], dp["pv"], dp["pks"], dp["pvs"], form, scale, 0.0, None)

    keep = {a: b.clone() for a, b in cache.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    for a in cache:
        cache[a].copy_(keep[a])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for a, b, c in new:
        q.copy_(a), k.copy_(b), v.copy_(c)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        held = {m: t.cpu() for m, t in cache.items()}
        want, top, score = cache_reference({"q": a, **held, **x}, (pos + 1).cpu(), form, scale, 0.0, None, P)
        near(got, want, top, score, kind)
        assert torch.equal(got, step())
        codes, scales = encode(b, form)
        for i in range(B):
            assert torch.equal(held["k"][i, :, int(pos[i])], codes[i, 0]) and torch.equal(held["ks"][i, :, int(pos[i])], scales[i, 0])
            assert bool((held["k"][i, :, int(pos[i]) + 1:] == 255).all())
        pos += 1


def test_calls_on_another_stream_and_at_once(ops):
    q, k, v, *rest = masked_inputs(MASKED[7], torch.float16)
    args = (0.0625, False, 50.0, *rest)
    want = run_masked(ops, q, k, v, *args)
    dq, dk, dv = q.to(DEV), k.to(DEV), v.to(DEV)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(ops.attention_masked(dq, dk, dv, 0.0625, False, 50.0, None, None, None, None, None, None))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


# ---- refusals -----------------------------------------------------------------------------------------------------------------

def test_refusals(ops):
    z = lambda *s, kind=torch.bfloat16: torch.zeros(*s, dtype=kind, device=DEV)  # noqa: E731
    u8 = lambda *s: z(*s, kind=torch.uint8)  # noqa: E731
    i32 = lambda *s: z(*s, kind=torch.int32)  # noqa: E731
    good = dict(k=z(2, 3, 2, 64), v=None, pos=i32(2), count=None, k_codes=u8(2, 2, 8, 64), k_scales=u8(2, 2, 8, 2), v_codes=None, v_scales=None, format="mxfp8")
    ops.cache_write(**good)
    for change, match in [
        (dict(format="int8"), "unknown cache format"), (dict(format="plain"), "unknown cache format"), (dict(format="mxfp4"), "codes of k must be"),
        (dict(k=z(2, 3, 2, 48), k_codes=u8(2, 2, 8, 48), k_scales=u8(2, 2, 8, 1)), "multiple of 32"), (dict(k=z(2, 3, 2, 64, kind=torch.float64)), "must be bfloat16"),
        (dict(pos=i32(3)), "pos must be"), (dict(pos=i32(2).long()), "pos must be"), (dict(count=i32(1)), "count must be"), (dict(v=z(2, 3, 2, 64)), "go together"),
        (dict(k=z(2, 3, 2, 72)[..., 1:65]), "16-byte aligned"), (dict(k=z(2, 3, 64, 2).transpose(2, 3)), "must be contiguous"),
        (dict(k_codes=u8(2, 2, 1, 64).expand(2, 2, 8, 64)), "overlap"), (dict(k_scales=u8(2, 2, 8, 3)), "scales of k must be"), (dict(pos=i32(2).cpu()), "GPU tensor|same device|backend"),
    ]:
        with pytest.raises((RuntimeError, NotImplementedError), match=match):
            ops.cache_write(**{**good, **change})
    with pytest.raises(RuntimeError, match="unknown cache format"):
        ops.cache_read(u8(1, 1, 4, 32), u8(1, 1, 4, 1), None, "plain", torch.float16)
    with pytest.raises(RuntimeError, match="must be bfloat16"):
        ops.cache_read(u8(1, 1, 4, 32), u8(1, 1, 4, 1), None, "mxfp8", torch.float64)
    with pytest.raises(RuntimeError, match="scales of the cache"):
        ops.cache_read(u8(1, 1, 4, 32), u8(1, 1, 4, 2), None, "mxfp8", torch.float16)

    def attn(**c):
        a = dict(q=z(2, 1, 4, 64), k=z(2, 2, 8, 64), v=z(2, 2, 8, 64), k_scales=None, v_scales=None, lens=i32(2), prefix_k=None, prefix_v=None,
                 prefix_k_scales=None, prefix_v_scales=None, format="plain", scale=1.0, cap=0.0, slopes=None)
        return ops.cache_attention(**{**a, **c})
    assert attn().shape == (2, 1, 4, 64) and not attn().any()
    for change, match in [
        (dict(q=z(2, 1, 3, 64)), "share"), (dict(q=z(2, 1, 4, 48), k=z(2, 2, 8, 48), v=z(2, 2, 8, 48)), "unsupported head dim"), (dict(cap=-1.0), "cap"),
        (dict(scale=math.nan), "finite"), (dict(lens=i32(3)), "lens must be"), (dict(k=z(2, 2, 8, 64, kind=torch.float16)), "q's type"), (dict(v=z(2, 2, 9, 64)), "v must be"),
        (dict(q=z(2, 1, 4, 64, kind=torch.float32)), "bfloat16, float16"), (dict(k_scales=u8(2, 2, 8, 2)), "scales go with"), (dict(format="mxfp8"), "scales go with"),
        (dict(prefix_k=z(2, 5, 64)), "go together"), (dict(prefix_k=z(2, 5, 64), prefix_v=z(2, 6, 64)), "prefix_v must be"), (dict(slopes=z(3, kind=torch.float32)), "slopes must be"),
        (dict(q=z(2, 1, 4, 72)[..., 4:68]), "16-byte aligned"), (dict(k=z(2, 2, 8, 72)[..., :64][..., :].as_strided((2, 2, 8, 64), (1160, 580, 70, 1))), "16-byte aligned"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            attn(**change)

    def masked(**c):
        a = dict(q=z(2, 5, 4, 64), k=z(2, 8, 2, 64), v=z(2, 8, 2, 64), scale=1.0, causal=True, cap=0.0, slopes=None, lens=None, q_start=None, prefix=None, q_doc=None, k_doc=None)
        return ops.attention_masked(**{**a, **c})
    assert masked().shape == (2, 5, 4, 64)
    assert masked(q=z(2, 0, 4, 64)).shape == (2, 0, 4, 64) and not masked(k=z(2, 0, 2, 64), v=z(2, 0, 2, 64)).any()
    for change, match in [
        (dict(q=z(2, 5, 3, 64)), "share"), (dict(q=z(2, 5, 4, 60), k=z(2, 8, 2, 60), v=z(2, 8, 2, 60)), "multiple of 8"), (dict(v=z(2, 9, 2, 64)), "expected"),
        (dict(k=z(1, 8, 2, 64), v=z(1, 8, 2, 64)), "does not go with"), (dict(q_doc=i32(2, 5)), "go together"), (dict(q_doc=i32(2, 5), k_doc=i32(2, 5)), "k_doc must be"),
        (dict(causal=False, prefix=i32(2)), "causal"), (dict(cap=math.inf), "finite"), (dict(q=z(2, 5, 4, 64, kind=torch.float32)), "bfloat16, float16"),
        (dict(k=z(2, 8, 2, 64, kind=torch.float16)), "one type"), (dict(v=z(2, 8, 64, 2).transpose(2, 3)), "contiguous"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            masked(**change)
