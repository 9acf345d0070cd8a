"""Measured cases of the token-cache operators: quantised cache write / read, attention over a cache (few new tokens per
sequence, optionally behind a prefix that the whole batch shares) and masked attention (tanh cap, distance bias, causal, prefix
and document masks).

``run`` makes one pass: the plain form (elementary torch operations in fp32, rounded once at the end) where ``own`` is false, the
calls a user makes of ``torch.ops.det_sam2`` where it is true.

Formats of a cache: "plain" holds the 16-bit values themselves; "mxfp8" (e4m3) and "mxfp4" (e2m1, two codes a byte, the even
element in the low half) hold groups of 32 along the head dimension with one power-of-two scale byte each (value 2^(byte - 127)):
the smallest scale, at least 2^-126, for which no element of the group is over the code's largest value (448 resp. 6).
"""
import math

import torch

own = False

MAXIMUM = {"mxfp8": 448.0, "mxfp4": 6.0}
MANTISSA = {"mxfp8": 3, "mxfp4": 1}
SMALLEST = {"mxfp8": -6, "mxfp4": 0}          # exponent of the code's smallest normal value
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FP4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # one decoding step of 16 sequences puts its keys and values into the cache: the smallest call, latency
        dict(name="append_token", op="append", B=16, T=1, H=8, D=128, C=2048, pair=True, ragged=False, type="bf16", format="mxfp8"),
        # prompts of different lengths enter a 4-bit cache, some behind tokens that are there already
        dict(name="append_prompts", op="append", B=6, T=3001, H=8, D=128, C=4099, pair=True, ragged=True, type="fp16", format="mxfp4"),
        # the memory bank of 16 objects, 7 frames of 4096 tokens of 64 features, into 8 bits and back
        dict(name="bank_frames", op="append", B=16, T=28672, H=1, D=64, C=28672, pair=False, ragged=False, type="bf16", format="mxfp8"),
        # one sequence, one token: latency
        dict(name="decode_one", op="decode", B=1, T=1, Hq=32, Hkv=8, D=128, C=2048, low=1501, P=0, type="bf16", format="plain", cap=0.0, alibi=False),
        # a serving batch of sequences of very different lengths over an 8-bit cache
        dict(name="decode_batch", op="decode", B=32, T=1, Hq=32, Hkv=8, D=128, C=8192, low=65, P=0, type="bf16", format="mxfp8", cap=0.0, alibi=False),
        # two long contexts in 4 bits, four tokens at a time (a draft being verified), capped scores
        dict(name="decode_long", op="decode", B=2, T=4, Hq=16, Hkv=4, D=64, C=131073, low=100003, P=0, type="fp16", format="mxfp4", cap=30.0, alibi=False),
        # 64 answers behind one long instruction text
        dict(name="prefix_batch", op="decode", B=64, T=1, Hq=32, Hkv=8, D=128, C=512, low=33, P=8192, type="bf16", format="plain", cap=0.0, alibi=False),
        # seven streams behind one preloaded 8-bit bank, distance bias, one key head of 256
        dict(name="prefix_odd", op="decode", B=7, T=2, Hq=8, Hkv=1, D=256, C=77, low=2, P=1001, type="bf16", format="mxfp8", cap=0.0, alibi=True),
        # a training-length prompt with capped scores
        dict(name="causal_capped", op="masked", B=2, Lq=4096, Lk=4096, Hq=16, Hkv=8, D=128, type="bf16", causal=True, cap=50.0, alibi=False, docs=0, prefix=0, pad=0),
        # packed documents, each token sees its own document's past
        dict(name="documents", op="masked", B=1, Lq=8190, Lk=8190, Hq=16, Hkv=16, D=64, type="fp16", causal=True, cap=0.0, alibi=True, docs=13, prefix=0, pad=37),
        # a frame's 4096 tokens against a bank of 7 frames and 16 pointers of 4 tokens, older memories weigh less
        dict(name="memory", op="masked", B=1, Lq=4096, Lk=28736, Hq=4, Hkv=1, D=64, type="fp16", causal=False, cap=0.0, alibi=True, docs=0, prefix=0, pad=0),
        # a short chunk behind a bidirectional prefix, heads of 72
        dict(name="prefix_mask", op="masked", B=3, Lq=77, Lk=333, Hq=16, Hkv=16, D=72, type="fp16", causal=True, cap=0.0, alibi=False, docs=0, prefix=101, pad=5),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "masked", "masked"])
    kind = rng.choice(["bf16", "fp16"])
    if op == "append":
        form = rng.choice(["mxfp8", "mxfp4"])
        B, H, D = _log(rng, 1, 24), rng.choice([1, 2, 3, 8, 16]), rng.choice([32, 64, 96, 128, 256])
        pair = rng.random() < 0.5
        T = _log(rng, 1, max(2, min(30000, (28 << 20) // (B * H * D * (2 if pair else 1)))))
        return dict(op=op, B=B, T=T, H=H, D=D, C=T + _log(rng, 1, 1100), pair=pair, ragged=rng.random() < 0.5,
                    type=rng.choice(["bf16", "fp16", "fp32"]), format=form)
    if op == "decode":
        form = rng.choice(["plain", "mxfp8", "mxfp4"])
        Hkv, D = rng.choice([1, 2, 4, 8]), rng.choice([32, 64, 96, 128, 256])
        G, B, T = rng.choice([1, 2, 3, 4, 8]), _log(rng, 1, 48), rng.choice([1, 1, 1, 2, 3, 5])
        P = _log(rng, 17, 9000) if rng.random() < 0.5 else 0
        C = max(T + 1, _log(rng, 8, max(16, min(140000, (200 << 20) // (B * Hkv * D)))))
        return dict(op=op, B=B, T=T, Hq=G * Hkv, Hkv=Hkv, D=D, C=C, low=rng.randint(T, C), P=P, type=kind, format=form,
                    cap=rng.choice([0.0, 0.0, 15.0, 30.0, 50.0]), alibi=rng.random() < 0.3)
    Hkv, D, G, B = rng.choice([1, 2, 4, 8]), rng.choice([32, 64, 72, 96, 128, 256]), rng.choice([1, 2, 3, 4]), rng.choice([1, 1, 2, 3])
    causal = rng.random() < 0.7
    Lk = _log(rng, 1, 8200)
    Lq = Lk if causal and rng.random() < 0.7 else _log(rng, 1, Lk if causal else 4500)
    while B * Hkv * G * Lq * Lk * max(D, 64) > 1 << 35:
        B, G, Lq = max(1, B // 2), max(1, G // 2), max(1, Lq - Lq // 3)
    docs = rng.choice([0, 0, 2, 7, 30]) if Lq == Lk else 0
    return dict(op=op, B=B, Lq=Lq, Lk=Lk, Hq=G * Hkv, Hkv=Hkv, D=D, type=kind, causal=causal, cap=rng.choice([0.0, 0.0, 20.0, 50.0]),
                alibi=rng.random() < 0.4, docs=docs, prefix=rng.randint(1, Lk) if causal and not docs and rng.random() < 0.4 else 0,
                pad=rng.randint(0, Lk // 8))


# ---- sizes that follow from a case alone ----

def _spread(low, high, n):
    """n whole numbers from low to high, both ends among them."""
    return [high] if n == 1 else [low + (high - low) * i // (n - 1) for i in range(n)]


def _documents(c):
    """The document of each position: lengths that grow, then padding of no document (-1)."""
    n, L = c["docs"], c["Lk"] - c["pad"]
    ends = [L * (i + 1) * (i + 2) // (n * (n + 1)) for i in range(n)]
    ids, begin = [], 0
    for i, e in enumerate(ends):
        ids += [i] * (e - begin)
        begin = e
    return ids + [-1] * c["pad"]


def _pairs(c):
    """Visible (query, key) pairs of one head of the whole batch."""
    if c["docs"]:
        ids, n = _documents(c), {}
        for i in ids:
            if i >= 0:
                n[i] = n.get(i, 0) + 1
        return c["B"] * sum(x * (x + 1) // 2 if c["causal"] else x * x for x in n.values())
    keys = [c["Lk"] - c["pad"] * b // max(1, c["B"] - 1) if c["B"] > 1 else c["Lk"] - c["pad"] for b in range(c["B"])]
    if not c["causal"]:
        return sum(keys) * c["Lq"]
    begin = c["Lk"] - c["Lq"]
    return sum(min(n, max(begin + i + 1, c["prefix"])) for n in keys for i in range(c["Lq"]))


def _row_bytes(c):
    return {"plain": 2 * c["D"], "mxfp8": c["D"] + c["D"] // 32, "mxfp4": c["D"] // 2 + c["D"] // 32}[c["format"]]


def work(case):
    c = case
    size = 4 if c["type"] == "fp32" else 2
    if c["op"] == "append":
        rows = sum(_spread(c["T"] // 2, c["T"], c["B"])) if c["ragged"] else c["B"] * c["T"]
        back = sum(x + y for x, y in zip(*_placed(c))) if c["ragged"] else c["B"] * c["T"]
        whole = c["B"] * c["C"] if c["ragged"] else c["B"] * c["T"]
        n = c["H"] * (2 if c["pair"] else 1)
        # read the new rows, write their codes; read the codes that are there, write their values
        return {"bytes": n * (rows * (c["D"] * size + _row_bytes(c)) + back * _row_bytes(c) + whole * c["D"] * size), "flops": n * (rows + back) * c["D"] * 4}
    if c["op"] == "decode":
        keys = sum(_spread(c["low"], c["C"], c["B"]))
        held = (keys + c["P"]) * c["Hkv"] * 2 * _row_bytes(c)
        return {"bytes": held + 2 * size * c["B"] * c["T"] * c["Hq"] * c["D"], "flops": 4 * c["T"] * c["Hq"] * c["D"] * (keys + c["B"] * c["P"])}
    return {"bytes": size * c["D"] * c["B"] * (2 * c["Lq"] * c["Hq"] + 2 * c["Lk"] * c["Hkv"]), "flops": 4 * c["D"] * c["Hq"] * _pairs(c)}


def _placed(c):
    """Ragged appends: how many tokens of each sequence are there before, and how many come."""
    count = _spread(c["T"] // 2, c["T"], c["B"])
    return [(c["C"] - n) * (b + 1) // c["B"] for b, n in enumerate(count)], count


# ---- inputs ----

def _values(g, *shape):
    """Activations as a projection leaves them: normal, with some channels several times the others."""
    x = torch.randn(*shape, generator=g, device="cuda")
    return x * torch.exp(0.6 * torch.randn(shape[-1], generator=g, device="cuda"))


def _encode(x, form):
    """[..., D] fp32 -> codes and scale bytes, for the caches that a case finds filled."""
    groups = x.unflatten(-1, (-1, 32))
    most = groups.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(most.double().clamp(min=2.0 ** -140) / MAXIMUM[form])
    e = torch.where(m == 0.5, e - 1, e).clamp(-126, 127)
    y = torch.ldexp(groups, -e).flatten(-2)
    scales = (e.squeeze(-1) + 127).to(torch.uint8)
    if form == "mxfp8":
        return y.to(torch.float8_e4m3fn).view(torch.uint8), scales
    steps = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=x.device)
    code = torch.bucketize(y.abs(), steps).to(torch.uint8) + torch.where(y < 0, 8, 0).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scales


def _filled(g, c, *lead):
    x = _values(g, *lead, c["D"])
    if c["format"] == "plain":
        return x.to(TYPES[c["type"]]), None
    return _encode(x, c["format"])


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    order = torch.randperm(c["B"], generator=g, device="cuda")
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    s = {"case": c}
    kind = TYPES[c["type"]]
    if c["op"] == "append":
        B, T, H, D, C = (c[k] for k in "BTHDC")
        n = 2 if c["pair"] else 1
        s["new"] = [_values(g, B, T, H, D).to(kind) for _ in range(n)]
        if c["ragged"]:
            pos, count = (ints(v)[order] for v in _placed(c))
            s.update(pos=pos, count=count, lens=pos + count)
        else:
            s.update(pos=torch.full((B,), C - T, dtype=torch.int32, device="cuda"), count=None, lens=None)
        filled = [_encode(_values(g, B, H, C, D), c["format"]) for _ in range(n)]
        s["codes"], s["scales"] = [f[0] for f in filled], [f[1] for f in filled]
    elif c["op"] == "decode":
        B, Hkv = c["B"], c["Hkv"]
        s["q"] = torch.randn(B, c["T"], c["Hq"], c["D"], generator=g, device="cuda").to(kind)
        s["k"], s["ks"] = _filled(g, c, B, Hkv, c["C"])
        s["v"], s["vs"] = _filled(g, c, B, Hkv, c["C"])
        s["pk"], s["pks"] = _filled(g, c, Hkv, c["P"]) if c["P"] else (None, None)
        s["pv"], s["pvs"] = _filled(g, c, Hkv, c["P"]) if c["P"] else (None, None)
        s["lens"] = ints(_spread(c["low"], c["C"], B))[order]
        s["slopes"] = _slopes(c)
        s["scale"] = c["D"] ** -0.5
    else:
        B, Lq, Lk = c["B"], c["Lq"], c["Lk"]
        s["q"] = torch.randn(B, Lq, c["Hq"], c["D"], generator=g, device="cuda").to(kind)
        s["k"] = _values(g, B, Lk, c["Hkv"], c["D"]).to(kind)
        s["v"] = _values(g, B, Lk, c["Hkv"], c["D"]).to(kind)
        s["slopes"] = _slopes(c)
        s["scale"] = c["D"] ** -0.5
        s["docs"] = ints(_documents(c)).expand(B, Lk).contiguous() if c["docs"] else None
        short = [c["pad"] * b // max(1, B - 1) if B > 1 else c["pad"] for b in range(B)]
        s["lens"] = ints([Lk - x for x in short])[order] if c["pad"] and not c["docs"] else None
        s["start"] = ints([Lk - Lq] * B) if c["causal"] and Lq != Lk else None
        s["prefix"] = ints([c["prefix"]] * B) if c["prefix"] else None
    return s


def _slopes(c):
    if not c["alibi"]:
        return None
    return torch.exp2(-8.0 * torch.arange(1, c["Hq"] + 1, device="cuda", dtype=torch.float32) / c["Hq"])


# ---- one pass ----

def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": _own_append, "decode": _own_decode, "masked": _own_masked}[op](state)
    return {"append": _plain_append, "decode": _plain_decode, "masked": _plain_masked}[op](state)


def _ops():
    from det_sam2_amd import _capi
    return _capi.load_torch_ops()


def _own_append(s):
    c, ops = s["case"], _ops()
    pair = c["pair"]
    ops.cache_write(s["new"][0], s["new"][1] if pair else None, s["pos"], s["count"], s["codes"][0], s["scales"][0],
                    s["codes"][1] if pair else None, s["scales"][1] if pair else None, c["format"])
    at = 0 if c["ragged"] else c["C"] - c["T"]
    return [ops.cache_read(x[:, :, at:], y[:, :, at:], s["lens"], c["format"], TYPES[c["type"]]) for x, y in zip(s["codes"], s["scales"])]


def _own_decode(s):
    c = s["case"]
    return _ops().cache_attention(s["q"], s["k"], s["v"], s["ks"], s["vs"], s["lens"], s["pk"], s["pv"], s["pks"], s["pvs"], c["format"], s["scale"], c["cap"], s["slopes"])


def _own_masked(s):
    c = s["case"]
    return _ops().attention_masked(s["q"], s["k"], s["v"], s["scale"], c["causal"], c["cap"], s["slopes"], s["lens"], s["start"], s["prefix"], s["docs"], s["docs"])


def _rounded(x, form):
    """The values that the codes of x [..., D] stand for."""
    groups = x.float().unflatten(-1, (-1, 32))
    m, e = torch.frexp(groups.abs().amax(-1, keepdim=True).double().clamp(min=2.0 ** -140) / MAXIMUM[form])
    e = torch.where(m == 0.5, e - 1, e).clamp(-126, 127)
    y = torch.ldexp(groups, -e)
    step = (torch.frexp(y)[1] - 1).clamp(min=SMALLEST[form]) - MANTISSA[form]
    return torch.ldexp(torch.round(torch.ldexp(y, -step)), step + e).flatten(-2)


def _decoded(codes, scales, form):
    """Codes and scale bytes -> fp32 values."""
    if form == "plain":
        return codes.float()
    if form == "mxfp8":
        y = codes.view(torch.float8_e4m3fn).float()
    else:
        table = torch.tensor(FP4 + tuple(-v for v in FP4), device=codes.device)
        y = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), -1).flatten(-2)
    return (y.unflatten(-1, (-1, 32)) * torch.exp2(scales.float() - 127).unsqueeze(-1)).flatten(-2)


def _plain_append(s):
    c = s["case"]
    kind = TYPES[c["type"]]
    new = [_rounded(x, c["format"]).to(kind).transpose(1, 2) for x in s["new"]]
    if not c["ragged"]:
        return new
    at = torch.arange(c["C"], device="cuda")
    t = at - s["pos"].unsqueeze(1)                                                       # [B,C]: which new token lies there
    comes = ((t >= 0) & (t < s["count"].unsqueeze(1)))[:, None, :, None]
    there = (at < s["lens"].unsqueeze(1))[:, None, :, None]
    index = t.clamp(0, c["T"] - 1)[:, None, :, None].expand(-1, c["H"], -1, c["D"])
    old = [_decoded(x, y, c["format"]).to(kind) for x, y in zip(s["codes"], s["scales"])]
    zero = torch.zeros((), dtype=kind, device="cuda")
    return [torch.where(comes, x.gather(2, index), torch.where(there, y, zero)) for x, y in zip(new, old)]


def _softmax(x):
    """Softmax over the last axis; a row with nothing to see is zero."""
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    return p / p.sum(-1, keepdim=True).clamp(min=1e-30)


def _plain_decode(s):
    c = s["case"]
    B, T, Hkv, D, P, C = (c[k] for k in ("B", "T", "Hkv", "D", "P", "C"))
    G = c["Hq"] // Hkv
    q = s["q"].float().view(B, T, Hkv, G, D).permute(0, 2, 3, 1, 4) * s["scale"]           # [B,Hkv,G,T,D]
    k, v = _decoded(s["k"], s["ks"], c["format"]), _decoded(s["v"], s["vs"], c["format"])
    x = q.reshape(B, Hkv, G * T, D) @ k.transpose(2, 3)
    if P:
        pk, pv = _decoded(s["pk"], s["pks"], c["format"]), _decoded(s["pv"], s["pvs"], c["format"])
        rows = q.permute(1, 0, 2, 3, 4).reshape(Hkv, B * G * T, D)
        x = torch.cat(((rows @ pk.transpose(1, 2)).view(Hkv, B, G * T, P).transpose(0, 1), x), -1)
    x = x.view(B, Hkv, G, T, P + C)
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    at = P + s["lens"].view(B, 1) - T + torch.arange(T, device="cuda")                     # position of each query
    key = torch.arange(P + C, device="cuda")
    if s["slopes"] is not None:
        x = x - s["slopes"].view(1, Hkv, G, 1, 1) * (at.unsqueeze(2) - key).float()[:, None, None]
    x = x.masked_fill((key > at.unsqueeze(2))[:, None, None], -math.inf)
    p = _softmax(x).view(B, Hkv, G * T, P + C)
    o = p[..., P:] @ v
    if P:
        rows = p[..., :P].transpose(0, 1).reshape(Hkv, B * G * T, P)
        o = o + (rows @ pv).view(Hkv, B, G * T, D).transpose(0, 1)
    return o.view(B, Hkv, G, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, c["Hq"], D).to(s["q"].dtype)


def _plain_masked(s):
    c = s["case"]
    B, Lq, Lk, Hkv, D = (c[k] for k in ("B", "Lq", "Lk", "Hkv", "D"))
    G = c["Hq"] // Hkv
    q = s["q"].float().view(B, Lq, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * Lq, D) * s["scale"]
    k, v = s["k"].float().transpose(1, 2), s["v"].float().transpose(1, 2)
    x = (q @ k.transpose(2, 3)).view(B, Hkv, G, Lq, Lk)
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    key = torch.arange(Lk, device="cuda")
    start = s["start"] if s["start"] is not None else torch.zeros(B, dtype=torch.int32, device="cuda")
    at = start.view(B, 1) + torch.arange(Lq, device="cuda")
    if s["slopes"] is not None:
        x = x - s["slopes"].view(1, Hkv, G, 1, 1) * (at.unsqueeze(2) - key).abs().float()[:, None, None]
    seen = torch.ones(B, Lq, Lk, dtype=torch.bool, device="cuda")
    if c["causal"]:
        seen = key <= at.unsqueeze(2)
        if s["prefix"] is not None:
            seen = seen | (key < s["prefix"].view(B, 1, 1))
    if s["lens"] is not None:
        seen = seen & (key < s["lens"].view(B, 1, 1))
    if s["docs"] is not None:
        seen = seen & (s["docs"].unsqueeze(2) == s["docs"].unsqueeze(1)) & (s["docs"] >= 0).unsqueeze(2)
    p = _softmax(x.masked_fill(~seen[:, None, None], -math.inf)).view(B, Hkv, G * Lq, Lk)
    return (p @ v).view(B, Hkv, G, Lq, D).permute(0, 3, 1, 2, 4).reshape(B, Lq, c["Hq"], D).to(s["q"].dtype)


# ---- 64 bits, from the definition ----

def _exact_scale(most, form):
    """The smallest power of two, at least 2^-126, that brings the group's largest value to the code's range."""
    e = torch.ceil(torch.log2(most.clamp(min=1e-300) / MAXIMUM[form])) - 1
    for _ in range(2):                                    # log2 may be off by one at a power of two
        e = torch.where(MAXIMUM[form] * torch.exp2(e) < most, e + 1, e)
    return torch.exp2(e.clamp(min=-126))


def _grid(form, device):
    """All values of the code, in order, and which of them have an even code (where a tie goes)."""
    if form == "mxfp4":
        low = list(FP4)
    else:
        low = [m / 8 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)][:-1]
    return torch.tensor(low, dtype=torch.float64, device=device)


def _exact_codes(x, form):
    groups = x.double().unflatten(-1, (-1, 32))
    scale = _exact_scale(groups.abs().amax(-1, keepdim=True), form)
    grid, y = _grid(form, x.device), (groups / scale).abs()
    above = torch.searchsorted(grid, y).clamp(1, grid.numel() - 1)
    lower, upper = grid[above - 1], grid[above]
    up = (y - lower > upper - y) | ((y - lower == upper - y) & (above % 2 == 0))
    return (torch.where(up, upper, lower) * torch.sign(groups) * scale).flatten(-2)


def _exact_values(codes, scales, form):
    if form == "plain":
        return codes.double()
    low = _grid(form, codes.device)
    half = torch.zeros(8 if form == "mxfp4" else 128, dtype=torch.float64, device=codes.device)
    half[:low.numel()] = low
    table = torch.cat((half, -half))
    if form == "mxfp4":
        codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    return table[codes.int()] * (2.0 ** (scales.double() - 127)).repeat_interleave(32, -1)


def _exact_rows(x, seen, v):
    """exp(x) v over the seen keys, over the sum of exp(x); x [...,R,N], seen the same or broadcast, v [...,N,D]."""
    x = torch.where(seen, x, torch.full_like(x, -math.inf))
    top = torch.nan_to_num(x.max(-1, keepdim=True).values, neginf=0.0)
    w = (x - top).exp()
    total = w.sum(-1, keepdim=True)
    return torch.where(total > 0, torch.matmul(w, v) / torch.where(total > 0, total, torch.ones_like(total)), torch.zeros((), dtype=torch.float64, device=x.device))


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "append":
        out = []
        for new, codes, scales in zip(s["new"], s["codes"], s["scales"]):
            if not c["ragged"]:
                out.append(_exact_codes(new, c["format"]).permute(0, 2, 1, 3).contiguous())
                continue
            full = _exact_values(codes, scales, c["format"])
            for b in range(c["B"]):
                begin, n = int(s["pos"][b]), int(s["count"][b])
                full[b, :, begin:begin + n] = _exact_codes(new[b, :n], c["format"]).permute(1, 0, 2)
                full[b, :, begin + n:] = 0
            out.append(full)
        return out
    G = c["Hq"] // c["Hkv"]
    slopes = s["slopes"].double() if s["slopes"] is not None else torch.zeros(c["Hq"], dtype=torch.float64, device="cuda")
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b in range(c["B"]):
        for h in range(c["Hkv"]):
            q = s["q"][b, :, h * G:(h + 1) * G].double()                                   # [T,G,D]
            if c["op"] == "decode":
                n = int(s["lens"][b])
                pick = lambda t, i: None if t is None else t[i]  # noqa: E731
                k = _exact_values(s["k"][b, h, :n], pick(s["ks"], (b, h, slice(n))), c["format"])
                v = _exact_values(s["v"][b, h, :n], pick(s["vs"], (b, h, slice(n))), c["format"])
                if c["P"]:
                    k = torch.cat((_exact_values(s["pk"][h], pick(s["pks"], h), c["format"]), k))
                    v = torch.cat((_exact_values(s["pv"][h], pick(s["pvs"], h), c["format"]), v))
                place = torch.arange(k.shape[0], device="cuda")
                at = k.shape[0] - c["T"] + torch.arange(c["T"], device="cuda")
                seen = place[None, :] <= at[:, None]
            else:
                k, v = s["k"][b, :, h].double(), s["v"][b, :, h].double()
                place = torch.arange(c["Lk"], device="cuda")
                at = torch.arange(c["Lq"], device="cuda") + (int(s["start"][b]) if s["start"] is not None else 0)
                seen = torch.ones(c["Lq"], c["Lk"], dtype=torch.bool, device="cuda")
                if c["causal"]:
                    seen = place[None, :] <= at[:, None]
                    if c["prefix"]:
                        seen = torch.logical_or(seen, place[None, :] < c["prefix"])
                if s["lens"] is not None:
                    seen = torch.logical_and(seen, place[None, :] < int(s["lens"][b]))
                if c["docs"]:
                    mine = s["docs"][b]
                    seen = seen & (mine[:, None] == mine[None, :]) & (mine >= 0)[None, :]
            for j in range(G):
                x = torch.matmul(q[:, j], k.t()) * s["scale"]
                if c["cap"]:
                    x = torch.tanh(x / c["cap"]) * c["cap"]
                x = x - slopes[h * G + j] * (at[:, None] - place[None, :]).abs().double()
                out[b, :, h * G + j] = _exact_rows(x, seen, v)
    return out
