"""Token cache and attention entry points without a GPU: what the C entries refuse before any launch, calls with nothing to do, the
sizes of the workspaces, and that the torch ops have no CPU path."""
import ctypes as C

import pytest
import torch

from det_sam2_amd import _capi

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="the pointers below are no GPU memory; on a GPU the refusals are tested with tensors")

BF16, F16, F32 = range(3)
FAKE = 1 << 20                                      # aligned, never read: every call below is refused or has nothing to do


@pytest.fixture(scope="module")
def lib():
    return _capi.load()


def strided(*s, p=FAKE):
    return _capi.Ds2Strided(p, *s)


def refused(lib, rc, match):
    text = lib.ds2_last_error().decode()
    assert rc == 1 and match in text, (rc, text)


def write(lib, n=1, x=None, codes=None, scales=None, B=2, T=3, H=2, D=64, capacity=8, pos=FAKE, count=None, type=BF16, format=1):
    two = C.POINTER(_capi.Ds2Strided)
    arr = lambda a, s: (_capi.Ds2Strided * 2)(a or strided(*s), a or strided(*s))  # noqa: E731
    return lib.ds2_op_cache_write(n, C.cast(arr(x, (T * H * D, H * D, D)), two), C.cast(arr(codes, (H * capacity * D, capacity * D, D)), two),
                                  C.cast(arr(scales, (H * capacity * D // 32, capacity * D // 32, D // 32)), two), B, T, H, D, capacity, pos, count, type, format, None)


@pytest.mark.parametrize("change,match", [
    (dict(n=0), "one or two"), (dict(n=3), "one or two"), (dict(B=-1), "bad sizes"), (dict(T=-1), "bad sizes"), (dict(H=0), "bad sizes"), (dict(capacity=-1), "bad sizes"),
    (dict(D=48), "multiple of 32"), (dict(D=0), "multiple of 32"), (dict(D=4128), "multiple of 32"), (dict(type=3), "unknown type"), (dict(format=0), "unknown format"),
    (dict(format=3), "unknown format"), (dict(pos=None), "pos is missing"), (dict(x=strided(64, 64, 64, p=None)), "null pointer"), (dict(x=strided(64, 64, 64, p=FAKE + 2)), "16-byte"),
    (dict(x=strided(64, 60, 64)), "16-byte"), (dict(codes=strided(1024, 512, 60)), "16-byte"), (dict(B=1 << 20, T=1 << 20), "too many rows"),
])
def test_cache_write_refuses(lib, change, match):
    refused(lib, write(lib, **change), match)


@pytest.mark.parametrize("change", [dict(B=0), dict(T=0), dict(capacity=0), dict(B=0, pos=None)])
def test_cache_write_of_nothing_is_no_launch(lib, change):
    assert write(lib, **change) == 0


def read(lib, codes=strided(1024, 512, 64), scales=strided(32, 16, 2), out=strided(1024, 512, 64), B=2, H=2, C_=8, D=64, lens=None, type=BF16, format=1):
    return lib.ds2_op_cache_read(codes and C.byref(codes), scales and C.byref(scales), out and C.byref(out), B, H, C_, D, lens, type, format, None)


@pytest.mark.parametrize("change,match", [
    (dict(codes=None), "null argument"), (dict(B=-1), "bad sizes"), (dict(H=0), "bad sizes"), (dict(D=33), "multiple of 32"), (dict(type=-1), "unknown type"), (dict(format=0), "unknown format"),
    (dict(out=strided(1024, 512, 64, p=None)), "null pointer"), (dict(out=strided(1024, 512, 64, p=FAKE + 8)), "16-byte"), (dict(codes=strided(1024, 512, 72)), "16-byte"),
    (dict(C_=1 << 30), "too many rows"),
])
def test_cache_read_refuses(lib, change, match):
    refused(lib, read(lib, **change), match)


def test_cache_read_of_nothing_is_no_launch(lib):
    assert read(lib, B=0) == 0 and read(lib, C_=0) == 0


def cache_args(**c):
    a = _capi.Ds2CacheAttentionArgs(B=2, T=1, Hq=8, Hkv=2, D=64, capacity=100, prefix_len=0, type=BF16, format=0, scale=1.0, cap=0.0, q=strided(512, 512, 64), k=strided(12800, 6400, 64),
                                    v=strided(12800, 6400, 64), k_scales=strided(400, 200, 2), v_scales=strided(400, 200, 2), prefix_k=strided(0, 6400, 64), prefix_v=strided(0, 6400, 64),
                                    prefix_k_scales=strided(0, 200, 2), prefix_v_scales=strided(0, 200, 2), lens=FAKE, out=FAKE)
    for k, v in c.items():
        setattr(a, k, v)
    return a


def cache_call(lib, work=FAKE, work_bytes=1 << 40, **c):
    return lib.ds2_op_cache_attention(C.byref(cache_args(**c)), work, work_bytes, None)


@pytest.mark.parametrize("change,match", [
    (dict(B=-1), "negative size"), (dict(T=-1), "negative size"), (dict(capacity=-1), "negative size"), (dict(prefix_len=-1), "negative size"), (dict(Hkv=0), "share"), (dict(Hq=9), "share"),
    (dict(Hq=1), "share"), (dict(D=72), "head dim"), (dict(D=512), "head dim"), (dict(type=F32), "bf16 or fp16"), (dict(format=4), "unknown format"), (dict(scale=float("inf")), "finite"),
    (dict(cap=float("nan")), "finite"), (dict(cap=-1.0), "finite"), (dict(cap=1e-37), "too small"), (dict(cap=1e-32, scale=-50.0), "too small"), (dict(capacity=(1 << 31) - 1), "too many tokens"), (dict(T=1 << 20), "too many tokens"), (dict(B=1 << 20, Hq=512), "too many rows"),
    (dict(q=strided(512, 512, 64, p=None)), "null pointer"), (dict(lens=None), "null pointer"), (dict(out=None), "null pointer"), (dict(out=FAKE + 8), "16-byte"), (dict(q=strided(512, 512, 60)), "16-byte"),
    (dict(k=strided(0, 0, 0, p=None)), "k is missing"), (dict(k=strided(12800, 6400, 60)), "16-byte"), (dict(v=strided(12800, 6400, 1 << 25)), "out of range"), (dict(v=strided(12800, 6400, -64)), "out of range"),
    (dict(format=1, k_scales=strided(0, 0, 0, p=None)), "missing"), (dict(prefix_len=7, prefix_v=strided(0, 0, 0, p=None)), "missing"),
    (dict(prefix_len=7, format=2, prefix_k_scales=strided(0, 0, 0, p=None)), "missing"),
])
def test_cache_attention_refuses(lib, change, match):
    refused(lib, cache_call(lib, **change), match)
    if match not in ("null pointer", "16-byte", "out of range", "missing", "k is missing"):
        assert lib.ds2_op_cache_attention_work_bytes(C.byref(cache_args(**change))) == 0


def test_cache_attention_wants_its_workspace(lib):
    need = lib.ds2_op_cache_attention_work_bytes(C.byref(cache_args(capacity=9000)))
    assert need > 0
    refused(lib, cache_call(lib, work_bytes=need - 1, capacity=9000), "workspace too small")
    refused(lib, cache_call(lib, work=None, capacity=9000), "workspace too small")
    refused(lib, cache_call(lib, work=FAKE + 8, capacity=9000), "workspace too small")
    refused(lib, lib.ds2_op_cache_attention(None, None, 0, None), "null argument")


def test_attention_over_nothing_is_no_launch(lib):
    assert cache_call(lib, B=0) == 0 and cache_call(lib, T=0) == 0
    assert masked_call(lib, B=0) == 0 and masked_call(lib, Lq=0) == 0


def masked_args(**c):
    a = _capi.Ds2AttentionMaskedArgs(B=2, Lq=5, Lk=9, Hq=8, Hkv=2, D=64, type=F16, causal=1, scale=1.0, cap=0.0, q=strided(2560, 512, 64), k=strided(1152, 128, 64), v=strided(1152, 128, 64), out=FAKE)
    for k, v in c.items():
        setattr(a, k, v)
    return a


def masked_call(lib, work=FAKE, work_bytes=1 << 40, **c):
    return lib.ds2_op_attention_masked(C.byref(masked_args(**c)), work, work_bytes, None)


@pytest.mark.parametrize("change,match", [
    (dict(B=-1), "negative size"), (dict(Lq=-1), "negative size"), (dict(Lk=-1), "negative size"), (dict(Hkv=0), "share"), (dict(Hq=7), "share"), (dict(D=4), "multiple of 8"), (dict(D=264), "multiple of 8"),
    (dict(type=F32), "bf16 or fp16"), (dict(scale=float("nan")), "finite"), (dict(cap=float("inf")), "finite"), (dict(cap=1e-37), "too small"), (dict(q_doc=FAKE), "go together"), (dict(causal=0, prefix=FAKE), "causal"),
    (dict(Lk=1 << 30), "too long"), (dict(Lq=(1 << 31) - 1), "too long"), (dict(B=1 << 24), "too many rows"), (dict(out=None), "16-byte"), (dict(q=strided(0, 0, 0, p=None)), "16-byte"),
    (dict(k=strided(1152, 132, 64)), "16-byte"), (dict(v=strided(1152, 1 << 23, 64)), "out of range"), (dict(k=strided(1152, -128, 64)), "out of range"),
])
def test_attention_masked_refuses(lib, change, match):
    refused(lib, masked_call(lib, **change), match)


def test_attention_masked_wants_its_workspace(lib):
    for c in (dict(q_doc=FAKE, k_doc=FAKE), dict(B=1, Lk=20000, causal=0)):
        need = lib.ds2_op_attention_masked_work_bytes(C.byref(masked_args(**c)))
        assert need > 0
        refused(lib, masked_call(lib, work_bytes=need - 1, **c), "workspace too small")
        refused(lib, masked_call(lib, work=None, **c), "workspace too small")


def test_workspaces_hold_their_parts(lib):
    """Over the whole range of sizes: no size overflows, and a workspace stays within what its parts can need (a share or a part of the
    keys writes one fp32 row and two statistics for each of its rows)."""
    for D in (32, 64, 96, 128, 256):
        for B in (1, 7, 64, 1000):
            for T, G, H in ((1, 1, 1), (1, 4, 8), (5, 8, 2), (300, 1, 4)):
                for C_ in (0, 1, 500, 5000, 1 << 20):
                    for P in (0, 1, 700, 100000):
                        a = cache_args(B=B, T=T, Hq=G * H, Hkv=H, D=D, capacity=C_, prefix_len=P)
                        n = lib.ds2_op_cache_attention_work_bytes(C.byref(a))
                        rows, group = B * T * G * H, 64 if T * G > 16 else 16
                        streams = B * H * -(-T * G // 16)
                        segments = (1024 + streams) * group * (D + 2) * 4 + streams * 8
                        parts = -(-P // 32) * rows * (D + 2) * 4                     # a part of the prefix is 32 keys or more
                        assert 0 <= n <= segments + parts + 256, (D, B, T, G, H, C_, P, n)
    for D in (8, 72, 128, 256):
        for B, Lq, Lk, G, H in ((1, 1, 1, 1, 1), (1, 77, 40000, 2, 2), (3, 4096, 4096, 4, 1), (2, 1, 1 << 20, 8, 4)):
            n = lib.ds2_op_attention_masked_work_bytes(C.byref(masked_args(B=B, Lq=Lq, Lk=Lk, Hq=G * H, Hkv=H, D=D)))
            assert 0 <= n <= 64 * B * Lq * G * H * (D + 2) * 4, (D, B, Lq, Lk, G, H, n)


def test_torch_ops_have_no_cpu_path():
    ops = _capi.load_torch_ops()
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)  # noqa: E731
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(NotImplementedError):
        ops.cache_write(bf(1, 2, 1, 32), None, i, None, u8(1, 1, 4, 32), u8(1, 1, 4, 1), None, None, "mxfp8")
    with pytest.raises(NotImplementedError):
        ops.cache_read(u8(1, 1, 4, 32), u8(1, 1, 4, 1), None, "mxfp8", torch.bfloat16)
    with pytest.raises(NotImplementedError):
        ops.cache_attention(bf(1, 1, 1, 32), bf(1, 1, 4, 32), bf(1, 1, 4, 32), None, None, i, None, None, None, None, "plain", 1.0, 0.0, None)
    with pytest.raises(NotImplementedError):
        ops.attention_masked(bf(1, 1, 1, 32), bf(1, 4, 1, 32), bf(1, 4, 1, 32), 1.0, False, 0.0, None, None, None, None, None, None)
