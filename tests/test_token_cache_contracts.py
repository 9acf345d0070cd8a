"""What the C entries of the token cache and its attention promise about sizes, without a GPU: workspaces that go by the sizes alone, calls
that are too large for one launch or one index, and the registers of the built kernels."""
import ctypes as C
import os
import re
import struct
import subprocess

import pytest
import torch

from det_sam2_amd import _capi
from test_token_cache_host import FAKE, cache_args, cache_call, lib, masked_args, masked_call, read, refused, strided, write  # noqa: F401

no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="the pointers are no GPU memory")


def test_the_workspace_goes_by_the_sizes_alone(lib):  # noqa: F811
    """Whatever the strides: a caller sizes it once."""
    for D in (32, 64, 96, 128, 256):
        for B, T, G, H in ((64, 2, 4, 2), (2, 64, 8, 1), (1, 512, 4, 2), (1, 1, 8, 8), (16, 16, 2, 8), (300, 3, 1, 2)):
            for P in (0, 500, 9000, 65536):
                for C_ in (0, 40, 512, 5000):
                    sizes = dict(B=B, T=T, Hq=G * H, Hkv=H, D=D, capacity=C_, prefix_len=P)
                    row = G * H * D
                    need = {lib.ds2_op_cache_attention_work_bytes(C.byref(cache_args(q=q, **sizes)))
                            for q in (strided(T * row, row, D), strided(row, B * row, D), strided(0, row, D), strided(2 * T * row, row, D), strided(T * row, D, T * D), strided(0, 0, 0, p=None))}
                    assert len(need) == 1, (sizes, need)


@no_gpu
def test_documents_of_no_keys_need_no_memory(lib):  # noqa: F811
    """The documents of an empty key axis are an empty tensor, which lies nowhere: what is refused below is the missing output, the next check."""
    for q_doc in (FAKE, None):
        refused(lib, masked_call(lib, Lk=0, q_doc=q_doc, k_doc=None, out=None), "output rows")
        assert lib.ds2_op_attention_masked_work_bytes(C.byref(masked_args(Lk=0, q_doc=q_doc, k_doc=None))) == 0
    refused(lib, masked_call(lib, Lk=1, q_doc=FAKE, k_doc=None, out=None), "go together")


@no_gpu
@pytest.mark.parametrize("change", [dict(B=1 << 22, H=4, T=1, D=32), dict(B=1 << 12, H=1, T=1 << 15, D=4096), dict(n=2, B=1 << 23, H=1, T=1, D=32)])
def test_a_write_of_more_rows_than_a_launch_holds_is_refused(lib, change):  # noqa: F811
    refused(lib, write(lib, **change), "too many rows")


@no_gpu
@pytest.mark.parametrize("change", [dict(B=1 << 22, H=4, C_=1, D=32), dict(B=1 << 12, H=1, C_=1 << 15, D=4096)])
def test_a_read_of_more_rows_than_a_launch_holds_is_refused(lib, change):  # noqa: F811
    refused(lib, read(lib, **change), "too many rows")


@no_gpu
@pytest.mark.parametrize("change,match", [
    (dict(B=1 << 20, Hq=8, Hkv=8, Lq=1, Lk=1), "too many rows"),                            # 2^23 workgroups of 512 threads
    (dict(B=1, Hq=1, Hkv=1, Lq=1 << 30, D=8), "too long"),                                  # a position that no 32-bit number holds
    (dict(B=1, Hq=1, Hkv=1, Lq=(1 << 30) + (1 << 29), D=8), "too long"),
    (dict(B=1 << 22, Hq=1, Hkv=1, Lq=1, Lk=1024, D=8, q_doc=FAKE, k_doc=FAKE), "too many keys"),   # 2^26 tiles of documents, a workgroup of 64 threads each
])
def test_prompts_beyond_a_launch_are_refused(lib, change, match):  # noqa: F811
    refused(lib, masked_call(lib, **change), match)


@no_gpu
def test_a_cache_beyond_a_launch_is_refused(lib):  # noqa: F811
    refused(lib, cache_call(lib, B=1 << 20, Hq=4, Hkv=4, T=1, capacity=1, prefix_len=1 << 20, format=1), "too many")


@pytest.mark.parametrize("Lq,Lk,Hq,Hkv,D,least", [(16, 1 << 20, 4, 1, 64, 200), (64, 1 << 18, 4, 1, 128, 200), (16, 1 << 18, 8, 2, 128, 100), (16, 1 << 17, 4, 1, 256, 100), (16, 1 << 18, 4, 1, 256, 200)])
def test_few_rows_over_many_keys_are_split_over_the_chip(lib, Lq, Lk, Hq, Hkv, D, least):  # noqa: F811
    """256 compute units: as many parts as there are units for each tile of rows, as far as the model of the split goes (the workspace tells)."""
    n = lib.ds2_op_attention_masked_work_bytes(C.byref(masked_args(B=1, Lq=Lq, Lk=Lk, Hq=Hq, Hkv=Hkv, D=D, causal=0)))
    parts = n / (Lq * Hq * (D + 2) * 4)
    assert parts == int(parts) and least <= parts <= 256 // Hkv


# ---- the built kernels ----------------------------------------------------------------------------------------------------------

READELF = "/opt/rocm/llvm/bin/llvm-readelf"


def kernels(path):
    """name and place of each kernel -> its entry in the metadata of the library's gfx950 code objects"""
    raw, magic, at, out = open(path, "rb").read(), b"__CLANG_OFFLOAD_BUNDLE__", 0, {}
    while (at := raw.find(magic, at)) >= 0:
        (count,), p = struct.unpack_from("<Q", raw, at + 24), at + 32
        for _ in range(count):
            offset, size, n = struct.unpack_from("<QQQ", raw, p)
            name, p = raw[p + 24:p + 24 + n], p + 24 + n
            if b"gfx950" in name and size:
                text = subprocess.run([READELF, "--notes", "-"], input=raw[at + offset:at + offset + size], stdout=subprocess.PIPE, check=True).stdout.decode()
                for entry in re.split(r"\n  - (?=\.agpr_count)", text)[1:]:
                    out[re.search(r"\.name:\s+(\S+)", entry).group(1), at] = entry
        at += len(magic)
    return out


@pytest.mark.skipif(not os.path.exists(READELF), reason="no llvm-readelf")
def test_the_attention_kernels_hold_no_accumulator_registers(lib):  # noqa: F811
    """hipcc has left out wait states in front of copies from accumulator registers, and has put copies into them in front of the restored lane
    mask of a divergent branch.  Launch bounds keep these kernels out of those registers; a rebuild that does not is seen here."""
    found = {n: e for n, e in kernels(_capi.LIB_PATH).items() if any(k in n[0] for k in ("k_attn_masked", "k_cache_attn", "k_attn_join"))}
    assert len([n for n in found if "k_attn_masked" in n[0]]) >= 92 and len([n for n in found if "k_cache_attn" in n[0]]) >= 30
    number = lambda e, key: int(re.search(rf"\.{key}:\s+(\d+)", e).group(1))  # noqa: E731
    for name, entry in found.items():
        assert number(entry, "agpr_count") == 0, name
        assert number(entry, "vgpr_count") <= 256, name
