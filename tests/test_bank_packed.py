"""Preload-bank files whose memory features are rows of a quantised token cache (bank_io, version 2): the file on the CPU, the way
through VideoProcessor and the kernels on the GPU."""
import json
import os
import struct

import pytest
import torch

from det_sam2_amd import bank_io
from test_bank_io import _state
from test_hip_token_cache import decode, encode


def cpu_pack(features, form):
    codes, scales = encode(features.unsqueeze(1), form)
    return codes.to(torch.uint8), scales.to(torch.uint8)


@pytest.mark.parametrize("form", ["mxfp8", "mxfp4"])
def test_packed_file_round_trip(tmp_path, form):
    st, g = _state(2)
    fpn2 = {0: torch.randn(4096, 256, generator=g)}
    plain, path = str(tmp_path / "plain.ds2"), str(tmp_path / "bank.ds2")
    bank_io.save_bank(plain, st, "sam2.1_hiera_t", fpn2.get)
    hdr = bank_io.save_bank(path, st, "sam2.1_hiera_t", fpn2.get, form, cpu_pack)
    assert hdr["version"] == 2 and hdr["features"] == form
    saved = (512 - (264 if form == "mxfp8" else 136)) * 1024 * 2 * 3        # two objects, three entries with features
    assert abs(os.path.getsize(plain) - os.path.getsize(path) - saved) < 4096
    got = bank_io.load_bank(path)
    assert got["obj_ids"] == [4, 9] and torch.equal(got["preload_fpn2"][0], fpn2[0])
    for key in ("cond_frame_outputs", "non_cond_frame_outputs"):
        for t, out in got["output_dict"][key].items():
            ref = st["output_dict"][key][t]
            codes, scales = cpu_pack(ref["maskmem_features"], form)
            assert out["maskmem_features"] is None and out["maskmem_format"] == form
            assert torch.equal(out["maskmem_codes"], codes) and torch.equal(out["maskmem_scales"], scales)
            for k in bank_io.ENTRY_TENSORS[1:]:
                assert torch.equal(out[k], ref[k])
    again = str(tmp_path / "again.ds2")                                      # a state that nobody has unpacked is saved as it is
    bank_io.save_bank(again, got, "sam2.1_hiera_t", lambda t: got["preload_fpn2"].get(t), form, cpu_pack)
    assert open(again, "rb").read() == open(path, "rb").read()
    with pytest.raises(ValueError, match="unpack them"):
        bank_io.save_bank(again, got, "sam2.1_hiera_t")


def test_a_bf16_file_is_what_it_was(tmp_path):
    st, _ = _state(1)
    a, b = str(tmp_path / "a"), str(tmp_path / "b")
    hdr = bank_io.save_bank(a, st, "m")
    bank_io.save_bank(b, st, "m", None, "bf16", cpu_pack)
    assert hdr["version"] == 1 and "features" not in hdr and open(a, "rb").read() == open(b, "rb").read()


def test_packed_file_refusals(tmp_path):
    st, _ = _state(1)
    path = str(tmp_path / "bank.ds2")
    with pytest.raises(ValueError, match="must be one of"):
        bank_io.save_bank(path, st, "m", None, "int8", cpu_pack)
    with pytest.raises(ValueError, match="packing function"):
        bank_io.save_bank(path, st, "m", None, "mxfp8")
    hdr = bank_io.save_bank(path, st, "m", None, "mxfp8", cpu_pack)
    raw = open(path, "rb").read()

    def rewritten(change):
        h = json.loads(json.dumps(hdr))
        change(h)
        js = json.dumps(h).encode()
        (n,) = struct.unpack("<Q", raw[8:16])
        payload = raw[(16 + n + 63) // 64 * 64:]
        with open(path, "wb") as f:
            f.write(raw[:8] + struct.pack("<Q", len(js)) + js + b"\0" * ((-(16 + len(js))) % 64) + payload)

    for change, match in [(lambda h: h.update(features="int8"), "unsupported"), (lambda h: h.pop("features"), "unsupported"), (lambda h: h.update(version=3), "unsupported"),
                          (lambda h: h.update(features="mxfp4"), "unexpected shapes"),
                          (lambda h: h["entries"][0]["tensors"]["maskmem_codes"].update(dtype="bf16", shape=[1, 1, 4096, 32]), "unexpected shapes")]:
        rewritten(change)
        with pytest.raises(ValueError, match=match):
            bank_io.load_bank(path)
    from det_sam2_amd.det_sam2_RT import VideoProcessor
    with pytest.raises(ValueError, match="bank_format"):
        VideoProcessor(bank_format="fp8")


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["mxfp8", "mxfp4"])
def test_pack_and_unpack_on_the_gpu(form):
    from det_sam2_amd.hip_model import HipOps
    hip = HipOps("cuda:0")
    x = torch.randn(3, 4096, 64, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    codes, scales = hip.pack_features(x, form)
    want = cpu_pack(x, form)
    assert torch.equal(codes.cpu(), want[0]) and torch.equal(scales.cpu(), want[1])
    y = hip.unpack_features(codes.cpu(), scales.cpu(), form)                  # from the host, as a file is read
    assert y.dtype == torch.bfloat16 and torch.equal(y.cpu().double(), decode(*want, form).squeeze(1))
    assert torch.equal(hip.unpack_features(*hip.pack_features(y, form), form), y)      # what has been rounded once stays
    with pytest.raises(ValueError, match="cache format"):
        hip.cache_alloc(1, 1, 4, 64, "plain")
    with pytest.raises(ValueError, match="multiple of 32"):
        hip.cache_alloc(1, 1, 4, 40, "mxfp8")


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["mxfp8", "mxfp4"])
def test_a_packed_bank_is_preloaded(tmp_path, form):
    """A bank of three frames, saved packed, holds in a fresh VideoProcessor exactly the rounded features of the first one, and four
    new frames are tracked on it."""
    from det_sam2_amd.synth import SyntheticDetector, synthetic_frame
    from test_hip_e2e import _vp
    from oracle.make_goldens import PRELOAD_A, PRELOAD_B
    strip = lambda c: {k: v for k, v in c.items() if k != "skip_classes"}  # noqa: E731
    bank = str(tmp_path / "bank.ds2")
    a = _vp(SyntheticDetector(2), "bf16x3k", save_inference_state_path=bank, bank_format=form, **strip(PRELOAD_A))
    a.run(frames=[synthetic_frame(t) for t in range(3)])
    b = _vp(SyntheticDetector(2), "bf16x3k", load_inference_state_path=bank, **strip(PRELOAD_B))
    segs = b.run(frames=[synthetic_frame(100 + i) for i in range(4)])
    assert sorted(segs) == [0, 1, 2, 3] and all(len(s) == 2 for s in segs.values())
    seen = 0
    for key in ("cond_frame_outputs", "non_cond_frame_outputs"):
        for t, out in a.inference_state["output_dict"][key].items():
            if out.get("maskmem_features") is None or t not in b.inference_state["output_dict"][key]:
                continue
            got = b.inference_state["output_dict"][key][t]
            want = decode(*cpu_pack(out["maskmem_features"].cpu(), form), form).squeeze(1)
            assert "maskmem_codes" not in got and torch.equal(got["maskmem_features"].cpu().double(), want)
            seen += 1
    assert seen >= 1
