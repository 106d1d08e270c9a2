"""What the decoder operators' path does on the host, without a GPU: claims, the lanes of typed feeds, and models with typed
inputs through the loader."""
import os
import shutil
import subprocess

import numpy as np
import pytest

from oxionnx_b200 import _ffi
from oxionnx_b200.graph import Graph, Node
from oxionnx_b200.onnx_io import Model, write_onnx
from oxionnx_b200.session import accepts_resident_slot, is_supported_op


def test_claims():
    for op in ("MatMulNBits", "OxiPagedCacheAppend", "OxiPagedAttention"):
        assert is_supported_op(op)
    assert accepts_resident_slot("MatMulNBits", 0) and not accepts_resident_slot("MatMulNBits", 1)
    assert not any(accepts_resident_slot(op, slot) for op in ("OxiPagedCacheAppend", "OxiPagedAttention") for slot in range(10))


def test_type_names():
    assert _ffi.dtype_code("bfloat16") == _ffi.DT_BF16 and _ffi.dtype_code("int32") == _ffi.DT_I32
    assert _ffi.dtype_code(np.uint8) == _ffi.DT_U8 and _ffi.dtype_code(np.dtype(np.int8)) == _ffi.DT_I8
    assert _ffi.dtype_code(np.float32) == _ffi.DT_F32 and _ffi.dtype_code(np.float16) == _ffi.DT_F32  # by name only


def test_bf16_lanes_are_rounded_to_nearest_even():
    torch = pytest.importorskip("torch")
    g = np.random.default_rng(3)
    bits = g.integers(0, 2**32, 200_000, dtype=np.uint64).astype(np.uint32)
    bits[:6] = [0x3F808000, 0x3F818000, 0x7F7FFFFF, 0x7F800000, 0xFF800000, 0x7F800001]
    a = bits.view(np.float32)
    got = _ffi.lanes_of(a, _ffi.DT_BF16)
    want = torch.from_numpy(a.copy()).bfloat16().view(torch.int16).numpy().view(np.uint16)
    nan = np.isnan(a)
    assert got.dtype == np.uint16 and np.array_equal(got[~nan], want[~nan])
    assert ((got[nan] & 0x7F80) == 0x7F80).all() and ((got[nan] & 0x7F) != 0).all()


def test_lanes_keep_their_shapes():
    a = np.arange(6, dtype=np.float64).reshape(2, 3).T
    for code, kind in ((_ffi.DT_F16, np.float16), (_ffi.DT_BF16, np.uint16), (_ffi.DT_I32, np.int32), (_ffi.DT_F32, np.float32)):
        b = _ffi.lanes_of(a, code)
        assert b.shape == (3, 2) and b.dtype == kind and b.flags.c_contiguous


def test_models_carry_typed_inputs_and_packed_weights():
    w = np.arange(64 * 2 * 16, dtype=np.uint32).astype(np.uint8).reshape(64, 2, 16)
    node = Node("MatMulNBits", "linear", ["x", "w", "s"], ["y"], {"K": 64, "N": 64, "bits": 4, "block_size": 32})
    data = write_onnx(Graph([node], ["x"], ["y"]), {"w": w, "s": np.ones((64, 2), np.float16)}, {"x": ((2, 64), np.float16)})
    m = Model.from_bytes(data)
    assert m.inputs() == [("x", (2, 64), _ffi.DT_F16)]
    assert m.optimize(1) == 0 and m.nodes()[0].op == "MatMulNBits"
    lanes, code = m.initializers()["w"]
    assert code == _ffi.DT_U8 and np.array_equal(lanes, w.astype(np.float32))


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_the_prompt_kernels_runs_cover_every_tile_once(tmp_path):
    exe = str(tmp_path / "prompt_schedule_check")
    src = os.path.join(os.path.dirname(os.path.abspath(__file__)), "host_checks", "prompt_schedule_check.cpp")
    subprocess.run(["g++", "-O2", "-std=c++17", "-o", exe, src], check=True)
    out = subprocess.run([exe, "400"], capture_output=True, text=True)
    fields = out.stdout.split()
    assert out.returncode == 0 and int(fields[0]) > 10_000 and int(fields[2]) == 0, out.stdout
