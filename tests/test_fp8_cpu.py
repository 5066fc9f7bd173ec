"""CPU: the restated 8-bit format, and what the operators on it refuse."""
import ctypes as C
import math
import re
from pathlib import Path

import numpy as np
import pytest
import torch

from tests import fp8_reference as R
from vila_b200 import _lib, ops

E4M3 = torch.float8_e4m3fn


def test_restated_numbers_are_e4m3():
    every = torch.arange(256, dtype=torch.uint8).view(E4M3).float()
    every = every[~every.isnan()].double()
    assert np.array_equal(R.e4m3(every.numpy()), every.numpy())
    y = torch.cat([torch.linspace(-450, 450, 4001), torch.linspace(-0.05, 0.05, 4001)]).float()
    assert torch.equal(torch.from_numpy(R.e4m3(y.double().numpy())), y.to(E4M3).double())


def test_restated_ties_and_scales():
    x = torch.zeros(1, 128)
    x[0, :6] = torch.tensor([448.0, 17.0, 19.0, -17.0, 2.0 ** -10, -0.0])
    codes, scales = R.quantise(x)
    assert scales.tolist() == [[1.0]]
    assert codes[0, :6].tolist() == [448.0, 16.0, 20.0, -16.0, 0.0, -0.0] and math.copysign(1, codes[0, 5].item()) == -1
    tops = torch.tensor([[0.0], [1e-45], [2.0 ** -126 * 448], [3e38], [math.inf], [math.nan]])
    got = R.quantise(tops)[1].flatten()
    assert got[:3].tolist() == [2.0 ** -126] * 3 and got[3] == np.float32(np.float32(3e38) / np.float32(448)) and got[4:].isnan().all()


def test_number_is_off_by_at_most_half_a_step():
    x = torch.randn(64, 200, generator=torch.Generator().manual_seed(1), dtype=torch.float32)
    codes, scales = R.quantise(x)
    s = R.per_element(scales, 1, 64, 200)
    v = R.values(codes, scales)
    assert ((v - x.double()).abs() <= torch.maximum(v.abs() * 2.0 ** -4, s * 2.0 ** -10) * (1 + 2.0 ** -20)).all()


def weight(rows=4, cols=64):
    return ops.Fp8(torch.zeros(rows, cols).to(E4M3), torch.ones(1, 1), 128)


def test_host_tensors_are_refused():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    q = weight()
    for call in (lambda: ops.fp8_quantize(x), lambda: ops.fp8_dequantize(q), lambda: ops.fp8_linear(x, q), lambda: ops.fp8_rmsnorm(x, None, 1e-6),
                 lambda: ops.fp8_pack(q.codes, q.scales)):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()


def test_matrices_that_do_not_fit_are_refused():
    codes = torch.zeros(130, 144).to(E4M3)
    ops.Fp8(codes, torch.ones(2, 2), 128)
    ops.Fp8(codes[:, :130], torch.ones(2, 2), 128)
    ops.Fp8(codes, torch.ones(2, 132)[:, :130].T, 1)
    for scales, rows in ((torch.ones(2, 1), 128), (torch.ones(1, 2), 128), (torch.ones(2, 2).double(), 128), (torch.ones(130, 2), 128), (torch.ones(2, 2), 1)):
        with pytest.raises(RuntimeError, match="scales must be float32"):
            ops.Fp8(codes, scales, rows)
    with pytest.raises(RuntimeError, match="block_rows=64"):
        ops.Fp8(codes, torch.ones(3, 2), 64)
    with pytest.raises(RuntimeError, match="float8_e4m3fn"):
        ops.Fp8(codes.view(torch.uint8), torch.ones(2, 2), 128)
    with pytest.raises(RuntimeError, match="as the kernels read them"):
        ops.Fp8(codes, torch.ones(130, 2), 1)                           # rows of scales apart
    with pytest.raises(RuntimeError, match="as the kernels read them"):
        ops.Fp8(codes, torch.ones(2, 130).T, 1)                         # 130 is no multiple of 4
    with pytest.raises(RuntimeError, match="as the kernels read them"):
        ops.Fp8(codes, torch.ones(2, 2).T, 128)
    with pytest.raises(RuntimeError, match="16-byte boundaries"):
        ops.Fp8(torch.zeros(130, 143).to(E4M3), torch.ones(2, 2), 128)
    with pytest.raises(RuntimeError, match="16-byte boundaries"):
        ops.Fp8(torch.zeros(144, 130).to(E4M3).T, torch.ones(2, 2), 128)
    with pytest.raises(RuntimeError, match="16-byte boundaries"):
        ops.Fp8(torch.zeros(1, 130).to(E4M3), torch.ones(1, 2), 128)    # the last row's last 16 bytes are not there


def test_what_a_linear_layer_takes():
    x, q = torch.zeros(4, 64), weight()
    for a, w in ((q, q), (x.numpy(), q), (ops.Fp8(torch.zeros(4, 64).to(E4M3), torch.ones(1, 4).T, 1), x)):
        with pytest.raises(RuntimeError, match="a must be Fp8 rows"):
            ops.fp8_linear(a, w)
    assert q.shape == (4, 64) and q.nbytes == 4 * 64 + 4


@pytest.mark.skipif(torch.cuda.is_available(), reason="CPU-only behaviour")
def test_entry_points_fail_without_a_device():
    lib = _lib.load()
    assert lib.vila_fp8_quantize(None, 0, 0, None, 0, None, 0, 1, 32, 1, None) != 0 and b"no CUDA device" in lib.vila_last_error()
    assert lib.vila_fp8_dequantize(None, 0, None, 0, None, 0, 0, 1, 32, 1, None) != 0
    assert lib.vila_fp8_rmsnorm(_lib.Fp8RmsnormParams(rows=1, cols=32), None) != 0
    assert lib.vila_fp8_linear(C.byref(_lib.Fp8LinearParams()), None) != 0


def test_no_parameters_want_no_workspace():
    lib = _lib.load()
    assert lib.vila_fp8_linear_scratch(None) == 0 and lib.vila_fp8_linear_scratch(C.byref(_lib.Fp8LinearParams())) == 0
    assert lib.vila_fp8_rmsnorm(None, None) != 0 and lib.vila_fp8_linear(None, None) != 0 and lib.vila_fp8_linear_tries(None, 5, None) != 0


@pytest.mark.parametrize("name, struct", [("vila_fp8_linear_params", _lib.Fp8LinearParams), ("vila_fp8_rmsnorm_params", _lib.Fp8RmsnormParams)])
def test_parameter_structs_follow_the_header(name, struct):
    text = (Path(__file__).resolve().parent.parent / "include" / "vila_b200.h").read_text()
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, flags=re.S).group(1)
    fields = []
    for decl in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";"):
        if decl.strip():
            names = decl.strip().split(",")
            fields += [names[0].split()[-1].lstrip("*")] + [n.strip().lstrip("*") for n in names[1:]]
    assert fields == [f[0] for f in struct._fields_]
