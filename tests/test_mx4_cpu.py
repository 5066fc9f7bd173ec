"""CPU: the restated microscaled format, and what the operators on it refuse."""
import ctypes as C
import math

import pytest
import torch

from tests import mx4_reference as R
from vila_b200 import _lib, ops


def test_restated_values_and_ties():
    x = torch.tensor([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9, -0.25, -5.0, 6.0, 4.0, -0.0]])
    codes, scales = R.quantise(x)
    assert scales.tolist() == [[127]] and codes.shape == (1, 16)
    want = [0, 1, 1, 2, 2, 4, 4, 6, 0, -4, 6, 4, 0]
    got = R.values(codes, scales, 13)
    assert got.tolist() == [[float(v) for v in want]]
    assert math.copysign(1, got[0, 8].item()) == -1 and math.copysign(1, got[0, 12].item()) == -1


def test_restated_scales():
    x = torch.tensor([[1.0], [1.9999], [2.0], [2.0 ** -126], [2.0 ** -149], [0.0], [3e38], [math.inf], [math.nan]])
    assert R.quantise(x)[1].flatten().tolist() == [125, 125, 126, 0, 0, 0, 252, 255, 255]


def test_number_is_off_by_at_most_an_eighth_of_the_blocks_scale_range():
    # half a step is 1 (in units of the scale) between 4 and 6, and 7.99 is cut to 6: never more than 2 units
    x = torch.randn(64, 96, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    codes, scales = R.quantise(x)
    unit = torch.exp2(scales.double() - 127).repeat_interleave(32, 1)
    assert ((R.values(codes, scales, 96) - x).abs() <= 2 * unit).all()


def test_host_tensors_are_refused():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    q = ops.Mx4(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(1024, dtype=torch.uint8), 64)
    for call in (lambda: ops.mx4_quantize(x), lambda: ops.mx4_dequantize(q), lambda: ops.mx4_linear(x, q), lambda: ops.mx4_matmul(q, q),
                 lambda: ops.mx4_pack(q.codes, torch.zeros(4, 2, dtype=torch.uint8), 64), lambda: ops.mx4_unpack(q)):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()


@pytest.mark.parametrize("codes, scales, cols", [
    ((4, 32), 1024, 65),        # 65 columns are three blocks
    ((4, 32), 1024, 32),        # 32 columns are one
    ((4, 32), 512, 64),         # column tiles of 128 come in twos
    ((129, 32), 1024, 64),      # two row tiles
    ((4, 32), 1024, 0),
])
def test_sizes_that_do_not_fit_are_refused(codes, scales, cols):
    with pytest.raises(RuntimeError, match="must be contiguous uint8"):
        ops.Mx4(torch.zeros(codes, dtype=torch.uint8), torch.zeros(scales, dtype=torch.uint8), cols)


def test_types_and_strides_that_do_not_fit_are_refused():
    with pytest.raises(RuntimeError, match="codes must be contiguous"):
        ops.Mx4(torch.zeros(4, 32, dtype=torch.int8), torch.zeros(1024, dtype=torch.uint8), 64)
    with pytest.raises(RuntimeError, match="codes must be contiguous"):
        ops.Mx4(torch.zeros(4, 64, dtype=torch.uint8)[:, ::2], torch.zeros(1024, dtype=torch.uint8), 64)
    q = ops.Mx4(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(1024, dtype=torch.uint8), 64)
    assert q.shape == (4, 64) and q.nbytes == 4 * 32 + 1024
    with pytest.raises(RuntimeError, match="Mx4"):
        ops.mx4_matmul(torch.zeros(4, 64), q)


@pytest.mark.skipif(torch.cuda.is_available(), reason="CPU-only behaviour")
def test_entry_points_fail_without_a_device():
    lib = _lib.load()
    assert lib.vila_mx4_quantize(None, 0, 0, None, None, 1, 32, None) != 0 and b"no CUDA device" in lib.vila_last_error()
    assert lib.vila_mx4_dequantize(None, None, None, 0, 0, 1, 32, None) != 0
    assert lib.vila_mx4_scales(None, None, 1, 32, 1, None) != 0
    assert lib.vila_mx4_linear(C.byref(_lib.Mx4LinearParams()), None) != 0


def test_no_parameters_want_no_workspace():
    lib = _lib.load()
    assert lib.vila_mx4_linear_scratch(None) == 0
    assert lib.vila_mx4_linear(None, None) != 0 and lib.vila_mx4_linear_tries(None, 5, None) != 0


def test_parameter_struct_follows_the_header():
    import re
    from pathlib import Path
    text = (Path(__file__).resolve().parent.parent / "include" / "vila_b200.h").read_text()
    body = re.search(r"typedef struct vila_mx4_linear_params \{(.*?)\} vila_mx4_linear_params;", text, flags=re.S).group(1)
    fields = []
    for decl in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";"):
        if decl.strip():
            names = decl.strip().split(",")
            fields += [names[0].split()[-1].lstrip("*")] + [n.strip().lstrip("*") for n in names[1:]]
    assert fields == [f[0] for f in _lib.Mx4LinearParams._fields_]


def test_captured_steps_are_dropped_with_the_weights_that_they_read():
    from vila_b200.serving import TokenEngine

    class Model:
        device, dtype = "cpu", torch.float32
        latent_widths = state_shapes = staticmethod(dict)
        eager = 0

        def forward_step(self, batch, cache, layer_outputs=None):
            self.eager += 1
            return torch.zeros(batch.T, 4)

        def logits(self, x):
            return x

    class Graph:
        replays = 0

        def replay(self):
            self.replays += 1

    model, graph = Model(), Graph()
    engine = TokenEngine(model, 64, 1)
    engine._decode_seen[1] = 1
    engine._decode_graphs[1] = (graph, torch.zeros(0, dtype=torch.int32), torch.zeros(1, 4), torch.zeros(1, 4))
    engine._decode_step_graphed = lambda flat, sizes: (graph.replay(), torch.zeros(1, 4))
    engine.step([("a", [1], [0])])
    assert (graph.replays, model.eager) == (1, 0)
    model.weights_version = 1
    engine.step([("a", [2], [0])])
    assert (graph.replays, model.eager) == (1, 1) and not engine._decode_graphs
    engine.step([("a", [3], [0])])      # seen once: captured, then replayed again
    assert (graph.replays, model.eager) == (2, 1)


def test_weights_in_4_bits_are_refused_before_anything_is_loaded(tmp_path):
    import json
    from vila_b200.model.registry import load_language_model, quantize_weights
    (tmp_path / "config.json").write_text(json.dumps({"architecture": "Moronex"}))
    with pytest.raises(ValueError, match="4-bit weights are for"):
        load_language_model(tmp_path, weights="mx4")
    (tmp_path / "config.json").write_text(json.dumps({"architecture": "Nusovik"}))
    with pytest.raises(ValueError, match="in bfloat16"):
        load_language_model(tmp_path, dtype="float32", weights="mx4")
    with pytest.raises(ValueError, match="None or 'mx4'"):
        load_language_model(tmp_path, weights="int4")
    with pytest.raises(ValueError, match="does not hold weights in 4 bits"):
        quantize_weights(object())
