"""Every small model whose layers hold a matrix of attention or of a dense feed-forward loads with 4-bit weights, in both types (the rounding
itself needs a GPU and is left out here)."""
import importlib

import pytest
import torch

import qstream_b200 as qs
from qstream_b200.csrc import q4
from qstream_b200.errors import QsError, QStreamError

MODELS = [(name, which) for name in ("lutelorn", "fofinex", "sefuvik", "nutatar", "fotanex", "vofinex") for which in sorted(importlib.import_module(name + "_util").CONFIGS)]
# models of mixers and experts alone, whose matrices stay as they are stored
WIDE_ONLY = {("fofinex", "L"), ("sefuvik", "R"), ("nutatar", "G"), ("nutatar", "L"), ("nutatar", "M"), ("fotanex", "R"), ("fotanex", "S"), ("fotanex", "M")}


def rounded(weight, group=64):
    n, k = weight.shape
    codes, scales = q4.sizes(n, k, group)
    return q4.Weight4(torch.full(codes, 0x88, dtype=torch.uint8), torch.zeros(scales, dtype=torch.bfloat16), n, k, group)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name,which", MODELS)
def test_every_arrangement_takes_narrow_matrices(tmp_path, monkeypatch, name, which, dtype):
    monkeypatch.setattr(q4, "quantize", rounded)
    folder, _ = importlib.import_module(name + "_util").make_folder(tmp_path, which, dtype)
    load = lambda **kw: qs.load_model(folder, dtype=dtype, device="cpu", allow_mmap=False, **kw)       # noqa: E731
    if (name, which) in WIDE_ONLY:
        with pytest.raises(QStreamError) as e:
            load(weight_bits=4)
        assert e.value.code == QsError.UNSUPPORTED_ARCH
        return
    wide, narrow = load(), load(weight_bits=4, weight_group=32)
    assert narrow.runtime.narrowed and narrow.n_parameters == wide.n_parameters and narrow.weight_bytes < wide.weight_bytes


def test_what_a_key_takes_does_not_depend_on_how_the_matrices_are_held(tmp_path, monkeypatch):
    from util import make_folder
    monkeypatch.setattr(q4, "quantize", rounded)
    for dtype, size in (("float32", 4), ("bfloat16", 2)):
        folder, _ = make_folder(tmp_path, "A", dtype)
        for bits in (None, 4):
            mixer = qs.load_model(folder, dtype=dtype, device="cpu", allow_mmap=False, weight_bits=bits).blocks[0].mixer
            assert mixer.cache_bytes_per_key == size * mixer.spec.n_kv_heads * (mixer.spec.head_dim + mixer.spec.value_dim)


def test_a_matrix_that_no_product_takes_is_not_made():
    """Wider matrices are refused when they are rounded, so when a model is loaded, and not at its first step."""
    from qstream_b200.parts import Runtime
    wide = torch.zeros(2, q4.MAX_COLUMNS + 1)
    for make in (q4.quantize, Runtime(dtype=torch.float32, device=torch.device("cpu"), weight_group=64).matrix):
        with pytest.raises(QStreamError, match="32769 columns") as e:
            make(wide)
        assert e.value.code == QsError.QUANT_MISMATCH


@pytest.mark.parametrize("name,which", [m for m in MODELS if m[0] in ("lutelorn", "fotanex", "vofinex") and m not in WIDE_ONLY])
def test_the_bytes_of_a_narrow_model(tmp_path, monkeypatch, name, which):
    """What the wide model holds, less its matrices, and the narrow ones; rows that fill up a product are none of the wide model's."""
    from qstream_b200.parts import Part
    monkeypatch.setattr(q4, "quantize", rounded)
    folder, _ = importlib.import_module(name + "_util").make_folder(tmp_path, which, "float32")
    wide, narrow = (qs.load_model(folder, dtype="float32", device="cpu", allow_mmap=False, weight_bits=bits) for bits in (None, 4))
    stored = held = 0

    def look(part):
        nonlocal stored, held
        for key, value in vars(part).items():
            if isinstance(value, q4.Weight4):
                rows = part.gate_at + part.gate_rows if key == "w_qkv" else value.out_features
                stored, held = stored + 4 * rows * value.in_features, held + value.nbytes
            elif isinstance(value, Part):
                look(value)

    for block in narrow.blocks:
        look(block)
    assert narrow.weight_bytes == wide.weight_bytes - stored + held
