"""What microscaled weights refuse, and their definition; no GPU needed."""
import pathlib
import re

import numpy as np
import pytest
import torch

import plain_mx as plain
from alofa_b200 import mx
from alofa_b200.cli.generate import build_parser
from alofa_b200.config.engine_config import EngineConfig
from alofa_b200.errors import AlofaError
from alofa_b200.models.qwen2 import build_spec
from alofa_b200.parts.base import Runtime
from alofa_b200.parts.model import Model
import tiny


def refused(code, call, *args, **kw):
    with pytest.raises(AlofaError) as err:
        call(*args, **kw)
    assert err.value.code == code, err.value


def test_settings():
    EngineConfig(weight_format="mxfp4").validate()
    refused("invalid_argument", EngineConfig(weight_format="mxfp4", dtype="float32").validate)
    refused("invalid_argument", EngineConfig(weight_format="int4").validate)
    assert build_parser().parse_args(["--weight-format", "mxfp4"]).weight_format == "mxfp4"
    with pytest.raises(SystemExit):
        build_parser().parse_args(["--weight-format", "int4"])


def test_models_that_take_the_format():
    cpu, bf16 = torch.device("cpu"), torch.bfloat16
    spec = build_spec(tiny.CONFIGS["A"][0])
    model = Model(spec, Runtime(cpu, bf16, "mxfp4"))
    assert model.tensors().keys() == Model(spec, Runtime(cpu, bf16)).tensors().keys()
    refused("unsupported", Model, spec, Runtime(cpu, torch.float32, "mxfp4"))
    refused("unsupported", Model, spec, Runtime(cpu, bf16, "int4"))


def test_models_that_do_not():
    import tiny_kotutar
    from alofa_b200.config.registry import get_architecture

    arch = get_architecture("Kotutar")
    spec = arch.build_spec(arch.read_config(tiny_kotutar.CONFIGS["A"], "test"))
    refused("unsupported", Model, spec, Runtime(torch.device("cpu"), torch.bfloat16, "mxfp4"))


@pytest.mark.skipif(torch.cuda.is_available(), reason="for machines without a GPU")
def test_operators_need_a_gpu():
    x, u8 = torch.zeros(2, 128), torch.zeros(2, 128, dtype=torch.uint8)
    refused("unsupported", mx.quantize_rows, x)
    refused("unsupported", mx.pack_weight, x)
    refused("unsupported", mx.norm_rows, x, torch.ones(128), 1e-6)
    refused("unsupported", mx.MxRows, u8, torch.zeros(2, 4, dtype=torch.uint8), 128)
    refused("unsupported", mx.MxWeight.from_codes, u8, torch.zeros(2, 8, dtype=torch.uint8), 256)


def test_arguments_as_the_library_has_them():
    """Every entry point is declared with as many arguments, of the same sizes, as its source has: one more would go through unconverted, an address cut to 32 bits."""
    from alofa_b200.csrc import ops

    lib, kernels = ops.mx_library(), pathlib.Path(ops.__file__).parent / "kernels"
    found = re.findall(r"ALOFA_API int (alofa_mx_\w+)\(([^)]*)\)", "".join((kernels / name).read_text() for name in ("mx_rows.cu", "mx_gemm.cu")))
    assert len(found) == 9
    for name, args in found:
        kinds = ["c_void_p" if "*" in a else {"int": "c_int", "float": "c_float", "long long": "c_long"}[a.strip().rsplit(" ", 1)[0]] for a in args.split(",")]
        assert [{"c_longlong": "c_long"}.get(t.__name__, t.__name__) for t in getattr(lib, name).argtypes] == kinds, name


def test_the_definition():
    """Encoding is the nearest of all codes; what it gives is encoded to itself."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((7, 200)) * np.exp2(rng.integers(-20, 20, (7, 1)))
    for weights, half in ((False, 2.0**-4), (True, 2.0**-2)):
        v = plain.values(x, weights)
        largest = np.abs(np.pad(x, ((0, 0), (0, 24)))).reshape(7, -1, 32).max(-1).repeat(32, -1)[:, :200]
        # half a step of the number's own size, or of the block's smallest; what a weight clips is at most a quarter off
        assert (np.abs(v - x) <= np.maximum(half * np.abs(x), largest * (2.0**-3 if weights else 2.0**-17))).all()
        assert np.array_equal(plain.values(v, weights), v)
    assert plain.scale_bytes(np.array([448.0, 448.1, 1.75, 0.0, np.inf, np.nan]), False).tolist() == [127, 128, 119, 0, 255, 255]
    assert plain.scale_bytes(np.array([4.0, 6.0, 7.99, 8.0, 0.0]), True).tolist() == [127, 127, 127, 128, 0]
