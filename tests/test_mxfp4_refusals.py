"""Calls that the MXFP4 and AdamW entry points refuse, without a GPU."""

import ctypes

import pytest
import torch

from mirai_amd import AdapterAdamW, CompressedGroupedExperts, mxfp4_quantize
from mirai_amd import _native as nat
from mirai_amd import quant


def _rc(name, *args):
    return getattr(nat.load_library(), name)(*args)


BAD_QUANTIZE = [
    (1, 1, -1, 32, 32, 1, 1),   # rows
    (1, 1, 4, 0, 32, 1, 1),     # cols
    (1, 1, 4, 64, 32, 1, 1),    # rows overlap
    (1, 7, 4, 32, 32, 1, 1),    # type
    (0, 1, 4, 32, 32, 1, 1),    # null
    (16, 1, 4, 32, 32, 18, 1),  # codes alignment
]


@pytest.mark.parametrize("x,dtype,rows,cols,ldx,codes,scales", BAD_QUANTIZE)
def test_quantize_refuses(x, dtype, rows, cols, ldx, codes, scales):
    assert _rc("mx_mxfp4_quantize", x, dtype, rows, cols, ldx, codes, scales, None) == nat.MX_ERR_INVALID
    assert "mx_mxfp4_quantize" in nat.last_error()


def test_no_rows_are_no_work():
    assert _rc("mx_mxfp4_quantize", None, 1, 0, 32, 32, None, None, None) == 0
    assert _rc("mx_mxfp4_dequantize", None, None, 0, 32, None, 1, None) == 0
    assert _rc("mx_adamw_moments", None, None, 0, 1, None, None) == 0


def test_dequantize_refuses():
    for args in ((4, 1, -1, 32, 16, 1), (4, 1, 4, 0, 16, 1), (4, 1, 4, 32, 16, 9), (5, 1, 4, 32, 16, 1),
                 (4, None, 4, 32, 16, 1)):
        assert _rc("mx_mxfp4_dequantize", *args, None) == nat.MX_ERR_INVALID


def _linear(w, *, x=16, dt=1, offs=16, rows=4, E=2, out=16, odt=1, ws=256):
    return _rc("mx_mxfp4_grouped_linear", x, dt, offs, 0, rows, E, ctypes.byref(w) if w else None, out, odt,
               ws, None, None)


def test_grouped_linear_refuses():
    good = nat.MxWeight(nat.FMT_MXFP4, 16, 16, 128, 64)
    assert _linear(good, rows=0) == 0
    for w, kw in ((None, {}), (nat.MxWeight(nat.FMT_NF4, 16, 16, 128, 64), {}),
                  (nat.MxWeight(nat.FMT_MXFP4, 16, None, 128, 64), {}),
                  (nat.MxWeight(nat.FMT_MXFP4, 16, 16, 128, 96), {}),
                  (nat.MxWeight(nat.FMT_MXFP4, 16, 16, 12, 64), {}),
                  (nat.MxWeight(nat.FMT_MXFP4, 8, 16, 128, 64), {}),
                  (nat.MxWeight(nat.FMT_MXFP4, 16, 18, 128, 64), {}),
                  (good, {"rows": -1}), (good, {"rows": 1 << 31}), (good, {"E": 0}), (good, {"E": 9000}),
                  (good, {"dt": 3}), (good, {"odt": 3}), (good, {"x": None}), (good, {"offs": None}),
                  (good, {"out": None}), (good, {"out": 8}), (good, {"ws": None}), (good, {"ws": 8})):
        assert _linear(w, **kw) == nat.MX_ERR_INVALID, (w, kw)
    lib = nat.load_library()
    assert lib.mx_mxfp4_grouped_linear_workspace_size(-1, 2, 64) == 0
    assert lib.mx_mxfp4_grouped_linear_workspace_size(8, 0, 64) == 0
    assert (lib.mx_mxfp4_grouped_linear_workspace_size(4096, 8, 256)
            >= 4096 * (256 // 2 + 256 // 32))


def _config(**kw):
    base = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, step=1, dtype=0, state_bits=32,
                exp_avg=16, exp_avg_sq=16, exp_avg_e=16, exp_avg_sq_e=16)
    base.update(kw)
    return nat.MxAdamwConfig(**base)


def test_adamw_step_refuses():
    def rc(rows, **kw):
        table = (nat.MxAdamwTensor * max(len(rows), 1))(*rows)
        return _rc("mx_adamw_step", table, len(rows), ctypes.byref(_config(**kw)), None)

    assert rc([]) == 0
    good = (16, 16, 8, 0, 0)
    for rows, kw in (([good], {"dtype": 5}), ([good], {"state_bits": 16}), ([good], {"beta1": 1.0}),
                     ([good], {"beta2": -0.1}), ([good], {"beta2": float("nan")}), ([good], {"eps": -1.0}),
                     ([good], {"step": 0}), ([good], {"steps": 16, "scalars": None}),
                     ([good], {"exp_avg": None}), ([good], {"exp_avg_sq": 8}),
                     ([good], {"state_bits": 8, "exp_avg_e": None}), ([(16, 16, -1, 0, 0)], {}),
                     ([(None, 16, 8, 0, 0)], {}), ([(16, None, 8, 0, 0)], {}), ([(16, 16, 8, 64, 0)], {}),
                     ([(18, 16, 8, 0, 0)], {}), ([(16, 16, 8, 0, -1)], {}), ([(16, 16, 8, -128, 0)], {})):
        assert rc(rows, **kw) == nat.MX_ERR_INVALID, (rows, kw)
        assert "mx_adamw_step" in nat.last_error()


def test_adamw_moments_refuses():
    for args in ((16, 16, 100, 1, 16), (16, 16, -128, 1, 16), (4, 16, 128, 1, 16), (16, 16, 128, 1, 8),
                 (16, None, 128, 1, 16)):
        assert _rc("mx_adamw_moments", *args, None) == nat.MX_ERR_INVALID


def test_python_refusals():
    with pytest.raises(ValueError, match="floating-point"):
        mxfp4_quantize(torch.zeros(4, 32, dtype=torch.int32))
    with pytest.raises(ValueError, match="cols >= 1"):
        mxfp4_quantize(torch.zeros(4, 0))
    with pytest.raises(ValueError, match="cols >= 1"):
        mxfp4_quantize(torch.tensor(1.0))
    assert quant.normalize_quant_format("MXFP4") == "mxfp4"
    m = CompressedGroupedExperts.from_empty(num_experts=2, quant_format="mxfp4")
    with pytest.raises(ValueError, match="activations"):
        m.grouped_linear("w1", torch.zeros(2, 64), offsets=torch.zeros(2), activations="int8")
    n = CompressedGroupedExperts.from_empty(num_experts=2, quant_format="nf4")
    with pytest.raises(ValueError, match="quant_format"):
        n.grouped_linear("w1", torch.zeros(2, 64), offsets=torch.zeros(2), activations="mxfp4")
    with pytest.raises(ValueError, match="quant_format='mxfp4'"):
        n.load_packed_mxfp4("w1", codes=torch.zeros(1), scales=torch.zeros(1), shape=(2, 64, 64))
    with pytest.raises(ValueError, match="Unknown"):
        m.load_packed_mxfp4("nope", codes=torch.zeros(1), scales=torch.zeros(1), shape=(2, 64, 64))
    with pytest.raises(ValueError, match="experts"):
        m.load_packed_mxfp4("w1", codes=torch.zeros(1), scales=torch.zeros(1), shape=(3, 64, 64))


@pytest.mark.parametrize("kw", [{"lr": -1.0}, {"eps": -1.0}, {"betas": (0.9, 1.0)}, {"betas": (-0.1, 0.9)},
                                {"weight_decay": -1.0}, {"state_bits": 16}, {"lr": torch.tensor(1e-3)},
                                {"lr": torch.tensor(1e-3), "capturable": True}])
def test_optimizer_arguments(kw):
    with pytest.raises(ValueError):
        AdapterAdamW([torch.nn.Parameter(torch.zeros(4))], **kw)


def test_optimizer_parameters():
    p = torch.nn.Parameter(torch.zeros(4))
    with pytest.raises(ValueError, match="twice"), pytest.warns(UserWarning):
        AdapterAdamW([p, p])
    with pytest.raises(ValueError, match="bf16 or fp32"):
        AdapterAdamW([torch.nn.Parameter(torch.zeros(4, dtype=torch.float16))])
    with pytest.raises(ValueError, match="gaps or overlaps"):
        AdapterAdamW([torch.nn.Parameter(torch.zeros(4, 8)[:, :4])])
    AdapterAdamW([torch.nn.Parameter(torch.zeros(4, 8).t())])
