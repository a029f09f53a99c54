"""MXFP4 on the GPU against the numpy oracle: codec (bit for bit), the grouped
product with bf16 rows and its gradient, the product of two MXFP4 operands, and
the routed layer over MXFP4 experts."""

import numpy as np
import pytest
import torch

import mirai_amd
from mirai_amd import CompressedGroupedExperts, MXFP4Tensor, mxfp4_dequantize, mxfp4_quantize
from mirai_amd import quant
from mirai_amd import workloads as wl
from oracle import layer as olayer
from oracle import mxfp4 as omx

from helpers import assert_layer_close, build_module, oracle_loras

pytestmark = pytest.mark.gpu


def _np(t):
    return t.detach().float().cpu().numpy()


def _same(got, want):
    """Equal values and equal signs of zero, NaN in the same places."""
    assert np.array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    assert np.array_equal(got[ok], want[ok])
    assert np.array_equal(np.signbit(got[ok]), np.signbit(want[ok]))


def _check_codec(x):
    q = mxfp4_quantize(x)
    codes, scales = omx.quantize(_np(x).astype(np.float64))
    assert np.array_equal(q.scales.cpu().numpy(), scales)
    assert np.array_equal(q.codes.cpu().numpy(), codes)
    assert q.shape == tuple(x.shape)
    want = omx.dequantize(codes, scales, x.shape[-1])
    for dtype in (torch.bfloat16, torch.float32):
        got = mxfp4_dequantize(q, dtype=dtype)
        assert got.dtype == dtype and tuple(got.shape) == tuple(x.shape)
        _same(_np(got).astype(np.float64), want)


# ------------------------------------------------------------------- codec
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1), (1, 31), (3, 32), (5, 33), (7, 1000), (2, 3, 64), (1000,), (4099, 40),
                                   (2, 5, 3, 96), (33, 2048)])
def test_codec_shapes(shape, dtype):
    g = torch.Generator(device="cuda").manual_seed(sum(shape))
    x = torch.randn(shape, generator=g, device="cuda")
    x = x * torch.exp2(torch.randint(-30, 30, (*shape[:-1], 1), generator=g, device="cuda").float())
    _check_codec(x.to(dtype))


def test_codec_takes_every_bf16_value():
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    x = bits.view(torch.bfloat16)
    g = torch.Generator().manual_seed(5)
    # Each value as its block's largest, and below others.
    finite = x[torch.isfinite(x)]
    _check_codec(finite.view(-1, 1).expand(-1, 32).contiguous().cuda())
    _check_codec(finite[torch.randperm(finite.numel(), generator=g)][:65024].view(-1, 32).contiguous().cuda())
    mixed = finite[torch.randint(0, finite.numel(), (4096, 32), generator=g)]
    _check_codec(mixed.cuda())
    # One value per block beside a fixed largest one, for every spacing.
    rows = torch.zeros(finite.numel(), 32, dtype=torch.bfloat16)
    rows[:, 0], rows[:, 5] = 1.5, finite
    _check_codec(rows.cuda())


def test_codec_at_the_borders_of_rounding():
    mids = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=np.float32)
    near = np.concatenate([mids, np.nextafter(mids, np.float32(0)), np.nextafter(mids, np.float32(9)),
                           [6.0, np.nextafter(np.float32(6), np.float32(9)), 7.0, 7.9999995]]).astype(np.float32)
    for e in (-126, -125, -124, -60, 0, 60, 124, 125):
        x = np.zeros((2, 32), dtype=np.float32)
        x[0, :near.size] = near
        x[1] = -x[0]
        x[:, 31] = 4.0
        _check_codec(torch.from_numpy(np.ldexp(x, e).astype(np.float32)).cuda())


def test_codec_denormals_and_extremes():
    tiny = np.array([2.0 ** -149, 3 * 2.0 ** -149, 2.0 ** -130, 2.0 ** -127, 2.0 ** -126, 0.0, -0.0,
                     -2.0 ** -149], dtype=np.float32)
    x = np.resize(tiny, (4, 32)).astype(np.float32)
    x[1, 7] = 2.0 ** -124
    x[2, 7] = 3.4028235e38
    x[3] = 0
    _check_codec(torch.from_numpy(x).cuda())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_codec_poisons_one_block(bad, dtype):
    x = torch.randn(3, 100, device="cuda").to(dtype)
    x[1, 70] = bad
    _check_codec(x)
    got = mxfp4_dequantize(mxfp4_quantize(x))
    assert int(got.isnan().sum()) == 32


def test_codec_reads_scales_of_other_quantisers():
    codes = torch.randint(0, 256, (256, 16), dtype=torch.uint8, device="cuda")
    scales = torch.arange(256, dtype=torch.uint8, device="cuda").view(256, 1)
    want = omx.dequantize(codes.cpu().numpy(), scales.cpu().numpy(), 32)
    for dtype in (torch.float32, torch.bfloat16):
        got = _np(mxfp4_dequantize(MXFP4Tensor(codes, scales, 32), dtype=dtype)).astype(np.float64)
        big = np.abs(want) > 3.3895314e38  # beyond both types
        assert np.isinf(got[big]).all()
        _same(np.where(big, 0, got), np.where(big, 0, want))


def test_codec_strides_types_and_empty():
    base = torch.randn(64, 200, device="cuda")
    for x in (base[:, :100], base[:, 3:99], base[::2, :64], base.t(), base[:, ::2],
              base[:1].expand(5, 200), base.view(8, 8, 200)[:, 1:3, 4:68], base.half(), base.double()):
        q = mxfp4_quantize(x)
        ref = mxfp4_quantize(x.float().contiguous())
        assert torch.equal(q.codes, ref.codes) and torch.equal(q.scales, ref.scales)
    e = mxfp4_quantize(torch.empty(0, 3, 40, device="cuda"))
    assert e.shape == (0, 3, 40) and tuple(mxfp4_dequantize(e).shape) == (0, 3, 40)
    bad = mxfp4_quantize(base)
    with pytest.raises(ValueError, match="codes"):
        mxfp4_dequantize(MXFP4Tensor(bad.codes, bad.scales, 300))
    with pytest.raises(ValueError, match="dtype"):
        mxfp4_dequantize(bad, dtype=torch.float16)


# ---------------------------------------------------------- grouped product
def _module(E, out_f, in_f, seed=0, std=0.05):
    g = torch.Generator().manual_seed(1000 + seed)
    w = (torch.randn(E, out_f, in_f, generator=g) * std).bfloat16()
    m = CompressedGroupedExperts.from_empty(num_experts=E, quant_format="mxfp4")
    m.load_dense_weight("w1", w.cuda())
    wq = omx.roundtrip(w.float().numpy())
    assert np.array_equal(_np(m._dequantize("w1", dtype=torch.float32)), wq)
    return m, wq


def _reference(x, wq, ends):
    """(y, sum |x| |w|) in float64."""
    y = np.zeros((x.shape[0], wq.shape[1]))
    mag = np.zeros_like(y)
    start = 0
    for e, end in enumerate(ends):
        y[start:end] = x[start:end] @ wq[e].T
        mag[start:end] = np.abs(x[start:end]) @ np.abs(wq[e]).T
        start = max(start, end)
    return y, mag


def _bound(y, mag, K, dtype):
    """K fp32 additions (each off by at most a unit in the last place of the running
    sum, which never exceeds the sum of magnitudes), then the output's rounding."""
    acc = K * 2.0 ** -23 * mag
    return acc + (0 if dtype == torch.float32 else 2.0 ** -8 * (np.abs(y) + acc)) + 1e-30


CASES = [  # E, out, in, ends
    (1, 64, 64, [1]),
    (1, 72, 128, [33]),
    (3, 64, 192, [0, 0, 5]),
    (4, 136, 320, [1, 1, 34, 100]),
    (8, 256, 512, [64, 64, 200, 201, 201, 330, 459, 461]),
    (2, 520, 1088, [129, 300]),
    (5, 128, 64, [7, 263, 263, 520, 777]),
]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("activations,dtype", [("bf16", torch.bfloat16), ("mxfp4", torch.bfloat16),
                                               ("mxfp4", torch.float32)])
def test_grouped_linear(case, activations, dtype):
    E, out_f, in_f, ends = case
    m, wq = _module(E, out_f, in_f, seed=out_f)
    x = torch.randn(ends[-1], in_f, generator=torch.Generator().manual_seed(3)).to(dtype)
    x[0, : in_f // 2] *= 40
    xr = x.double().numpy()
    if activations == "mxfp4":
        xr = omx.roundtrip(xr)
    y, mag = _reference(xr, wq, ends)
    for odtype in (torch.int32, torch.int64):
        got = m.grouped_linear("w1", x.cuda(), offsets=torch.tensor(ends, dtype=odtype, device="cuda"),
                               activations=activations)
        assert got.dtype == dtype
        err = np.abs(_np(got).astype(np.float64) - y)
        assert (err <= _bound(y, mag, in_f, dtype)).all(), float((err - _bound(y, mag, in_f, dtype)).max())


# Rows and columns enough for the 256 x 256 tiles: last tiles of few rows, of few
# columns, of both; one to five stages of K, odd halves.
WIDE = [(1, 1720, 64, [20000]), (2, 1624, 192, [9000, 20800]), (4, 1624, 384, [100, 229, 12000, 21000]),
        (2, 2048, 128, [16513, 16640]), (3, 1544, 576, [0, 22000, 22129]), (1, 1288, 320, [26300])]


@pytest.mark.parametrize("case", WIDE, ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_mxfp4_product_of_many_rows(case, dtype):
    E, out_f, in_f, ends = case
    m, wq = _module(E, out_f, in_f, seed=out_f)
    x = torch.randn(ends[-1], in_f, generator=torch.Generator().manual_seed(3)).to(dtype)
    y, mag = _reference(omx.roundtrip(x.double().numpy()), wq, ends)
    offs = torch.tensor(ends, dtype=torch.int32, device="cuda")
    for _ in range(2):
        got = m.grouped_linear("w1", x.cuda(), offsets=offs, activations="mxfp4")
        err = np.abs(_np(got).astype(np.float64) - y)
        assert (err <= _bound(y, mag, in_f, dtype)).all(), float((err - _bound(y, mag, in_f, dtype)).max())
    some = m.grouped_linear("w1", x[:300].cuda(), offsets=offs.clamp(max=300), activations="mxfp4")
    assert torch.equal(some, got[:300])


@pytest.mark.parametrize("activations", ["bf16", "mxfp4"])
@pytest.mark.parametrize("E,out_f,in_f,ends", [(1, 64, 64, [1]), (4, 128, 320, [1, 1, 34, 100]),
                                               (3, 320, 128, [200, 200, 461])])
def test_grouped_linear_gradient(E, out_f, in_f, ends, activations):
    m, wq = _module(E, out_f, in_f, seed=7)
    x = torch.randn(ends[-1], in_f, device="cuda").bfloat16().requires_grad_(True)
    dy = torch.randn(ends[-1], out_f, generator=torch.Generator().manual_seed(4)).bfloat16()
    offs = torch.tensor(ends, dtype=torch.int32, device="cuda")
    y = m.grouped_linear("w1", x, offsets=offs, activations=activations)
    y.backward(dy.cuda())
    dx, mag = _reference(dy.double().numpy(), wq.transpose(0, 2, 1), ends)
    err = np.abs(_np(x.grad).astype(np.float64) - dx)
    assert (err <= _bound(dx, mag, out_f, torch.bfloat16)).all()
    with torch.no_grad():
        assert torch.equal(y, m.grouped_linear("w1", x, offsets=offs, activations=activations))


@pytest.mark.parametrize("activations", ["bf16", "mxfp4"])
def test_row_ends_may_be_refilled_before_the_backward(activations):
    m, wq = _module(2, 64, 128)
    offs = torch.tensor([3, 8], dtype=torch.int32, device="cuda")
    x = torch.randn(8, 128, device="cuda").bfloat16().requires_grad_(True)
    dy = torch.randn(8, 64, device="cuda").bfloat16()
    y = m.grouped_linear("w1", x, offsets=offs, activations=activations)
    offs.fill_(8)
    y.backward(dy)
    dx, mag = _reference(_np(dy).astype(np.float64), wq.transpose(0, 2, 1), [3, 8])
    assert (np.abs(_np(x.grad).astype(np.float64) - dx) <= _bound(dx, mag, 64, torch.bfloat16)).all()


@pytest.mark.parametrize("experts", [1, 3, 255, 256, 257, 1024, 1500])
def test_row_ends_of_many_experts(experts):
    g = torch.Generator().manual_seed(experts)
    counts = torch.randint(0, 4, (experts,), generator=g)
    counts[::3] = 0
    counts[0] = 300
    ends = counts.cumsum(0)
    m, wq = _module(experts, 64, 64, seed=experts)
    x = torch.randn(int(ends[-1]), 64, generator=g).bfloat16()
    for activations in ("bf16", "mxfp4"):
        got = m.grouped_linear("w1", x.cuda(), offsets=ends.cuda(), activations=activations)
        xr = x.double().numpy() if activations == "bf16" else omx.roundtrip(x.double().numpy())
        y, mag = _reference(xr, wq, ends.tolist())
        assert (np.abs(_np(got).astype(np.float64) - y) <= _bound(y, mag, 64, torch.bfloat16)).all()
    mirai_amd.check_route_errors()


def test_rows_give_the_same_bits_alone_and_together():
    m, _ = _module(2, 256, 512)
    x = torch.randn(700, 512, device="cuda").bfloat16()
    offs = torch.tensor([300, 700], dtype=torch.int32, device="cuda")
    for activations in ("bf16", "mxfp4"):
        full = m.grouped_linear("w1", x, offsets=offs, activations=activations)
        one = m.grouped_linear("w1", x[299:301], offsets=torch.tensor([1, 2], device="cuda"),
                               activations=activations)
        assert torch.equal(full[299:301], one), activations


def test_mxfp4_rows_with_nan_and_zeros():
    m, wq = _module(2, 64, 128)
    x = torch.randn(6, 128, device="cuda").bfloat16()
    x[1] = 0
    x[2, 5] = float("nan")
    x[4, 100] = float("inf")
    y = m.grouped_linear("w1", x, offsets=torch.tensor([3, 6], device="cuda"), activations="mxfp4")
    bad = y.isnan().all(dim=1)
    assert bad.tolist() == [False, False, True, False, True, False]
    assert not y[[0, 1, 3, 5]].isnan().any() and not y[1].any()


def test_mxfp4_offsets_that_do_not_match_are_reported():
    m, wq = _module(3, 64, 64)
    x = torch.randn(8, 64, device="cuda").bfloat16()
    whole = m.grouped_linear("w1", x, offsets=torch.tensor([2, 5, 8], device="cuda"), activations="mxfp4")
    mirai_amd.check_route_errors()
    for ends in ([2, 5, 7], [2, 1, 8], [2, 5, 9], [-1, 5, 8], [0, 0, 0]):
        for activations in ("mxfp4", "bf16"):
            m.grouped_linear("w1", x, offsets=torch.tensor(ends, device="cuda"), activations=activations)
            with pytest.raises(mirai_amd.RouteIndexError):
                mirai_amd.check_route_errors()
    again = m.grouped_linear("w1", x, offsets=torch.tensor([2, 5, 8], device="cuda"), activations="mxfp4")
    assert torch.equal(whole, again)
    mirai_amd.check_route_errors()


def test_mxfp4_refusals_on_the_gpu():
    m, _ = _module(2, 64, 64)
    x = torch.randn(4, 64, device="cuda").bfloat16()
    offs = torch.tensor([2, 4], device="cuda")
    with pytest.raises(ValueError, match="expects"):
        m.grouped_linear("w1", x[:, :32], offsets=offs, activations="mxfp4")
    with pytest.raises(ValueError, match="one inclusive row end"):
        m.grouped_linear("w1", x, offsets=offs[:1], activations="mxfp4")
    with pytest.raises(ValueError, match="floating"):
        m.grouped_linear("w1", x.int(), offsets=offs, activations="mxfp4")
    odd, _ = _module(2, 72, 64)
    with pytest.raises(ValueError, match="multiple of 64"):
        odd.grouped_linear("w1", x.clone().requires_grad_(True), offsets=offs, activations="mxfp4")
    m.attach_expert_lora(tensor_name="w1", adapter_name="t", rank=8, alpha=8.0)
    with pytest.raises(ValueError, match="adapter"):
        m.grouped_linear("w1", x, offsets=offs, activations="mxfp4")
    assert tuple(m.grouped_linear("w1", x[:0], offsets=offs * 0).shape) == (0, 64)
    with pytest.raises(ValueError, match="uint8"):
        m.load_packed_mxfp4("w1", codes=torch.zeros(7, dtype=torch.uint8, device="cuda"),
                            scales=torch.zeros(7, dtype=torch.uint8, device="cuda"), shape=(2, 64, 64))


def test_no_rows():
    m, _ = _module(2, 64, 64)
    x = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16)
    y = m.grouped_linear("w1", x, offsets=torch.zeros(2, dtype=torch.int32, device="cuda"), activations="mxfp4")
    assert tuple(y.shape) == (0, 64)


def test_packed_blocks_load_without_requantising():
    m, wq = _module(2, 64, 128)
    p = m.packed_weight("w1")
    n = CompressedGroupedExperts.from_empty(num_experts=2, quant_format="mxfp4")
    q = mxfp4_quantize(torch.from_numpy(wq).float().cuda())
    codes, scales = q.codes.view(2, 64, 4, 16).clone(), q.scales.clone()
    n.load_packed_mxfp4("w1", codes=codes, scales=scales, shape=(2, 64, 128))
    codes.zero_()
    assert np.array_equal(_np(n._dequantize("w1", dtype=torch.float32)), wq)
    assert n.packed_buffer_names("w1") == ("w1_mxfp4", "w1_mxfp4_scale")
    assert p.nbytes() == 2 * 64 * (64 + 4)
    assert torch.equal(n.packed_weight("w1").data, p.data)
    assert torch.equal(n.packed_weight("w1").scale, p.scale)
    one = quant.dequantize(p, experts=slice(1, 2), dtype=torch.float32)
    assert np.array_equal(_np(one)[0], wq[1])


def test_products_in_a_graph():
    m, _ = _module(4, 192, 256)
    x = torch.randn(300, 256, device="cuda").bfloat16()
    offs = torch.tensor([10, 10, 200, 300], dtype=torch.int32, device="cuda")

    def run():
        q = mxfp4_quantize(x)
        return (mxfp4_dequantize(q), m.grouped_linear("w1", x, offsets=offs, activations="mxfp4"))

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for seed in range(4):
        x.copy_(torch.randn(300, 256, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        want = run()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_products_on_a_side_stream():
    m, _ = _module(4, 192, 256)
    x = torch.randn(300, 256, device="cuda").bfloat16()
    offs = torch.tensor([10, 10, 200, 300], dtype=torch.int32, device="cuda")
    want = m.grouped_linear("w1", x, offsets=offs, activations="mxfp4")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = m.grouped_linear("w1", x, offsets=offs, activations="mxfp4")
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


@pytest.mark.parametrize("activations", ["bf16", "mxfp4"])
def test_rows_off_the_alignment(activations):
    m, _ = _module(2, 64, 128)
    buf = torch.randn(1 + 40 * 128, device="cuda").bfloat16()
    x = buf[1:].view(40, 128)
    offs = torch.tensor([7, 40], device="cuda")
    want = m.grouped_linear("w1", x.clone(), offsets=offs, activations=activations)
    assert torch.equal(m.grouped_linear("w1", x, offsets=offs, activations=activations), want)
    wide = torch.randn(40, 300, device="cuda").bfloat16()[:, 5:133]
    assert torch.equal(m.grouped_linear("w1", wide, offsets=offs, activations=activations),
                       m.grouped_linear("w1", wide.clone(), offsets=offs, activations=activations))
    grad = torch.randn(1 + 40 * 64, device="cuda").bfloat16()[1:].view(40, 64)
    out = []
    for dy in (grad, grad.clone()):
        leaf = x.clone().requires_grad_(True)
        m.grouped_linear("w1", leaf, offsets=offs, activations=activations).backward(dy)
        out.append(leaf.grad)
    assert torch.equal(*out)


@pytest.mark.parametrize("in_f", [64, 320, 384])
@pytest.mark.parametrize("rows", [2, 40, 300])
def test_infinite_rows_give_what_their_products_do(in_f, rows):
    """An infinity is not read twice where K ends in half a step of 128 columns."""
    m, wq = _module(2, 128, in_f)
    x = torch.randn(2 * rows, in_f, generator=torch.Generator().manual_seed(4)).bfloat16()
    x[0, in_f - 1] = float("inf")
    x[1, 0] = float("-inf")
    x[rows + 1, in_f - 64] = float("nan")
    y = _np(m.grouped_linear("w1", x.cuda(), offsets=torch.tensor([rows, 2 * rows], device="cuda")))
    with np.errstate(invalid="ignore"):
        want, _ = _reference(x.double().numpy(), wq.astype(np.float64), [rows, 2 * rows])
    assert np.array_equal(np.isnan(y), np.isnan(want))
    assert np.array_equal(np.isposinf(y), np.isposinf(want)) and np.array_equal(np.isneginf(y), np.isneginf(want))
    assert np.isposinf(y[0]).any() and np.isnan(y[rows + 1]).all() and np.isfinite(y[2:rows + 1]).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_bad_weights_spoil_their_column_only(bad):
    g = torch.Generator().manual_seed(0)
    w = (torch.randn(2, 128, 256, generator=g) * 0.05).bfloat16()
    w[1, 17, 100] = bad
    m = CompressedGroupedExperts.from_empty(num_experts=2, quant_format="mxfp4")
    m.load_dense_weight("w1", w.cuda())
    for rows in (3, 150):
        x = torch.randn(2 * rows, 256, generator=g).bfloat16().cuda()
        offs = torch.tensor([rows, 2 * rows], device="cuda")
        for activations in ("bf16", "mxfp4"):
            y = m.grouped_linear("w1", x, offsets=offs, activations=activations)
            want = torch.zeros(2 * rows, 128, dtype=torch.bool, device="cuda")
            want[rows:, 17] = True
            assert torch.equal(y.isnan(), want), (rows, activations)


def test_more_than_32_bits_of_elements():
    rows, cols = 2 ** 21 + 300, 2112
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    ends = x[:5], x[-300:]
    for t in ends:
        t.normal_()
    q = mxfp4_quantize(x)
    back = mxfp4_dequantize(q)
    for t, c, s, v in ((x[:5], q.codes[:5], q.scales[:5], back[:5]),
                       (x[-300:], q.codes[-300:], q.scales[-300:], back[-300:])):
        part = mxfp4_quantize(t.clone())
        assert torch.equal(part.codes, c) and torch.equal(part.scales, s)
        assert torch.equal(mxfp4_dequantize(part), v)
    assert not q.codes[5:-300].any() and not back[5:-300].any()
    del q, back
    m, _ = _module(2, 64, cols)
    y = m.grouped_linear("w1", x, offsets=torch.tensor([3, rows], device="cuda"), activations="mxfp4")
    assert torch.equal(y[-300:], m.grouped_linear("w1", x[-300:].clone(), offsets=torch.tensor([0, 300], device="cuda"),
                                                  activations="mxfp4"))
    assert torch.equal(y[:5], m.grouped_linear("w1", x[:5].clone(), offsets=torch.tensor([3, 5], device="cuda"),
                                               activations="mxfp4"))
    assert not y[5:-300].any()


def test_weights_past_32_bits_of_bytes():
    E, out_f, in_f = 520, 4096, 4160
    w = torch.zeros(E, out_f, in_f, dtype=torch.bfloat16, device="cuda")
    w[-1].normal_(std=0.05)
    m = CompressedGroupedExperts.from_empty(num_experts=E, quant_format="mxfp4")
    m.load_dense_weight("w1", w)
    one = CompressedGroupedExperts.from_empty(num_experts=1, quant_format="mxfp4")
    one.load_dense_weight("w1", w[-1:].clone())
    del w
    assert m.packed_weight("w1").data.numel() > 2 ** 32
    for rows in (3, 300):
        x = torch.randn(rows, in_f, device="cuda").bfloat16()
        dy = torch.randn(rows, out_f, device="cuda").bfloat16()
        for activations in ("bf16", "mxfp4"):
            got = []
            for module, zeros in ((m, E - 1), (one, 0)):
                leaf = x.clone().requires_grad_(True)
                offs = torch.tensor([0] * zeros + [rows], device="cuda")
                y = module.grouped_linear("w1", leaf, offsets=offs, activations=activations)
                y.backward(dy)
                got.append((y.detach().float(), leaf.grad.float()))
            # Other launches may add in another order: fp32 sums and one bf16 rounding a
            # side, 2^-8 of the value each, and as much again for the sums.
            for a, b in zip(*got):
                assert float((a - b).abs().max()) <= 2 ** -6 * float(b.abs().max())
                assert float(b.abs().max()) > 0.5


# ------------------------------------------------------------- routed layer
def test_other_paths_run_over_mxfp4_experts():
    """Every path of the module over MXFP4 experts against the same module over their
    values in bf16 (the same products; other tiles add them in another order)."""
    from mirai_amd import route_topk
    w = wl.Workload("mxpaths", 16, 300, 256, 192, 8, 2, 8, 16.0, "mxfp4", torch.bfloat16)
    dense, lora = wl.dense_weights(w), wl.lora_factors(w)
    m = build_module(w, dense, lora)
    values = {k: torch.from_numpy(omx.roundtrip(t.float().numpy())).bfloat16() for k, t in dense.items()}
    b = build_module(wl.Workload("mxpaths", 16, 300, 256, 192, 8, 2, 8, 16.0, "bf16", torch.bfloat16), values, lora)
    x = wl.tokens(w).cuda()
    idx, scores = route_topk(wl.router_logits(w).cuda(), w.top_k)
    counts = torch.tensor([10, 0, 150, 3, 37, 0, 99, 1], device="cuda")
    picks = torch.stack([torch.randperm(300, device="cuda")[:40] for _ in range(8)]).unsqueeze(0)
    weight = torch.rand(1, 8, 40, device="cuda")
    with torch.no_grad():
        for f in (lambda e: e.run_direct_routed(x, scores, idx), lambda e: e.run_for_loop(x, counts),
                  lambda e: e.run_expert_choice_routed(x, weight, picks, tokens_per_sample=300)):
            assert_layer_close(f(m), f(b))
    assert torch.equal(m.w1, values["w1"].cuda())


def _grad_close(got, want):
    """The backward's bound against another order of sums: mean 5e-3, 3e-2 of the largest."""
    got, want = got.detach().float(), want.detach().float()
    diff = (got - want).abs()
    assert float(diff.sum()) <= 5e-3 * float(want.abs().sum())
    assert float(diff.max()) <= 3e-2 * float(want.abs().max())


def test_heads_of_experts_over_mxfp4():
    """MAGI-2's groups, forward and backward, against the same values in bf16."""
    from mirai_amd import Magi2GroupedExperts
    H, E, d, f, S = 2, 4, 128, 192, 70
    g = torch.Generator().manual_seed(2)
    shapes = {"W_gate": (H * E, d, f), "W_up": (H * E, d, f), "W_down": (H * E, f, d)}
    dense = {k: (torch.randn(s, generator=g) * 0.08).bfloat16() for k, s in shapes.items()}
    values = {k: torch.from_numpy(omx.roundtrip(t.transpose(1, 2).float().numpy())).bfloat16().transpose(1, 2)
              .contiguous() for k, t in dense.items()}
    probs = torch.rand(H, S, 2, generator=g).cuda()
    idx = torch.stack([torch.randperm(E, generator=g)[:2] for _ in range(H * S)]).view(H, S, 2).cuda()
    x = torch.randn(S, H, d, generator=g).bfloat16().cuda()
    dy = torch.randn(S, H, d, generator=g).bfloat16().cuda()
    got = []
    for fmt, w in (("mxfp4", dense), ("bf16", values)):
        m = Magi2GroupedExperts.from_dense(*(w[k].cuda() for k in shapes), num_heads=H, quant_format=fmt)
        leaf = x.clone().requires_grad_(True)
        y = m.execute(leaf, probs, idx)
        y.backward(dy)
        got.append((y, leaf.grad))
    assert_layer_close(got[0][0].detach(), got[1][0].detach())
    _grad_close(got[0][1], got[1][1])


def test_chunks_and_expert_choice_train_over_mxfp4():
    from mirai_amd import MoETokenChunkPolicy, fused_chunk_runner, route_topk
    w = wl.Workload("mxchunk", 17, 300, 256, 192, 8, 2, 8, 16.0, "mxfp4", torch.bfloat16)
    dense, lora = wl.dense_weights(w), wl.lora_factors(w)
    values = {k: torch.from_numpy(omx.roundtrip(t.float().numpy())).bfloat16() for k, t in dense.items()}
    m = build_module(w, dense, lora)
    b = build_module(wl.Workload("mxchunk", 17, 300, 256, 192, 8, 2, 8, 16.0, "bf16", torch.bfloat16), values, lora)
    x, dy = wl.tokens(w).cuda(), wl.upstream_grad(w).cuda()
    idx, scores = route_topk(wl.router_logits(w).cuda(), w.top_k)
    picks = torch.stack([torch.randperm(300, device="cuda")[:40] for _ in range(8)]).unsqueeze(0)
    weight = torch.rand(1, 8, 40, device="cuda")
    policy = MoETokenChunkPolicy(token_chunk_size=128)

    def step(e, f):
        leaf = x.clone().requires_grad_(True)
        for ad in e.expert_lora.values():
            ad.lora_a.grad = ad.lora_b.grad = None
        y = f(e, leaf)
        y.backward(dy)
        return [y.detach(), leaf.grad, *(p.grad.clone() for p in e.expert_lora.parameters())]

    for f in (lambda e, t: e.run_direct_routed(t, scores, idx),
              lambda e, t: policy.execute(t, scores, idx, runner=fused_chunk_runner(e), training=True),
              lambda e, t: e.run_expert_choice_routed(t, weight, picks, tokens_per_sample=300)):
        got, want = step(m, f), step(b, f)
        assert_layer_close(got[0], want[0])
        for a, c in zip(got[1:], want[1:]):
            _grad_close(a, c)


@pytest.mark.parametrize("tokens,rank,hidden", [(1, 0, 256), (9, 16, 256), (200, 16, 256), (700, 40, 256),
                                                (1, 16, 320), (90, 0, 320), (700, 16, 320)])
def test_routed_layer_and_its_gradients(tokens, rank, hidden):
    w = wl.Workload("mxfp4", 14, tokens, hidden, 192, 8, 2, max(rank, 8), 16.0, "mxfp4", torch.bfloat16)
    dense, lora = wl.dense_weights(w), wl.lora_factors(w) if rank else None
    m = build_module(w, dense, lora)
    ow = {k: torch.from_numpy(omx.roundtrip(t.float().numpy())).bfloat16() for k, t in dense.items()}
    from mirai_amd import route_topk
    idx, scores = route_topk(wl.router_logits(w).cuda(), w.top_k)
    x = wl.tokens(w)
    xg = x.cuda().requires_grad_(True)
    out = m.run_direct_routed(xg, scores, idx)
    leaves = {k: (a.clone().requires_grad_(True), b.clone().requires_grad_(True), s)
              for k, (a, b, s) in oracle_loras(w, lora).items()}
    xo = x.clone().requires_grad_(True)
    ref = olayer.layer_forward(xo, scores.cpu(), idx.cpu(), ow, leaves, w.experts)
    assert_layer_close(out, ref)
    dy = wl.upstream_grad(w)
    out.backward(dy.cuda())
    ref.backward(dy)
    pairs = [(xg.grad, xo.grad)]
    for k, (a, b, _) in leaves.items():
        pairs += [(m.expert_lora[k].lora_a.grad, a.grad), (m.expert_lora[k].lora_b.grad, b.grad)]
    for got, want in pairs:
        rel = float((got.float().cpu() - want.float()).abs().sum() / want.float().abs().sum().clamp_min(1e-30))
        assert rel <= 1e-2
