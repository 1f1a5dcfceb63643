"""Activations in 8-bit integers and their products with int8 weights.

Codes and scales are held to their definition bit for bit.  A product's integer sum is exact; what follows is a conversion, a product and
a fused multiply-add in fp32 and one rounding to the output's type, each off by at most half a step: 3 * 2^-24 of |sum * scales|,
2^-24 of the result and eps / 2 of it (and half of the type's smallest step where the result is below its normal range)."""
import copy
import io
import warnings

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

import if_i_could_turn_back_time_b200 as jq
from if_i_could_turn_back_time_b200 import _lib, checkpoint, ops

DEV = "cuda"
gpu = pytest.mark.gpu
DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def _codes(v):
    """Codes and scales of fp32 rows [n, K], by their definition, on the CPU."""
    v = v.cpu()
    size = v.abs().amax(-1)
    good = torch.isfinite(size)                                    # (NaN counts as the largest)
    s = torch.where(good, size, 0.0).clamp(min=2.0 ** -100) / torch.full_like(size, 127.0)
    q = torch.where(good[:, None], torch.round(v / s[:, None]).clamp(-127, 127), 0.0).to(torch.int8)
    return q, torch.where(good, s, torch.nan)


def _same(a, b):
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(0), b.nan_to_num(0))


def _product(q, s, pw, bias, dtype):
    """(result, bound) in 64 bits of codes [n, K] with their scales."""
    total = q.double() @ pw.qweight[:, :pw.K].double().T           # (below 2^53: exact)
    y = total * pw.scales.double() * s.double()[:, None]
    part = y.abs()
    if bias is not None:
        y = y + bias.double()
    fin = torch.finfo(dtype)
    bound = 3 * 2.0 ** -24 * part + (2.0 ** -24 + fin.eps / 2) * (y.abs() + part * 2.0 ** -22) + fin.smallest_normal * fin.eps / 2
    return y, bound


def _near(got, want, bound):
    assert got.shape == want.shape
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), (off / bound).max().item()


def _weight(N, K, seed=0, had=0):
    gen = torch.Generator(DEV).manual_seed(seed)
    return jq.pack_weight(torch.randn(N, K, device=DEV, generator=gen) * (torch.rand(N, 1, device=DEV, generator=gen) + 0.5), jq.QuantSpec("int8", 0, had))


# ------------------------------------------------------------------------------------------------------------ quantising

@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,K", [(1, 1), (3, 7), (5, 8), (2, 31), (70, 100), (9, 256), (1, 1000), (400, 1000), (6, 1024), (400, 1032), (1, 8192), (301, 4100),
                                    (500, 4096), (3, 32768), (2, 32776), (300, 11008), (400, 12296), (3, 28672), (2, 98304), (2, 131064), (2, 131071), (66000, 1100)])
def test_codes_are_those_of_the_definition(rows, K, dtype):
    gen = torch.Generator(DEV).manual_seed(rows + K)
    x = torch.randn(rows, K, device=DEV, generator=gen)
    x[:, ::13] *= 9
    x = (x * torch.rand(rows, 1, device=DEV, generator=gen)).to(dtype)
    got = ops.quantize_rows(x)
    q, s = _codes(x.float())
    assert got.codes.shape == (rows, K) and got.codes.stride(0) % 32 == 0 and got.dtype == dtype and got.had_block == 0
    assert torch.equal(got.scales.cpu(), s) and torch.equal(got.codes.cpu(), q)
    for out in DTYPES:
        want = (q.float() * s[:, None]).to(out)
        assert torch.equal(got.dequantize(out).cpu(), want)
    assert got.dequantize().dtype == dtype


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,K", [(1, 128), (400, 128), (7, 384), (600, 1024), (3, 4096), (330, 11008), (300, 12416), (2, 32768), (3, 33024), (5, 130944)])
def test_rotated_codes(rows, K, dtype):
    """The rotation has the bits of ops.fwht_block."""
    x = torch.randn(rows, K, device=DEV, generator=torch.Generator(DEV).manual_seed(K)).to(dtype)
    x[:, 5] *= 30
    got = ops.quantize_rows(x, had_block=128)
    q, s = _codes(ops.fwht_block(x, 128))
    assert got.had_block == 128 and torch.equal(got.scales.cpu(), s) and torch.equal(got.codes.cpu(), q)
    wide = torch.empty(rows, K + 3, dtype=dtype, device=DEV)[:, 3:]                  # rows that are not of 16-byte pieces
    wide.copy_(x)
    again = ops.quantize_rows(wide, 128)
    assert torch.equal(again.scales, got.scales) and torch.equal(again.codes, got.codes)


@gpu
def test_quotients_at_the_border_of_two_codes():
    """Values half a step from a code and their neighbours of fp32, at scales of many sizes: where the products with the reciprocals
    on both sides of it disagree."""
    size = torch.tensor([127.0, 254.0, 1.0, 3.3, 1e-20, 7e18, 2.0 ** -100, 126.99999, 0.1], device=DEV)
    half = torch.arange(-126.5, 127, 1, device=DEV)
    x = half * (size / 127)[:, None]
    x = torch.cat([torch.nextafter(x, torch.full_like(x, -torch.inf)), x, torch.nextafter(x, torch.full_like(x, torch.inf)), size[:, None]], 1)
    got = ops.quantize_rows(x)
    q, s = _codes(x)
    assert torch.equal(got.codes.cpu(), q) and torch.equal(got.scales.cpu(), s)


@gpu
@pytest.mark.parametrize("K", [24, 1003, 9000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_go_wrong(K, dtype):
    x = torch.randn(400, K, device=DEV).to(dtype)
    x[0] = 0
    x[1, K // 2] = torch.nan
    x[2, K - 1] = torch.inf
    x[3, 0] = -torch.inf
    x[4] = torch.finfo(dtype).max
    x[5] = torch.finfo(dtype).tiny / 4
    x[6] = torch.nan
    x[7, 1:] = 0
    for t in (x, x[:8]):
        got = ops.quantize_rows(t)
        q, s = _codes(t.float())
        assert _same(got.scales.cpu(), s) and torch.equal(got.codes.cpu(), q)
        assert torch.isnan(got.scales[[1, 2, 3, 6]]).all() and torch.isfinite(got.scales[[0, 4, 5, 7]]).all()
        pw = _weight(40, K)
        y = ops.linear(t, pw)
        assert torch.isnan(y[[1, 2, 3, 6]]).all() and bool((y[0] == 0).all()) and torch.isfinite(y[[0, 5, 7]]).all() and torch.isfinite(y[8:]).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_leading_dims_of_rows(dtype):
    raw = torch.randn(3, 40, 600, device=DEV).to(dtype)
    for x in (raw[:, :, 1:257], raw[:, ::3, 8:520], raw[1, :, 3:300], raw.transpose(1, 2)[:, :, :40], raw[:1].expand(2, 40, 600), raw[0, 0, :77], raw[:, 0],
              raw[:, :0], torch.randn(1, 600, device=DEV).expand(5, 600).to(dtype)):
        got = ops.quantize_rows(x)
        q, s = _codes(x.float().reshape(-1, x.shape[-1]))
        assert got.codes.shape == x.shape and got.scales.shape == x.shape[:-1]
        assert torch.equal(got.codes.reshape(-1, x.shape[-1]).cpu(), q) and torch.equal(got.scales.reshape(-1).cpu(), s)
        assert got.dequantize().shape == x.shape


# -------------------------------------------------------------------------------------------------------------- products

ROWS = (1, 2, 15, 16, 17, 33, 64, 65, 129, 257, 700)


@gpu
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("N,K", [(1, 1), (7, 100), (300, 784), (128, 128), (129, 130), (1003, 4100), (4096, 512)])
def test_linear_against_64_bits(rows, N, K):
    gen = torch.Generator(DEV).manual_seed(rows + N + K)
    pw = _weight(N, K)
    x = torch.randn(rows, K, device=DEV, generator=gen)
    x *= torch.rand(rows, 1, device=DEV, generator=gen) * 3
    for i, dtype in enumerate(DTYPES):
        bias = torch.randn(N, device=DEV, generator=gen) if (rows + i) % 2 else None
        xs = x.to(dtype)
        rows8 = ops.quantize_rows(xs)
        y = ops.linear(xs, pw, bias)
        _near(y, *_product(rows8.codes, rows8.scales, pw, bias, dtype))
        assert y.dtype == dtype and torch.equal(ops.linear(rows8, pw, bias), y)
        other = DTYPES[i - 1]
        _near(ops.linear(xs, pw, bias, out_dtype=other), *_product(rows8.codes, rows8.scales, pw, bias, other))


@gpu
@pytest.mark.parametrize("rows,N,K", [(1, 11008, 4096), (3, 32003, 2048), (48, 8192, 8192), (1, 256, 131071), (300, 130, 131040), (2048, 4096, 1024),
                                      (4097, 1000, 784), (1111, 2304, 3333), (9000, 640, 384), (3000, 9001, 640)])
def test_linear_of_larger_sizes(rows, N, K):
    pw = _weight(N, K)
    x = torch.randn(rows, K, device=DEV, generator=torch.Generator(DEV).manual_seed(N)).bfloat16()
    rows8 = ops.quantize_rows(x)
    y = ops.linear(x, pw)
    _near(y, *_product(rows8.codes, rows8.scales, pw, None, torch.bfloat16))
    some = torch.tensor([0, rows - 1, rows // 2, rows // 3], device=DEV)         # a row's result does not depend on the rows beside it
    assert torch.equal(ops.linear(x[some], pw), y[some])
    assert ops.check_status() == 0


@gpu
@pytest.mark.parametrize("rows,N,K", [(1, 4096, 4096), (1, 130, 65536), (2, 200, 32768), (3, 11008, 4096), (5, 40000, 1024), (8, 300, 8192), (16, 1000, 4096),
                                      (16, 70, 4104), (7, 64, 104), (4, 3000, 8)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_few_tokens(rows, N, K, dtype):
    """Values and rows of codes give the same bits; a row that is not finite, or nothing but zeros, stays by itself."""
    pw = _weight(N, K)
    x = torch.randn(rows, K, device=DEV, generator=torch.Generator(DEV).manual_seed(K)).to(dtype)
    x[:, ::7] *= 5
    bias = torch.randn(N, device=DEV)
    x[-1] *= 1e-3
    rows8 = ops.quantize_rows(x)
    y = ops.linear(x, pw, bias)
    _near(y, *_product(rows8.codes, rows8.scales, pw, bias, dtype))
    assert torch.equal(y, ops.linear(rows8, pw, bias))
    x[0, K // 2] = torch.nan
    if rows > 1:
        x[1] = 0
    again = ops.linear(x, pw, bias)
    assert torch.isnan(again[0]).all() and torch.equal(again[2:], y[2:]) and (rows == 1 or torch.equal(again[1], bias.to(dtype)))
    assert ops.check_status() == 0


@gpu
def test_largest_sums_do_not_overflow():
    """Codes of -128 (which no row of quantize_rows has) at the longest row: 2^31 - 2^14, still exact."""
    K = _lib.JQ_INT8_MAX_K
    q = torch.full((3, (K + 31) // 32 * 32), -128, dtype=torch.int8, device=DEV)
    pw = jq.PackedWeight(jq.QuantSpec("int8", 0, 0), 3, K, q, torch.ones(3, device=DEV), None)
    y = ops.linear(ops.QuantizedRows(q[:, :K], torch.ones(3, device=DEV), torch.float32), pw)
    assert bool((y == float(16384 * K)).all())                     # 2^31 - 2^14: a number of fp32


@gpu
@pytest.mark.parametrize("rows", [1, 40, 400])
def test_extreme_scales(rows):
    """Neither product of the scales leaves fp32's range before the result does."""
    x = torch.randn(rows, 256, device=DEV)
    x[0] *= 1e36
    w = torch.randn(64, 256, device=DEV)
    w[:32] *= 1e-25
    w[32:] *= 1e-36
    pw = jq.pack_weight(w, jq.QuantSpec("int8", 0, 0))
    rows8 = ops.quantize_rows(x)
    y, bound = _product(rows8.codes, rows8.scales, pw, None, torch.float32)
    _near(ops.linear(x, pw), y, bound + 2.0 ** -149 * 2)           # (a subnormal product and result are off by half of 2^-149 each)


@gpu
@pytest.mark.parametrize("rows", [1, 20, 300])
def test_rotated_linear_undoes_the_weights_rotation(rows):
    """W x = (W H)(H x): against the unquantised product, off by the rounding of both operands: half a step of 1/127 of a row's largest
    value (about 4 times the typical one) each, independent over K: (4 / 127 / sqrt(12)) sqrt(2) = 0.013 of the result's size."""
    K, N = 512, 96
    w = torch.randn(N, K, device=DEV, generator=torch.Generator(DEV).manual_seed(1))
    x = torch.randn(rows, K, device=DEV, generator=torch.Generator(DEV).manual_seed(2))
    pw = jq.pack_weight(w, jq.QuantSpec("int8", 0, 128))
    y = ops.linear(x, pw)
    want = x.double() @ w.double().T
    assert ((y - want).norm() / want.norm()).item() < 0.02
    rows8 = ops.quantize_rows(x, 128)
    _near(y, *_product(rows8.codes, rows8.scales, pw, None, torch.float32))


@gpu
@pytest.mark.parametrize("rows", [1, 33, 300])
def test_rotated_linear_of_values_anywhere(rows):
    """A contiguous activation that does not begin at a 16-byte boundary."""
    pw = _weight(72, 256, had=128)
    flat = torch.randn(rows * 256 + 1, device=DEV).bfloat16()
    x = flat[1:].view(rows, 256)
    assert torch.equal(ops.linear(x, pw), ops.linear(x.clone(), pw)) and torch.equal(ops.linear(x, _weight(72, 256)), ops.linear(x.clone(), _weight(72, 256)))


@gpu
def test_captured_before_any_other_call():
    """A thread and stream that have no scratch buffer yet: the captured calls' own outlast them."""
    import threading
    pw = _weight(200, 384)
    x = torch.randn(300, 384, device=DEV)
    rows8, found = ops.quantize_rows(x), []
    want = ops.linear(x, pw)
    torch.cuda.synchronize()

    def work():
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                a, b = ops.linear(x, pw), ops.linear(rows8, pw)
            more = ops.linear(x[:3], pw)
            for _ in range(2):
                a.zero_()
                b.zero_()
                graph.replay()
            stream.synchronize()
            found.extend([a.clone(), b.clone(), more.clone(), ops.check_status(raise_on_error=False)])

    t = threading.Thread(target=work)
    t.start()
    t.join()
    assert torch.equal(found[0], want) and torch.equal(found[1], want) and torch.equal(found[2], want[:3]) and found[3] == 0


@gpu
def test_rows_of_codes_that_lie_otherwise():
    pw = _weight(70, 200)
    x = torch.randn(4, 6, 200, device=DEV)
    rows8 = ops.quantize_rows(x)
    want = ops.linear(x, pw)
    assert want.shape == (4, 6, 70) and torch.equal(ops.linear(rows8, pw), want)
    tight = rows8.codes.contiguous()                               # rows 200 bytes apart: not a multiple of 16
    assert torch.equal(ops.linear(ops.QuantizedRows(tight, rows8.scales, torch.float32), pw), want)
    turned = rows8.codes.transpose(0, 1), rows8.scales.transpose(0, 1)
    assert torch.equal(ops.linear(ops.QuantizedRows(*turned, torch.float32), pw), want.transpose(0, 1))
    shifted = torch.empty(24 * 224 + 1, dtype=torch.int8, device=DEV)[1:].view(24, 224)[:, :200]
    shifted.copy_(rows8.codes.reshape(24, 200))
    assert torch.equal(ops.linear(ops.QuantizedRows(shifted, rows8.scales.reshape(24), torch.float32), pw), want.reshape(24, 70))
    one = ops.QuantizedRows(rows8.codes[:1, :1].expand(3, 1, 200), rows8.scales[:1, :1].expand(3, 1), torch.float32)
    assert torch.equal(ops.linear(one, pw), want[:1, :1].expand(3, 1, 70))
    assert torch.equal(one.dequantize(), rows8.dequantize()[:1, :1].expand(3, 1, 200))
    assert ops.linear(ops.quantize_rows(x[:0]), pw).shape == (0, 6, 70) and ops.linear(x[:0], pw).shape == (0, 6, 70)
    assert ops.linear(x[0, 0], pw).shape == (70,) and torch.equal(ops.linear(rows8, pw, out_dtype=torch.bfloat16), want.bfloat16())


@gpu
@pytest.mark.parametrize("rows", [1, 40, 500])
def test_streams_graphs_and_calls_behind_one_another(rows):
    pw, small = _weight(512, 640), _weight(64, 512, 3)
    x = torch.randn(rows, 640, device=DEV).bfloat16()
    want = ops.linear(ops.linear(x, pw), small)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(ops.linear(ops.linear(x, pw), small), want)
        rows8 = ops.quantize_rows(x)
        ops.linear(rows8, pw)
    torch.cuda.current_stream().wait_stream(side)
    held, graphs = x.clone(), []
    for _ in range(2):                                             # two graphs captured one after the other, replayed on two streams
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = ops.linear(ops.linear(held, pw), small)
            z = ops.linear(ops.quantize_rows(held), pw)
        graphs.append((graph, y, z))
    other = torch.randn(rows, 640, device=DEV).bfloat16()
    held.copy_(other)
    want, first = ops.linear(ops.linear(other, pw), small), ops.linear(other, pw)
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
    torch.cuda.synchronize()
    for _, y, z in graphs:
        assert torch.equal(y, want) and torch.equal(z, first)
    assert ops.check_status() == 0


@gpu
def test_memory_behind_and_beside_the_output_is_left_alone():
    lib = _lib.load()
    for rows, N in ((1, 7), (17, 130), (300, 257)):
        pw = _weight(N, 100)
        rows8 = ops.quantize_rows(torch.randn(rows, 100, device=DEV))
        y = torch.full((rows * N + 64,), 7.0, device=DEV)
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        assert lib.jq_int8_matmul(pw.qweight.data_ptr(), pw.scales.data_ptr(), rows8.codes.data_ptr(), rows8.codes.stride(0), rows8.scales.data_ptr(), None,
                                  y[32:].data_ptr(), N, 100, rows, 0, status.data_ptr(), None) == 0
        assert bool((y[:32] == 7).all()) and bool((y[32 + rows * N:] == 7).all()) and status.item() == 0
        assert torch.equal(y[32:32 + rows * N].view(rows, N), ops.linear(rows8, pw))


# ---------------------------------------------------------------------------------------------------- layers and packing

def test_packing_on_the_cpu():
    w = torch.randn(5, 50)
    w[0] = 0
    w[1, ::2] = 0
    w[2, 3] = torch.nan
    pw = jq.pack_weight(w, jq.QuantSpec("int8", 0))
    q, s = _codes(w)
    assert pw.qweight.dtype == torch.int8 and pw.qweight.shape == (5, 64) and pw.codebook is None
    assert torch.equal(pw.qweight[:, :50], q) and _same(pw.scales, s) and bool((pw.qweight[:, 50:] == 0).all())
    assert bool((pw.qweight[1, :50:2] == 0).all()) and pw.nbytes() == 5 * 64 + 20
    part = pw.rows(1, 3)
    assert torch.equal(part.qweight, pw.qweight[1:3]) and part.N == 2
    assert jq.algorithmic_bytes(jq.QuantSpec("int8", 0), 10, 100, 2, 2, 2) == 1000 + 40 + 400 + 40


def test_refusals_of_specs_and_layers():
    with pytest.raises(ValueError, match="group_size"):
        jq.QuantSpec("int8", 32)
    with pytest.raises(ValueError, match="bitwidth"):
        jq.JenksQuantLinear(nn.Linear(64, 8), 4, fmt="int8")
    with pytest.raises(ValueError, match="bitwidth"):
        jq.JenksQuantLinear(nn.Linear(64, 8), 8)
    with pytest.raises(ValueError, match="bitwidth"):
        jq.JenksQuantConv2d(nn.Conv2d(3, 8, 3), 4, fmt="int8")
    with pytest.raises(ValueError, match="rotation block"):
        jq.pack_weight(torch.randn(4, 100), jq.QuantSpec("int8", 0, 128))
    with pytest.raises(ValueError, match="1 to 131071"):
        jq.pack_weight(torch.empty(1, 131072), jq.QuantSpec("int8", 0))
    pw = jq.pack_weight(torch.randn(4, 100), jq.QuantSpec("int8", 0))
    with pytest.raises(ValueError, match="4-bit"):
        ops.GroupedGemv([pw], 1)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.linear(torch.randn(2, 100), pw)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.quantize_rows(torch.randn(2, 100))
    with pytest.raises(RuntimeError, match="128"):
        ops.quantize_rows(torch.randn(2, 100), 128)
    with pytest.raises(RuntimeError, match="rows of 1"):
        ops.quantize_rows(torch.randn(2, 0))
    with pytest.raises(RuntimeError, match="dtype"):
        ops.quantize_rows(torch.randn(2, 8).double())
    with pytest.raises(RuntimeError, match="unfold|laid out"):
        ops.conv2d(torch.randn(1, 4, 9, 9), jq.pack_weight(torch.randn(4, 36), jq.QuantSpec("int8", 0)), None, (3, 3), (1, 1), (0, 0), (1, 1))


def test_refusals_of_the_library():
    """Bad arguments are turned away before anything is launched; no GPU is needed."""
    lib, p = _lib.load(), torch.zeros(4096, dtype=torch.uint8).data_ptr()
    assert lib.jq_quantize_rows(None, 8, 1, 8, 0, 0, p, 32, p, None) == -1
    for rows, K, had, stride in ((0, 8, 0, 32), (1, 0, 0, 32), (1, 131072, 0, 131072), (1, 100, 128, 128), (1, 128, 64, 128), (1, 40, 0, 32)):
        assert lib.jq_quantize_rows(p, K, rows, K, had, 0, p, stride, p, None) == -2
    assert lib.jq_quantize_rows(p, 8, 1, 8, 0, 3, p, 32, p, None) == -4
    assert lib.jq_quantize_rows(p, 8, 1, 8, 0, 0, p + 8, 32, p, None) == -3 and lib.jq_quantize_rows(p, 8, 1, 8, 0, 0, p, 24, p, None) == -3
    assert lib.jq_quantize_rows(p + 4, 128, 1, 128, 128, 0, p, 128, p, None) == -3 and lib.jq_quantize_rows(p, 130, 2, 128, 128, 0, p, 128, p, None) == -3
    assert lib.jq_dequantize_rows(p, 24, p, 1, 8, p, 0, None) == -3 and lib.jq_dequantize_rows(p, 32, p, 1, 8, p, 5, None) == -4
    assert lib.jq_int8_scratch_bytes(3, 100) == 256 + 3 * 128 and lib.jq_int8_scratch_bytes(0, 4) == 0
    assert lib.jq_int8_linear(p, p, p, None, p, 4, 8, 1, 0, 0, 0, p, 8, p, None) == -6
    assert lib.jq_int8_linear(p, p, None, None, p, 4, 8, 1, 0, 0, 0, p, 4096, p, None) == -1
    assert lib.jq_int8_linear(p, p, p, None, p, 4, 131072, 1, 0, 0, 0, p, 4096, p, None) == -2
    assert lib.jq_int8_linear(p + 8, p, p, None, p, 4, 8, 1, 0, 0, 0, p, 4096, p, None) == -3
    assert lib.jq_int8_matmul(p, p, p, 24, p, None, p, 4, 8, 1, 0, p, None) == -3
    assert lib.jq_int8_matmul(p, p, p, 32, p, None, p + 1, 4, 8, 1, 1, p, None) == -3
    assert lib.jq_int8_matmul(p, p, p, 32, p, None, p, 4, 8, 1, 9, p, None) == -4
    assert lib.jq_int8_matmul(p, p, p, 0, p, None, p, 4, 8, 1, 0, p, None) == -2
    assert lib.jq_int8_matmul(p, p, p, 32, p, None, p, 4, 8, 1, 0, None, None) == -1


@gpu
def test_refusals_of_rows_and_weights():
    pw, rot = _weight(8, 128), _weight(8, 128, had=128)
    x = torch.randn(2, 128, device=DEV)
    rows8 = ops.quantize_rows(x)
    four = jq.pack_weight(torch.randn(8, 128), jq.QuantSpec("gf4", 128)).to(DEV)
    for call, text in ((lambda: ops.linear(rows8, rot), "had_block"), (lambda: ops.linear(ops.quantize_rows(x, 128), pw), "had_block"),
                       (lambda: ops.linear(rows8, four), "gf4"), (lambda: ops.linear(rows8, _weight(8, 64)), "K=64"),
                       (lambda: ops.linear(rows8, pw, out_dtype=torch.float64), "dtype"),
                       (lambda: ops.linear(x, pw, torch.zeros(9, device=DEV)), "bias"), (lambda: ops.linear(x, pw, torch.zeros(8)), "CUDA"),
                       (lambda: ops.linear(rows8._replace(scales=rows8.scales[:1]), pw), "scales"),
                       (lambda: ops.linear(rows8._replace(codes=rows8.codes.float()), pw), "int8"),
                       (lambda: ops.linear(x, jq.PackedWeight(pw.spec, 8, 128, pw.qweight.float(), pw.scales, None)), "int8 weight"),
                       (lambda: ops.linear(x, jq.PackedWeight(pw.spec, 8, 100, pw.qweight, pw.scales, None)), "K=100"),
                       (lambda: ops.linear(x, jq.PackedWeight(pw.spec, 8, 128, pw.qweight, pw.scales.half(), None)), "fp32 scales"),
                       (lambda: rows8.dequantize(torch.float64), "dtype"), (lambda: ops.linear(x.double(), pw), "dtype")):
        with pytest.raises(RuntimeError, match=text):
            call()


@gpu
@pytest.mark.parametrize("had", [0, 128])
def test_packing_on_the_gpu_is_that_on_the_cpu(had):
    w = torch.randn(37, 1152) * 0.1
    a, b = jq.pack_weight(w, jq.QuantSpec("int8", 0, had)), jq.pack_weight(w.to(DEV), jq.QuantSpec("int8", 0, had))
    assert torch.equal(a.qweight, b.qweight.cpu()) and torch.equal(a.scales, b.scales.cpu())
    dense = ops.dequantize(b)
    assert torch.equal(dense.cpu(), a.qweight[:, :1152].float() * a.scales[:, None])


@gpu
def test_layers_checkpoints_and_copies():
    model = nn.Sequential(nn.Flatten(), nn.Linear(784, 300), nn.ReLU(), nn.Linear(300, 100), nn.ReLU(), nn.Linear(100, 10))
    q = jq.quantize_module(model, 8, fmt="int8").to(DEV)
    x = torch.randn(33, 1, 28, 28, device=DEV)

    def plain(h, layers):
        for m in layers:
            if isinstance(m, jq.JenksQuantLinear):
                q8, s = _codes(h)
                h = (q8.to(DEV).float() * s.to(DEV)[:, None]).double() @ m.weight.double().T + m.bias.double()
                h = h.float()
            else:
                h = m(h)
        return h

    y = q(x)
    # fp32 between the layers: a hidden value off by 2^-22 may cross the border of two codes, a step of 1/127 of the largest in one of 100
    assert ((y - plain(x, q)).abs().max() / y.abs().max()).item() < 0.02
    for m in q:
        if isinstance(m, jq.JenksQuantLinear):
            m.commit()
    assert torch.equal(q(x), y) and torch.equal(copy.deepcopy(q)(x), y)
    state = checkpoint.pack_state_dict(model.state_dict(), jq.QuantSpec("int8", 0))
    buf = io.BytesIO()
    torch.save(state, buf)
    buf.seek(0)
    loaded = checkpoint.load_packed_into(copy.deepcopy(model), torch.load(buf)).to(DEV)
    assert torch.equal(loaded(x), y) and loaded[1].spec == jq.QuantSpec("int8", 0, 0)
    with warnings.catch_warnings(record=True) as told:
        warnings.simplefilter("always")
        state = checkpoint.pack_state_dict(model.state_dict(), jq.QuantSpec("int8", 0, 128))
    assert len(told) == 3 and checkpoint.packed_weight_from(state, "1").spec == jq.QuantSpec("int8", 0, 0)


@gpu
def test_convolution_and_traced_call():
    conv = nn.Conv2d(6, 20, 3, stride=2, padding=1)
    q = jq.JenksQuantConv2d(conv, 8, fmt="int8").to(DEV)
    x = torch.randn(5, 6, 21, 17, device=DEV)
    y = q(x)
    fields = F.unfold(x, 3, 1, 1, 2).transpose(1, 2)
    q8, s = _codes(fields.reshape(-1, 54))
    want, bound = _product(q8.to(DEV), s.to(DEV), q.packed, q.bias, torch.float32)
    _near(y.flatten(2).transpose(1, 2).reshape(-1, 20), want, bound)
    pw = _weight(48, 256)
    z = torch.randn(7, 256, device=DEV)
    assert torch.equal(torch.ops.jq.linear(z, pw.qweight, pw.scales, None, None, pw.spec.fmt_id, 48, 256, 0, 0, -1), ops.linear(z, pw))


@gpu
def test_the_example_decoder_with_int8_weights():
    """Its log probabilities stand within 0.2 of a plain decoder's with the same dequantised weights and unquantised activations, keys and
    values: a row's codes are off by half a step of 1/127 of its largest value (four times the typical one), 0.9 % of a product's size;
    some ten products, with bf16 between them, move logits of spread 0.6 by a few hundredths, as 8-bit keys and values do."""
    import os
    import sys
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    import decode
    from test_example_decode import _plain_logits
    torch.manual_seed(0)
    model = decode.packed(decode.Decoder(2, 512, 8, 2, 1024, 1000), "int8")
    assert model.layers[0].q.spec.fmt == "int8" and model.layers[0].q._parameters["weight"] is None
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 1000, (n,), generator=gen).tolist() for n in (5, 170, 1)]
    answers, scored, logprobs, _ = decode.generate(model, prompts, 4, block_size=32)
    at = 0
    for i, p in enumerate(prompts):
        full = torch.tensor(p + answers[i].tolist(), device=DEV)
        lp = torch.log_softmax(_plain_logits(model, full), -1)
        want = lp[:-1].gather(1, full[1:, None])[:, 0]
        assert len(p) == 1 or (scored[at:at + len(p) - 1] - want[:len(p) - 1]).abs().max().item() < 0.2
        at += len(p)
        assert (logprobs[i, :, 0] - want[len(p) - 1:]).abs().max().item() < 0.2


# ------------------------------------------------------------------------------------------- rotations that leave fp32's range

def _overflowing(rows, K, dtype):
    """Rows of which some have a NaN or an infinity, and some leave fp32's range only within the rotation."""
    x = torch.randn(rows, K, device=DEV, generator=torch.Generator(DEV).manual_seed(K)).to(dtype)
    top = min(torch.finfo(dtype).max, 3e38)
    signs = torch.tensor([1, -1, 1, -1, 1, -1, -1, 1], device=DEV, dtype=torch.float32)
    x[0] = 0
    x[0, :8] = (top * signs).to(dtype)                              # odd places end as NaN, even ones as 0, none as an infinity
    x[1] = (top * signs).to(dtype).repeat(K // 8)
    x[2, K // 2] = torch.nan
    x[3, K - 1] = torch.inf
    x[4, 0], x[4, 1] = torch.inf, -torch.inf
    x[5] = top
    x[6] = 0
    x[6, K - 8:] = (top * signs).to(dtype)                          # the last block only
    x[7, ::2] = -top
    return x


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,K", [(8, 128), (400, 256), (400, 512), (8, 1024), (400, 1024), (9, 4096), (400, 4096), (8, 16384), (400, 16384), (8, 33024)])
def test_rotated_rows_that_go_wrong(rows, K, dtype):
    """What the rotation makes of a row decides: a NaN or an infinity among its values, also one that only the rotation's sums make of
    finite values, gives the scale NaN and codes 0, and the product's row is NaN."""
    x = _overflowing(rows, K, dtype)
    got = ops.quantize_rows(x, 128)
    q, s = _codes(ops.fwht_block(x, 128))
    assert _same(got.scales.cpu(), s) and torch.equal(got.codes.cpu(), q)
    lost = [2, 3, 4] if dtype == torch.float16 else [0, 1, 2, 3, 4, 5, 6, 7]
    assert torch.isnan(got.scales[lost]).all() and torch.isfinite(got.scales[8:]).all()
    if K <= 4096:
        y = ops.linear(x, _weight(40, K, had=128))
        assert torch.isnan(y[lost]).all() and torch.isfinite(y[8:]).all()


@gpu
@pytest.mark.parametrize("K", [128, 1024])
def test_rotated_weights_that_go_wrong_are_packed_as_on_the_cpu(K):
    w = _overflowing(12, K, torch.float32)
    spec = jq.QuantSpec("int8", 0, 128)
    a, b = jq.pack_weight(w.cpu(), spec), jq.pack_weight(w, spec)
    assert _same(a.scales, b.scales.cpu()) and torch.equal(a.qweight, b.qweight.cpu()) and torch.isnan(a.scales[:8]).all()


# A kernel that lets what is behind it start at once and ends `ns` nanoseconds later, or after 4 million pauses
_PAUSE = b"""
.version 8.0
.target sm_90
.address_size 64
.visible .entry pause(.param .u64 ns) {
    .reg .u64 want, begin, now;
    .reg .u32 i;
    .reg .pred p;
    ld.param.u64 want, [ns];
    griddepcontrol.launch_dependents;
    mov.u64 begin, %globaltimer;
    mov.u32 i, 0;
again:
    nanosleep.u32 1000;
    mov.u64 now, %globaltimer;
    sub.u64 now, now, begin;
    setp.ge.u64 p, now, want;
    @p bra done;
    add.u32 i, i, 1;
    setp.lt.u32 p, i, 4000000;
    @p bra again;
done:
    ret;
}
"""


@gpu
@pytest.mark.parametrize("rows,N,K", [(1, 256, 4096), (40, 300, 256), (256, 4096, 4096), (300, 512, 16384), (2000, 1000, 512)])
def test_products_behind_a_kernel_that_lasts(rows, N, K):
    """A product that starts while the kernel in front of it runs on for a second: its bounded waits (a quarter of a second) begin behind
    that kernel, in the forms that share K too (4096 x 4096 of 256 rows)."""
    import ctypes
    pw = _weight(N, K)
    rows8 = ops.quantize_rows(torch.randn(rows, K, device=DEV))
    want = ops.linear(rows8, pw)
    cuda, module, entry = ctypes.CDLL("libcuda.so.1"), ctypes.c_void_p(), ctypes.c_void_p()
    assert cuda.cuModuleLoadData(ctypes.byref(module), ctypes.c_char_p(_PAUSE)) == 0
    try:
        assert cuda.cuModuleGetFunction(ctypes.byref(entry), module, b"pause") == 0
        ns = ctypes.c_uint64(10 ** 9)
        args = (ctypes.c_void_p * 1)(ctypes.cast(ctypes.byref(ns), ctypes.c_void_p))
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert cuda.cuLaunchKernel(entry, 1, 1, 1, 32, 1, 1, 0, stream, args, None) == 0
        y = ops.linear(rows8, pw)
        torch.cuda.synchronize()
        assert ops.check_status(raise_on_error=False) == 0 and torch.equal(y, want)
    finally:
        cuda.cuModuleUnload(module)


@gpu
@pytest.mark.parametrize("rows,N,K", [(1, 64, 256), (40, 64, 256), (400, 64, 256), (300, 4096, 4096), (2000, 2001, 256), (3000, 4096, 384)])
def test_scales_whose_product_with_the_sum_leaves_the_range(rows, N, K):
    """Channels so large that the sum times their scale is no number of fp32, tokens so small that the result is one.  Such channels
    have one rounding more than others, the third of 2^-24 that the bound counts."""
    gen = torch.Generator(DEV).manual_seed(N)
    x = torch.randn(rows, K, device=DEV, generator=gen) * 1e-28
    x[rows // 2] *= 1e-20                                           # below the least scale: codes 0
    w = torch.randn(N, K, device=DEV, generator=gen)
    w[::3] *= 1e36
    w[1::3] *= 1e25
    w[-1] = 3e38
    bias = torch.randn(N, device=DEV, generator=gen)
    pw = jq.pack_weight(w, jq.QuantSpec("int8", 0, 0))
    rows8 = ops.quantize_rows(x)
    for b in (None, bias):
        y, bound = _product(rows8.codes, rows8.scales, pw, b, torch.float32)
        assert y.abs().max().item() < 1e38
        _near(ops.linear(rows8, pw, b), y, bound)
    w[2], w[5] = torch.nan, torch.inf
    rows8.scales[rows // 2] = torch.nan
    pw = jq.pack_weight(w, jq.QuantSpec("int8", 0, 0))
    y = ops.linear(rows8, pw)
    good = torch.ones(N, dtype=torch.bool, device=DEV)
    good[[2, 5]] = False
    assert torch.isnan(y[:, [2, 5]]).all() and torch.isnan(y[rows // 2]).all() and torch.isfinite(y[:rows // 2][:, good]).all()


def test_arrays_off_their_elements_boundary_are_refused():
    """Scales, biases, outputs and status words that a kernel would access at a misaligned address; no GPU is needed."""
    lib, p = _lib.load(), torch.zeros(8192, dtype=torch.uint8).data_ptr()
    assert p % 16 == 0
    for dtype, off in ((0, 1), (0, 2), (1, 1), (2, 1)):
        assert lib.jq_quantize_rows(p + off, 8, 1, 8, 0, dtype, p, 32, p, None) == -3
        assert lib.jq_dequantize_rows(p, 32, p, 1, 8, p + off, dtype, None) == -3
        assert lib.jq_int8_linear(p, p, p + off, None, p, 4, 8, 1, 0, dtype, 0, p, 4096, p, None) == -3
        assert lib.jq_int8_matmul(p, p, p, 32, p, None, p + off, 4, 8, 1, dtype, p, None) == -3
    for off in (1, 2, 3):
        assert lib.jq_quantize_rows(p, 8, 1, 8, 0, 0, p, 32, p + off, None) == -3 and lib.jq_dequantize_rows(p, 32, p + off, 1, 8, p, 0, None) == -3
        for at in range(4):                                        # the channels' scales, the rows', the bias, the status word
            cs, ts, bias, status = (p + off if i == at else p for i in range(4))
            assert lib.jq_int8_matmul(p, cs, p, 32, ts, bias, p, 4, 8, 1, 0, status, None) == -3
            assert at == 1 or lib.jq_int8_linear(p, cs, p, bias, p, 4, 8, 1, 0, 0, 0, p, 4096, status, None) == -3


def test_sizes_that_leave_32_bits_are_refused():
    """Rows whose count the kernels' arithmetic could not hold, and rows of codes longer than the format has; no GPU is needed."""
    lib, p = _lib.load(), torch.zeros(4096, dtype=torch.uint8).data_ptr()
    for rows in (_lib.JQ_INT8_MAX_ROWS + 1, 2 ** 31 - 1):
        assert lib.jq_quantize_rows(p, 0, rows, 8, 0, 0, p, 32, p, None) == -2 and lib.jq_dequantize_rows(p, 32, p, rows, 8, p, 0, None) == -2
        assert lib.jq_int8_matmul(p, p, p, 32, p, None, p, 4, 8, rows, 0, p, None) == -2
        assert lib.jq_int8_linear(p, p, p, None, p, 4, 8, rows, 0, 0, 0, p, 1 << 60, p, None) == -2
        with pytest.raises(RuntimeError, match="32 bits"):
            ops._rows_of(torch.zeros(1, 8).expand(rows, 8), 8, "x")
    for K in (_lib.JQ_INT8_MAX_K + 1, 2 ** 31 - 1):
        assert lib.jq_dequantize_rows(p, 1 << 32, p, 1, K, p, 0, None) == -2 and lib.jq_int8_scratch_bytes(1, K) == 0


# Rows, N and K of two products for each form that the rule may take: (pair, tile, split) -> odd N, and rows of y of 16 bytes
FORMS = {
    (0, 16, 1): ((2, 133, 205), (2, 132, 202)), (0, 16, 2): ((2, 6285, 657), (3, 6300, 668)), (0, 16, 3): ((3, 131, 513), (4, 132, 520)),
    (0, 16, 4): ((3, 133, 391), (4, 132, 394)), (0, 16, 8): ((2, 131, 915), (3, 132, 911)), (0, 32, 1): ((19, 137, 212), (17, 132, 206)),
    (0, 32, 2): ((397, 385, 1219), (398, 400, 1229)), (0, 32, 3): ((134, 402, 1035), (294, 160, 1025)), (0, 32, 4): ((17, 131, 777), (19, 136, 774)),
    (0, 32, 8): ((17, 131, 936), (21, 132, 921)), (0, 64, 1): ((34, 666, 905), (33, 584, 1060)), (0, 64, 2): ((521, 649, 3212), (511, 780, 3315)),
    (0, 64, 3): ((449, 522, 2230), (258, 948, 2191)), (0, 64, 4): ((270, 398, 1806), (264, 396, 1863)), (0, 64, 8): ((34, 393, 1572), (33, 376, 1631)),
    (0, 128, 1): ((71, 18998, 205), (65, 20332, 203)), (0, 128, 2): ((85, 8439, 14591), (120, 8516, 14510)), (0, 128, 3): ((75, 4838, 7733), (85, 4868, 7903)),
    (0, 128, 4): ((342, 1033, 16203), (265, 1164, 17033)), (0, 128, 8): ((265, 389, 21122), (210, 560, 21015)), (1, 128, 1): ((68, 666, 904), (69, 488, 1245)),
    (1, 128, 2): ((331, 1033, 3592), (275, 1180, 3402)), (1, 256, 1): ((10016, 131, 209), (196, 9600, 205)), (1, 256, 2): ((520, 1398, 15160), (332, 2068, 14862)),
    (1, 256, 4): ((442, 1182, 17757), (390, 1308, 17729))}


def _form(N, K, rows):
    import ctypes
    found = [ctypes.c_int() for _ in range(3)]
    assert _lib.load().jq_int8_form(N, K, rows, *(ctypes.byref(v) for v in found)) == 0
    return tuple(v.value for v in found)


def test_the_products_below_reach_every_form():
    """On a device of 148 SMs, as where there is none; the kernels, tiles and splits are all that the rule can choose from."""
    if torch.cuda.is_available() and torch.cuda.get_device_properties(0).multi_processor_count != 148:
        pytest.skip("another number of SMs")
    every = {(0, tile, split) for tile in (16, 32, 64, 128) for split in (1, 2, 3, 4, 8)} | {(1, 128, 1), (1, 128, 2), (1, 256, 1), (1, 256, 2), (1, 256, 4)}
    assert set(FORMS) == every
    for form, cases in FORMS.items():
        assert [_form(N, K, rows) for rows, N, K in cases] == [form, form]
    for bad in ((0, 8, 1), (8, 0, 1), (8, 8, 0), (8, _lib.JQ_INT8_MAX_K + 1, 1), (8, 8, _lib.JQ_INT8_MAX_ROWS + 1), ((1 << 28) + 1, 8, 1)):
        with pytest.raises(AssertionError):
            _form(*bad)
    assert _lib.load().jq_int8_form(8, 8, 1, None, None, None) == -1


@gpu
@pytest.mark.parametrize("form", sorted(FORMS))
def test_every_form_against_64_bits(form):
    for i, (rows, N, K) in enumerate(FORMS[form]):
        gen = torch.Generator(DEV).manual_seed(N + K)
        pw = _weight(N, K)
        x = torch.randn(rows, K, device=DEV, generator=gen) * (torch.rand(rows, 1, device=DEV, generator=gen) + 0.1)
        bias = torch.randn(N, device=DEV, generator=gen)
        for dtype in DTYPES:
            xs, b = x.to(dtype), bias if (i == 0) == (dtype == torch.bfloat16) else None
            rows8 = ops.quantize_rows(xs)
            y = ops.linear(xs, pw, b)
            _near(y, *_product(rows8.codes, rows8.scales, pw, b, dtype))
            assert torch.equal(ops.linear(rows8, pw, b), y)
        # captured, replayed on another stream; and into memory whose surroundings stay as they are
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph):
            again, direct = ops.linear(xs, pw, b), ops.linear(rows8, pw, b)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph.replay()
        side.synchronize()
        assert torch.equal(again, y) and torch.equal(direct, y)
        room = torch.full((rows * N + 64,), 7.0, dtype=dtype, device=DEV)
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        assert _lib.load().jq_int8_matmul(pw.qweight.data_ptr(), pw.scales.data_ptr(), rows8.codes.data_ptr(), rows8.codes.stride(0), rows8.scales.data_ptr(),
                                          ops._addr(b), room[32:].data_ptr(), N, K, rows, _lib.JQ_BF16, status.data_ptr(), None) == 0
        assert bool((room[:32] == 7).all()) and bool((room[32 + rows * N:] == 7).all()) and status.item() == 0
        assert torch.equal(room[32:32 + rows * N].view(rows, N), y)
    assert ops.check_status(raise_on_error=False) == 0


@gpu
@pytest.mark.parametrize("had", [0, 128])
@pytest.mark.parametrize("dtype,out", [(torch.bfloat16, None), (torch.float32, None), (torch.float16, torch.float32), (torch.float32, torch.bfloat16)])
def test_activations_in_parts(monkeypatch, had, dtype, out):
    """Rows beyond what a call's scratch holds go in parts of a multiple of 256, each into its own rows of the output."""
    pw = _weight(130, 384, had=had)
    x, bias = torch.randn(700, 384, device=DEV).to(dtype), torch.randn(130, device=DEV)
    want = ops.linear(x, pw, bias, out_dtype=out)
    calls, linear = [], _lib.load().jq_int8_linear
    monkeypatch.setattr(_lib.load(), "jq_int8_linear", lambda *a: calls.append(a[7]) or linear(*a))
    monkeypatch.setattr(ops, "MAX_ROWS_SCRATCH", 300 * 384)
    graph = torch.cuda.CUDAGraph()
    for leading in ((700,), (7, 100)):
        assert torch.equal(ops.linear(x.view(*leading, 384), pw, bias, out_dtype=out), want.view(*leading, 130))
    with torch.cuda.graph(graph):
        y = ops.linear(x, pw, bias, out_dtype=out)
    assert calls == [256, 256, 188] * 3
    other = torch.randn(700, 384, device=DEV).to(dtype)
    x.copy_(other)
    for _ in range(2):
        y.zero_()
        graph.replay()
    monkeypatch.undo()
    assert torch.equal(y, ops.linear(other, pw, bias, out_dtype=out)) and ops.check_status(raise_on_error=False) == 0


@gpu
def test_rows_sharded_over_ranks():
    """A world of one, and the slices that two ranks would have, side by side."""
    import torch.distributed as dist
    from if_i_could_turn_back_time_b200 import dist as sharded
    pw, x, bias = _weight(96, 200), torch.randn(5, 200, device=DEV), torch.randn(96)
    want = ops.linear(x, pw, bias.to(DEV))
    two = [sharded.shard_rows(pw, rank, 2) for rank in range(2)]
    assert torch.equal(torch.cat([ops.linear(x, part, bias[48 * i:48 * i + 48].to(DEV)) for i, part in enumerate(two)], -1), want)
    dist.init_process_group("gloo", store=dist.HashStore(), rank=0, world_size=1)
    try:
        layer = sharded.RowShardedLinear(jq.PackedWeight(pw.spec, 96, 200, pw.qweight.cpu(), pw.scales.cpu(), None), bias, device=DEV)
        assert torch.equal(layer(x), want)
    finally:
        dist.destroy_process_group()


@gpu
def test_linear_under_torch_compile():
    """One opaque operation in the traced graph, the same bits."""
    pw, x, bias = _weight(72, 200), torch.randn(3, 5, 200, device=DEV).bfloat16(), torch.randn(72, device=DEV)
    traced = []

    def backend(graph, _):
        traced.append([str(n.target) for n in graph.graph.nodes if n.op == "call_function"])
        return graph.forward

    for out in (None, torch.float32):
        call = torch.compile(lambda t: ops.linear(t, pw, bias, out_dtype=out) + 1, backend=backend, fullgraph=True)
        assert torch.equal(call(x), ops.linear(x, pw, bias, out_dtype=out) + 1)
    layer = jq.JenksQuantLinear(nn.Linear(200, 72), 8, fmt="int8").to(DEV)
    layer.commit()
    assert torch.equal(torch.compile(layer, backend=backend, fullgraph=True)(x), layer(x))
    assert len(traced) == 3 and all(sum("jq.linear" in n for n in names) == 1 for names in traced)


@gpu
@pytest.mark.parametrize("rotate", [0, 128])
def test_a_norm_its_codes_and_their_products_repeat_themselves(rotate):
    """Every pass over the same inputs gives the same bits."""
    x, residual = (torch.randn(512, 1024, device=DEV).bfloat16() for _ in range(2))
    weights = [_weight(n, 1024, n, rotate) for n in (1024, 256, 256)]

    def chain():
        h, r = ops.residual_norm(x, residual, quantize=True, had_block=rotate)
        return [h.codes, h.scales, r] + [ops.linear(h, w) for w in weights]

    first = chain()
    for _ in range(50):
        assert all(torch.equal(a, b) for a, b in zip(chain(), first))
