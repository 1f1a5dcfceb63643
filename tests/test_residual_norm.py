"""The norms around a block against 64 bits.

Bounds.  A sum over a row is formed by at most 32 additions in a thread and ten between threads: a sum of squares is off by 45 * 2^-24 of
itself with its division, its reciprocal root (2^-22) by half of that and 2^-22, N(v) = v * root by two roundings more: 2^-18 of
itself.  A mean is off by 45 * 2^-24 of the mean size.  Errors of what a norm is given pass through it times 1 / rms, and through the root
by their own rms.  Every output is rounded once: eps / 2 of its type, and half of the type's smallest step."""
import math

import pytest
import torch

import if_i_could_turn_back_time_b200 as jq
from if_i_could_turn_back_time_b200 import _lib, ops
from oracle import formats

DEV = "cuda"
gpu = pytest.mark.gpu
DTYPES = (torch.float32, torch.float16, torch.bfloat16)
U = 2.0 ** -24


def _norm64(v, e, kind, weight, bias, eps):
    """(N(v) weight + bias, bound on its error) in 64 bits, v being off by e."""
    if kind == "layer":
        mean = v.mean(-1, keepdim=True)
        d = 45 * U * v.abs().mean(-1, keepdim=True)
        c = v - mean
        e = e + e.mean(-1, keepdim=True) + d + U * c.abs()
        v = c
    inv = 1 / (v.square().mean(-1, keepdim=True) + eps).sqrt()
    n = v * inv
    off = e * inv + n.abs() * (e.square().mean(-1, keepdim=True).sqrt() * inv + 2.0 ** -18)
    if weight is not None:
        n, off = n * weight.double(), off * weight.double().abs()
    if bias is not None:
        n = n + bias.double()
    return n, off * (1 + 2.0 ** -10) + 2 * U * n.abs() + 2.0 ** -148


def _expected(x, residual, weight, bias, post_weight, post_bias, gate, scale, eps, kind):
    """((h, its bound), (r, its bound)) before the outputs' rounding."""
    u = x.double()
    e = torch.zeros_like(u)
    if post_weight is not None:
        u, e = _norm64(u, e, kind, post_weight, post_bias, eps)
    f = scale * (1 if gate is None else gate.double())
    r = u * f
    e = e * (f if isinstance(f, float) else f.abs()) * (1 if not isinstance(f, float) or f > 0 else -1) + 4 * U * r.abs()
    if residual is not None:
        r = r + residual.double()
    e = e + U * r.abs()
    return _norm64(r, e, kind, weight, bias, eps), (r, e)


def _near(got, want, off, what):
    fin = torch.finfo(got.dtype)
    bound = off + fin.eps / 2 * (want.abs() + off) + fin.smallest_normal * fin.eps / 2
    d = (got.double() - want).abs()
    assert got.shape == want.shape and bool((d <= bound).all()), (what, (d / bound).max().item())


def _check(x, residual=None, weight=None, bias=None, *, post_weight=None, post_bias=None, gate=None, scale=1.0, eps=1e-6, kind="rms", had=0):
    args = dict(post_weight=post_weight, post_bias=post_bias, gate=gate, scale=scale, eps=eps, kind=kind)
    (h, eh), (r, er) = _expected(x, residual, weight, bias, **args)
    got = ops.residual_norm(x, residual, weight, bias, **args)
    assert got.h.dtype == x.dtype and got.r.dtype == (x if residual is None else residual).dtype
    _near(got.h, h, eh, "h")
    _near(got.r, r, er, "r")
    q = ops.residual_norm(x, residual, weight, bias, quantize=True, had_block=had, **args)
    assert torch.equal(q.r, got.r)
    rows = q.h
    assert rows.dtype == x.dtype and rows.had_block == had and rows.codes.shape == x.shape and rows.scales.shape == x.shape[:-1]
    if had:                                              # sums of 128 with signs, over sqrt(128); eight roundings on the way
        H = torch.from_numpy(formats.hadamard_matrix(128)).double().to(DEV)
        H = H / H[0, 0].abs() / math.sqrt(128)
        blocks = lambda t: t.reshape(*t.shape[:-1], -1, 128)                                                       # noqa: E731
        eh = ((blocks(eh) + 8 * U * blocks(h.abs())) @ H.abs()).reshape(h.shape)
        h = (blocks(h) @ H).reshape(h.shape)
    s = rows.scales.double()
    size, loose = h.abs().amax(-1).clamp(min=2.0 ** -100) / 127, eh.amax(-1) / 127
    assert bool(((s - size).abs() <= loose + 2 * U * size).all())
    step = (rows.codes.double() * s[..., None] - h).abs()        # half a step, the quotient's rounding, and what h is off by
    assert bool((step <= s[..., None] * (0.5 + 128 * U) + eh + loose[..., None]).all())
    return got


def _inputs(shape, dtype, rdtype=None, wdtype=None, seed=0):
    gen = torch.Generator(DEV).manual_seed(seed + shape[-1])
    rnd = lambda *s: torch.randn(*s, device=DEV, generator=gen)                                                     # noqa: E731
    x, res = rnd(*shape) * 0.5, rnd(*shape) * 2 + 0.3
    x[..., ::17] *= 6
    vec = [(rnd(shape[-1]) * 0.2 + 1).to(wdtype or dtype) if i % 2 == 0 else rnd(shape[-1]).to(wdtype or dtype) for i in range(4)]
    return x.to(dtype), res.to(rdtype or dtype), vec


WIDTHS = (1, 7, 8, 31, 64, 100, 197, 256, 264, 768, 1000, 1024, 1032, 2050, 4096, 5025, 8192, 11008, 16384, 20001, 32768)


@gpu
@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_against_64_bits(width, kind):
    for rows in (1, 3, 301):
        for dtype, rdtype, wdtype in ((torch.float32, None, None), (torch.float16, None, torch.float32), (torch.bfloat16, None, None),
                                      (torch.bfloat16, torch.float32, torch.bfloat16), (torch.float16, torch.float32, torch.float16)):
            x, res, (w, b, pw, pb) = _inputs((rows, width), dtype, rdtype, wdtype, rows)
            had = 128 if width % 128 == 0 and rows != 3 else 0
            _check(x, res, w, kind=kind, had=had)
            _check(x, res, w, b, post_weight=pw, post_bias=pb, scale=0.7071, kind=kind, had=had, eps=1e-5)
            if rows == 3:
                _check(x, res, kind=kind)
                _check(x, None, None, b, gate=w, scale=-0.5, kind=kind)
                _check(x, res, w, None, post_weight=pw, gate=pb, kind=kind)


@gpu
@pytest.mark.parametrize("width", [64, 100, 1152])
def test_gates_of_every_shape(width):
    G, T = 5, 83
    for dtype in (torch.bfloat16, torch.float32):
        x, res, (w, b, pw, _) = _inputs((G, T, width), dtype)
        gen = torch.Generator(DEV).manual_seed(1)
        rnd = lambda *s: torch.randn(*s, device=DEV, generator=gen)                                                 # noqa: E731
        gates = [rnd(()), rnd(1), rnd(width), rnd(T, 1), rnd(T, width), rnd(G, 1, 1), rnd(G, 1, width), rnd(G, T, 1), rnd(G, T, width), rnd(1, T, width),
                 rnd(G, 1, 6 * width)[..., width:2 * width], rnd(G, 1, width * 2)[..., 1:2 * width:2], rnd(G, T, 3)[..., 1:2], rnd(width, 1, G).permute(2, 1, 0),
                 rnd(G, 1, width + 1)[..., 1:], rnd(T, G, width).transpose(0, 1)]
        for gate in gates:
            _check(x, res, w, gate=gate.to(dtype if gate.numel() % 2 else torch.float16), scale=0.5)
        y = x.view(G, 1, T, width)
        _check(y, res.view(y.shape), w, gate=rnd(G, 2, 1, width)[:, 1:].half())
        four = x[:4, :82].reshape(2, 2, 82, width)                        # a gate that changes along the first and third dim only
        _check(four, None, w, b, gate=rnd(2, 1, 82, 1), post_weight=pw)
        _check(four, None, w, gate=rnd(2, 1, 82, width))


@gpu
def test_rotated_rows_of_every_layout():
    """Rows that are to be rotated are copied where they are not of 16-byte pieces, vectors where they are of another 16-bit type."""
    x, res, (w, b, pw, pb) = _inputs((6, 50, 256), torch.float16)
    same = ops.residual_norm(x, res, w, b, post_weight=pw, gate=pb, quantize=True, had_block=128)
    wide = lambda t: torch.empty(*t.shape[:-1], t.shape[-1] + 3, dtype=t.dtype, device=DEV)[..., 3:].copy_(t)                  # noqa: E731
    for args in ((wide(x), wide(res), wide(w), wide(b), wide(pw), wide(pb)), (x, wide(res), w, b, pw, pb), (x, res, w, b, pw, wide(pb.expand(6, 50, 256))),
                 (x, res, wide(w), b, pw, pb), (x.transpose(0, 1).contiguous().transpose(0, 1), res, w, b, pw, pb)):
        got = ops.residual_norm(args[0], args[1], args[2], args[3], post_weight=args[4], gate=args[5], quantize=True, had_block=128)
        assert torch.equal(got.r, same.r) and torch.equal(got.h.codes, same.h.codes) and torch.equal(got.h.scales, same.h.scales)
    _check(x, res, w.bfloat16(), b.bfloat16(), gate=pb.bfloat16(), had=128)
    _check(x, res, w.float(), gate=pb.bfloat16().view(1, 1, 256).expand(6, 1, 256), had=128)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_leading_dims_and_alignment(dtype):
    raw = torch.randn(3, 50, 700, device=DEV).to(dtype)
    other = torch.randn(3, 50, 700, device=DEV).to(dtype)
    vec = torch.randn(1000, device=DEV).to(dtype)
    for cut in (lambda t: t[:, :, 1:257], lambda t: t[:, ::3, 8:520], lambda t: t[1, :, 3:300], lambda t: t.transpose(1, 2)[:, :, :48], lambda t: t[:1].expand(2, 50, 700),
                lambda t: t[0, 0, :96], lambda t: t[:, :0]):
        x, res = cut(raw), cut(other)
        for at in (0, 1, 8):
            w = vec[at:at + x.shape[-1]]
            if x.numel():
                got = _check(x, res, w, w, post_weight=w)
            else:
                got = ops.residual_norm(x, res, w)
            assert got.h.is_contiguous() and got.r.is_contiguous() and got.h.shape == got.r.shape == x.shape
    x = raw[:, :, :256]
    got = ops.residual_norm(x, weight=vec[:256])
    assert got.r is x                                                       # nothing to add: the stream is the input


@gpu
@pytest.mark.parametrize("width", [40, 100, 2048])
def test_rows_that_go_wrong(width):
    """A row with NaN or infinity stays by itself; zeros, sizes at the types' ends and eps 0."""
    for dtype in DTYPES:
        for kind in ("rms", "layer"):
            x, res, (w, b, pw, _) = _inputs((330, width), dtype)
            x[0], res[0] = 0, 0
            x[1, 3] = torch.nan
            res[2, width - 1] = torch.inf
            x[3], res[3] = 1e-7, 0
            x[4] = 3.0 if kind == "layer" else x[4]
            res[4] = 0
            bad = torch.tensor([1, 2], device=DEV)
            for rows in (330, 7):
                good = torch.tensor([i for i in range(rows) if i not in (1, 2)], device=DEV)
                for post in (None, pw):
                    got = ops.residual_norm(x[:rows], res[:rows], w, b, post_weight=post, kind=kind)
                    q = ops.residual_norm(x[:rows], res[:rows], w, b, post_weight=post, kind=kind, quantize=True)
                    assert torch.isnan(got.h[bad]).any(-1).all() and torch.isnan(q.h.scales[bad]).all() and bool((q.h.codes[bad] == 0).all())
                    alone = ops.residual_norm(x[good], res[good], w, b, post_weight=post, kind=kind)
                    if rows == 330:
                        assert torch.equal(got.h[good], alone.h) and torch.equal(got.r[good], alone.r)
                    _check(x[good], res[good], w, b, post_weight=post, kind=kind)
    z = torch.zeros(2, width, device=DEV)
    assert torch.isnan(ops.residual_norm(z, eps=0.0).h).all() and bool((ops.residual_norm(z).h == 0).all())


@gpu
def test_a_large_mean_is_taken_out_first():
    """Layer norm of values around 1000 with a spread of 1: the variance comes from what is left without the mean."""
    x = torch.randn(40, 4096, device=DEV) + 1000
    got = _check(x, kind="layer")
    want = torch.nn.functional.layer_norm(x.double(), (4096,), eps=1e-6)
    assert (got.h - want).abs().max().item() < 0.01                          # (the mean is off by 45 * 2^-24 * 1000 at most)


@gpu
@pytest.mark.parametrize("rows", [1, 64, 600])
def test_the_way_into_three_products(rows):
    """Norm, codes and products together: the products are exactly those of the codes."""
    x, res, (w, _, pw, _) = _inputs((rows, 1024), torch.bfloat16)
    gen = torch.Generator(DEV).manual_seed(9)
    weights = [jq.pack_weight(torch.randn(n, 1024, device=DEV, generator=gen), jq.QuantSpec("int8", 0, 128)) for n in (1024, 200, 57)]
    h, r = ops.residual_norm(x, res, w, post_weight=pw, quantize=True, had_block=128)
    for pk in weights:
        y = ops.linear(h, pk, out_dtype=torch.float32)
        total = h.codes.double() @ pk.qweight.double().T
        want = total * pk.scales.double() * h.scales.double()[:, None]
        assert bool(((y - want).abs() <= 4 * U * want.abs()).all())
        assert ops.linear(h, pk).dtype == torch.bfloat16 and torch.equal(ops.linear(h, pk), y.bfloat16())
    dense = ops.residual_norm(x, res, w, post_weight=pw)
    assert torch.equal(dense.r, r)
    y = ops.linear(dense.h, weights[0], out_dtype=torch.float32)            # through 16 bits: the codes' rounding is what differs
    full = ops.linear(h, weights[0], out_dtype=torch.float32)
    assert ((y - full).norm() / full.norm()).item() < 0.02


@gpu
@pytest.mark.parametrize("rows", [2, 700])
def test_streams_and_graphs(rows):
    x, res, (w, b, pw, pb) = _inputs((rows, 640), torch.bfloat16)
    pk = jq.pack_weight(torch.randn(96, 640, device=DEV), jq.QuantSpec("int8", 0))

    def step(x, res):
        h, r = ops.residual_norm(x, res, w, b, post_weight=pw, post_bias=pb, gate=w, scale=0.5, quantize=True)
        y = ops.linear(h, pk)
        return y, ops.residual_norm(x, r, w, kind="layer")

    side = torch.cuda.Stream()
    want = step(x, res)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x, res)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1].h, want[1].h)
    graph, held = torch.cuda.CUDAGraph(), x.clone()
    with torch.cuda.graph(graph):
        out = step(held, res)
    held.copy_(x * 2)
    graph.replay()
    want = step(x * 2, res)
    assert torch.equal(out[0], want[0]) and torch.equal(out[1].h, want[1].h) and torch.equal(out[1].r, want[1].r)


def test_refusals():
    x = torch.randn(2, 3, 100)
    w = torch.randn(100)
    for call, text in ((lambda: ops.residual_norm(x), "CUDA"), (lambda: ops.residual_norm(x, x[:1]), "residual"), (lambda: ops.residual_norm(x, x.half()), "residual"),
                       (lambda: ops.residual_norm(x.half(), x.bfloat16()), "residual"), (lambda: ops.residual_norm(x, weight=w[:9]), "one dtype"),
                       (lambda: ops.residual_norm(x, weight=w, bias=w.half()), "one dtype"), (lambda: ops.residual_norm(x, post_bias=w), "post_weight"),
                       (lambda: ops.residual_norm(x, kind="batch"), "kind"), (lambda: ops.residual_norm(x, had_block=128), "had_block"),
                       (lambda: ops.residual_norm(x, quantize=True, had_block=128), "had_block"), (lambda: ops.residual_norm(x, scale=math.inf), "scale"),
                       (lambda: ops.residual_norm(x, eps=-1.0), "eps"), (lambda: ops.residual_norm(x, eps=math.nan), "eps"),
                       (lambda: ops.residual_norm(x, scale=math.nan), "scale"), (lambda: ops.residual_norm(x.double()), "dtype|CUDA"),
                       (lambda: ops.residual_norm(x, gate=w.double()), "gate"),
                       (lambda: ops.residual_norm(torch.randn(2, 0)), "rows of 1"), (lambda: ops.residual_norm(torch.empty(1, 32769)), "32768")):
        with pytest.raises(RuntimeError, match=text):
            call()


def test_refusals_of_the_library():
    lib, p = _lib.load(), torch.zeros(4096, dtype=torch.uint8).data_ptr()

    def call(**change):
        n = _lib.jq_norm(x=p, h=p, stride_x=64, rows=1, width=64, gate_inner_rows=1, scale=1.0, eps=1e-6)
        for k, v in change.items():
            setattr(n, k, v)
        import ctypes
        return lib.jq_residual_norm(ctypes.byref(n), None)

    assert lib.jq_residual_norm(None, None) == -1 and call(x=None) == -1 and call(h=None) == -1 and call(codes=p) == -1
    assert call(rows=0) == -2 and call(width=0) == -2 and call(width=32769) == -2 and call(had_block=128) == -2 and call(gate=p, gate_inner_rows=0) == -2
    assert call(codes=p, scales=p, stride_codes=48) == -2 and call(codes=p, scales=p, stride_codes=72) == -3 and call(codes=p + 4, scales=p, stride_codes=64) == -3
    assert call(codes=p, scales=p, stride_codes=128, width=128, had_block=128, x=p + 4) == -3
    assert call(x_dtype=3) == -4 and call(residual_dtype=1) == -4 and call(weight_dtype=-1) == -4 and call(kind=2) == -5


@gpu
def test_refusals_on_the_gpu():
    x = torch.randn(2, 64, device=DEV)
    w = torch.nn.Parameter(torch.ones(64, device=DEV))
    with pytest.raises(RuntimeError, match="backward"):
        ops.residual_norm(x, weight=w)
    with torch.no_grad():
        ops.residual_norm(x, weight=w)
    with pytest.raises(RuntimeError, match="broadcast"):
        ops.residual_norm(x, gate=torch.ones(3, 64, device=DEV))
    with pytest.raises(RuntimeError, match="broadcast"):
        ops.residual_norm(x, gate=torch.ones(1, 2, 64, device=DEV))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.residual_norm(x, gate=torch.ones(64))


@gpu
@pytest.mark.parametrize("width", [128, 1024, 8192])
def test_rotations_that_leave_the_range(width):
    """Normed values whose rotation leaves fp32's range: the row's scale is NaN, as by quantising the rotated values."""
    signs = torch.tensor([1, -1, 1, -1, 1, -1, -1, 1], device=DEV, dtype=torch.float32)
    x = torch.ones(5, width, device=DEV)
    x[3] = torch.nan
    for weight, lost in ((3e38 * signs.repeat(width // 8), [0, 1, 2, 3, 4]), (torch.full((width,), 3e38, device=DEV), [0, 1, 2, 3, 4]), (signs.repeat(width // 8), [3])):
        rows = ops.residual_norm(x, weight=weight, quantize=True, had_block=128).h
        assert torch.isnan(rows.scales[lost]).all() and bool((rows.codes[lost] == 0).all())
        assert int(torch.isnan(rows.scales).sum()) == len(lost)


def test_arrays_off_their_elements_boundary_are_refused():
    import ctypes
    lib, p = _lib.load(), torch.zeros(4096, dtype=torch.uint8).data_ptr()
    assert p % 16 == 0

    def call(**change):
        n = _lib.jq_norm(x=p, residual=p, h=p, r=p, stride_x=8, stride_residual=8, rows=1, width=8, gate_inner_rows=1, scale=1.0, eps=1e-6)
        for k, v in change.items():
            setattr(n, k, v)
        return lib.jq_residual_norm(ctypes.byref(n), None)

    arrays = {"x": "x_dtype", "h": "x_dtype", "residual": "residual_dtype", "r": "residual_dtype", "weight": "weight_dtype", "bias": "weight_dtype",
              "post_weight": "weight_dtype", "post_bias": "weight_dtype", "gate": "gate_dtype"}
    for name in arrays:
        for off in (1, 2, 3):
            assert call(**{name: p + off}) == -3
        for dtype in (1, 2):
            assert call(**{"x_dtype": dtype, "residual_dtype": dtype, arrays[name]: dtype, name: p + 1}) == -3
    assert call(codes=p, scales=p + 2, stride_codes=16) == -3
    assert call(reserved=1) == -2


def test_rows_that_leave_32_bits_are_refused():
    import ctypes
    p = torch.zeros(4096, dtype=torch.uint8).data_ptr()
    for rows in (_lib.JQ_INT8_MAX_ROWS + 1, 2 ** 31 - 1):
        n = _lib.jq_norm(x=p, h=p, rows=rows, width=8, gate_inner_rows=1, scale=1.0, eps=1e-6)
        assert _lib.load().jq_residual_norm(ctypes.byref(n), None) == -2
