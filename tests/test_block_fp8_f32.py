"""Block-scaled 8-bit rows whose scales are held in 32 bits, and products that leave in
32 bits, against the formulas in 64 bits.

Half a step of f32 is 2^-24 of the value, of e4m3 2^-4, or 2^-10 of a scale below
its smallest normal value, of bf16 2^-8.
"""

import math

import pytest
import torch

from vilbert_multi_task_amd.ops import functional as F_ops

gpu = pytest.mark.gpu
BF, F32, F64, E4 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn
EPS = 1e-6
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]


def _ceil(n, by=128):
    return -(-n // by)


def _normal(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def _spread(scales, k):
    return scales.repeat_interleave(128, -1)[..., :k]


def _scales64(y):
    """The scales that rows of y have."""
    a = y.abs()
    a = torch.where(torch.isfinite(a), a, 0.0)
    parts = [a[..., i:i + 128].amax(-1) for i in range(0, y.shape[-1], 128)]
    return (torch.stack(parts, -1) / 448).clamp(min=2.0 ** -100)


def _check_rows(q, scales, y64, off):
    """q and f32 scales against y64, of which the quantised values were `off` (a
    bound for each) before they were rounded."""
    k = y64.shape[-1]
    assert q.dtype == E4 and scales.dtype == F32
    assert q.shape == y64.shape and scales.shape == (*y64.shape[:-1], _ceil(k))
    q, s64 = q.cpu().to(F64), _scales64(y64)
    pad = torch.nn.functional.pad(off, (0, _ceil(k) * 128 - k)).unflatten(-1, (-1, 128)).amax(-1)
    s = scales.cpu().to(F64)
    # the largest value is `pad` off, the division by 448 half a step
    assert ((s - s64).abs() <= pad / 448 + 2.0 ** -24 * (s64 + pad / 448)).all()
    s = _spread(s, k)
    # the reciprocal and the product move a value by two half steps of f32
    half = torch.maximum(2.0 ** -4 * (y64.abs() + off), 2.0 ** -10 * s)
    assert ((q * s - y64).abs() <= half * (1 + 2.0 ** -20) + off).all()


ROWS = [(1, 1), (3, 129), (7, 15), (38, 1024), (2, 8193)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,k", ROWS)
def test_quantiser(rows, k, dtype, device):
    x = _normal(rows, k, seed=rows + k).to(dtype)
    x[-1, k // 2:] *= 2.0 ** -14  # below e4m3's normal values
    q, s = F_ops.quantize_fp8_block(x.to(device), scale_dtype=F32)
    _check_rows(q, s, x.to(F64), torch.zeros(rows, k, dtype=F64))
    rq, rs = F_ops.quantize_fp8_block(x, scale_dtype=F32)
    assert torch.equal(s.cpu(), rs) and torch.equal(q.cpu().float(), rq.float())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,k", [(1, 1), (129, 127), (257, 1000)])
def test_weight_quantiser(rows, k, dtype, device):
    w = _normal(rows, k, seed=rows).to(dtype)
    q, s = F_ops.quantize_fp8_block_weight(w.to(device), scale_dtype=F32)
    assert q.shape == (rows, k) and s.dtype == F32 and s.shape == (_ceil(rows), _ceil(k))
    for i in range(_ceil(rows)):
        for j in range(_ceil(k)):
            part = (slice(128 * i, 128 * i + 128), slice(128 * j, 128 * j + 128))
            v = w[part].float()
            assert s[i, j].cpu() == v.abs().max() / 448  # one rounding
            assert torch.equal(q.cpu()[part].float(), (v * (1 / s[i, j].cpu())).to(E4).float())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_quantisers_at_the_ends_of_their_range(dtype, device):
    x = _normal(6, 256, seed=3)
    x[0], x[1], x[2, :128] = 0, 1e-37, 3e38
    x[3, 5], x[3, 7], x[4, 200], x[5, :128] = math.inf, math.nan, -math.inf, math.nan
    x = x.to(dtype)
    for op in (F_ops.quantize_fp8_block, F_ops.quantize_fp8_block_weight):
        q, s = op(x.to(device), scale_dtype=F32)
        assert torch.isfinite(s).all()
        nan = torch.isnan(q.float()).cpu()
        assert torch.equal(nan, ~torch.isfinite(x))
        rq, rs = op(torch.where(nan, 0.0, x).to(dtype), scale_dtype=F32)
        assert torch.equal(s.cpu(), rs)
        assert torch.equal(torch.where(nan, 0.0, q.cpu().float()), rq.float())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("with_res", [False, True])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,k", ROWS)
def test_norms(rows, k, dtype, with_res, device):
    x = _normal(rows, k, seed=k + 1).to(dtype)
    res = (3 * _normal(rows, k, seed=k + 2)).to(dtype) if with_res else None
    w = (1 + 0.2 * _normal(k, seed=k + 3)).to(dtype)
    b = (0.2 * _normal(k, seed=k + 4)).to(dtype)
    gx, gw, gb = (t.to(device) for t in (x, w, b))
    gr = res.to(device) if with_res else None

    t = (x + res if with_res else x).to(F64)  # in x's type
    y64 = t / torch.sqrt(t.square().mean(-1, keepdim=True) + EPS) * w.to(F64)
    got = F_ops.rms_norm_fp8_block(gx, gw, EPS, residual=gr, scale_dtype=F32)
    # a sum of k squares, by 64 a lane, 6 + 16 for the row, and single roundings
    _check_rows(got[0], got[1], y64, 96 * 2.0 ** -24 * y64.abs())
    if with_res:
        assert torch.equal(got[2].cpu().to(F64), t)

    t = x.to(F64) + (res.to(F64) if with_res else 0.0)
    d = t - t.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(d.square().mean(-1, keepdim=True) + 1e-5)
    y64 = d * r * w.to(F64) + b.to(F64)
    size = (t.abs() + t.abs().mean(-1, keepdim=True)) * r * w.to(F64).abs() + y64.abs() + b.to(F64).abs()
    y, q, s = F_ops.layer_norm_fp8_block(gx, gw, gb, 1e-5, residual=gr, scale_dtype=F32)
    assert y.dtype == dtype
    _check_rows(q, s, y64, 96 * 2.0 ** -24 * size)


@pytest.mark.parametrize("device", DEVICES)
def test_other_scale_types_are_refused(device):
    x, w = torch.zeros(2, 8, device=device), torch.ones(8, device=device)
    for call in (
        lambda t: F_ops.quantize_fp8_block(x, scale_dtype=t),
        lambda t: F_ops.quantize_fp8_block_weight(x, scale_dtype=t),
        lambda t: F_ops.rms_norm_fp8_block(x, w, EPS, scale_dtype=t),
        lambda t: F_ops.layer_norm_fp8_block(x, w, w, EPS, scale_dtype=t),
    ):
        for t in (torch.float16, torch.float64, torch.float8_e4m3fn):
            with pytest.raises(RuntimeError, match="scale_dtype"):
                call(t)


# --- the products ---------------------------------------------------------------


def _rows8(m, k, seed=0):
    x = _normal(m, k, seed=seed) * (1 + 9 * (_normal(k, seed=seed + 1) > 1.5))
    return F_ops.quantize_fp8_block(x, scale_dtype=F32)


def _weight8(n, k, seed=0):
    return F_ops.quantize_fp8_block_weight(_normal(n, k, seed=seed) / math.sqrt(k), scale_dtype=F32)


def _operands(m, n, k, device, seed=0):
    return [t.to(device) for t in (*_rows8(m, k, seed=seed + m + k), *_weight8(n, k, seed=seed + n + k + 1))]


def _product64(x8, xs, w8, ws, bias, gelu):
    """y, and a bound of what a sum in 32 bits is off: 128 products, which are exact, in
    a block, the blocks, what teams and waves join, the scales and the bias, each at
    most a half step of the sum of all sizes."""
    k, n = x8.shape[-1], w8.shape[0]
    x = x8.to(F64) * _spread(xs.to(F64), k)
    w = w8.to(F64) * _spread(ws.to(F64).repeat_interleave(128, 0)[:n], k)
    y, size = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        y, size = y + bias.to(F64), size + bias.to(F64).abs()
    off = (128 + _ceil(k) + 24) * 2.0 ** -24 * size
    if gelu:
        # GELU's slope is at most 1.13, its own value good to 2^-18 of |y|
        off = 1.13 * off + 2.0 ** -18 * y.abs()
        y = y * 0.5 * torch.erfc(-y / math.sqrt(2))
    return y.cpu(), off.cpu()


# on the GPU: every kernel that has few or many rows, its edges, ragged widths
PRODUCTS = [
    (1, 1, 1), (2, 16, 15), (16, 127, 16), (7, 300, 1000), (38, 768, 768), (17, 129, 100),
    (101, 1024, 1024), (256, 1601, 130), (600, 1030, 300), (1616, 1601, 128), (2500, 1000, 257),
    (4100, 1030, 300), (9000, 640, 1024),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("gelu,with_bias", [(False, False), (True, True)])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_products_in_32_bits(m, n, k, gelu, with_bias, device):
    if device == "cpu" and m * n * k > 1e8:
        m = 33
    a = _operands(m, n, k, device)
    b = _normal(n, seed=5).to(device) if with_bias else None
    y64, off = _product64(*a, b, gelu)
    y = F_ops.fp8_block_linear(*a, b, gelu=gelu, out_dtype=F32)
    assert y.dtype == F32 and y.shape == (m, n)
    assert ((y.cpu().to(F64) - y64).abs() <= off + 2.0 ** -24 * y64.abs()).all()
    q, s = F_ops.fp8_block_linear_fp8(*a, b, gelu=gelu)
    _check_rows(q, s, y64, off)
    # to bf16: the 8-bit instruction, 7 losses of 2^-13 of the largest in each eight
    # products, at most 7 * 2^-13 of all their sizes
    y = F_ops.fp8_block_linear(*a, b, gelu=gelu)
    size = off / (128 + _ceil(k) + 24) * 2.0 ** 24
    assert y.dtype == BF
    assert ((y.cpu().to(F64) - y64).abs() <= 7 * 2.0 ** -13 * size + off + 2.0 ** -8 * (y64.abs() + off)).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("m,n,k", [(3, 40, 128), (40, 300, 384), (300, 1000, 512), (2500, 1000, 130), (4100, 1030, 256)])
def test_nothing_is_dropped_beside_a_large_product(m, n, k, device):
    """One product of 448 * 448 in each block beside multiples of 2^-4: every partial sum
    is a multiple of 2^-4 below 2^20, exact in 32 bits in whatever order."""
    g = torch.Generator().manual_seed(m)
    x = torch.randint(-7, 8, (m, k), generator=g) / 4.0
    w = torch.randint(-7, 8, (n, k), generator=g) / 4.0
    x[:, 5::128], w[:, 5::128] = 448, 448
    x8, w8 = x.to(E4).to(device), w.to(E4).to(device)
    y = (x.double() @ w.double().t()).float()
    assert (y.double() == x.double() @ w.double().t()).all()
    for scales in (BF, F32):
        xs = torch.ones(m, _ceil(k), dtype=scales, device=device)
        ws = torch.ones(_ceil(n), _ceil(k), dtype=scales, device=device)
        assert torch.equal(F_ops.fp8_block_linear(x8, xs, w8, ws, out_dtype=F32).cpu(), y)
    _, s = F_ops.fp8_block_linear_fp8(x8, xs, w8, ws)
    parts = [y[:, i:i + 128].abs().amax(-1) for i in range(0, n, 128)]
    assert torch.equal(s.cpu(), torch.stack(parts, -1) / 448)


@gpu
@pytest.mark.parametrize("m,n,k", PRODUCTS + [
    (2049, 2100, 1000), (16500, 257, 128), (16300, 1024, 384), (4097, 3200, 512), (33000, 640, 1024)])
def test_scales_in_either_type_give_the_same(m, n, k):
    """Scales that bf16 holds, in f32: the same products, bit for bit."""
    x8, xs, w8, ws = _operands(m, n, k, "cuda")
    xs, ws = xs.to(BF), ws.to(BF)
    b = _normal(n, seed=5).cuda()
    for gelu in (False, True):
        for out in (BF, F32):
            want = F_ops.fp8_block_linear(x8, xs, w8, ws, b, gelu, out)
            assert torch.equal(F_ops.fp8_block_linear(x8, xs.float(), w8, ws.float(), b, gelu, out), want)


@gpu
def test_gelu_in_32_bits():
    """Of a bias alone, so that nothing else is rounded: 1.3e-6 of its value down to -4,
    1.4e-5 to -8, 1.3e-3 to -12.9, and the exponential's and the difference's steps."""
    n = 8192
    b = torch.linspace(-12.9, 12.9, n)
    for m in (1, 40, 300, 2000):  # kernels of few, some and many rows
        x8, w8 = torch.zeros(m, 128, device="cuda").to(E4), torch.zeros(n, 128, device="cuda").to(E4)
        xs, ws = torch.ones(m, 1, device="cuda"), torch.ones(n // 128, 1, device="cuda")
        y = F_ops.fp8_block_linear(x8, xs, w8, ws, b.cuda(), gelu=True, out_dtype=F32)[-1].cpu().to(F64)
        v = b.to(F64)
        y64 = v * 0.5 * torch.erfc(-v / math.sqrt(2))
        tol = torch.where(v >= -4, 2.0 ** -18, torch.where(v >= -8, 2.0 ** -15, 2.0 ** -9))
        assert ((y - y64).abs() <= tol * y64.abs()).all()
    ends = torch.tensor([math.inf, -math.inf, math.nan, -20.0, 20.0, 0.0])
    y = F_ops.fp8_block_linear(x8[:1], xs[:1], w8[:6], ws[:1], ends.cuda(), gelu=True, out_dtype=F32)[0].cpu()
    assert y[0] == math.inf and y[1] == 0 and torch.isnan(y[2]) and y[3] == 0 and y[4] == 20 and y[5] == 0


@gpu
@pytest.mark.parametrize("m", [5, 40, 400, 5000])
def test_exact_products_keep_nan_in_its_row_and_column(m):
    a = _operands(m, 300, 400, "cuda")
    want = F_ops.fp8_block_linear(*a, out_dtype=F32)
    a[0].view(torch.uint8)[3, 399] = 0x7F
    a[2].view(torch.uint8)[200, 0] = 0xFF
    nan = torch.zeros_like(want, dtype=torch.bool)
    nan[3], nan[:, 200] = True, True
    got = F_ops.fp8_block_linear(*a, out_dtype=F32)
    assert torch.equal(torch.isnan(got), nan) and torch.equal(got[~nan], want[~nan])
    q, s = F_ops.fp8_block_linear_fp8(*a)
    assert torch.equal(torch.isnan(q.float()), nan) and torch.isfinite(s).all()


@pytest.mark.parametrize("device", DEVICES)
def test_products_of_scales_wherever_they_lie(device):
    x8, xs, w8, ws = _operands(12, 130, 300, device)
    want = F_ops.fp8_block_linear(x8, xs, w8, ws, out_dtype=F32)
    across = F_ops.fp8_block_linear(x8, xs.t().contiguous().t(), w8, ws.t().contiguous().t(), out_dtype=F32)
    assert torch.equal(across, want)
    wide = torch.full((12, 7), math.nan, device=device)
    wide[:, 2:5] = xs
    assert torch.equal(F_ops.fp8_block_linear(x8, wide[:, 2:5], w8, ws, out_dtype=F32), want)
    got = F_ops.fp8_block_linear(x8.view(3, 4, 300), xs.view(3, 4, 3), w8, ws, out_dtype=F32)
    assert torch.equal(got, want.view(3, 4, 130))
    y64, off = _product64(x8, xs, w8, ws, None, False)
    got = F_ops.fp8_block_linear(x8[7], xs[7], w8, ws, out_dtype=F32).cpu().to(F64)
    assert got.shape == (130,) and ((got - y64[7]).abs() <= off[7] + 2.0 ** -24 * y64[7].abs()).all()
    y8, s = F_ops.fp8_block_linear_fp8(x8[:0], xs[:0], w8, ws)
    assert y8.shape == (0, 130) and s.shape == (0, 2) and s.dtype == F32
    assert F_ops.fp8_block_linear(x8[:0], xs[:0], w8, ws, out_dtype=F32).shape == (0, 130)


@pytest.mark.parametrize("device", DEVICES)
def test_product_types_are_refused(device):
    x8, xs, w8, ws = _operands(3, 130, 256, device)
    for op in (F_ops.fp8_block_linear, F_ops.fp8_block_linear_fp8):
        for a in ((x8, xs.to(BF), w8, ws), (x8, xs, w8, ws.to(BF)), (x8, xs.half(), w8, ws.half()),
                  (x8, xs.double(), w8, ws.double())):
            with pytest.raises(RuntimeError, match=op.__name__ + ": scales must be both"):
                op(*a)
    for t in (torch.float16, torch.float64, E4):
        with pytest.raises(RuntimeError, match="out_dtype"):
            F_ops.fp8_block_linear(x8, xs, w8, ws, out_dtype=t)


@gpu
def test_exact_products_on_streams_and_in_graphs():
    m, n, k = 4100, 384, 300
    a = _operands(m, n, k, "cuda")
    b = _normal(n, seed=5).cuda()

    def both():
        return (F_ops.fp8_block_linear(*a, b, gelu=True, out_dtype=F32), F_ops.fp8_block_linear(*a, b),
                *F_ops.fp8_block_linear_fp8(*a, b))

    want = [t.clone() for t in both()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = both()
        graphs.append((g, out))
    results = [other]
    for _ in range(3):
        for g, _ in graphs:
            g.replay()
        results.append(both())
        torch.cuda.synchronize()
        results += [[t.clone() for t in out] for _, out in graphs]
    for got in results:
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(got, want))


@gpu
def test_exact_outputs_past_32_bits():
    m, n = 70001, 32000
    x8, xs, w8, ws = _operands(4, n, 32, "cuda")
    big = torch.zeros(m, 32, dtype=torch.uint8, device="cuda")
    big[-4:] = x8.view(torch.uint8)
    scales = torch.ones(m, 1, device="cuda")
    scales[-4:] = xs
    y64, off = _product64(x8, xs, w8, ws, None, False)
    y = F_ops.fp8_block_linear(big.view(E4), scales, w8, ws, out_dtype=F32)
    assert ((y[-4:].cpu().to(F64) - y64).abs() <= off + 2.0 ** -24 * y64.abs()).all()
    del y
    q, s = F_ops.fp8_block_linear_fp8(big.view(E4), scales, w8, ws)
    _check_rows(q[-4:], s[-4:], y64, off)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("m,n,k", [(5, 128, 128), (40, 300, 300), (600, 1030, 300), (2500, 1000, 128), (4100, 1030, 300), (16300, 1024, 384)])
def test_scales_whose_product_passes_the_range(m, n, k, device):
    """What is nothing stays nothing, however large the scales beside it are."""
    if device == "cpu":
        m = 5
    x8, xs, w8, ws = _operands(m, n, k, device)
    b = _normal(n, seed=5).to(device)
    cases = [(BF, BF), (BF, F32), (F32, BF), (F32, F32)]  # scales, results
    want = [F_ops.fp8_block_linear(x8, xs.to(s), w8, ws.to(s), b, out_dtype=o) for s, o in cases]
    x8.view(torch.uint8)[3] = 0
    xs[3], ws[0] = 6e35, 1000.0
    xs[1], ws[-1, -1] = 2.0 ** -100, 2.0 ** -100
    small = x8.view(torch.uint8).clone()
    small[1, k // 128 * 128 if k % 128 else k - 128:] = 0  # and where a product is 2^-200
    x8 = small.view(E4)
    for (s, o), ref in zip(cases, want):
        y = F_ops.fp8_block_linear(x8, xs.to(s), w8, ws.to(s), b, out_dtype=o)
        assert torch.equal(y[3], b.to(o))
        # rows of ordinary scales are what they were, where W's are
        at = slice(128, (n - 1) // 128 * 128)
        assert torch.equal(y[4, at], ref[4, at]) and not torch.isnan(y).any()
    xs[3, 0] = math.nan  # a scale that is none is not hidden
    assert torch.isnan(F_ops.fp8_block_linear(x8, xs, w8, ws, b)[3]).all()
    assert torch.isnan(F_ops.fp8_block_linear(x8, xs, w8, ws, b, out_dtype=F32)[3]).all()


@gpu
@pytest.mark.parametrize("m", [1, 40, 300, 2000, 8192])  # kernels of few, some, many and very many rows
def test_gelu_to_bf16(m):
    """Of a bias alone: 2^-17 of its value down to -4, 2^-14 down to -6, 2^-10 down to -8,
    and an absolute error of 1e-14 below, each before bf16's half step."""
    n = 8192
    b = torch.linspace(-15, 15, n)
    x8, w8 = torch.zeros(m, 256, device="cuda").to(E4), torch.zeros(n, 256, device="cuda").to(E4)
    xs, ws = torch.ones(m, 2, device="cuda", dtype=BF), torch.ones(n // 128, 2, device="cuda", dtype=BF)
    y = F_ops.fp8_block_linear(x8, xs, w8, ws, b.cuda(), gelu=True)[-1].cpu().to(F64)
    v = b.to(F64)
    y64 = v * 0.5 * torch.erfc(-v / math.sqrt(2))
    tol = torch.where(v >= -4, 2.0 ** -17, torch.where(v >= -6, 2.0 ** -14, 2.0 ** -10)) * y64.abs()
    tol = torch.where(v >= -8, tol, 1e-14)
    assert ((y - y64).abs() <= tol + 2.0 ** -8 * (y64.abs() + tol)).all()
