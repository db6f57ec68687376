"""The 8-bit row operators (include/zf_int8.h) on the GPU against their definitions in 64 bits, at the sizes, layouts and
values where they can go wrong. Tolerances follow from the operators' roundings (u = 2^-24, one fp32 rounding)."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF16 = 2.0 ** -8  # one bf16 rounding: 8 significant bits, so 1 + 2^-8 lies halfway between 1 and its successor 1 + 2^-7
EPS = 1e-6


@pytest.fixture(scope='module')
def backend():
    import ZipNeRFCudaBackend
    return ZipNeRFCudaBackend


def generator(seed, device='cuda'):
    return torch.Generator(device=device).manual_seed(seed)


def rows(n, d, seed, dtype=torch.float32, stride=None, offset=0):
    """Rows with columns of different size and every seventh row zero, as a view with the given row stride and offset."""
    gen = generator(seed)
    x = torch.randn(n, d, device='cuda', generator=gen) * torch.randn(d, device='cuda', generator=gen).mul(0.7).exp()
    x[3::7] = 0
    stride = stride or d
    base = torch.full((n * stride + offset,), 9.0, device='cuda', dtype=dtype)
    view = base[offset:].as_strided((n, d), (stride, 1), offset)
    view.copy_(x)
    return view


def scale_of(largest, power_of_two):
    """64-bit: the step of rows whose largest magnitudes are given (zero for rows of zeros)"""
    step = (largest / 127).clamp(min=2.0 ** -126)
    if power_of_two:
        step = torch.exp2(torch.ceil(torch.log2(step)))
    return torch.where(largest > 0, step, torch.zeros_like(step))


def codes_of(values, scales):
    return torch.round(values / torch.where(scales > 0, scales, torch.ones_like(scales))[:, None])


def code_rows(n, d, seed, power_of_two=True):
    """Random codes in a padded buffer whose padding holds other values, and scales; every fifth row zero."""
    gen = generator(seed)
    buffer = torch.randint(-127, 128, (n, (d + 15) // 16 * 16), device='cuda', generator=gen, dtype=torch.int8)
    scales = torch.exp2(torch.randint(-9, 2, (n,), device='cuda', generator=gen).float())
    if not power_of_two:
        scales *= torch.rand(n, device='cuda', generator=gen) + 0.5
    scales[2::5] = 0
    buffer[2::5, :d] = 0
    return buffer[:, :d], scales


SIZES = [(1, 1), (1, 8), (3, 7), (5, 64), (33, 65), (7, 256), (9, 257), (4, 1000), (5, 1024), (3, 1025), (2, 4096), (3, 4099), (2, 8192), (2, 8193), (1, 70001)]


@pytest.mark.parametrize('power_of_two', [False, True])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('n,d', SIZES)
def test_quantize_rows(backend, n, d, dtype, power_of_two):
    x = rows(n, d, n + d, dtype)
    codes, scales = backend.quantize_rows(x, power_of_two)
    assert codes.shape == (n, d) and codes.dtype == torch.int8 and codes.stride(0) % 16 == 0
    wanted = scale_of(x.double().abs().amax(1), power_of_two)
    # one rounding of the quotient
    assert ((scales.double() - wanted).abs() <= U * wanted).all()
    if power_of_two:
        assert torch.equal(codes.double(), codes_of(x.double(), wanted))  # x / scale is exact
    # half a step, and the roundings of the scale, its reciprocal and the product (at most 127 steps, 3 u each)
    error = (codes.double() * scales.double()[:, None] - x.double()).abs()
    assert (error <= scales.double()[:, None] * (0.5 + 127 * 4 * U)).all()
    # restored: one rounding to the output's type (of the fp32 product)
    for out_type, unit in ((torch.float32, 2 * U), (torch.bfloat16, BF16 + 2 * U)):
        exact = codes.double() * scales.double()[:, None]
        restored = backend.dequantize_rows(codes, scales, out_type)
        assert restored.dtype == out_type and restored.shape == (n, d)
        assert ((restored.double() - exact).abs() <= unit * exact.abs()).all()
    if power_of_two:
        assert torch.equal(backend.dequantize_rows(codes, scales).double(), codes.double() * scales.double()[:, None])


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('d,stride,offset', [(96, 104, 0), (96, 99, 0), (96, 96, 3), (256, 256, 1), (100, 128, 8), (1500, 1501, 5)])
def test_strided_rows(backend, d, stride, offset, dtype):
    """Row strides and offsets on and off the 16-byte grid give the same bits as contiguous rows"""
    x = rows(21, d, 5, dtype, stride, offset)
    r = rows(21, d, 6, dtype, stride, offset)
    for got, wanted in zip(backend.quantize_rows(x), backend.quantize_rows(x.contiguous())):
        assert torch.equal(got, wanted)
    w = torch.rand(d, device='cuda', generator=generator(1)) + 0.5
    # the reduction's order depends on the access width: codes may differ where a value lies within u of a tie
    a, b = backend.rms_norm_int8(x, r, w, EPS), backend.rms_norm_int8(x.contiguous(), r.contiguous(), w, EPS)
    assert torch.equal(a[2], b[2])
    assert ((a[3] - b[3]).abs() <= 8 * U * b[3]).all() and (a[0].int() - b[0].int()).abs().max() <= 1


@pytest.mark.parametrize('bad', [float('nan'), float('inf'), -float('inf')])
@pytest.mark.parametrize('d', [5, 64, 200, 700, 1800, 5000, 9000])
def test_rows_that_are_not_finite(backend, d, bad):
    x = rows(6, d, d)
    x[1, d - 1] = bad
    codes, scales = backend.quantize_rows(x)
    assert scales[1].isnan() and not codes[1].any() and backend.dequantize_rows(codes, scales)[1].isnan().all()
    keep = [0, 2, 3, 4, 5]
    assert scales[keep].isfinite().all()
    codes, scales, total, rstd = backend.rms_norm_int8(x, torch.zeros_like(x))
    assert scales[1].isnan() and rstd[1].isnan() and not codes[1].any() and scales[keep].isfinite().all()
    assert torch.equal(total[1, :-1], x[1, :-1])
    # finite, but the sum of squares is not
    x[1] = 1e25
    codes, scales, _, rstd = backend.rms_norm_int8(x)
    assert scales[1].isnan() and rstd[1].isnan() and scales[keep].isfinite().all()


def test_the_smallest_values(backend):
    """Rows of subnormals: the scale stays a normal number, nothing is flushed"""
    x = torch.tensor([[2.0 ** -126, -(2.0 ** -127), 2.0 ** -149, 0.0], [0.0] * 4, [3.0e38, -1.0, 1.0e37, 0.0]], device='cuda')
    codes, scales = backend.quantize_rows(x)
    assert scales.tolist()[:2] == [2.0 ** -126, 0.0]
    assert codes[0].tolist() == [1, 0, 0, 0] and codes[1].tolist() == [0] * 4 and codes[2].tolist() == [127, 0, 4, 0]  # -0.5 rounds to even


@pytest.mark.parametrize('power_of_two,weight', [(False, True), (True, False)])
@pytest.mark.parametrize('types', [('f', None), ('b', None), ('f', 'f'), ('f', 'b'), ('b', 'f'), ('b', 'b')])
@pytest.mark.parametrize('n,d', SIZES)
def test_rms_norm_int8(backend, n, d, types, power_of_two, weight):
    names = {'f': torch.float32, 'b': torch.bfloat16}
    x = rows(n, d, 11, names[types[0]])
    r = rows(n, d, 12, names[types[1]]) if types[1] else None
    w = torch.rand(d, device='cuda', generator=generator(3)) + 0.5 if weight else None
    codes, scales, total, rstd = backend.rms_norm_int8(x, r, w, EPS, power_of_two)
    h = x.double() if r is None else x.double() + r.double()
    if r is None:
        assert total is None
    else:
        assert torch.equal(total, (x.float() + r.float()).to(r.dtype))
    norm = (h.square().mean(1) + EPS).rsqrt()
    # the fp32 sum of h (u), its square (2 u), sums in chains of at most d / 32 + 32, quotient, sum and root: (d / 32 + 40) u
    unit = (d / 32 + 40) * U
    assert ((rstd.double() - norm).abs() <= unit * norm).all()
    y = h * norm[:, None] * (1.0 if w is None else w.double())
    largest = y.abs().amax(1)
    # the sum's own rounding: u (|x| + |r|) against the largest magnitude of the row
    cancel = 0 if r is None else ((x.double().abs() + r.double().abs()) * norm[:, None] * (1.0 if w is None else w.double())).amax(1) * U
    slack = (unit + 4 * U) * largest + cancel
    if power_of_two:
        live = largest > 0
        assert (torch.frexp(scales[live])[0] == 0.5).all()
        assert (scales.double() >= (largest - slack) / 127).all() and (scales.double() <= 2 * (largest + slack) / 127).all()
    else:
        assert ((scales.double() - largest / 127).abs() <= slack / 127 + U * largest).all()
    error = (codes.double() * scales.double()[:, None] - y).abs()
    assert (error <= scales.double()[:, None] * (0.5 + 127 * 4 * U) + slack[:, None]).all()


def test_rms_norm_of_zeros_and_of_no_rows(backend):
    x = torch.zeros(3, 40, device='cuda', dtype=torch.bfloat16)
    codes, scales, total, rstd = backend.rms_norm_int8(x, x.float(), None, 0.25)
    assert not codes.any() and not scales.any() and not total.any() and (rstd == 2).all() and total.dtype == torch.float32
    none = x[:0]
    codes, scales, total, rstd = backend.rms_norm_int8(none, none)
    assert codes.shape == (0, 40) and scales.shape == (0,) and total.shape == (0, 40) and rstd.shape == (0,)
    assert backend.quantize_rows(none)[0].shape == (0, 40) and backend.dequantize_rows(codes, scales).shape == (0, 40)
    assert backend.rms_norm_int8_backward(none, codes, scales, rstd).shape == (0, 40)
    w_codes, w_scales = backend.quantize_rows(torch.ones(8, 40, device='cuda'))
    assert backend.int8_linear(codes, scales, w_codes, w_scales).shape == (0, 8)
    grad_weight = torch.ones(8, 40, device='cuda')
    backend.int8_weight_grad(torch.zeros(0, 8, device='cuda', dtype=torch.bfloat16), codes, scales, grad_weight)
    assert (grad_weight == 1).all()


LINEAR = [(1, 1, 1), (1, 16, 8), (1, 1024, 1024), (2, 37, 5), (3, 4000, 130), (15, 283, 131), (16, 288, 257), (17, 64, 3), (64, 128, 64), (100, 96, 500),
          (127, 513, 96), (128, 256, 256), (129, 272, 300), (300, 1, 40), (1000, 2048, 24), (1111, 77, 1025), (4133, 283, 61), (20000, 256, 256)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('n,k,o', LINEAR)
def test_int8_linear(backend, n, k, o, dtype):
    codes, scales = code_rows(n, k, n + k, power_of_two=False)
    w_codes, w_scales = code_rows(o, k, o, power_of_two=False)
    bias = torch.randn(o, device='cuda', generator=generator(2)) if o % 2 else None
    relu = n % 3 != 0
    out = backend.int8_linear(codes, scales, w_codes, w_scales, bias, relu, dtype)
    assert out.dtype == dtype and out.shape == (n, o)
    # whole sums below 2^53 are exact in float64
    product = (codes.double() @ w_codes.double().t()) * scales.double()[:, None] * w_scales.double()
    wanted = product if bias is None else product + bias.double()
    # the integer's conversion, two products, the bias and the rounding of the result
    slack = 3 * U * product.abs() + U * wanted.abs() + (BF16 if dtype == torch.bfloat16 else U) * wanted.abs()
    wanted = wanted.clamp(min=0) if relu else wanted
    assert ((out.double() - wanted).abs() <= slack * (1 + 1e-3)).all()


def test_int8_linear_extremes(backend):
    """The largest sums (all codes -128 and 127, k = 131071), and rows and weights whose scale is NaN"""
    k = 131071
    codes = torch.full((3, k + 1), -128, device='cuda', dtype=torch.int8)[:, :k]
    codes[1] = 127
    one = torch.ones(3, device='cuda')
    out = backend.int8_linear(codes, one, codes, one, None, False, torch.float32)
    exact = torch.tensor([[16384.0, -16256.0, 16384.0], [-16256.0, 16129.0, -16256.0], [16384.0, -16256.0, 16384.0]], dtype=torch.float64) * k
    assert torch.equal(out.cpu(), exact.float())
    with pytest.raises(RuntimeError, match='ZipNeRF: int8_linear: more than 131071'):
        wide = torch.zeros(2, k + 1, device='cuda', dtype=torch.int8)
        backend.int8_linear(wide, one[:2], wide, one[:2])
    small = torch.ones(200, 64, device='cuda', dtype=torch.int8)
    scales, w_scales = torch.ones(200, device='cuda'), torch.ones(70, device='cuda')
    scales[150], w_scales[69] = float('nan'), float('nan')
    out = backend.int8_linear(small, scales, small[:70], w_scales, None, True)
    bad = out.isnan()
    assert bad[150].all() and bad[:, 69].all() and bad.sum() == 70 + 199


def test_int8_linear_reads_row_slices(backend):
    """Codes as rows and 16-column slices of larger buffers; output bits do not depend on the other rows"""
    codes, scales = code_rows(400, 512, 8)
    w_codes, w_scales = code_rows(96, 512, 9)
    part = backend.int8_linear(codes[37:301, 32:331], scales[37:301], w_codes[5:70, 32:331], w_scales[5:70], None, False, torch.float32)
    whole = backend.int8_linear(codes[:, 32:331].contiguous().new_zeros(400, 304)[:, :299].copy_(codes[:, 32:331]), scales,
                                w_codes.new_zeros(96, 304)[:, :299].copy_(w_codes[:, 32:331]), w_scales, None, False, torch.float32)
    assert torch.equal(part, whole[37:301, 5:70])
    with pytest.raises(RuntimeError, match='16-byte aligned'):
        backend.int8_linear(codes[:, 8:40], scales, w_codes[:, 8:40], w_scales)


WEIGHT_GRAD = [(1, 1, 1), (1, 16, 8), (5, 37, 3), (31, 64, 64), (64, 256, 256), (100, 283, 61), (129, 128, 128), (1000, 96, 300), (4133, 283, 61),
               (4133, 56, 64), (3000, 700, 520), (70000, 256, 256), (70001, 40, 257)]


@pytest.mark.parametrize('power_of_two', [True, False])
@pytest.mark.parametrize('n,k,o', WEIGHT_GRAD)
def test_int8_weight_grad(backend, n, k, o, power_of_two):
    codes, scales = code_rows(n, k, n + k, power_of_two)
    g = rows(n, o, o, torch.bfloat16)
    before = torch.randn(o, k, device='cuda', generator=generator(4))
    grad_weight, grad_bias = before.clone(), torch.ones(o, device='cuda')
    backend.int8_weight_grad(g, codes, scales, grad_weight, grad_bias)
    x = codes.double() * scales.double()[:, None]
    wanted, terms = g.double().t() @ x + before.double(), g.double().abs().t() @ x.abs()
    # products of bf16 numbers are exact in fp32; sums of n of them in fp32, in chains of at most n / 8 + 1000 steps that may
    # truncate (2 u each); a scale that is no power of two rounds each value to bf16 once
    unit = min(n, n / 8 + 1000) * 2 * U + (0 if power_of_two else BF16)
    assert ((grad_weight.double() - wanted).abs() <= unit * terms + 2 * U * (wanted.abs() + before.abs())).all()
    bias, bias_terms = g.double().sum(0) + 1, g.double().abs().sum(0)
    assert ((grad_bias.double() - bias).abs() <= min(n, n / 8 + 1000) * U * bias_terms + 2 * U * (bias.abs() + 1)).all()
    # without the bias, and again: the same bits
    again = before.clone()
    backend.int8_weight_grad(g, codes, scales, again)
    assert torch.equal(again, grad_weight)
    assert backend.int8_status(torch.device('cuda:0')).item() == 0


@pytest.mark.parametrize('o,stride,offset', [(64, 72, 0), (64, 67, 0), (64, 64, 1), (61, 61, 0), (61, 64, 0), (300, 301, 3)])
def test_int8_weight_grad_reads_strided_gradients(backend, o, stride, offset):
    """Gradients on and off the 16-byte grid: the sums of the definition"""
    codes, scales = code_rows(777, 130, 1)
    g = rows(777, o, 2, torch.bfloat16, stride, offset)
    grad_weight, grad_bias = torch.zeros(o, 130, device='cuda'), torch.zeros(o, device='cuda')
    backend.int8_weight_grad(g, codes, scales, grad_weight, grad_bias)
    x = codes.double() * scales.double()[:, None]
    assert ((grad_weight.double() - g.double().t() @ x).abs() <= 777 * 2 * U * (g.double().abs().t() @ x.abs())).all()
    assert ((grad_bias.double() - g.double().sum(0)).abs() <= 777 * U * g.double().abs().sum(0)).all()


def test_int8_weight_grad_is_the_slope_of_int8_linear(backend):
    """Differences: moving one weight code by two steps moves the loss by two steps of the gradient (the layer is linear)"""
    n, k, o = 150, 70, 40
    codes, scales = code_rows(n, k, 1)
    w_codes, w_scales = code_rows(o, k, 2)
    w_codes.clamp_(-126, 126)
    w_scales.fill_(0.5)
    g = rows(n, o, 3, torch.bfloat16)
    grad_weight = torch.zeros(o, k, device='cuda')
    backend.int8_weight_grad(g, codes, scales, grad_weight)
    for at in [(0, 0), (17, 33), (39, 69)]:
        losses = []
        for step in (1, -1):
            moved = w_codes.new_zeros(o, 80)[:, :k].copy_(w_codes)
            moved[at] += step
            out = backend.int8_linear(codes, scales, moved, w_scales, None, False, torch.float32).double()
            losses.append((out * g.double()).sum())
        slope = (losses[0] - losses[1]) / (2 * 0.5)
        terms = (g.double()[:, at[0]].abs() * (codes.double()[:, at[1]] * scales.double()).abs()).sum()
        # sums below 2^24 with power-of-two scales: the layer's outputs are exact, so only the gradient's own sum rounds
        assert (grad_weight[at].double() - slope).abs() <= n * 2 * U * terms


@pytest.mark.parametrize('types', [('f', None), ('b', None), ('f', 'f'), ('f', 'b'), ('b', 'f'), ('b', 'b')])
@pytest.mark.parametrize('n,d', SIZES)
def test_rms_norm_int8_backward(backend, n, d, types):
    names = {'f': torch.float32, 'b': torch.bfloat16}
    g = rows(n, d, 1, names[types[0]])
    gr = rows(n, d, 2, names[types[1]]) if types[1] else None
    codes, scales = code_rows(n, d, 3, power_of_two=False)
    rstd = torch.rand(n, device='cuda', generator=generator(4)) + 0.1
    out = backend.rms_norm_int8_backward(g, codes, scales, rstd, gr)
    y = codes.double() * scales.double()[:, None]
    mean = (g.double() * y).mean(1, keepdim=True)
    terms = (g.double() * y).abs().mean(1, keepdim=True)
    wanted = rstd.double()[:, None] * (g.double() - y * mean)
    # y (u), the sum of products in chains of at most d / 32 + 32, the quotient; then the difference, the product, the sum
    slack = rstd.double()[:, None] * ((d / 32 + 40) * U * y.abs() * terms + 4 * U * (g.double().abs() + (y * mean).abs()))
    if gr is not None:
        wanted = wanted + gr.double()
        slack = slack + U * gr.double().abs()
    assert out.dtype == (g.dtype if gr is None else gr.dtype)
    slack = slack + (BF16 if out.dtype == torch.bfloat16 else U) * (wanted.abs() + slack)
    assert ((out.double() - wanted).abs() <= slack * (1 + 1e-3)).all()


@pytest.mark.parametrize('stride,offset', [(104, 0), (99, 0), (96, 3)])
def test_rms_norm_int8_backward_reads_strided_gradients(backend, stride, offset):
    codes, scales = code_rows(23, 96, 3)
    rstd = torch.rand(23, device='cuda') + 0.1
    g, gr = rows(23, 96, 1, torch.bfloat16, stride, offset), rows(23, 96, 2, torch.float32, stride, offset)
    a, b = backend.rms_norm_int8_backward(g, codes, scales, rstd, gr), backend.rms_norm_int8_backward(g.contiguous(), codes, scales, rstd, gr.contiguous())
    # the dot product's order depends on the access width
    y = codes.double().abs() * scales.double()[:, None]
    slack = rstd.double()[:, None] * (100 * U * y * (g.double().abs() * y).mean(1, keepdim=True) + 8 * U * g.double().abs()) + 4 * U * gr.double().abs()
    assert ((a.double() - b.double()).abs() <= slack).all()


def test_rms_norm_int8_backward_is_the_slope_of_the_norm(backend):
    """Differences of the norm in 64 bits, at rows that the codes hold exactly: with y = codes * scale, rstd = 1 and
    eps = 1 - mean(y^2), the row h = y has the norm y."""
    n, d = 6, 90
    codes, _ = code_rows(n, d, 5)
    codes[2::5] = codes[0]
    scales = torch.full((n,), 2.0 ** -7, device='cuda')
    y = codes.double() * 2.0 ** -7
    eps = 1 - y.square().mean(1)
    assert (eps > 0).all()
    g = torch.randn(n, d, device='cuda', generator=generator(6))
    out = backend.rms_norm_int8_backward(g, codes, scales, torch.ones(n, device='cuda'))
    direction = torch.randn(n, d, device='cuda', generator=generator(7), dtype=torch.float64)

    def loss(h):
        return (g.double() * h * (h.square().mean(1) + eps).rsqrt()[:, None]).sum(1)

    step = 1e-5
    slope = (loss(y + step * direction) - loss(y - step * direction)) / (2 * step)
    # third-order terms of the difference (step^2) and the kernel's roundings, against sums of d terms of size about 1
    assert ((out.double() * direction).sum(1) - slope).abs().max() <= 1e-7 + d * 16 * U * 4


def test_operators_run_on_the_current_stream(backend):
    """On another stream, behind work that the inputs depend on"""
    stream = torch.cuda.Stream()
    x = rows(3000, 512, 1, torch.bfloat16)
    w_codes, w_scales = backend.quantize_rows(rows(256, 512, 2))
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        late = x
        for _ in range(20):
            late = late * 1.0
        codes, scales, total, rstd = backend.rms_norm_int8(late, late, None, EPS, True)
        out = backend.int8_linear(codes, scales, w_codes, w_scales)
        grad = torch.zeros(256, 512, device='cuda')
        backend.int8_weight_grad(out, codes, scales, grad)
    stream.synchronize()
    codes2, scales2, total2, rstd2 = backend.rms_norm_int8(x, x, None, EPS, True)
    out2 = backend.int8_linear(codes2, scales2, w_codes, w_scales)
    grad2 = torch.zeros(256, 512, device='cuda')
    backend.int8_weight_grad(out2, codes2, scales2, grad2)
    assert torch.equal(codes, codes2) and torch.equal(scales, scales2) and torch.equal(out, out2) and torch.equal(grad, grad2)


def test_offsets_past_32_bits(backend):
    """More than 2^31 elements: the last rows of the operators equal those of a call on these rows alone"""
    n, d = 8_400_011, 256
    x = torch.zeros(n, d, device='cuda', dtype=torch.bfloat16)
    x[-3:] = rows(3, d, 1, torch.bfloat16)
    codes, scales, total, rstd = backend.rms_norm_int8(x, x, None, EPS, True)
    last = backend.rms_norm_int8(x[-3:], x[-3:], None, EPS, True)
    assert torch.equal(codes[-3:], last[0]) and torch.equal(scales[-3:], last[1]) and torch.equal(total[-3:], last[2])
    del total
    w_codes, w_scales = code_rows(264, d, 2)
    out = backend.int8_linear(codes, scales, w_codes, w_scales)
    assert torch.equal(out[-3:], backend.int8_linear(last[0], last[1], w_codes, w_scales)) and not out[:-3].any()
    grad_weight, grad_bias = torch.zeros(264, d, device='cuda'), torch.zeros(264, device='cuda')
    backend.int8_weight_grad(out, codes, scales, grad_weight, grad_bias)
    y = last[0].double() * last[1].double()[:, None]
    wanted = out[-3:].double().t() @ y
    assert ((grad_weight.double() - wanted).abs() <= 16 * U * (out[-3:].double().abs().t() @ y.abs())).all()
    assert ((grad_bias.double() - out[-3:].double().sum(0)).abs() <= 8 * U * out[-3:].double().abs().sum(0)).all()
    del out
    back = backend.rms_norm_int8_backward(x, codes, scales, rstd, x)
    assert torch.equal(back[-3:], backend.rms_norm_int8_backward(x[-3:], last[0], last[1], last[3], x[-3:])) and not back[:-3].any()
    del back
    assert torch.equal(backend.dequantize_rows(codes, scales)[-3:], backend.dequantize_rows(last[0], last[1]))


def test_the_sum_and_the_gradient_in_place(backend):
    """Through the C ABI: the sum over the residual's own memory, the norm's gradient over the upstream gradient's"""
    import ctypes

    from zipnerf_b200 import capi
    lib = capi.load()
    stream = torch.cuda.current_stream().cuda_stream
    for n, d in [(37, 256), (5, 99), (3, 3000), (2, 9000)]:
        x, r = rows(n, d, 1, torch.bfloat16), rows(n, d, 2)
        wanted = backend.rms_norm_int8(x, r, None, EPS)
        codes = torch.empty(n, (d + 15) // 16 * 16, device='cuda', dtype=torch.int8)[:, :d]
        scales, rstd, total = torch.empty_like(wanted[1]), torch.empty_like(wanted[3]), r.clone()
        args = capi.zf_rms_norm_int8_args(x.data_ptr(), capi.ZF_BFLOAT16, d, total.data_ptr(), capi.ZF_FLOAT32, d, None, n, d, EPS, 0, codes.data_ptr(),
                                          codes.stride(0), scales.data_ptr(), total.data_ptr(), d, rstd.data_ptr())
        capi.check(lib.zf_rms_norm_int8(ctypes.byref(args), stream))
        assert all(torch.equal(a, b) for a, b in zip((codes, scales, total, rstd), wanted))
        g = rows(n, d, 3)
        wanted = backend.rms_norm_int8_backward(g, codes, scales, rstd, None)
        args = capi.zf_rms_norm_int8_backward_args(g.data_ptr(), capi.ZF_FLOAT32, d, codes.data_ptr(), codes.stride(0), scales.data_ptr(), rstd.data_ptr(),
                                                   None, 0, 0, n, d, g.data_ptr(), d)
        capi.check(lib.zf_rms_norm_int8_backward(ctypes.byref(args), stream))
        assert torch.equal(g, wanted)


def test_refusals(backend):
    x = rows(4, 32, 1)
    codes, scales = backend.quantize_rows(x)
    with pytest.raises(RuntimeError, match='ZipNeRF: x must be float32 or bfloat16'):
        backend.quantize_rows(x.half())
    with pytest.raises(RuntimeError, match='ZipNeRF: x has an invalid layout'):
        backend.quantize_rows(x.t())
    with pytest.raises(RuntimeError, match='ZipNeRF: x must be a 2D cuda tensor'):
        backend.quantize_rows(x[0])
    with pytest.raises(RuntimeError, match='ZipNeRF: the output must be'):
        backend.dequantize_rows(codes, scales, torch.float16)
    with pytest.raises(RuntimeError, match='ZipNeRF: scales has the wrong size'):
        backend.dequantize_rows(codes, scales[:3])
    with pytest.raises(RuntimeError, match='ZipNeRF: codes must be int8'):
        backend.dequantize_rows(x, scales)
    with pytest.raises(RuntimeError, match='ZipNeRF: residual has an invalid layout'):
        backend.rms_norm_int8(x, x[:3])
    with pytest.raises(RuntimeError, match='ZipNeRF: weight has the wrong size'):
        backend.rms_norm_int8(x, None, scales)
    with pytest.raises(RuntimeError, match='ZipNeRF: rms_norm_int8: eps must be positive'):
        backend.rms_norm_int8(x, None, None, 0.0)
    with pytest.raises(RuntimeError, match='ZipNeRF: weight_codes has an invalid layout'):
        backend.int8_linear(codes, scales, codes[:, :16], scales)
    with pytest.raises(RuntimeError, match='ZipNeRF: grad must be bfloat16'):
        backend.int8_weight_grad(x, codes, scales, torch.zeros(32, 32, device='cuda'))
    with pytest.raises(RuntimeError, match='ZipNeRF: grad_weight has the wrong size'):
        backend.int8_weight_grad(x.bfloat16(), codes, scales, torch.zeros(32, 33, device='cuda'))
    with pytest.raises(RuntimeError, match='16-byte aligned'):
        backend.dequantize_rows(torch.zeros(4, 20, dtype=torch.int8, device='cuda'), scales)
