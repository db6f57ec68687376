"""The 8-bit row operators (include/zf_int8.h) on the GPU at the edges of their tiles, layouts and values, against their
definitions in 64 bits. Tolerances follow from the operators' roundings (u = 2^-24, one fp32 rounding)."""
from __future__ import annotations

import pytest
import torch

from test_gpu_int8 import BF16, EPS, U, backend, code_rows, generator, rows  # noqa: F401  (backend is a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('o', [1, 3, 9, 61, 127, 129, 257])
@pytest.mark.parametrize('n', [129, 130, 140, 193])
def test_weight_grad_of_narrow_odd_layers(backend, n, o):  # noqa: F811
    """Gradients off the 16-byte grid with whole 64-sample stages between the first and the last, in a tensor that ends with
    its last element: a pair's second CTA has no columns up to 128 outputs, one at 129"""
    k = 70
    codes, scales = code_rows(n, k, n + o)
    g = rows(n, o, o, torch.bfloat16)
    grad_weight, grad_bias = torch.zeros(o, k, device='cuda'), torch.zeros(o, device='cuda')
    backend.int8_weight_grad(g, codes, scales, grad_weight, grad_bias)
    x = codes.double() * scales.double()[:, None]
    # exact products; sums of n terms in fp32 that may truncate (2 u a step)
    assert ((grad_weight.double() - g.double().t() @ x).abs() <= n * 2 * U * (g.double().abs().t() @ x.abs())).all()
    assert ((grad_bias.double() - g.double().sum(0)).abs() <= n * U * g.double().abs().sum(0)).all()
    assert backend.int8_status(g.device).item() == 0


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('n,k,o', [(33, 16, 1), (33, 16, 3), (65, 40, 7), (97, 33, 5), (129, 40, 7), (161, 16, 1), (289, 16, 3), (257, 40, 1)])
def test_linear_with_a_last_group_of_few_bytes(backend, n, k, o, dtype):  # noqa: F811
    """Outputs whose rows lie back to back off the 16-byte grid, where the last 32-row group holds one row: 2 to 28 bytes"""
    codes, scales = code_rows(n, k, n + k, power_of_two=False)
    w_codes, w_scales = code_rows(o, k, o, power_of_two=False)
    bias = torch.randn(o, device='cuda', generator=generator(2))
    out = backend.int8_linear(codes, scales, w_codes, w_scales, bias, False, dtype)
    product = (codes.double() @ w_codes.double().t()) * scales.double()[:, None] * w_scales.double()
    wanted = product + bias.double()
    # the integer's conversion, two products, the bias and the rounding of the result
    slack = 3 * U * product.abs() + U * wanted.abs() + (BF16 if dtype == torch.bfloat16 else U) * wanted.abs()
    assert ((out.double() - wanted).abs() <= slack * (1 + 1e-3)).all()
    assert backend.int8_status(codes.device).item() == 0


@pytest.mark.parametrize('n,d', [(1001, 40), (4133, 256), (3001, 512), (2501, 283), (777, 1000), (501, 4096), (301, 8000), (33, 9001)])
def test_outputs_over_inputs_with_teams_past_the_last_row(backend, n, d):  # noqa: F811
    """Through the C ABI, where many teams work at once and the last of them has rows past the end: the sum over the
    residual, the gradient over either upstream gradient, with the bits of a call into memory of its own"""
    import ctypes

    from zipnerf_b200 import capi
    lib = capi.load()
    stream = torch.cuda.current_stream().cuda_stream
    for dtype, tag in ((torch.float32, capi.ZF_FLOAT32), (torch.bfloat16, capi.ZF_BFLOAT16)):
        x, r = rows(n, d, 1, torch.bfloat16), rows(n, d, 2, dtype)
        wanted = backend.rms_norm_int8(x, r, None, EPS, True)
        codes = torch.empty(n, (d + 15) // 16 * 16, device='cuda', dtype=torch.int8)[:, :d]
        scales, rstd, total = torch.empty_like(wanted[1]), torch.empty_like(wanted[3]), r.clone()
        args = capi.zf_rms_norm_int8_args(x.data_ptr(), capi.ZF_BFLOAT16, d, total.data_ptr(), tag, d, None, n, d, EPS, 1, codes.data_ptr(),
                                          codes.stride(0), scales.data_ptr(), total.data_ptr(), d, rstd.data_ptr())
        capi.check(lib.zf_rms_norm_int8(ctypes.byref(args), stream))
        assert all(torch.equal(a, b) for a, b in zip((codes, scales, total, rstd), wanted))
        g, gr = rows(n, d, 3, dtype), rows(n, d, 4, dtype)
        wanted = backend.rms_norm_int8_backward(g, codes, scales, rstd, gr)
        for over in (0, 1):
            operands = [g.clone(), gr.clone()]
            out = operands[over]
            args = capi.zf_rms_norm_int8_backward_args(operands[0].data_ptr(), tag, d, codes.data_ptr(), codes.stride(0), scales.data_ptr(), rstd.data_ptr(),
                                                       operands[1].data_ptr(), tag, d, n, d, out.data_ptr(), d)
            capi.check(lib.zf_rms_norm_int8_backward(ctypes.byref(args), stream))
            assert torch.equal(out, wanted)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('n,d', [(20000, 256), (4000, 1000), (4001, 283), (3000, 98), (500, 4097), (301, 5002), (100, 9001)])
def test_codes_are_the_rounded_quotients(backend, n, d, dtype):  # noqa: F811
    """Without power-of-two scales too: codes = the fp32 quotient x / scale to the nearest integer, ties to even. Rows hold
    many values at and beside a half step, where another rounding of the quotient gives the neighbouring code."""
    x = torch.randn(n, d, device='cuda', generator=generator(d))
    half_steps = torch.randint(-127, 127, (n, d), device='cuda', generator=generator(n)).float() + 0.5
    largest = x.abs().amax(1, keepdim=True)
    x[:, ::2] = (half_steps * (largest / 127))[:, ::2].clamp(-largest, largest)
    x = x.to(dtype)
    codes, scales = backend.quantize_rows(x, False)
    # a 64-bit quotient of fp32 numbers rounded to fp32 is the fp32 quotient: 53 >= 2 * 24 + 2 bits
    assert torch.equal(scales, (x.double().abs().amax(1) / 127).float())
    assert torch.equal(codes.float(), torch.round((x.double() / scales.double()[:, None]).float()))


@pytest.mark.parametrize('n', [20, 150])
def test_the_largest_sums_on_the_tensor_cores(backend, n):  # noqa: F811
    """Codes -128 and 127 over 131,071 inputs in tiles of one CTA and of a pair: sums of up to 2^31 - 16,384, exact"""
    k = 131071
    codes = torch.full((n, k + 1), -128, device='cuda', dtype=torch.int8)[:, :k]
    codes[1::3] = 127
    w_codes = torch.full((33, k + 1), -128, device='cuda', dtype=torch.int8)[:, :k]
    w_codes[::2] = 127
    scales, w_scales = torch.ones(n, device='cuda'), torch.ones(33, device='cuda')
    out = backend.int8_linear(codes, scales, w_codes, w_scales, None, False, torch.float32)
    exact = codes[:, :1].double() * w_codes[:, 0].double() * k  # every input has the same codes
    assert torch.equal(out, exact.float())
    assert backend.int8_status(codes.device).item() == 0


def test_operators_in_a_captured_graph(backend):  # noqa: F811
    """A forward and backward captured once and replayed on other inputs: the bits of plain calls, the weight gradient's
    early-launched join among them"""
    n, d, o = 3000, 256, 131
    x, g = rows(n, d, 1, torch.bfloat16), rows(n, o, 2, torch.bfloat16)
    w_codes, w_scales = code_rows(o, d, 3, power_of_two=False)
    grad_weight, grad_bias = torch.zeros(o, d, device='cuda'), torch.zeros(o, device='cuda')

    def step():
        codes, scales, total, rstd = backend.rms_norm_int8(x, x, None, EPS, True)
        out = backend.int8_linear(codes, scales, w_codes, w_scales, None, True)
        grad_weight.zero_()
        grad_bias.zero_()
        backend.int8_weight_grad(g, codes, scales, grad_weight, grad_bias)
        back = backend.rms_norm_int8_backward(total, codes, scales, rstd, x)
        return [codes, scales, total, rstd, out, back, grad_weight, grad_bias]

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (4, 5):
        x.copy_(rows(n, d, seed, torch.bfloat16))
        g.copy_(rows(n, o, seed + 2, torch.bfloat16))
        graph.replay()
        replayed = [t.clone() for t in captured]
        for got, wanted in zip(replayed, step()):
            assert torch.equal(got, wanted)
    del graph
