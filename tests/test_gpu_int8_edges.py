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
