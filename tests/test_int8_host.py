"""The 8-bit row operators' argument checks (include/zf_int8.h), which run before any launch: sizes, layouts, alignment,
types, workspaces; and the binding's refusals of tensors on the CPU. No GPU needed."""
from __future__ import annotations

import ctypes

import pytest
import torch

FAKE = 1 << 20  # a 16-byte aligned address that is never dereferenced


def lib():
    from zipnerf_b200 import capi
    return capi, capi.load()


def refused(name, args, message):
    capi, library = lib()
    assert getattr(library, name)(ctypes.byref(args), None) == capi.ZF_ERROR_INVALID_ARGUMENT
    assert message.encode() in library.zf_last_error(), library.zf_last_error()


def fields(base, **changed):
    return type(base)(*[changed.get(name, getattr(base, name)) for name, _ in base._fields_])


def test_quantize_rows_refusals():
    capi, library = lib()
    good = capi.zf_quantize_rows_args(FAKE, capi.ZF_BFLOAT16, 256, 10, 256, 0, FAKE, 256, FAKE)
    for changed, message in [(dict(n=-1), 'sizes'), (dict(d=0), 'sizes'), (dict(n=1 << 31), 'sizes'), (dict(x=None), 'invalid x'),
                             (dict(x=FAKE + 1), 'invalid x'), (dict(x_dtype=7), 'invalid x'), (dict(x_stride=255), 'invalid x'),
                             (dict(codes=None), '16-byte'), (dict(codes=FAKE + 8), '16-byte'), (dict(codes_stride=264), '16-byte'),
                             (dict(codes_stride=240), '16-byte'), (dict(scales=None), '16-byte')]:
        refused('zf_quantize_rows', fields(good, **changed), message)
    assert library.zf_quantize_rows(None, None) == capi.ZF_ERROR_INVALID_ARGUMENT
    assert library.zf_quantize_rows(ctypes.byref(fields(good, n=0, x=None, codes=None)), None) == capi.ZF_OK


def test_dequantize_rows_refusals():
    capi, library = lib()
    good = capi.zf_dequantize_rows_args(FAKE, 256, FAKE, 10, 256, FAKE, capi.ZF_BFLOAT16, 256)
    for changed, message in [(dict(d=-3), 'sizes'), (dict(codes=FAKE + 4), '16-byte'), (dict(codes_stride=257), '16-byte'), (dict(scales=None), '16-byte'),
                             (dict(out=None), 'output'), (dict(out_dtype=2), 'output'), (dict(out_stride=200), 'output')]:
        refused('zf_dequantize_rows', fields(good, **changed), message)
    assert library.zf_dequantize_rows(ctypes.byref(fields(good, n=0, out=None)), None) == capi.ZF_OK


def test_rms_norm_int8_refusals():
    capi, library = lib()
    good = capi.zf_rms_norm_int8_args(FAKE, capi.ZF_BFLOAT16, 256, FAKE, capi.ZF_FLOAT32, 256, FAKE, 10, 256, 1e-6, 0, FAKE, 256, FAKE, FAKE, 256, FAKE)
    for changed, message in [(dict(d=0), 'sizes'), (dict(eps=0.0), 'eps'), (dict(eps=-1e-6), 'eps'), (dict(eps=float('nan')), 'eps'),
                             (dict(eps=float('inf')), 'eps'), (dict(sum=None), 'go together'), (dict(residual=None), 'go together'),
                             (dict(x_stride=3), 'invalid x'), (dict(residual_dtype=9), 'residual'), (dict(residual=FAKE + 2), 'residual'),
                             (dict(sum_stride=10), 'residual'), (dict(codes_stride=250), '16-byte'), (dict(scales=None), '16-byte')]:
        refused('zf_rms_norm_int8', fields(good, **changed), message)
    assert library.zf_rms_norm_int8(ctypes.byref(fields(good, n=0)), None) == capi.ZF_OK


def test_rms_norm_int8_backward_refusals():
    capi, library = lib()
    good = capi.zf_rms_norm_int8_backward_args(FAKE, capi.ZF_BFLOAT16, 256, FAKE, 256, FAKE, FAKE, FAKE, capi.ZF_BFLOAT16, 256, 10, 256, FAKE, 256)
    for changed, message in [(dict(n=-5), 'sizes'), (dict(grad=None), 'grad'), (dict(grad_dtype=5), 'grad'), (dict(grad_residual_stride=5), 'grad_residual'),
                             (dict(codes=FAKE + 1), '16-byte'), (dict(rstd=None), '16-byte'), (dict(grad_x=None), 'grad_x'), (dict(grad_x_stride=100), 'grad_x')]:
        refused('zf_rms_norm_int8_backward', fields(good, **changed), message)
    assert library.zf_rms_norm_int8_backward(ctypes.byref(fields(good, n=0)), None) == capi.ZF_OK


def test_int8_linear_refusals():
    capi, library = lib()
    good = capi.zf_int8_linear_args(FAKE, 256, FAKE, FAKE, 256, FAKE, FAKE, 10, 256, 64, 0, FAKE, capi.ZF_BFLOAT16, 64, FAKE)
    for changed, message in [(dict(out=0), 'sizes'), (dict(in_=0), 'sizes'), (dict(n=(1 << 31) - 1), 'sizes'), (dict(out=1 << 31), 'sizes'),
                             (dict(in_=131072, codes_stride=1 << 18, weight_stride=1 << 18), 'overflow'), (dict(codes_stride=248), '16-byte'),
                             (dict(weight_codes=FAKE + 2), '16-byte'), (dict(weight_stride=128), '16-byte'), (dict(weight_scales=None), 'scales'),
                             (dict(status=None), 'status'), (dict(output=None), 'output'), (dict(output_dtype=3), 'output'), (dict(output_stride=60), 'output')]:
        refused('zf_int8_linear', fields(good, **changed), message)
    assert library.zf_int8_linear(ctypes.byref(fields(good, n=0)), None) == capi.ZF_OK


def test_int8_weight_grad_refusals():
    capi, library = lib()
    size = library.zf_int8_weight_grad_workspace_size(1000, 256, 64)
    assert size >= 0 and library.zf_int8_weight_grad_workspace_size(0, 256, 64) == 0
    good = capi.zf_int8_weight_grad_args(FAKE, 64, FAKE, 256, FAKE, 1000, 256, 64, FAKE, FAKE, FAKE, size, FAKE)
    for changed, message in [(dict(in_=0), 'sizes'), (dict(n=1 << 31), 'sizes'), (dict(grad=None), 'grad'), (dict(grad_stride=63), 'grad'),
                             (dict(codes_stride=255), '16-byte'), (dict(scales=None), 'scales'), (dict(grad_weight=None), 'grad_weight'),
                             (dict(status=None), 'status'), (dict(workspace_bytes=size - 1), 'workspace'), (dict(workspace=FAKE + 4), 'workspace')]:
        refused('zf_int8_weight_grad', fields(good, **changed), message)
    assert library.zf_int8_weight_grad(ctypes.byref(fields(good, n=0)), None) == capi.ZF_OK


def test_the_binding_refuses_cpu_tensors():
    import ZipNeRFCudaBackend as backend
    x, codes, scales = torch.zeros(4, 32), torch.zeros(4, 32, dtype=torch.int8), torch.zeros(4)
    for call in [lambda: backend.quantize_rows(x), lambda: backend.dequantize_rows(codes, scales), lambda: backend.rms_norm_int8(x),
                 lambda: backend.rms_norm_int8_backward(x, codes, scales, scales), lambda: backend.int8_linear(codes, scales, codes, scales),
                 lambda: backend.int8_weight_grad(x.bfloat16(), codes, scales, torch.zeros(32, 32))]:
        with pytest.raises(RuntimeError, match='ZipNeRF: '):
            call()


def test_the_status_is_a_cuda_device_s():
    import ZipNeRFCudaBackend as backend
    with pytest.raises(RuntimeError, match='ZipNeRF: the status belongs to a cuda device'):
        backend.int8_status(torch.device('cpu'))
    with pytest.raises(RuntimeError, match='ZipNeRF: no such cuda device'):
        backend.int8_status(torch.device('cuda', 63))


def test_every_operator_is_reachable_by_name():
    import ZipNeRFCudaBackend
    from ZipNeRFCudaBackend import _C
    from ZipNeRFCudaBackend.torch_bindings import pipeline
    for name in ['quantize_rows', 'dequantize_rows', 'rms_norm_int8', 'rms_norm_int8_backward', 'int8_linear', 'int8_weight_grad', 'int8_status']:
        assert getattr(ZipNeRFCudaBackend, name) is getattr(_C, name) is getattr(pipeline, name)
        assert name in ZipNeRFCudaBackend.__all__
