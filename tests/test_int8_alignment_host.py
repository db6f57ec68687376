"""The 8-bit row operators' C entries (include/zf_int8.h) refuse pointers off their element's alignment, which would fault on
the device, before any launch. No GPU needed."""
from __future__ import annotations

import ctypes

import pytest

from test_int8_host import FAKE, fields, refused


def good(name):
    from zipnerf_b200 import capi
    b, f = capi.ZF_BFLOAT16, capi.ZF_FLOAT32
    return {'zf_quantize_rows': lambda: capi.zf_quantize_rows_args(FAKE, b, 256, 10, 256, 0, FAKE, 256, FAKE),
            'zf_dequantize_rows': lambda: capi.zf_dequantize_rows_args(FAKE, 256, FAKE, 10, 256, FAKE, b, 256),
            'zf_rms_norm_int8': lambda: capi.zf_rms_norm_int8_args(FAKE, b, 256, FAKE, f, 256, FAKE, 10, 256, 1e-6, 0, FAKE, 256, FAKE, FAKE, 256, FAKE),
            'zf_rms_norm_int8_backward': lambda: capi.zf_rms_norm_int8_backward_args(FAKE, b, 256, FAKE, 256, FAKE, FAKE, FAKE, b, 256, 10, 256, FAKE, 256),
            'zf_int8_linear': lambda: capi.zf_int8_linear_args(FAKE, 256, FAKE, FAKE, 256, FAKE, FAKE, 10, 256, 64, 0, FAKE, b, 64, FAKE),
            'zf_int8_weight_grad': lambda: capi.zf_int8_weight_grad_args(FAKE, 64, FAKE, 256, FAKE, 1000, 256, 64, FAKE, FAKE, FAKE, 1 << 40, FAKE)}[name]()


POINTERS = {'zf_quantize_rows': ['scales'], 'zf_dequantize_rows': ['scales'], 'zf_rms_norm_int8': ['scales', 'weight', 'rstd'],
            'zf_rms_norm_int8_backward': ['scales', 'rstd'], 'zf_int8_linear': ['scales', 'weight_scales', 'bias', 'status'],
            'zf_int8_weight_grad': ['grad', 'scales', 'grad_weight', 'grad_bias', 'status']}


@pytest.mark.parametrize('name,pointer', [(name, pointer) for name, pointers in POINTERS.items() for pointer in pointers])
def test_misaligned_pointers_are_refused(name, pointer):
    for offset in (1,) if pointer == 'grad' else (1, 2):
        refused(name, fields(good(name), **{pointer: FAKE + offset}), 'misaligned')
