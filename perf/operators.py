"""Cases of the 8-bit row operators: the add + RMS norm with 8-bit output, the 8-bit linear layer, 8-bit activation
checkpoints, and the two backward passes that read them (a linear layer's weight gradient, the norm's input gradient).

All of them share one format, int8 rows: codes (int8 [n, d], row stride a multiple of 16) and one fp32 scale per row;
the values are codes * scale. `own = False` computes every operator from elementary torch operations in fp32, rounded
once at the end; `own = True` calls the framework's operators. Codes are returned as the values they stand for (bf16)."""
import math
import sys
from pathlib import Path

import torch

own = False

EPS = 1e-6
SAMPLES = 2097152  # NeRF-level samples of one training step: 65,536 rays x 32 intervals
TYPES = {'bf16': torch.bfloat16, 'f32': torch.float32}


def listed():
    return [
        # the norm over the 32 samples of a single ray: a call that does almost nothing, where latency counts
        dict(name='norm one ray', op='norm', n=32, d=256, type='bf16', residual=True, weight=True, pow2=False),
        # the norm over a training step's samples at the view layers' width, codes that the backward will read
        dict(name='norm training batch', op='norm', n=SAMPLES, d=256, type='bf16', residual=True, weight=False, pow2=True),
        # one row through a 1024-wide layer: the weights' bytes and latency
        dict(name='linear one row', op='linear', n=1, k=1024, o=1024, type='bf16', bias=True, relu=False),
        # a view layer of the training batch, 256 to 256 with ReLU
        dict(name='linear training batch', op='linear', n=SAMPLES, k=256, o=256, type='bf16', bias=True, relu=True),
        # a wide layer, bound by arithmetic
        dict(name='linear wide', op='linear', n=8192, k=4096, o=4096, type='bf16', bias=False, relu=False),
        # ragged everywhere: 283 inputs (bottleneck 256 + encoded direction 27), odd rows and outputs, fp32 out
        dict(name='linear ragged', op='linear', n=57003, k=283, o=131, type='f32', bias=True, relu=True),
        # storing and restoring the activations of a training step's layer
        dict(name='checkpoint training batch', op='checkpoint', n=SAMPLES, d=256, type='bf16', pow2=True),
        # the same on a chunk of an odd width in fp32
        dict(name='checkpoint odd', op='checkpoint', n=4133, d=283, type='f32', pow2=False),
        # weight and bias gradient of a view layer over the training batch
        dict(name='weight grad training batch', op='weight_grad', n=SAMPLES, k=256, o=256, bias=True),
        # a small ragged layer over a chunk of rows
        dict(name='weight grad ragged', op='weight_grad', n=4133, k=283, o=61, bias=False),
        # the norm's backward over the training batch, with the residual stream's gradient
        dict(name='norm backward training batch', op='norm_backward', n=SAMPLES, d=256, type='bf16', residual=True),
        # and on a chunk of an odd width in fp32
        dict(name='norm backward odd', op='norm_backward', n=4133, d=1001, type='f32', residual=False),
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(['norm', 'linear', 'linear', 'checkpoint', 'weight_grad', 'weight_grad', 'norm_backward'])
    elements = SAMPLES * 256
    if op in ('linear', 'weight_grad'):
        k, o = _log_uniform(rng, 16, 4096), _log_uniform(rng, 8, 4096)
        most = min(SAMPLES, elements // max(k, o), elements * 256 // (k * o))
        n = _log_uniform(rng, 1, most)
        if op == 'weight_grad':
            return dict(op=op, n=n, k=k, o=o, bias=rng.random() < 0.5)
        return dict(op=op, n=n, k=k, o=o, type=rng.choice(['bf16', 'f32']), bias=rng.random() < 0.5, relu=rng.random() < 0.5)
    d = _log_uniform(rng, 16, 8192)
    case = dict(op=op, n=_log_uniform(rng, 1, min(SAMPLES, elements // (2 * d))), d=d, type=rng.choice(['bf16', 'f32']))
    if op == 'norm':
        case |= dict(residual=rng.random() < 0.5, weight=rng.random() < 0.5, pow2=rng.random() < 0.5)
    elif op == 'checkpoint':
        case |= dict(pow2=rng.random() < 0.5)
    else:
        case |= dict(residual=rng.random() < 0.5)
    return case


def _activations(n, d, gen, dtype):
    """Rows of a residual stream: normal, columns of different size, a few rows of zeros (samples outside the scene)."""
    x = torch.empty(n, d, device='cuda').normal_(generator=gen)
    x *= torch.empty(d, device='cuda').normal_(generator=gen).mul_(0.5).exp_()
    x[torch.rand(n, device='cuda', generator=gen) < 0.02] = 0
    return x.to(dtype)


def _upstream(n, d, gen, dtype):
    """Upstream gradients: rows of very different size (a sample's compositing weight), some of them zero."""
    g = torch.empty(n, d, device='cuda').normal_(generator=gen)
    row = torch.empty(n, 1, device='cuda').normal_(generator=gen).mul_(1.5).exp_()
    row[torch.rand(n, device='cuda', generator=gen) < 0.1] = 0
    return g.mul_(row).mul_(1e-3).to(dtype)


def _scales(largest, pow2):
    """The step of a row from its largest magnitude: largest / 127, or the smallest power of two that is no less."""
    scale = largest / torch.full_like(largest, 127)  # a quotient: a plain number would be multiplied by its reciprocal
    if pow2:
        mantissa, exponent = torch.frexp(scale)
        scale = torch.ldexp(torch.ones_like(scale), exponent - (mantissa == 0.5).to(exponent.dtype))
    return torch.where(largest == 0, 0.0, scale.clamp(min=2.0 ** -126))


def _codes(x, pow2):
    """Codes (as floats) and scales of the rows of x."""
    scale = _scales(x.abs().amax(1), pow2)
    return (x / torch.where(scale == 0, 1.0, scale)[:, None]).round_(), scale


def _stored(codes):
    """Codes as a program holds them: int8, the row stride a multiple of 16."""
    n, d = codes.shape
    out = torch.zeros(n, (d + 15) // 16 * 16, dtype=torch.int8, device='cuda')
    out[:, :d] = codes
    return out[:, :d]


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    op, n = case['op'], case['n']
    s = dict(case)
    if op == 'norm':
        s['x'] = _activations(n, case['d'], gen, TYPES[case['type']])
        s['r'] = _activations(n, case['d'], gen, TYPES[case['type']]) if case['residual'] else None
        s['w'] = torch.empty(case['d'], device='cuda').uniform_(0.5, 1.5, generator=gen) if case['weight'] else None
    elif op == 'checkpoint':
        s['x'] = _activations(n, case['d'], gen, TYPES[case['type']])
    elif op == 'linear':
        codes, s['scales'] = _codes(_activations(n, case['k'], gen, torch.float32), False)
        s['codes'] = _stored(codes)
        bound = math.sqrt(6.0 / case['k'])
        codes, s['w_scales'] = _codes(torch.empty(case['o'], case['k'], device='cuda').uniform_(-bound, bound, generator=gen), False)
        s['w_codes'] = _stored(codes)
        s['b'] = torch.empty(case['o'], device='cuda').uniform_(-0.3, 0.3, generator=gen) if case['bias'] else None
    elif op == 'weight_grad':
        s['g'] = _upstream(n, case['o'], gen, torch.bfloat16)
        codes, s['scales'] = _codes(_activations(n, case['k'], gen, torch.float32), True)
        s['codes'] = _stored(codes)
    else:
        s['g'] = _upstream(n, case['d'], gen, TYPES[case['type']])
        s['gr'] = _upstream(n, case['d'], gen, TYPES[case['type']]) if case['residual'] else None
        h = _activations(n, case['d'], gen, torch.float32)
        s['rstd'] = torch.rsqrt(h.square().mean(1) + EPS)
        codes, s['scales'] = _codes(h * s['rstd'][:, None], True)
        s['codes'] = _stored(codes)
    return s


# the plain forms, in fp32


def _norm_plain(s):
    h = s['x'].float()
    if s['r'] is not None:
        h = h + s['r'].float()
    rstd = 1.0 / torch.sqrt((h * h).mean(1) + EPS)
    y = h * rstd[:, None]
    if s['w'] is not None:
        y = y * s['w']
    codes, scales = _codes(y, s['pow2'])
    out = {'values': (codes * scales[:, None]).to(torch.bfloat16), 'rstd': rstd}
    if s['r'] is not None:
        out['sum'] = h.to(s['r'].dtype)
    return out


def _linear_plain(s):
    out = s['codes'].float() @ s['w_codes'].float().t()
    out = out * s['scales'][:, None] * s['w_scales']
    if s['b'] is not None:
        out = out + s['b']
    if s['relu']:
        out = torch.where(out < 0, 0.0, out)
    return out.to(TYPES[s['type']])


def _checkpoint_plain(s):
    codes, scales = _codes(s['x'].float(), s['pow2'])
    return (codes * scales[:, None]).to(torch.bfloat16)


def _weight_grad_plain(s):
    g = s['g'].float()
    out = {'weight': g.t() @ (s['codes'].float() * s['scales'][:, None])}
    if s['bias']:
        out['bias'] = g.sum(0)
    return out


def _norm_backward_plain(s):
    g = s['g'].float()
    y = s['codes'].float() * s['scales'][:, None]
    out = s['rstd'][:, None] * (g - y * (g * y).mean(1, keepdim=True))
    if s['gr'] is not None:
        out = out + s['gr'].float()
    return out.to(s['g'].dtype)


# the framework's operators

_module = None


def _backend():
    global _module
    if _module is None:
        package = str(Path(__file__).resolve().parent.parent / 'fused-zipnerf_b200')
        if package not in sys.path:
            sys.path.insert(0, package)
        import ZipNeRFCudaBackend
        _module = ZipNeRFCudaBackend
    return _module


def _norm_own(s):
    b = _backend()
    codes, scales, total, rstd = b.rms_norm_int8(s['x'], s['r'], s['w'], EPS, s['pow2'])
    out = {'values': b.dequantize_rows(codes, scales), 'rstd': rstd}
    if total is not None:
        out['sum'] = total
    return out


def _linear_own(s):
    return _backend().int8_linear(s['codes'], s['scales'], s['w_codes'], s['w_scales'], s['b'], s['relu'], TYPES[s['type']])


def _checkpoint_own(s):
    b = _backend()
    return b.dequantize_rows(*b.quantize_rows(s['x'], s['pow2']))


def _weight_grad_own(s):
    out = {'weight': torch.zeros(s['o'], s['k'], device='cuda')}
    if s['bias']:
        out['bias'] = torch.zeros(s['o'], device='cuda')
    _backend().int8_weight_grad(s['g'], s['codes'], s['scales'], out['weight'], out.get('bias'))
    return out


def _norm_backward_own(s):
    return _backend().rms_norm_int8_backward(s['g'], s['codes'], s['scales'], s['rstd'], s['gr'])


_PLAIN = {'norm': _norm_plain, 'linear': _linear_plain, 'checkpoint': _checkpoint_plain, 'weight_grad': _weight_grad_plain,
          'norm_backward': _norm_backward_plain}
_OWN = {'norm': _norm_own, 'linear': _linear_own, 'checkpoint': _checkpoint_own, 'weight_grad': _weight_grad_own,
        'norm_backward': _norm_backward_own}


def run(state):
    return (_OWN if own else _PLAIN)[state['op']](state)


def work(case):
    op, n = case['op'], case['n']
    size = {'bf16': 2, 'f32': 4}[case.get('type', 'bf16')]
    if op == 'norm':
        # x (and the residual stream in and out) in the inputs' type; codes and scales out and, restored, as bf16; rstd
        rows = n * case['d']
        return {'bytes': rows * (size * (3 if case['residual'] else 1) + 1 + 2) + 8 * n + (4 * case['d'] if case['weight'] else 0),
                'flops': 8.0 * rows}
    if op == 'checkpoint':
        return {'bytes': n * case['d'] * (size + 1 + 2) + 4 * n, 'flops': 3.0 * n * case['d']}
    if op == 'linear':
        k, o = case['k'], case['o']
        return {'bytes': n * k + o * k + 4 * n + 4 * o * (2 if case['bias'] else 1) + n * o * size, 'flops': 2.0 * n * k * o}
    if op == 'weight_grad':
        k, o = case['k'], case['o']
        return {'bytes': 2 * n * o + n * k + 4 * n + 4 * o * k + (4 * o if case['bias'] else 0), 'flops': 2.0 * n * k * o}
    return {'bytes': n * case['d'] * (size * (3 if case['residual'] else 2) + 1) + 8 * n, 'flops': 7.0 * n * case['d']}


def exact(case, seed):
    """The operators' definitions in 64 bits."""
    s = prepare(case, seed)
    s = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in s.items()}

    def stepped(rows):
        top = rows.abs().max(dim=1, keepdim=True).values
        step = top / 127
        if s['pow2']:
            # log2 is exact at powers of two, so the ceiling is the smallest exponent that covers the step
            step = torch.exp2(torch.ceil(torch.log2(step)))
        step = torch.clamp(step, min=2.0 ** -126)
        return torch.where(top > 0, torch.round(rows / step) * step, torch.zeros_like(rows))

    if s['op'] == 'norm':
        h = s['x'] if s['r'] is None else s['x'] + s['r']
        norm = (h.pow(2).sum(dim=1) / s['d'] + EPS).pow(-0.5)
        out = {'values': stepped(torch.einsum('nd,n->nd', h, norm) * (1.0 if s['w'] is None else s['w'])), 'rstd': norm}
        return out if s['r'] is None else out | {'sum': h}
    if s['op'] == 'checkpoint':
        return stepped(s['x'])
    if s['op'] == 'linear':
        out = torch.diag_embed(s['w_scales']) @ s['w_codes'] if s['o'] <= 256 else s['w_codes'] * s['w_scales'].unsqueeze(1)
        out = (s['codes'] * s['scales'].unsqueeze(1)).matmul(out.transpose(0, 1))
        if s['b'] is not None:
            out += s['b']
        return torch.clamp(out, min=0) if s['relu'] else out
    if s['op'] == 'weight_grad':
        out = {'weight': (s['g'] * s['scales'].unsqueeze(1)).transpose(0, 1).matmul(s['codes'])}
        return out | {'bias': torch.ones(1, s['n'], dtype=torch.float64, device='cuda').matmul(s['g'])[0]} if s['bias'] else out
    y = torch.einsum('nd,n->nd', s['codes'], s['scales'])
    dot = torch.einsum('nd,nd->n', s['g'], y) / s['d']
    out = torch.einsum('n,nd->nd', s['rstd'], s['g'] - torch.einsum('n,nd->nd', dot, y))
    return out if s['gr'] is None else out + s['gr']
