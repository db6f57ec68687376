"""The residual decoder on the 8-bit row operators (zipnerf_b200/trunk.py) on the GPU: outputs against the same network in
float32 torch with rounding at the same places, gradients against the backward formulas in float64 at the forward's own
codes and ReLU masks (another forward's masks differ wherever a pre-activation lies within its rounding of zero), and a
short fit."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def in_steps(x, power_of_two):
    largest = x.abs().amax(1, keepdim=True)
    step = largest / 127
    if power_of_two:
        step = torch.exp2(torch.ceil(torch.log2(step)))
    step = torch.where(largest > 0, step, torch.ones_like(step))
    return torch.round(x / step) * step


def reference_forward(trunk, params, features):
    def layer(name, x):
        weight, bias = trunk.view(params, name)
        return x @ in_steps(weight, False).t() + bias

    def norm(h):
        return in_steps(h * (h.square().mean(1, keepdim=True) + 1e-6).rsqrt(), True)

    def bf16(x):
        return x.bfloat16().float()

    h = bf16(layer('in', in_steps(features, True)))
    for i in range(trunk.blocks):
        z = bf16(torch.relu(layer(f'{i}.up', norm(h))))
        h = bf16(h + bf16(layer(f'{i}.down', in_steps(z, True))))
    return layer('out', norm(h))


def reference_backward(trunk, params, context, grad_outputs):
    """float64: the gradients by layer name (weight, bias) and the features', straight through the roundings to codes"""
    kept = {name: c for (name, _, _), c in zip(trunk.layers, context)}
    grads = {}

    def inputs(name):
        return kept[name][0].double() * kept[name][1].double()[:, None]

    def weight(name):
        return in_steps(trunk.view(params, name)[0], False).double()

    def through_layer(name, g):
        grads[name] = (g.t() @ inputs(name), g.sum(0))
        return g @ weight(name)

    def through_norm(name, g):
        y, rstd = inputs(name), kept[name][2].double()[:, None]
        return rstd * (g - y * (g * y).mean(1, keepdim=True))

    g = through_norm('out', through_layer('out', grad_outputs.double()))
    for i in reversed(range(trunk.blocks)):
        grad_z = through_layer(f'{i}.down', g)
        pre = inputs(f'{i}.up') @ weight(f'{i}.up').t() + trunk.view(params, f'{i}.up')[1].double()
        g = g + through_norm(f'{i}.up', through_layer(f'{i}.up', grad_z * (pre > 0)))
    return grads, through_layer('in', g)


@pytest.mark.parametrize('n,width,hidden,blocks', [(1, 64, 128, 1), (333, 64, 128, 2), (4133, 96, 264, 3)])
def test_trunk_matches_its_formulas(cuda_device, n, width, hidden, blocks):
    import ZipNeRFCudaBackend as backend
    from zipnerf_b200.trunk import ResidualTrunk
    trunk = ResidualTrunk(56, width, hidden, blocks, 8)
    generator = torch.Generator(device=cuda_device).manual_seed(n)
    params = torch.zeros(trunk.numel, device=cuda_device)
    trunk.initialize(params, generator)
    for name, _, _ in trunk.layers:
        trunk.view(params, name)[1].uniform_(-0.2, 0.2, generator=generator)
    features = torch.randn(n, 56, device=cuda_device, generator=generator).bfloat16()
    grad_outputs = torch.randn(n, 8, device=cuda_device, generator=generator).bfloat16()
    packed = trunk.pack(params)
    outputs, context = trunk.forward(features, packed, True)
    grads = torch.zeros_like(params)
    grad_features = trunk.backward(grad_outputs, packed, context, grads)
    again, none = trunk.forward(features, trunk.pack(params, training=False), False)
    assert none == [] and torch.equal(again, outputs)
    expected = reference_forward(trunk, params, features.float())

    def rel(a, b):
        return ((a.double() - b.double()).norm() / b.double().norm().clamp(min=1e-12)).item()

    # the forwards differ where a value lies near a rounding boundary (fp32 order), by one step of 1/64 to 1/127 of a row's
    # largest value for a small share of the values
    assert rel(outputs, expected) < 2e-2
    # the backwards differ by the bf16 roundings of the gradients and of the weights in the data gradients: 2^-9 each on
    # average, some ten in sequence
    wanted, wanted_features = reference_backward(trunk, params, context, grad_outputs)
    errors = {name: max(rel(trunk.view(grads, name)[i], wanted[name][i]) for i in range(2)) for name, _, _ in trunk.layers}
    errors['features'] = rel(grad_features, wanted_features)
    assert max(errors.values()) < 5e-2, errors
    assert backend.int8_status(cuda_device).item() == 0


def test_trunk_keeps_a_byte_per_activation(cuda_device):
    from zipnerf_b200.trunk import ResidualTrunk
    trunk = ResidualTrunk(56, 256, 512, 2, 8)
    params = torch.zeros(trunk.numel, device=cuda_device)
    trunk.initialize(params, torch.Generator(device=cuda_device).manual_seed(0))
    _, context = trunk.forward(torch.randn(1000, 56, device=cuda_device), trunk.pack(params), True)
    # inputs (stride 64), two blocks of a norm and a hidden layer, the last norm; a scale each, and a norm's rstd
    assert trunk.kept_bytes(context) == 1000 * (64 + 2 * (256 + 512) + 256 + 4 * 6 + 4 * 3)


def test_trunk_fits(cuda_device):
    from zipnerf_b200 import trunk
    losses = trunk.main(['--samples', '4096', '--steps', '60', '--width', '64', '--hidden', '128', '--blocks', '2', '--lr', '3e-3'])
    assert sum(losses[-5:]) < 0.5 * sum(losses[:5])


def test_trunk_refusals():
    from zipnerf_b200.trunk import ResidualTrunk
    for widths in [(57, 64, 64, 1, 8), (56, 60, 64, 1, 8), (56, 64, 64, 1, 4), (56, 64, 64, -1, 8), (0, 64, 64, 1, 8)]:
        with pytest.raises(RuntimeError, match='ZipNeRF: trunk widths'):
            ResidualTrunk(*widths)
    with pytest.raises(RuntimeError, match='at most 512'):
        ResidualTrunk(hidden=520)
    trunk = ResidualTrunk(56, 64, 64, 1, 8)
    with pytest.raises(RuntimeError, match='ZipNeRF: invalid trunk features'):
        trunk.forward(torch.zeros(3, 55), {}, False)
    with pytest.raises(RuntimeError, match='needs the context'):
        trunk.backward(torch.zeros(3, 8), {}, [], torch.zeros(trunk.numel))
