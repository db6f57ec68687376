"""A residual decoder on the 8-bit row operators (include/zf_int8.h): the operators together as a training or rendering
loop uses them. The reference's NeRF MLP has no residual layers (nerf_mlp.h:31-73); this is an addition for scenes that
want a deeper decoder behind the NeRF grid's features.

    h_0 = features W_in^T + b_in
    h_{l+1} = h_l + relu(norm(h_l) W_up^T + b_up) W_down^T + b_down         blocks l = 0 .. blocks - 1
    outputs = norm(h_blocks) W_out^T + b_out

Every layer runs in 8 bits: the norms write int8 rows (adding the last block's update on the way), the hidden layers are
quantized by rows, and the weights, fp32 masters, are quantized by output rows in `pack`. The norms have no gain of their
own: it would multiply the columns of the next weight, which is trained anyway (as the reference folds its bottleneck,
nerf_mlp.cu:186-234).

Training keeps one code per activation, the very operands of the forward's products, and two floats per row: 8 bits
instead of the 16 of a bf16 record. The backward passes gradients straight through the rounding to codes and reads the
codes: weight gradients by `int8_weight_grad`, the norms by `rms_norm_int8_backward`. The ReLU masks come from running the
up layer again on its codes, which gives the forward's bits. Data gradients are plain bf16 products with the weights'
restored values. Forward and backward only enqueue: a caller reads `int8_status` where it synchronises, as the fit below does.

    python -m zipnerf_b200.trunk --samples 65536 --steps 100       # fits random features to a fixed random decoder
"""
from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import torch

if str(Path(__file__).resolve().parent.parent) not in sys.path:  # ZipNeRFCudaBackend sits beside this package
    sys.path.append(str(Path(__file__).resolve().parent.parent))

EPS = 1e-6


class ResidualTrunk:
    """The decoder's parameter layout, its packed 8-bit weights, forward and backward. Widths are multiples of 8, the
    hidden width at most 512 (the widest layer of `relu_backward_`)."""

    def __init__(self, n_features: int = 56, width: int = 256, hidden: int = 512, blocks: int = 4, n_outputs: int = 8) -> None:
        if n_features <= 0 or blocks < 0 or width <= 0 or hidden <= 0 or n_outputs <= 0 or n_features % 8 or width % 8 or hidden % 8 or n_outputs % 8:
            raise RuntimeError('ZipNeRF: trunk widths must be positive multiples of 8')
        if hidden > 512:
            raise RuntimeError('ZipNeRF: the trunk\'s hidden width is at most 512')
        self.n_features, self.width, self.hidden, self.blocks, self.n_outputs = n_features, width, hidden, blocks, n_outputs
        self.layers = [('in', width, n_features)]
        for i in range(blocks):
            self.layers += [(f'{i}.up', hidden, width), (f'{i}.down', width, hidden)]
        self.layers.append(('out', n_outputs, width))
        self.offsets, n = {}, 0
        for name, rows, columns in self.layers:
            self.offsets[name] = n
            n += rows * columns + rows
        self.numel = n  # a multiple of 8, as every width is

    def view(self, buffer: torch.Tensor, name: str) -> tuple[torch.Tensor, torch.Tensor]:
        """Weight [rows, columns] and bias [rows] of a layer as views of the flat buffer."""
        rows, columns = next((r, c) for n, r, c in self.layers if n == name)
        a = self.offsets[name]
        return buffer[a:a + rows * columns].view(rows, columns), buffer[a + rows * columns:a + rows * columns + rows]

    def initialize(self, buffer: torch.Tensor, generator: torch.Generator) -> None:
        """He-uniform weights; the down layers start small so that the blocks start near the identity. Zero biases."""
        buffer.zero_()
        for name, _, columns in self.layers:
            bound = math.sqrt(6.0 / columns) * (0.1 if name.endswith('down') else 1.0)
            self.view(buffer, name)[0].uniform_(-bound, bound, generator=generator)

    def pack(self, params: torch.Tensor, training: bool = True) -> dict:
        """The weights as int8 rows; for training also their restored values in bf16 (the data gradients' operands)."""
        import ZipNeRFCudaBackend as backend
        packed = {}
        for name, _, _ in self.layers:
            weight, bias = self.view(params, name)
            codes, scales = backend.quantize_rows(weight)
            packed[name] = (codes, scales, bias, backend.dequantize_rows(codes, scales) if training else None)
        return packed

    def forward(self, features: torch.Tensor, packed: dict, training: bool):
        """features [n, n_features] (bf16 or float32) -> outputs [n, n_outputs] float32, and the context of the backward:
        the codes, scales and norms' rstd of every layer's input (empty without training)."""
        import ZipNeRFCudaBackend as backend
        if features.dim() != 2 or features.shape[1] != self.n_features:
            raise RuntimeError('ZipNeRF: invalid trunk features')
        context = []

        def layer(name, codes, scales, rstd=None, relu=False, dtype=torch.bfloat16):
            if training:
                context.append((codes, scales, rstd))
            weight_codes, weight_scales, bias, _ = packed[name]
            return backend.int8_linear(codes, scales, weight_codes, weight_scales, bias, relu, dtype)

        h = layer('in', *backend.quantize_rows(features, True))
        update = None
        for i in range(self.blocks + 1):
            # power-of-two scales: the backward's products of these codes are exact
            if update is None:
                codes, scales, _, rstd = backend.rms_norm_int8(h, None, None, EPS, True)
            else:
                codes, scales, h, rstd = backend.rms_norm_int8(update, h, None, EPS, True)
            if i == self.blocks:
                return layer('out', codes, scales, rstd, dtype=torch.float32), context
            z = layer(f'{i}.up', codes, scales, rstd, relu=True)
            update = layer(f'{i}.down', *backend.quantize_rows(z, True))

    def backward(self, grad_outputs: torch.Tensor, packed: dict, context: list, grads: torch.Tensor) -> torch.Tensor:
        """grads (flat float32, the parameter layout) += the parameters' gradients; returns the features' gradient in
        bf16. grad_outputs [n, n_outputs] bf16."""
        import ZipNeRFCudaBackend as backend
        if len(context) != len(self.layers):
            raise RuntimeError('ZipNeRF: the trunk\'s backward needs the context of its training forward')
        kept = {name: c for (name, _, _), c in zip(self.layers, context)}

        def weight_grad(name, grad, bias=True):
            weight, bias_grad = self.view(grads, name)
            backend.int8_weight_grad(grad, kept[name][0], kept[name][1], weight, bias_grad if bias else None)
            return grad @ packed[name][3]

        g = backend.rms_norm_int8_backward(weight_grad('out', grad_outputs), *kept['out'])
        for i in reversed(range(self.blocks)):
            # g is the gradient of the stream behind the block, and so of the block's update
            grad_z = weight_grad(f'{i}.down', g)
            codes, scales, rstd = kept[f'{i}.up']
            weight_codes, weight_scales, bias, _ = packed[f'{i}.up']
            z = backend.int8_linear(codes, scales, weight_codes, weight_scales, bias, True)
            backend.relu_backward_(grad_z, z, self.view(grads, f'{i}.up')[1])  # the mask, and the bias gradient
            g = backend.rms_norm_int8_backward(weight_grad(f'{i}.up', grad_z, bias=False), codes, scales, rstd, g)
        return weight_grad('in', g)

    def kept_bytes(self, context: list) -> int:
        """Device bytes of a training forward's context."""
        return sum(t.shape[0] * t.stride(0) * t.element_size() if t.dim() == 2 else t.numel() * t.element_size()
                   for entry in context for t in entry if t is not None)


def main(argv=None) -> list[float]:
    parser = argparse.ArgumentParser(description='Fits the residual decoder to a fixed random decoder of its own shape.')
    parser.add_argument('--samples', type=int, default=65536)
    parser.add_argument('--steps', type=int, default=100)
    parser.add_argument('--width', type=int, default=256)
    parser.add_argument('--hidden', type=int, default=512)
    parser.add_argument('--blocks', type=int, default=4)
    parser.add_argument('--lr', type=float, default=1e-3)
    args = parser.parse_args(argv)
    import ZipNeRFCudaBackend as backend
    device = torch.device('cuda')
    generator = torch.Generator(device=device).manual_seed(0)
    trunk = ResidualTrunk(width=args.width, hidden=args.hidden, blocks=args.blocks)
    teacher, params = torch.zeros(trunk.numel, device=device), torch.zeros(trunk.numel, device=device)
    trunk.initialize(teacher, generator)
    trunk.initialize(params, generator)
    grads = torch.zeros_like(params)
    optimizer = backend.Adam([params], [grads], [1.0], [[]], 0.0, backend.grid_max_value, 0.9, 0.99, 1e-15, torch.zeros(0, device=device))
    teacher_packed = trunk.pack(teacher, training=False)
    losses = []
    for step in range(args.steps):
        features = torch.randn(args.samples, trunk.n_features, generator=generator, device=device).bfloat16()
        target, _ = trunk.forward(features, teacher_packed, training=False)
        packed = trunk.pack(params)
        outputs, context = trunk.forward(features, packed, training=True)
        error = outputs - target
        losses.append(error.square().mean())
        trunk.backward((error * (2.0 / error.numel())).bfloat16(), packed, context, grads)
        optimizer.step(args.lr)  # zeroes the gradients
    losses = [loss.item() for loss in losses]
    if backend.int8_status(torch.device('cuda', torch.cuda.current_device())).item() != 0:
        raise RuntimeError('ZipNeRF: a bounded wait of an 8-bit kernel ran out')
    if args.steps > 0:
        print(f'loss {losses[0]:.4f} -> {losses[-1]:.4f} in {args.steps} steps; {trunk.kept_bytes(context) / 2 ** 20:.1f} MiB kept per forward')
    return losses


if __name__ == '__main__':
    main()
