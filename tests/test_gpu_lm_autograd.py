"""GPU: the norms and rotation under autograd, by the function that a trainer wraps around the pair of calls."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


class QKNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved):
        from kbb200 import lm

        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.how = eps, interleaved
        return lm.qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)

    @staticmethod
    def backward(ctx, dq_out, dk_out):
        from kbb200 import lm

        grads = lm.qk_norm_rope_backward(dq_out.contiguous(), dk_out.contiguous(), *ctx.saved_tensors, *ctx.how)
        return *grads, None, None, None, None, None


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradients_of_a_loss(interleaved, cuda_device):
    """A loss through the function against the same in 64 bits and elementary operations.  fp32: each gradient within
    2^-16 of the sum of its terms' magnitudes, a few hundred roundings."""
    from kbb200 import lm

    T, hq, hkv, d, r = 33, 6, 2, 64, 48
    g = torch.Generator(device=cuda_device).manual_seed(0)
    packed = torch.randn(T, (hq + 2 * hkv) * d, device=cuda_device, generator=g)
    w = [1 + 0.3 * torch.randn(d, device=cuda_device, generator=g) for _ in range(2)]
    cos, sin = lm.rope_tables(200, r, device=cuda_device)
    pos = torch.randint(0, 200, (T,), device=cuda_device, generator=g)
    mix = [torch.randn(T, h, d, device=cuda_device, generator=g) for h in (hq, hkv)]

    def loss(fn, packed, w, mix):
        q, k = packed[:, : hq * d].view(T, hq, d), packed[:, hq * d: (hq + hkv) * d].view(T, hkv, d)
        zq, zk = fn(q, k, *w)
        return (zq * mix[0]).sum() + (zk * mix[1]).tanh().sum()

    def plain(q, k, wq, wk):
        c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]

        def one(x, wx):
            y = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * wx
            a, b = (y[..., 0:r:2], y[..., 1:r:2]) if interleaved else (y[..., : r // 2], y[..., r // 2: r])
            u, v = a * c - b * s, b * c + a * s
            turned = torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)
            return torch.cat((turned, y[..., r:]), -1)

        return one(q, wq), one(k, wk)

    leaves = [packed.requires_grad_(), *(x.requires_grad_() for x in w)]
    loss(lambda q, k, *w: QKNormRope.apply(q, k, *w, cos, sin, pos, 1e-6, interleaved), packed, w, mix).backward()
    exact = [x.detach().double().requires_grad_() for x in leaves]
    loss(plain, exact[0], exact[1:], [m.double() for m in mix]).backward()
    for a, b, terms in zip(leaves, exact, (8.0, 8.0 * T * hq, 8.0 * T * hkv)):
        assert float((a.grad.double() - b.grad).abs().max()) < 2.0 ** -16 * terms
