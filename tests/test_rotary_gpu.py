"""GPU: rotary positions against the fp64 definition, and their gradients."""

import numpy as np
import pytest
import torch

from oracle import serving as OS
from tests.conftest import SEED

pytestmark = pytest.mark.gpu


def _randn(shape, dev, seed, dtype):
    return torch.randn(shape, generator=torch.Generator(device=dev).manual_seed(seed), device=dev).to(dtype)


def check(y, x, pos, f, amplitude, interleaved, inverse=False):
    """|y - exact| <= half a step of the type (relative eps / 2, and half the
    smallest subnormal), plus 8 x 2^-24 of the pair's magnitude: cos and sin are
    within 4 x 2^-24 (the reduced angle's rounding and the series'), two
    products, a sum and the amplitude round once each."""
    n = f.numel()
    xs = x.double().cpu().numpy()
    ref = OS.rotate(xs, pos.cpu().numpy() if pos.dim() == 1 else pos.cpu().numpy()[:, None], f.cpu().numpy(), amplitude,
                    interleaved, inverse)
    pair = np.abs(xs).copy()
    i1, i2 = (np.arange(0, 2 * n, 2), np.arange(1, 2 * n, 2)) if interleaved else (np.arange(n), np.arange(n, 2 * n))
    both = pair[..., i1] + pair[..., i2]
    pair[..., i1] = pair[..., i2] = both
    info = torch.finfo(y.dtype)
    tol = info.eps / 2 * np.abs(ref) + amplitude * pair * 8 * 2.0 ** -24 * (1 + info.eps) + info.smallest_normal * info.eps / 2
    assert y.shape == x.shape and y.dtype == x.dtype
    err = np.abs(y.double().cpu().numpy() - ref)
    assert (err <= tol).all(), f"worst {np.max(err / tol):.3f} of the tolerance"


CASES = [  # B, S, Hq, Hkv, D, rotated, dtype, interleaved, head major, int64, amplitude
    (1, 1, 1, 1, 64, 64, torch.float16, False, True, False, 1.0),
    (32, 1, 32, 8, 128, 128, torch.float16, False, False, False, 1.0),
    (2, 77, 8, 2, 128, 128, torch.bfloat16, True, False, True, 1.2),
    (3, 33, 5, 1, 64, 16, torch.float16, True, True, False, 1.0),
    (3, 33, 5, 1, 64, 16, torch.float32, False, False, True, 0.7),
    (2, 65, 3, 3, 80, 20, torch.float16, False, False, False, 1.0),   # pairs and heads of odd sizes: one at a time
    (2, 65, 3, 3, 80, 20, torch.bfloat16, True, True, False, 1.0),
    (1, 9, 2, 1, 6, 2, torch.float32, True, False, False, 1.0),
    (1, 5, 2, 1, 1024, 1024, torch.float16, False, False, False, 1.0),
    (2, 513, 16, 16, 64, 64, torch.float32, False, True, False, 1.0),
    (4, 300, 64, 8, 128, 128, torch.float16, True, False, False, 1.0),
]


@pytest.mark.parametrize("B,S,Hq,Hkv,D,R,dtype,interleaved,head_major,wide,amplitude", CASES)
def test_rotary(cuda, B, S, Hq, Hkv, D, R, dtype, interleaved, head_major, wide, amplitude):
    import torch_spyre_amd as tsa

    f, _ = tsa.rotary_frequencies(R, base=500000.0, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(SEED + 1)
    pos = torch.randint(-5000, 1 << 20, (B, S), generator=g, device=cuda, dtype=torch.int64 if wide else torch.int32)
    shape = (lambda H: (B, H, S, D)) if head_major else (lambda H: (B, S, H, D))
    q, k = _randn(shape(Hq), cuda, SEED + 2, dtype), _randn(shape(Hkv), cuda, SEED + 3, dtype)
    if not head_major:
        q, k = q.transpose(1, 2), k.transpose(1, 2)
    yq, yk = tsa.rotary_embedding(q, k, pos, f, amplitude, interleaved)
    assert yq.stride() == q.stride() and yk.stride() == k.stride()
    check(yq, q, pos, f, amplitude, interleaved)
    check(yk, k, pos, f, amplitude, interleaved)
    back = tsa.rotary_embedding(q, None, pos, f, amplitude, interleaved, inverse=True)
    check(back, q, pos, f, amplitude, interleaved, inverse=True)
    one = tsa.rotary_embedding(k, None, pos[0], f, amplitude, interleaved)  # one row of positions for all
    check(one, k, pos[0], f, amplitude, interleaved)


def test_strides_and_alignment(cuda):
    """Slices of a packed projection, unaligned views, a transposed feature, an
    expanded batch; nothing besides the result is written."""
    import torch_spyre_amd as tsa

    f, _ = tsa.rotary_frequencies(64, device=cuda)
    pos = torch.arange(1000, 1019, dtype=torch.int32, device=cuda).expand(2, 19)
    packed = _randn((2, 19, 6, 64), cuda, SEED + 4, torch.float16)
    q, k = packed[:, :, :4].transpose(1, 2), packed[:, :, 4:5].transpose(1, 2)
    before = packed.clone()
    yq, yk = tsa.rotary_embedding(q, k, pos, f)
    check(yq, q, pos, f, 1.0, False)
    check(yk, k, pos, f, 1.0, False)
    assert torch.equal(packed, before)
    flat = _randn((2 * 3 * 19 * 64 + 1,), cuda, SEED + 5, torch.float16)
    odd = flat[1:].view(2, 3, 19, 64)
    check(tsa.rotary_embedding(odd, None, pos, f), odd, pos, f, 1.0, False)
    rows = _randn((2, 3, 19, 67), cuda, SEED + 6, torch.float16)[..., 2:66]
    check(tsa.rotary_embedding(rows, None, pos, f, interleaved=True), rows, pos, f, 1.0, True)
    turned = _randn((2, 3, 64, 19), cuda, SEED + 7, torch.float16).transpose(2, 3)
    check(tsa.rotary_embedding(turned, None, pos, f), turned, pos, f, 1.0, False)
    wide = _randn((1, 3, 19, 64), cuda, SEED + 8, torch.float16).expand(2, 3, 19, 64)
    check(tsa.rotary_embedding(wide, None, pos, f), wide, pos, f, 1.0, False)
    backwards = torch.arange(18, -1, -1, device=cuda)
    check(tsa.rotary_embedding(odd, None, backwards[::1], f), odd, backwards, f, 1.0, False)


def test_empty(cuda):
    import torch_spyre_amd as tsa

    f, _ = tsa.rotary_frequencies(64, device=cuda)
    for B, H, S in ((0, 2, 3), (2, 2, 0), (2, 0, 3)):
        q = torch.empty((B, H, S, 64), dtype=torch.float16, device=cuda)
        y = tsa.rotary_embedding(q, None, torch.zeros((B, S), dtype=torch.int32, device=cuda), f)
        assert y.shape == q.shape


@pytest.mark.parametrize("dtype,interleaved,R", [(torch.float32, False, 64), (torch.float32, True, 16),
                                                 (torch.bfloat16, False, 32), (torch.float16, True, 64)])
def test_gradient(cuda, dtype, interleaved, R):
    """The gradient is the inverse rotation of the cotangent, and (fp32)
    agrees with differences of the loss."""
    import torch_spyre_amd as tsa

    f, _ = tsa.rotary_frequencies(R, device=cuda)
    pos = torch.arange(7, 18, device=cuda)
    q = _randn((2, 11, 4, 64), cuda, SEED + 9, dtype).transpose(1, 2).requires_grad_()
    k = _randn((2, 11, 2, 64), cuda, SEED + 10, dtype).transpose(1, 2).requires_grad_()
    dq, dk = _randn(q.shape, cuda, SEED + 11, dtype), _randn(k.shape, cuda, SEED + 12, dtype)
    yq, yk = tsa.rotary_embedding(q, k, pos, f, 1.3, interleaved)
    gq, gk = torch.autograd.grad((yq, yk), (q, k), (dq, dk), retain_graph=True)
    check(gq, dq, pos, f, 1.3, interleaved, inverse=True)
    check(gk, dk, pos, f, 1.3, interleaved, inverse=True)
    only, = torch.autograd.grad(yk, (k,), (dk,))
    assert torch.equal(only, gk)
    if dtype == torch.float32:
        # The map is linear, so a difference of step 1 is the derivative; its
        # error is the rounding of y (2^-24 of |y| <= 6) summed over 2 features.
        e = torch.zeros_like(q)
        e[1, 2, 3, 5] = 1.0
        step = tsa.rotary_embedding((q + e).detach(), None, pos, f, 1.3, interleaved) - yq.detach()
        assert abs((step * dq).sum().item() - gq[1, 2, 3, 5].item()) <= 64 * 12 * 2.0 ** -24 * dq.abs().max().item()


def test_second_gradient_and_leaves(cuda):
    import torch_spyre_amd as tsa

    f, _ = tsa.rotary_frequencies(64, device=cuda)
    pos = torch.arange(5, device=cuda)
    q = _randn((1, 2, 5, 64), cuda, SEED + 13, torch.float32).requires_grad_()
    y = tsa.rotary_embedding(q, None, pos, f)
    assert y.requires_grad
    g, = torch.autograd.grad(y.square().sum() / 2, q, create_graph=True)  # the rotation is orthogonal: g = q
    assert torch.allclose(g, q, atol=1e-5)
    h, = torch.autograd.grad(g.sum(), q)
    assert torch.allclose(h, torch.ones_like(q), atol=1e-5)
    k = _randn((1, 1, 5, 64), cuda, SEED + 14, torch.float32)
    yq, yk = tsa.rotary_embedding(q.detach(), k, pos, f)
    assert not yq.requires_grad and not yk.requires_grad
    yq, yk = tsa.rotary_embedding(q, k, pos, f)
    assert yq.requires_grad
    g, = torch.autograd.grad((yq.sum() + yk.sum()), q)
    assert torch.isfinite(g).all()


def test_graph(cuda):
    """A captured call follows its inputs through replays, eager work between them."""
    import torch_spyre_amd as tsa

    f, _ = tsa.rotary_frequencies(128, device=cuda)
    q, k = _randn((4, 8, 1, 128), cuda, SEED + 15, torch.float16), _randn((4, 2, 1, 128), cuda, SEED + 16, torch.float16)
    pos = torch.zeros((4, 1), dtype=torch.int32, device=cuda)
    tsa.rotary_embedding(q, k, pos, f)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        yq, yk = tsa.rotary_embedding(q, k, pos, f)
    for step in range(4):
        pos.fill_(1000 * step + 3)
        q.add_(0.125)
        g.replay()
        torch.cuda.synchronize()
        eq, ek = tsa.rotary_embedding(q, k, pos, f)
        assert torch.equal(yq, eq) and torch.equal(yk, ek)


def test_refusals(cuda):
    import torch_spyre_amd as tsa

    f, _ = tsa.rotary_frequencies(64, device=cuda)
    q = torch.zeros((2, 3, 5, 64), dtype=torch.float16, device=cuda)
    pos = torch.zeros((2, 5), dtype=torch.int32, device=cuda)
    bad = [
        dict(q=q[0]), dict(q=q.double()), dict(k=q.float()), dict(k=q[:, :, :4]), dict(k=q.cpu()),
        dict(positions=pos.float()), dict(positions=pos[:, :4]), dict(positions=pos.cpu()), dict(positions=pos[None]),
        dict(frequencies=f.float()), dict(frequencies=f.cpu()), dict(frequencies=f[:0]),
        dict(frequencies=torch.cat((f, f))), dict(frequencies=torch.stack((f, f), 1)[:, 0]),
        dict(frequencies=f.clone().requires_grad_()),
    ]
    for change in bad:
        args = {"q": q, "k": q, "positions": pos, "frequencies": f} | change
        with pytest.raises((ValueError, TypeError)):
            tsa.rotary_embedding(**args)
    with pytest.raises(NotImplementedError):
        tsa.rotary_embedding(q.cpu(), None, pos.cpu(), f.cpu())
