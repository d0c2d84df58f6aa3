"""Forward-mode derivatives of the rotation: it is linear in q and k, so the
tangent of a result is the rotation of the operand's.  On the CPU behind the
operator's own autograd entry, with a plain kernel in place of the GPU's, and
on the GPU."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from tests.conftest import SEED


def plain(q, k, positions, frequencies, amplitude=1.0, interleaved=False, inverse=False):
    """The rotation in elementary operations."""
    theta = positions.double().unsqueeze(-1) * frequencies
    if theta.dim() == 3:
        theta = theta.unsqueeze(1)
    c, s = (amplitude * theta.cos()).float(), (amplitude * theta.sin()).float() * (-1 if inverse else 1)
    n = frequencies.numel()

    def turn(x):
        a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
        a, b = a * c - b * s, b * c + a * s
        y = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
        return torch.cat((y, x[..., 2 * n:]), -1).to(x.dtype)

    return turn(q), q.new_empty((0,)) if k is None else turn(k)


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request):
    import torch_spyre_amd  # noqa: F401

    if request.param == "cuda":
        yield request.getfixturevalue("cuda")
        return
    lib = torch.library.Library("spyre", "IMPL")
    lib.impl("rotary", plain, "CPU")
    try:
        yield torch.device("cpu")
    finally:
        lib._destroy()


def operands(dev, interleaved):
    def randn(*shape):
        g = torch.Generator().manual_seed(SEED + shape[1])
        return torch.randn(shape, generator=g).to(dev)

    q, k, tq, tk = randn(2, 4, 5, 64), randn(2, 2, 5, 64), randn(2, 4, 5, 64).flip(0), randn(2, 2, 5, 64).flip(0)
    pos = torch.arange(3, 8, device=dev)
    f = (10000.0 ** (-torch.arange(16, dtype=torch.float64) / 16)).to(dev)
    return q, k, tq, tk, pos, f, {"amplitude": 1.25, "interleaved": interleaved}


@pytest.mark.parametrize("interleaved", [False, True])
def test_dual_numbers(dev, interleaved):
    """Tangents of q, of k and of both; results without one where the operand
    has none; the values themselves as ever."""
    import torch_spyre_amd as tsa

    q, k, tq, tk, pos, f, how = operands(dev, interleaved)
    yq, yk = tsa.rotary_embedding(q, k, pos, f, **how)
    dq, dk = tsa.rotary_embedding(tq, tk, pos, f, **how)
    for has_q, has_k in ((True, True), (True, False), (False, True)):
        with fwAD.dual_level():
            a = fwAD.make_dual(q, tq) if has_q else q
            b = fwAD.make_dual(k, tk) if has_k else k
            (pq, gq), (pk, gk) = (fwAD.unpack_dual(x) for x in tsa.rotary_embedding(a, b, pos, f, **how))
            assert torch.equal(pq, yq) and torch.equal(pk, yk)
            assert torch.equal(gq, dq) if has_q else gq is None
            assert torch.equal(gk, dk) if has_k else gk is None
            if has_q:
                p, t = fwAD.unpack_dual(tsa.rotary_embedding(a, None, pos, f, inverse=True, **how))
                assert torch.equal(p, tsa.rotary_embedding(q, None, pos, f, inverse=True, **how))
                assert torch.equal(t, tsa.rotary_embedding(tq, None, pos, f, inverse=True, **how))
    with fwAD.dual_level(), fwAD._set_fwd_grad_enabled(False):
        p = tsa.rotary_embedding(fwAD.make_dual(q, tq), None, pos, f, **how)
        assert fwAD.unpack_dual(p).tangent is None


@pytest.mark.parametrize("grad", [False, True])
def test_with_and_without_gradients(dev, grad):
    """Under no_grad, and where the operands or the tangents take gradients
    (which pass through both results)."""
    import torch_spyre_amd as tsa

    q, k, tq, tk, pos, f, how = operands(dev, False)
    dq, dk = tsa.rotary_embedding(tq, tk, pos, f, **how)
    if not grad:
        with torch.no_grad(), fwAD.dual_level():
            y, _ = tsa.rotary_embedding(fwAD.make_dual(q, tq), k, pos, f, **how)
            assert torch.equal(fwAD.unpack_dual(y).tangent, dq)
        return
    for t in (q, tq, k):
        t.requires_grad_()
    with fwAD.dual_level():
        a, b = tsa.rotary_embedding(fwAD.make_dual(q, tq), fwAD.make_dual(k, tk), pos, f, **how)
        (pq, gq), (pk, gk) = fwAD.unpack_dual(a), fwAD.unpack_dual(b)
        assert torch.equal(gq.detach(), dq) and torch.equal(gk.detach(), dk) and pq.requires_grad and gq.requires_grad
        got = torch.autograd.grad((pq, pk, gq), (q, k, tq), (tq.detach(), tk, q.detach()))
    want = tsa.rotary_embedding(tq.detach(), tk, pos, f, inverse=True, **how)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(got[2], tsa.rotary_embedding(q.detach(), None, pos, f, inverse=True, **how))


def test_transforms(dev):
    """torch.func.jvp and jacfwd, of one operand and through both."""
    import torch_spyre_amd as tsa

    q, k, tq, tk, pos, f, how = operands(dev, False)
    y, t = torch.func.jvp(lambda x: tsa.rotary_embedding(x, None, pos, f, **how), (q,), (tq,))
    assert torch.equal(y, tsa.rotary_embedding(q, None, pos, f, **how))
    assert torch.equal(t, tsa.rotary_embedding(tq, None, pos, f, **how))
    _, (gq, gk) = torch.func.jvp(lambda x, z: tsa.rotary_embedding(x, z, pos, f, **how), (q, k), (tq, tk))
    assert torch.equal(gq, t) and torch.equal(gk, tsa.rotary_embedding(tk, None, pos, f, **how))
    small = q[:1, :1, :1].contiguous()
    jac = torch.func.jacfwd(lambda x: tsa.rotary_embedding(x, None, pos[:1], f, **how))(small)
    for i in (0, 7, 16, 40):
        e = torch.zeros_like(small)
        e[..., i] = 1
        assert torch.equal(jac[..., i].reshape(small.shape), tsa.rotary_embedding(e, None, pos[:1], f, **how))


def test_frequencies_take_no_tangent(dev):
    import torch_spyre_amd as tsa

    q, _, _, _, pos, f, how = operands(dev, False)
    with fwAD.dual_level(), pytest.raises(ValueError):
        tsa.rotary_embedding(q, None, pos, fwAD.make_dual(f, torch.ones_like(f)), **how)


def test_strides(dev):
    """Operands and tangents of other strides than each other's, a packed projection's among them."""
    import torch_spyre_amd as tsa

    q, k, tq, tk, pos, f, how = operands(dev, False)
    packed = torch.cat((q, k), 1).transpose(1, 2).contiguous()
    a, b = packed[:, :, :4].transpose(1, 2), packed[:, :, 4:].transpose(1, 2)
    with fwAD.dual_level():
        yq, yk = tsa.rotary_embedding(fwAD.make_dual(a, tq), fwAD.make_dual(b, tk), pos, f, **how)
        want = tsa.rotary_embedding(q, k, pos, f, **how) + tsa.rotary_embedding(tq, tk, pos, f, **how)
        got = [fwAD.unpack_dual(x) for x in (yq, yk)]
        for x, y in zip([g.primal for g in got] + [g.tangent for g in got], want):
            assert torch.equal(x, y)
