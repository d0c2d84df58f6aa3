"""GPU: lengths and strides of latent attention outside of what its tensors hold or its kernels reach."""

import math

import pytest
import torch

from tests.conftest import SEED
from tests.test_latent_gpu import randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128])
def test_negative_contexts_of_prompts(cuda, D):
    """They count as 0, also where there are fewer keys than queries: that is NaN."""
    import torch_spyre_amd as tsa

    B, T, keys = 6, 70, 66
    k, v, kr = randn((B, keys, 2, D), cuda, SEED), randn((B, keys, 2, D), cuda, SEED + 1), randn((B, keys, 64), cuda, SEED + 2)
    q = randn((B, T, 2, D + 64), cuda, SEED + 3)
    call = lambda ctx, n: tsa.latent_attention(q[..., :D], q[..., D:], k, kr, v, torch.tensor(ctx, dtype=torch.int32, device=cuda),  # noqa: E731
                                               torch.tensor(n, dtype=torch.int32, device=cuda), return_lse=True)
    n = [70, 67, 66, 3, 0, 70]
    want = call([0] * B, n)
    out, lse = call([-5, -1, -5, -(2**31), -7, -100], n)
    for b in range(B):
        if n[b] > keys:
            assert out[b, :n[b]].isnan().all() and lse[b, :n[b]].isnan().all()
            assert want[0][b, :n[b]].isnan().all()
            assert not out[b, n[b]:].any() and (lse[b, n[b]:] == -math.inf).all()
        else:
            assert torch.equal(out[b], want[0][b]) and torch.equal(lse[b], want[1][b])


@pytest.mark.parametrize("far", ["heads", "tokens", "rotated heads", "rotated tokens"])
@pytest.mark.parametrize("H", [2, 40])
def test_queries_far_apart(cuda, far, H):
    """Strides beyond the kernels' 31 bits, as a product batched over heads leaves them."""
    import torch_spyre_amd as tsa

    B, T, rank = 2, 3, 256
    cache, table = randn((8, 5, 64, 64), cuda, SEED), torch.tensor([[3, 1], [0, 7]], dtype=torch.int32, device=cuda)
    q, qr = randn((B, T, H, rank), cuda, SEED + 1, 0.5), randn((B, T, H, 64), cuda, SEED + 2)
    ctx = torch.tensor([70, 3], dtype=torch.int32, device=cuda)
    call = lambda q, qr: tsa.paged_latent_attention(q, qr, cache, table, ctx, 0.07, max_context_len=70, return_lse=True)  # noqa: E731
    want = call(q, qr)
    x = qr if "rotated" in far else q
    F = x.shape[-1]
    step = ((1 << 30) + (H if "heads" in far else T) - 2) // ((H if "heads" in far else T) - 1) + 8 & ~7
    strides = (T * F, F, step, 1) if "heads" in far else (H * F, step, F, 1)
    room = torch.empty(sum((n - 1) * s for n, s in zip(x.shape, strides)) + 1, dtype=torch.float16, device=cuda)
    wide = room.as_strided(x.shape, strides)
    wide.copy_(x)
    out, lse = call(q, wide) if "rotated" in far else call(wide, qr)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


@pytest.mark.parametrize("far", [0, 1, 2])
@pytest.mark.parametrize("step", [(1 << 23) - 8, 1 << 23, (1 << 24) + 8])
def test_keys_far_apart(cuda, far, step):
    """Tokens of keys, rotated keys or values beyond the kernels' 31 bits, as [keys, B, H, D] has them."""
    import torch_spyre_amd as tsa

    T, keys, H, D = 5, 70, 2, 64
    k, v, kr = randn((1, keys, H, D), cuda, SEED), randn((1, keys, H, D), cuda, SEED + 1), randn((1, keys, 64), cuda, SEED + 2)
    q, ctx = randn((1, T, H, D + 64), cuda, SEED + 3), torch.tensor([keys - T], dtype=torch.int32, device=cuda)
    call = lambda k, kr, v: tsa.latent_attention(q[..., :D], q[..., D:], k, kr, v, ctx, return_lse=True)  # noqa: E731
    want = call(k, kr, v)
    x = [k, kr, v]
    like = x[far]
    room = torch.empty(keys * step, dtype=torch.float16, device=cuda)
    x[far] = room.as_strided(like.shape, (8, step) + like.stride()[2:])
    x[far].copy_(like)
    out, lse = call(*x)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    none = call(*(y[:, :0] for y in x)) if far == 0 else None  # no keys: the strides do not matter
    assert none is None or none[0].isnan().all()
