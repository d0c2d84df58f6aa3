"""GPU: lengths of latent attention outside of what its tensors hold."""

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
