"""GPU: attention of drafted tokens whose keys hold infinities, so that runs of
tokens score -inf: they weigh nothing, wherever a run begins."""

import pytest
import torch

from tests.conftest import SEED
from tests.test_quantized_gpu import table_of
from tests.test_tree_attention_gpu import check, logical, make_cache

pytestmark = pytest.mark.gpu


# Rows to a KV head: 12, 40, 64, 80, 100, 120, 160, 300.
@pytest.mark.parametrize("T,Hq,Hkv,D", [(3, 8, 2, 128), (10, 4, 1, 64), (16, 4, 1, 64), (20, 8, 2, 64), (25, 8, 2, 128),
                                        (30, 4, 1, 64), (40, 8, 2, 128), (150, 2, 1, 64)])
@pytest.mark.parametrize("ctx,runs", [
    (400, [(0, 32)]), (400, [(0, 64)]), (400, [(0, 150)]), (400, [(32, 64)]), (90, [(0, 90)]),
    (3000, [(0, 600), (900, 1700)])])
def test_runs_that_score_minus_infinity(cuda, T, Hq, Hkv, D, ctx, runs):
    import torch_spyre_amd as tsa

    W = (ctx + T + 63) // 64
    cache = make_cache("f16", W, Hkv, D, cuda, SEED + 1)
    table = table_of(1, W, W, cuda, SEED + 2)
    for first, end in runs:
        for t in range(first, end):
            cache.k[int(table[0, t // 64]), :, 0, t % 64, 0] = float("-inf")
    q = torch.randn((1, T, Hq, D), generator=torch.Generator(device=cuda).manual_seed(SEED + 3), device=cuda).half()
    q[..., 0] = q[..., 0].abs() + 0.125
    out, lse = tsa.paged_tree_attention(q, cache.k, cache.v, table, torch.tensor([ctx], dtype=torch.int32, device=cuda),
                                        max_context_len=ctx, return_lse=True)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    kl, vl = logical(cache, "f16")
    check(out, lse, q, kl, vl, table.cpu().numpy(), [ctx], [T], None)
