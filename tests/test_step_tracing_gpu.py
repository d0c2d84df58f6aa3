"""GPU: page plans, draft verification, the latent cache and latent attention through
the dispatcher's own checks (schema, fake kernels, traced form)."""

import pytest
import torch

from tests.conftest import SEED
from tests.test_latent_gpu import randn, table_of

pytestmark = pytest.mark.gpu


def cases(dev):
    ops, i32 = torch.ops.spyre, dict(dtype=torch.int32, device=dev)
    table, lens = table_of(2, 4, 12, dev, SEED), torch.tensor([100, 64], **i32)
    held, new = torch.tensor([2, 1], **i32), torch.tensor([5, 3], **i32)
    ring, cursor = torch.arange(12, **i32), torch.tensor([8, 12], dtype=torch.int64, device=dev)
    cache = randn((12, 5, 64, 64), dev, SEED + 1)
    p = torch.softmax(randn((2, 5, 300), dev, SEED + 2).float(), -1)
    q = torch.softmax(randn((2, 4, 300), dev, SEED + 3).float(), -1)
    x, u = torch.tensor([[5, 290, 0, 7], [299, 4, 4, 1]], device=dev), torch.tensor([[0.1, 0.9, 0.5, 0.2, 0.7]] * 2, device=dev)
    parents = torch.tensor([[-1, -1, 0, 1]] * 2, **i32)
    mask = torch.ones((5, 5), dtype=torch.bool, device=dev).tril()
    slots = torch.tensor([3, 70, -1], dtype=torch.int64, device=dev)
    kv = randn((2, 110, 3, 128), dev, SEED + 4)
    return {
        "plan_pages": (ops.plan_pages, (table, held, lens, new, ring, cursor, 6)),
        "plan_pages, packed": (ops.plan_pages, (table, held, lens, new, ring, cursor, -1, 9)),
        "release_pages": (ops.release_pages, (table, held, new, ring, cursor)),
        "verify_drafts": (ops.verify_drafts, (x, p, u)),
        "verify_drafts, q": (ops.verify_drafts, (x, p, u, q, None, new - 1)),
        "verify_drafts, tree": (ops.verify_drafts, (x, p, u, None, parents)),
        "latent_append": (ops.latent_append, (randn((3, 256), dev, SEED + 5), randn((3, 64), dev, SEED + 6), cache, slots)),
        "latent_read": (ops.latent_read, (cache, table, lens, 20, lens - 15)),
        "paged_latent_attention": (ops.paged_latent_attention,
                                   (randn((2, 5, 3, 256), dev, SEED + 7), randn((2, 5, 3, 64), dev, SEED + 8), cache, table, lens,
                                    0.1, mask, new, 100)),
        "latent_attention": (ops.latent_attention, (randn((2, 5, 3, 64), dev, SEED + 9), randn((2, 5, 3, 64), dev, SEED + 10),
                                                    kv[..., :64], randn((2, 110, 64), dev, SEED + 11), kv[..., 64:], lens, new)),
    }


NAMES = ["plan_pages", "plan_pages, packed", "release_pages", "verify_drafts", "verify_drafts, q", "verify_drafts, tree",
         "latent_append", "latent_read", "paged_latent_attention", "latent_attention"]


@pytest.mark.parametrize("name", NAMES)
def test_opcheck(cuda, name):
    op, args = cases(cuda)[name]
    torch.library.opcheck(op, args)
