"""CPU: drafted-token attention refuses more rows than its kernels can index,
before it touches a device.  The pointers here are never followed."""

import pytest

from tests.test_serving_refusals import ENOSPC, EUNSUPPORTED, L, TREE, call  # noqa: F401  (L: the fixture)


@pytest.mark.parametrize("T,Hq,Hkv,D,code", [
    (1 << 26, 1, 1, 128, EUNSUPPORTED), (1 << 27, 1, 1, 64, EUNSUPPORTED), (1 << 22, 16, 1, 128, EUNSUPPORTED),
    ((1 << 26) - (1 << 14), 1, 1, 128, EUNSUPPORTED), (1 << 20, 64, 1, 128, EUNSUPPORTED),
    (1 << 25, 1, 1, 128, ENOSPC), (1 << 26, 1, 1, 64, ENOSPC), (1 << 22, 8, 1, 128, ENOSPC), (1 << 25, 2, 2, 128, ENOSPC)])
def test_rows(L, T, Hq, Hkv, D, code):  # noqa: F811
    """32-bit indexes: rows x D / 4 items and the grid's stride past the last
    one.  What is allowed asks for its workspace; the rest has none."""
    sizes = dict(T=T, Hq=Hq, Hkv=Hkv, D=D)
    assert call(L.spyre_paged_tree_attn, TREE, sizes) == code
    need = L.spyre_paged_tree_attn_workspace_bytes(0, 1, T, Hq, Hkv, D, 100, 1)
    assert (need == 0) == (code == EUNSUPPORTED)
