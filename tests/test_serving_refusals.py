"""CPU: the C ABI of the rotary, 8-bit cache and draft attention refuses what it
does not handle before it touches a device, and the ops are registered with
their schemas, CUDA and fake kernels.  The pointers here are never followed."""

import ctypes

import pytest
import torch

PTR, ST = 4096, (ctypes.c_int64 * 3)(64, 64, 64)


@pytest.fixture(scope="module")
def L():
    from torch_spyre_amd import _lib

    return _lib.lib()


EINVAL, EUNSUPPORTED, ENOSPC = -1, -2, -3


def call(fn, args, change):
    a = dict(args) | change
    return fn(*a.values())


ROTARY = dict(q=PTR, qs=ST, qo=PTR, qos=ST, Hq=2, k=PTR, ks=ST, ko=PTR, kos=ST, Hkv=1, dt=5, pos=PTR, pb=4, sb=0, ss=1,
              f=PTR, pairs=32, amp=1.0, il=0, inv=0, B=1, S=1, D=64, stream=None)


@pytest.mark.parametrize("change,code", [
    ({"q": None}, EINVAL), ({"k": None}, EINVAL), ({"qo": None}, EINVAL), ({"pos": None}, EINVAL), ({"f": None}, EINVAL),
    ({"B": -1}, EINVAL), ({"D": 0}, EINVAL), ({"pairs": 33}, EINVAL), ({"pairs": 0}, EINVAL), ({"pb": 2}, EINVAL),
    ({"dt": 4}, EUNSUPPORTED), ({"pairs": 513, "D": 2048}, EUNSUPPORTED), ({"B": 1 << 16, "S": 1 << 16}, EUNSUPPORTED),
    ({"B": 0}, 0), ({"S": 0, "q": None}, 0), ({"Hq": 0, "Hkv": 0}, 0)])
def test_rotary(L, change, code):
    assert call(L.spyre_rotary, ROTARY, change) == code


APPEND = dict(q=PTR, qs=ST, qo=PTR, Hq=2, k=PTR, ks=ST, v=PTR, vs=ST, kc=PTR, vc=PTR, ksc=PTR, vsc=PTR, codes=1, bt=PTR,
              bts=4, pps=4, sl=PTR, slb=1, slt=1, pos=PTR, pb=4, psb=1, pst=1, f=PTR, pairs=32, amp=1.0, il=0, B=1, T=1,
              Hkv=1, D=64, page=64, pages=4, stream=None)


@pytest.mark.parametrize("change,code", [
    ({"k": None}, EINVAL), ({"vc": None}, EINVAL), ({"ksc": None}, EINVAL), ({"bt": None}, EINVAL), ({"sl": None}, EINVAL),
    ({"q": None}, EINVAL), ({"pos": None}, EINVAL), ({"f": None}, EINVAL), ({"codes": 0}, EINVAL), ({"codes": 3}, EINVAL),
    ({"Hkv": 0}, EINVAL), ({"pages": 0}, EINVAL), ({"k": PTR + 8}, EINVAL), ({"qo": PTR + 2}, EINVAL), ({"pb": 3}, EINVAL),
    ({"ks": (ctypes.c_int64 * 3)(64, 64, 60)}, EINVAL), ({"pairs": 33}, EINVAL), ({"pairs": 0}, EINVAL),
    ({"pairs": 4}, EUNSUPPORTED), ({"D": 96}, EUNSUPPORTED), ({"page": 32}, EUNSUPPORTED),
    ({"B": 1 << 20, "T": 1 << 20}, EUNSUPPORTED), ({"B": 0, "k": None}, 0), ({"T": 0, "k": None}, 0)])
def test_append(L, change, code):
    assert call(L.spyre_kv_quant_append, APPEND, change) == code


READ = dict(kc=PTR, vc=PTR, ks=PTR, vs=PTR, codes=2, bt=PTR, bts=4, pps=4, lens=PTR, start=None, k=PTR, v=PTR, B=1, Hkv=1,
            L=5, D=64, page=64, pages=4, stream=None)


@pytest.mark.parametrize("change,code", [
    ({"kc": None}, EINVAL), ({"vs": None}, EINVAL), ({"lens": None}, EINVAL), ({"v": None}, EINVAL), ({"codes": 0}, EINVAL),
    ({"L": -1}, EINVAL), ({"k": PTR + 4}, EINVAL), ({"D": 32}, EUNSUPPORTED), ({"page": 128}, EUNSUPPORTED),
    ({"B": 1 << 20, "L": 1 << 20}, EUNSUPPORTED), ({"B": 0, "kc": None}, 0), ({"L": 0, "kc": None}, 0)])
def test_read(L, change, code):
    assert call(L.spyre_kv_quant_read, READ, change) == code


TREE = dict(q=PTR, qs=ST, kc=PTR, vc=PTR, ks=None, vs=None, kind=0, bt=PTR, bts=4, pps=4, ctx=PTR, n=None, keys=1, mask=None,
            ms=None, out=PTR, lse=None, ws=None, wsb=0, B=1, T=2, Hq=2, Hkv=1, D=64, page=64, pages=4, max=100, scale=1.0,
            stream=None)


@pytest.mark.parametrize("change,code", [
    ({"q": None}, EINVAL), ({"kc": None}, EINVAL), ({"ctx": None}, EINVAL), ({"out": None}, EINVAL), ({"mask": PTR}, EINVAL),
    ({"kind": 1}, EINVAL), ({"kind": 5}, EINVAL), ({"Hq": 3, "Hkv": 2}, EINVAL), ({"Hkv": 0}, EINVAL), ({"max": -1}, EINVAL),
    ({"q": PTR + 8}, EINVAL), ({"out": PTR + 4}, EINVAL), ({"qs": (ctypes.c_int64 * 3)(64, 4, 64)}, EINVAL),
    ({"pages": 0}, EINVAL), ({"D": 256}, EUNSUPPORTED), ({"page": 16}, EUNSUPPORTED), ({"T": 1 << 30}, EUNSUPPORTED),
    ({"max": (1 << 31) - 2}, EUNSUPPORTED), ({"max": 1 << 20}, ENOSPC), ({"max": 1 << 20, "ws": PTR, "wsb": 64}, ENOSPC),
    ({"max": 1 << 20, "ws": PTR + 4, "wsb": 1 << 40}, ENOSPC), ({"B": 0, "q": None}, 0), ({"T": 0, "q": None}, 0)])
def test_tree(L, change, code):
    assert call(L.spyre_paged_tree_attn, TREE, change) == code


SCHEMAS = {
    "rotary": "spyre::rotary(Tensor q, Tensor? k, Tensor positions, Tensor frequencies, float amplitude=1., "
              "bool interleaved=False, bool inverse=False) -> (Tensor, Tensor)",
    "kv_quant_append": "spyre::kv_quant_append(Tensor k_new, Tensor v_new, Tensor(a!) k_cache, Tensor(b!) v_cache, "
                       "Tensor(c!) k_scale, Tensor(d!) v_scale, Tensor block_table, Tensor slots) -> ()",
    "rotary_kv_quant_append": "spyre::rotary_kv_quant_append(Tensor q, Tensor k_new, Tensor v_new, Tensor(a!) k_cache, "
                              "Tensor(b!) v_cache, Tensor(c!) k_scale, Tensor(d!) v_scale, Tensor block_table, "
                              "Tensor slots, Tensor positions, Tensor frequencies, float amplitude=1., "
                              "bool interleaved=False) -> Tensor",
    "kv_quant_read": "spyre::kv_quant_read(Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, "
                     "Tensor block_table, Tensor lens, int length, Tensor? start=None) -> (Tensor, Tensor)",
    "quant_paged_decode_attention": "spyre::quant_paged_decode_attention(Tensor q, Tensor k_cache, Tensor v_cache, "
                                    "Tensor k_scale, Tensor v_scale, Tensor block_table, Tensor context_lens, "
                                    "float? scale=None, int max_context_len=-1) -> (Tensor, Tensor)",
    "paged_tree_attention": "spyre::paged_tree_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, "
                            "Tensor context_lens, Tensor? tree_mask=None, Tensor? draft_lens=None, "
                            "Tensor? k_scale=None, Tensor? v_scale=None, float? scale=None, "
                            "int max_context_len=-1) -> (Tensor, Tensor)",
}


@pytest.mark.parametrize("name", sorted(SCHEMAS))
def test_schema_and_kernels(L, name):
    import torch_spyre_amd  # noqa: F401

    op = getattr(torch.ops.spyre, name).default
    assert str(op._schema) == SCHEMAS[name]
    assert torch._C._dispatch_has_kernel_for_dispatch_key(op.name(), "CUDA")
    assert not torch._C._dispatch_has_kernel_for_dispatch_key(op.name(), "CPU")
    assert torch._C._dispatch_has_kernel_for_dispatch_key(op.name(), "Meta")


def test_fake_shapes(L):
    from torch._subclasses.fake_tensor import FakeTensorMode

    import torch_spyre_amd  # noqa: F401

    with FakeTensorMode():
        e = lambda *s, t=torch.float16: torch.empty(s, dtype=t, device="cuda")  # noqa: E731
        q, k = torch.ops.spyre.rotary(e(2, 3, 8, 64).transpose(1, 2), e(2, 2, 3, 64).transpose(1, 2).transpose(1, 2),
                                      e(2, 8, t=torch.int32), e(32, t=torch.float64))
        assert q.shape == (2, 8, 3, 64) and q.stride() == (3 * 8 * 64, 64, 8 * 64, 1) and k.shape == (2, 2, 3, 64)
        f8, f32, i32 = torch.float8_e4m3fn, torch.float32, torch.int32
        cache = (e(4, 2, 4, 64, 16, t=f8), e(4, 2, 4, 64, 16, t=f8), e(4, 2, 64, t=f32), e(4, 2, 64, t=f32))
        k, v = torch.ops.spyre.kv_quant_read(*cache, e(2, 2, t=i32), e(2, t=i32), 100)
        assert k.shape == v.shape == (2, 2, 100, 64) and k.dtype == torch.float16
        out, lse = torch.ops.spyre.paged_tree_attention(e(2, 5, 4, 64), *cache[:2], e(2, 2, t=i32), e(2, t=i32), None, None,
                                                        *cache[2:])
        assert out.shape == (2, 5, 4, 64) and lse.shape == (2, 5, 4) and lse.dtype == f32
        out, lse = torch.ops.spyre.quant_paged_decode_attention(e(2, 4, 64), *cache, e(2, 2, t=i32), e(2, t=i32))
        assert out.shape == (2, 4, 64) and lse.shape == (2, 4)


def test_fake_strides_of_rotary(L):
    """Features lie next to each other in the results, as the kernel leaves them."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    import torch_spyre_amd  # noqa: F401

    with FakeTensorMode():
        e = lambda *s, t=torch.float16: torch.empty(s, dtype=t, device="cuda")  # noqa: E731
        q, k = torch.ops.spyre.rotary(e(2, 3, 64, 8).transpose(2, 3), e(2, 1, 8, 64).expand(2, 3, 8, 64), e(8, t=torch.int32),
                                      e(32, t=torch.float64))
        assert q.shape == (2, 3, 8, 64) and q.stride(-1) == 1 and k.shape == (2, 3, 8, 64) and k.stride(-1) == 1
