"""CPU: the C ABI of page plans, draft verification, the latent cache and latent
attention refuses what it does not handle before it touches a device, and the ops
are registered with their schemas, CUDA and fake kernels.  The pointers here are never
followed."""

import ctypes

import pytest
import torch

PTR = 4096
EINVAL, EUNSUPPORTED, ENOSPC = -1, -2, -3


def strides(*x):
    return (ctypes.c_int64 * len(x))(*x)


ST = strides(64, 64, 64)


@pytest.fixture(scope="module")
def L():
    from torch_spyre_amd import _lib

    return _lib.lib()


def call(fn, args, change):
    a = dict(args) | change
    return fn(*a.values())


PLAN = dict(bt=PTR, bts=4, pps=4, held=PTR, ctx=PTR, new=PTR, free=PTR, num=8, cursor=PTR, length=3, tokens=-1, pos=PTR, slots=PTR,
            starts=None, held_out=PTR, cursor_out=PTR, B=2, stream=None)


@pytest.mark.parametrize("change,code", [
    ({"bt": None}, EINVAL), ({"held": None}, EINVAL), ({"ctx": None}, EINVAL), ({"new": None}, EINVAL), ({"free": None}, EINVAL),
    ({"cursor": None}, EINVAL), ({"cursor_out": None}, EINVAL), ({"held_out": None}, EINVAL), ({"slots": None}, EINVAL),
    ({"tokens": 5}, EINVAL), ({"length": -1}, EINVAL), ({"length": -1, "tokens": 5}, EINVAL), ({"B": -1}, EINVAL),
    ({"pps": -1}, EINVAL), ({"num": -1}, EINVAL), ({"B": 4097}, EUNSUPPORTED), ({"pps": 1 << 31}, EUNSUPPORTED),
    ({"num": 1 << 31}, EUNSUPPORTED), ({"B": 2, "length": (1 << 30) + 1}, EUNSUPPORTED)])
def test_plan(L, change, code):
    assert call(L.spyre_plan_pages, PLAN, change) == code


RELEASE = dict(bt=PTR, bts=4, pps=4, held=PTR, lens=PTR, free=PTR, num=8, cursor=PTR, held_out=PTR, cursor_out=PTR, B=2, stream=None)


@pytest.mark.parametrize("change,code", [
    ({"bt": None}, EINVAL), ({"held": None}, EINVAL), ({"lens": None}, EINVAL), ({"free": None}, EINVAL), ({"cursor": None}, EINVAL),
    ({"held_out": None}, EINVAL), ({"B": -1}, EINVAL), ({"B": 5000}, EUNSUPPORTED), ({"pps": 1 << 31}, EUNSUPPORTED)])
def test_release(L, change, code):
    assert call(L.spyre_release_pages, RELEASE, change) == code


VERIFY = dict(tok=PTR, tb=8, tsb=5, tst=1, p=PTR, ps=strides(600, 100), q=None, qs=None, dt=6, u=PTR, usb=6, ust=1, par=None, pab=0,
              pat=0, lens=None, out=PTR, acc=PTR, path=PTR, ws=PTR, wsb=1 << 20, B=2, T=5, V=100, stream=None)


@pytest.mark.parametrize("change,code", [
    ({"tok": None}, EINVAL), ({"p": None}, EINVAL), ({"ps": None}, EINVAL), ({"u": None}, EINVAL), ({"out": None}, EINVAL),
    ({"acc": None}, EINVAL), ({"path": None}, EINVAL), ({"q": PTR}, EINVAL), ({"tb": 2}, EINVAL), ({"V": 0}, EINVAL),
    ({"B": -1}, EINVAL), ({"T": -1}, EINVAL), ({"dt": 7}, EUNSUPPORTED), ({"q": PTR, "qs": strides(1, 1), "par": PTR}, EUNSUPPORTED),
    ({"T": 1025}, EUNSUPPORTED), ({"B": 65536}, EUNSUPPORTED), ({"V": 1 << 30}, EUNSUPPORTED), ({"ws": None}, ENOSPC),
    ({"wsb": 39}, ENOSPC), ({"ws": PTR + 8}, ENOSPC), ({"B": 0, "tok": None}, 0)])
def test_verify(L, change, code):
    assert call(L.spyre_verify_drafts, VERIFY, change) == code


APPEND = dict(x=PTR, xs=256, r=PTR, rs=64, cache=PTR, slots=PTR, rows=3, rank=256, pages=4, stream=None)


@pytest.mark.parametrize("change,code", [
    ({"x": None}, EINVAL), ({"r": None}, EINVAL), ({"cache": None}, EINVAL), ({"slots": None}, EINVAL), ({"x": PTR + 8}, EINVAL),
    ({"rs": 60}, EINVAL), ({"rows": -1}, EINVAL), ({"pages": -1}, EINVAL), ({"rank": 128}, EUNSUPPORTED),
    ({"rows": 1 << 31}, EUNSUPPORTED), ({"rows": 0, "x": None}, 0), ({"pages": 0, "x": None}, 0)])
def test_append(L, change, code):
    assert call(L.spyre_latent_append_f16, APPEND, change) == code


READ = dict(cache=PTR, bt=PTR, bts=4, pps=4, lens=PTR, start=None, x=PTR, r=PTR, B=2, length=5, rank=512, pages=4, stream=None)


@pytest.mark.parametrize("change,code", [
    ({"cache": None}, EINVAL), ({"bt": None}, EINVAL), ({"lens": None}, EINVAL), ({"x": None}, EINVAL), ({"r": PTR + 4}, EINVAL),
    ({"length": -1}, EINVAL), ({"B": -1}, EINVAL), ({"rank": 576}, EUNSUPPORTED), ({"B": 1 << 20, "length": 1 << 20}, EUNSUPPORTED),
    ({"B": 0, "x": None}, 0), ({"length": 0, "x": None}, 0)])
def test_read(L, change, code):
    assert call(L.spyre_latent_read_f16, READ, change) == code


PAGED = dict(q=PTR, qs=ST, qr=PTR, qrs=ST, cache=PTR, bt=PTR, bts=4, pps=4, ctx=PTR, n=None, mask=None, ms=None, out=PTR, lse=None,
             ws=PTR, wsb=1 << 34, B=2, T=2, H=4, rank=512, pages=4, max=100, scale=1.0, stream=None)


@pytest.mark.parametrize("change,code", [
    ({"q": None}, EINVAL), ({"qr": None}, EINVAL), ({"cache": None}, EINVAL), ({"bt": None}, EINVAL), ({"ctx": None}, EINVAL),
    ({"out": None}, EINVAL), ({"mask": PTR}, EINVAL), ({"q": PTR + 8}, EINVAL), ({"out": PTR + 2}, EINVAL),
    ({"qs": strides(64, 4, 64)}, EINVAL), ({"qs": strides(64, 1 << 30, 64)}, EUNSUPPORTED),
    ({"qrs": strides(64, 64, -64)}, EUNSUPPORTED), ({"H": 0}, EINVAL), ({"pages": 0}, EINVAL), ({"max": -1}, EINVAL), ({"B": -1}, EINVAL),
    ({"rank": 384}, EUNSUPPORTED), ({"T": 1 << 30}, EUNSUPPORTED), ({"max": (1 << 31) - 66}, EUNSUPPORTED),
    ({"B": 1 << 20, "max": 1 << 20}, EUNSUPPORTED), ({"ws": None}, ENOSPC), ({"wsb": 64}, ENOSPC), ({"ws": PTR + 4}, ENOSPC),
    ({"B": 0, "q": None}, 0), ({"T": 0, "q": None}, 0)])
def test_paged_attention(L, change, code):
    assert call(L.spyre_paged_latent_attn, PAGED, change) == code


EXPANDED = dict(q=PTR, qs=ST, qr=PTR, qrs=ST, k=PTR, ks=ST, kr=PTR, krs=ST, v=PTR, vs=ST, ctx=PTR, n=None, out=PTR, lse=None, ws=None,
                wsb=0, B=1, T=600, H=128, D=128, keys=700, scale=1.0, stream=None)


@pytest.mark.parametrize("change,code", [
    ({"q": None}, EINVAL), ({"k": None}, EINVAL), ({"kr": None}, EINVAL), ({"v": None}, EINVAL), ({"ctx": None}, EINVAL),
    ({"out": None}, EINVAL), ({"k": PTR + 8}, EINVAL), ({"ks": strides(64, 4, 64)}, EINVAL), ({"krs": strides(64, 4, 1)}, EINVAL),
    ({"H": 0}, EINVAL), ({"keys": -1}, EINVAL), ({"D": 96}, EUNSUPPORTED), ({"ks": strides(64, 1 << 23, 64)}, EUNSUPPORTED),
    ({"vs": strides(64, -64, 64)}, EUNSUPPORTED), ({"keys": 1 << 30}, EUNSUPPORTED), ({"B": 1 << 20, "T": 1 << 20}, EUNSUPPORTED),
    ({"T": 1, "H": 1, "keys": 9000}, ENOSPC), ({"T": 1, "H": 1, "keys": 9000, "ws": PTR + 8, "wsb": 1 << 30}, ENOSPC),
    ({"B": 0, "q": None}, 0), ({"T": 0, "q": None}, 0)])
def test_expanded_attention(L, change, code):
    assert call(L.spyre_latent_attn, EXPANDED, change) == code


SCHEMAS = {
    "plan_pages": "spyre::plan_pages(Tensor(a!) block_table, Tensor held, Tensor context_lens, Tensor new_lens, Tensor free_pages, "
                  "Tensor cursor, int length=-1, int tokens=-1) -> (Tensor, Tensor, Tensor, Tensor, Tensor)",
    "release_pages": "spyre::release_pages(Tensor block_table, Tensor held, Tensor lens, Tensor(a!) free_pages, Tensor cursor) "
                     "-> (Tensor, Tensor)",
    "verify_drafts": "spyre::verify_drafts(Tensor draft_tokens, Tensor target_probs, Tensor uniforms, Tensor? draft_probs=None, "
                     "Tensor? parents=None, Tensor? draft_lens=None) -> (Tensor, Tensor, Tensor)",
    "latent_append": "spyre::latent_append(Tensor latent, Tensor k_rope, Tensor(a!) cache, Tensor slots) -> ()",
    "latent_read": "spyre::latent_read(Tensor cache, Tensor block_table, Tensor lens, int length, Tensor? start=None) "
                   "-> (Tensor, Tensor)",
    "paged_latent_attention": "spyre::paged_latent_attention(Tensor q, Tensor q_rope, Tensor cache, Tensor block_table, "
                              "Tensor context_lens, float scale, Tensor? tree_mask=None, Tensor? draft_lens=None, "
                              "int max_context_len=-1) -> (Tensor, Tensor)",
    "latent_attention": "spyre::latent_attention(Tensor q, Tensor q_rope, Tensor k, Tensor k_rope, Tensor v, Tensor context_lens, "
                        "Tensor? new_lens=None, float? scale=None) -> (Tensor, Tensor)",
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

    f16, f32, i32, i64 = torch.float16, torch.float32, torch.int32, torch.int64
    with FakeTensorMode():
        e = lambda *s, t=f16: torch.empty(s, dtype=t, device="cuda")  # noqa: E731
        lens, table, ops = e(2, t=i32), e(2, 4, t=i32), torch.ops.spyre
        ring = (e(9, t=i32), e(2, t=i64))
        pos, slots, held, cursor, starts = ops.plan_pages(table, lens, lens, lens, *ring, 5)
        assert pos.shape == slots.shape == (2, 5) and pos.dtype == i32 and slots.dtype == i64 and held.shape == (2,)
        assert cursor.shape == (2,) and cursor.dtype == i64 and starts.shape == (0,)
        pos, slots, _, _, starts = ops.plan_pages(table, lens, lens, lens, *ring, -1, 7)
        assert pos.shape == slots.shape == (7,) and starts.shape == (3,) and starts.dtype == i32
        held, cursor = ops.release_pages(table, lens, lens, *ring)
        assert held.shape == (2,) and cursor.shape == (2,) and cursor.dtype == i64
        out, kept, path = ops.verify_drafts(e(2, 3, t=i64), e(2, 4, 50, t=f32), e(2, 4, t=f32))
        assert out.shape == (2, 4) and out.dtype == i64 and kept.shape == (2,) and path.shape == (2, 3) and path.dtype == i32
        cache = e(4, 5, 64, 64)
        assert ops.latent_append(e(3, 256), e(3, 64), cache, e(3, t=i64)) is None
        x, r = ops.latent_read(cache, table, lens, 6)
        assert x.shape == (2, 6, 256) and r.shape == (2, 6, 64)
        out, lse = ops.paged_latent_attention(e(2, 3, 4, 256), e(2, 3, 4, 64), cache, table, lens, 0.1)
        assert out.shape == (2, 3, 4, 256) and lse.shape == (2, 3, 4) and lse.dtype == f32
        out, lse = ops.latent_attention(e(2, 3, 4, 64), e(2, 3, 4, 64), e(2, 9, 4, 64), e(2, 9, 64), e(2, 9, 4, 64), lens)
        assert out.shape == (2, 3, 4, 64) and lse.shape == (2, 3, 4) and lse.dtype == f32


def test_arguments_of_the_functions(L):
    import torch_spyre_amd as tsa

    x = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="either length or tokens"):
        tsa.plan_pages(x.view(1, 2), x, x, x, x, x)
    with pytest.raises(ValueError, match="either length or tokens"):
        tsa.plan_pages(x.view(1, 2), x, x, x, x, x, length=1, tokens=1)
    with pytest.raises(ValueError, match="negative"):
        tsa.plan_pages(x.view(1, 2), x, x, x, x, x, length=-1)
    with pytest.raises(ValueError, match="rank"):
        tsa.LatentKVCache(4, rank=128, device="cpu")
