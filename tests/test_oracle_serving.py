"""CPU: pins of the fp64 definitions that the rotary, 8-bit cache and draft
attention tests compare against, and of rotary_frequencies."""

import math

import numpy as np
import pytest
import torch

from oracle import attention as OA
from oracle import serving as OS
from tests.conftest import SEED


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation(interleaved):
    r = np.random.default_rng(SEED)
    x = r.standard_normal((3, 5, 8))
    quarter = OS.rotate(x, np.ones(5), [math.pi / 2, 0.0], interleaved=interleaved)
    a, b = (0, 1) if interleaved else (0, 2)
    assert np.allclose(quarter[..., a], -x[..., b], atol=1e-15) and np.allclose(quarter[..., b], x[..., a], atol=1e-15)
    assert np.array_equal(quarter[..., 4:], x[..., 4:])
    pos = r.integers(-100000, 100000, 5)
    f = r.uniform(0, 1, 4)
    y = OS.rotate(x, pos, f, 1.5, interleaved)
    assert np.allclose((y ** 2).sum(-1), 2.25 * (x ** 2).sum(-1))
    assert np.allclose(OS.rotate(y, pos, f, 1.0, interleaved, inverse=True), 1.5 * x)


def test_codes():
    numbers = np.unique(torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy())
    numbers = numbers[np.isfinite(numbers)].astype(np.float64)
    assert np.array_equal(OS.e4m3_nearest(numbers), numbers) and numbers.max() == 448
    between = np.random.default_rng(SEED).uniform(-448, 448, 4000)
    near = numbers[np.abs(between[:, None] - numbers).argmin(1)]
    assert np.array_equal(OS.e4m3_nearest(between), near)
    assert OS.e4m3_nearest(17.0) == 16.0 and OS.e4m3_nearest(19.0) == 20.0  # ties to even
    assert OS.e4m3_nearest(2.0 ** -10) == 0.0 and OS.e4m3_nearest(3 * 2.0 ** -10) == 2.0 ** -8
    for codes in ("e4m3", "int8"):
        c, s = OS.quantise(np.zeros((2, 16)), codes)
        assert not c.any() and np.array_equal(s, np.ones(2, np.float32))
        c, s = OS.quantise(np.array([[-3.0, 1.5, 0.0]]), codes)
        assert c[0, 0] == -OS.TOP[codes] and s[0] == np.float32(3.0 / OS.TOP[codes])


def test_attend_pins():
    r = np.random.default_rng(SEED)
    q, k, v = r.standard_normal((4, 6, 16)), r.standard_normal((2, 9, 16)), r.standard_normal((2, 9, 16))
    keep = OS.tree_keep(5, 4, 4)
    out, lse, _ = OS.attend(q, k, v, keep)
    mask = np.tril(np.ones((9, 9), bool))[5:]
    ref, rl = OA.sdpa_decomposition_fp64(q.transpose(1, 0, 2)[None], k[None], v[None], attn_mask=mask, return_lse=True)
    assert np.allclose(out, ref[0].transpose(1, 0, 2)) and np.allclose(lse, rl[0].T)
    keep[1] = False
    keep[2] = np.arange(9) == 7
    v[:, 6] = np.nan
    out, lse, _ = OS.attend(q, k, v, keep)
    assert not out[1].any() and np.all(np.isneginf(lse[1]))
    assert np.allclose(out[2], np.repeat(v[:, 7], 3, 0)) and np.isfinite(out[2]).all()
    assert OS.tree_keep(3, 2, 4)[2:].sum() == 0


def test_frequencies():
    import torch_spyre_amd as tsa

    i = torch.arange(64, dtype=torch.float64)
    plain, a = tsa.rotary_frequencies(128, device="cpu")
    assert plain.dtype == torch.float64 and a == 1.0
    assert torch.allclose(plain, 10000.0 ** (-i / 64), rtol=1e-15)
    linear, _ = tsa.rotary_frequencies(128, scaling="linear", factor=4.0, device="cpu")
    assert torch.equal(linear, plain / 4)
    ntk, _ = tsa.rotary_frequencies(128, scaling="ntk", factor=4.0, device="cpu")
    assert ntk[0] == 1.0 and abs(ntk[-1] * 4 / plain[-1] - 1) < 1e-12
    for kind, fast in (("yarn", 32.0), ("llama3", 4.0)):
        f, a = tsa.rotary_frequencies(128, scaling=kind, factor=8.0, original_positions=4096, device="cpu")
        turns = 4096 * plain / (2 * math.pi)
        ratio = f / plain
        assert torch.all(ratio[turns > 1.3 * fast] == 1.0) and torch.allclose(ratio[turns < 0.7], torch.tensor(0.125).double())
        assert torch.all(ratio.diff() <= 1e-15)
        assert a == (pytest.approx(0.1 * math.log(8.0) + 1) if kind == "yarn" else 1.0)
    assert tsa.rotary_frequencies(64, scaling="yarn", factor=2.0, amplitude=1.0, device="cpu")[1] == 1.0
    for bad in ({"rotary_dim": 63}, {"rotary_dim": 0}, {"rotary_dim": 64, "scaling": "other"},
                {"rotary_dim": 64, "factor": 0.0}, {"rotary_dim": 2, "scaling": "ntk"},
                {"rotary_dim": 64, "scaling": "yarn", "fast_turns": 1.0}):
        with pytest.raises(ValueError):
            tsa.rotary_frequencies(device="cpu", **bad)
