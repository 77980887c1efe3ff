"""The 64-bit restatement of the quantised cache against torch's own e4m3 type, against every e2m1 / e4m3 number, and
against its definition (no element further than half a step away, scale as small as it may be)."""
import numpy as np
import pytest
import torch

from oracle import ref_kvmx as K


def test_grids_are_the_types():
    every = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(K.GRID["mxfp8"], every)
    assert list(K.GRID["mxfp4"]) == [0, 0.5, 1, 1.5, 2, 3, 4, 6]


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
def test_codes_survive_a_round_trip(fmt):
    n = len(K.GRID[fmt])
    x = np.zeros((2 * n, 32))
    x[:n, 0], x[n:, 0] = K.GRID[fmt], -K.GRID[fmt]
    x[:, 1] = K.GRID[fmt][-1]                      # holds the scale at 1
    code, e = K.quantise(x, fmt)
    assert (e == 127).all()
    assert np.array_equal(K.values(K.pack(code, fmt), e, fmt), x)
    assert np.array_equal(code[:n, 0], np.arange(n))


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
def test_half_a_step_at_most_and_the_smallest_scale(fmt):
    g = np.random.RandomState(0)
    x = torch.from_numpy(g.randn(400, 64) * np.exp2(g.randint(-20, 20, (400, 1)))).bfloat16().double().numpy()
    code, e = K.quantise(x, fmt)
    v = K.values(K.pack(code, fmt), e, fmt)
    s = np.repeat(2.0 ** (e.astype(float) - 127), 32, -1)
    grid = np.append(K.GRID[fmt], 2 * K.EDGE[fmt] - K.GRID[fmt][-1])       # the step the largest code would have
    y = np.abs(x) / s
    lo = np.searchsorted(grid, y, side="right") - 1
    step = grid[np.minimum(lo + 1, len(grid) - 1)] - grid[lo]
    assert (np.abs(v - x) <= step * s / 2).all()
    top = np.abs(x).reshape(400, 2, 32).max(-1)
    assert (top <= K.EDGE[fmt] * 2.0 ** (e.astype(float) - 127)).all()
    assert (top > K.EDGE[fmt] * 2.0 ** (e.astype(float) - 128)).all()


def test_ties_zero_and_non_finite_blocks():
    x = np.zeros((1, 64))
    x[0, :8] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0]
    x[0, 8] = -0.0
    code, e = K.quantise(x, "mxfp4")
    assert list(code[0, :9]) == [0, 2, 2, 4, 4, 6, 6, 7, 8] and list(e[0]) == [127, 1]
    x[0, 40] = np.inf
    x[0, 0] = np.nan
    for fmt in K.GRID:
        code, e = K.quantise(x, fmt)
        assert (e == 255).all() and (code == 0).all()
        assert np.isnan(K.values(K.pack(code, fmt), e, fmt)).all()


def test_attention_of_one_key_is_its_value_and_of_none_zero():
    g = np.random.RandomState(1)
    q, k, v = g.randn(4, 64), g.randn(2, 1, 64), g.randn(2, 1, 64)
    out, _ = K.attend(q, k, v, 0.125)
    assert np.allclose(out, np.repeat(v[:, 0], 2, 0), rtol=1e-15)
    assert (K.attend(q, k[:, :0], v[:, :0], 0.125)[0] == 0).all()


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
def test_no_rows(fmt):
    code, e = K.quantise(np.zeros((2, 0, 64)), fmt)
    assert code.shape == (2, 0, 64) and e.shape == (2, 0, 2) and K.values(K.pack(code, fmt), e, fmt).shape == (2, 0, 64)


def test_weights_in_two_bf16_numbers():
    """What the bound of several query heads a kv head counts for them, and that it is not idle."""
    import torch
    w = 1 + torch.rand(1 << 20, generator=torch.Generator().manual_seed(0))
    w = torch.cat([w, 1 + 2.0 ** -8 - torch.arange(1, 1 << 15) * 2.0 ** -23])
    high = w.bfloat16().float()
    off = ((high + (w - high).bfloat16().float()).double() - w.double()).abs()
    assert 2.0 ** -18 < float(off.max()) <= 2.0 ** -17
    q, k, v = np.zeros((2, 64)), np.zeros((1, 1, 64)), np.ones((1, 1, 64))
    several, one = K.attend(q, k, v, 1.0)[1], K.attend(q[:1], k, v, 1.0)[1]
    assert np.allclose(several - one, 2.0 ** -17, rtol=1e-6)
