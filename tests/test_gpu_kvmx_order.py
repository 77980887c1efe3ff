"""The quantised cache's decode step with more workgroups than the chip holds, which takes long streams first; blocks with a
NaN in every core and form; repeated calls; the largest values whose sums stay finite."""
import numpy as np
import pytest
import torch

from oracle import ref_kvmx as K
from test_gpu_kvmx import FMT, attention_case, bf16_rows, check_attention, dev, put

pytestmark = pytest.mark.gpu
NAMES = ("k", "k_scale", "v", "v_scale")


@pytest.fixture(scope="module")
def ops():
    from mgen import ops as o
    return o


def many_streams(ops, fmt, B, H, KVH, D, L, seed):
    """Caches of B streams (eight different ones, repeated) with rows of every length up to L, and one new token a stream."""
    g = torch.Generator().manual_seed(seed)
    kv = ops.MXKV.empty(B, KVH, L, D, fmt, dev())
    rows = [bf16_rows(g, 8 * L, KVH * D, spread=1).to(dev()) for _ in range(2)]
    ops.kv_append_mx(*rows, KVH * D, KVH * D, kv, torch.zeros(8, dtype=torch.int32, device=dev()), 8, L)
    for n in NAMES:
        t = getattr(kv, n)
        for b in range(8, B):
            t[b] = t[b % 8]
    lens = torch.randint(1, L + 1, (B,), generator=g, dtype=torch.int32)
    lens[::5] = 700                                      # equal ones
    lens[2], lens[4] = L, 1
    pos, kv_len = lens - 1, lens.clone()
    kv_len[3::11] += 1                                   # streams whose lengths do not fit: zeros, nothing written
    pos[6::17] = torch.tensor([-1, L], dtype=torch.int32).repeat(B)[:pos[6::17].numel()]
    fits = (kv_len == pos + 1) & (pos >= 0) & (pos < L)
    qkv = bf16_rows(g, B, (H + 2 * KVH) * D, spread=1).to(dev())
    gains = [1 + 0.3 * torch.randn(D, generator=g).to(dev()) for _ in range(2)]
    cs = ops.rope_table((1.0 / 10000 ** (torch.arange(0, D, 2).float() / D)).to(dev()), L)
    return kv, qkv, gains, cs, pos.to(dev()), kv_len.to(dev()), fits.to(dev())


def copy_of(ops, kv):
    return ops.MXKV(*(getattr(kv, n).clone() for n in NAMES))


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("B,H,KVH,D,nsplit,step", [(150, 8, 8, 128, 1, 75), (150, 16, 8, 128, 1, 75), (140, 8, 8, 64, 1, 70),
                                                   (90, 16, 8, 64, 2, 45), (130, 20, 2, 128, 4, 65)])
def test_decode_step_takes_long_streams_first(ops, fmt, B, H, KVH, D, nsplit, step):
    """Outputs and caches have the bits of calls on parts of the batch, which take the streams as they are numbered; and the
    bits of a second call."""
    L, il = 1100, D == 64
    kv, qkv, (wq, wk), cs, pos, kv_len, fits = many_streams(ops, fmt, B, H, KVH, D, L, B + H)
    before, parts = copy_of(ops, kv), copy_of(ops, kv)
    ld = (H + 2 * KVH) * D
    ws = torch.empty(ops.attn_decode_workspace(B, H, D, nsplit), dtype=torch.float32, device=dev())
    out, again, want = (torch.full((B, H * D), 7.0, dtype=torch.bfloat16, device=dev()) for _ in range(3))

    def call(cache, o, b, e):
        ops.attn_decode_prep_mx(qkv[b:e], ld, wq, wk, cs, pos[b:e], 1e-6, il, cache.streams(b, e), kv_len[b:e], o[b:e], H * D,
                                ws, e - b, H, nsplit, D ** -0.5)

    call(kv, out, 0, B)
    for b in range(0, B, step):
        call(parts, want, b, min(b + step, B))
    assert torch.equal(out, want)
    at = torch.arange(B, device=dev())
    for n in NAMES:
        a, o = getattr(kv, n), getattr(before, n)
        assert torch.equal(a, getattr(parts, n)), n
        changed = (a != o).flatten(2).any(-1).any(1)
        assert not bool(changed[~fits].any()), n
        a = a.clone()
        a[at[fits], :, pos[fits].long()] = o[at[fits], :, pos[fits].long()]
        assert torch.equal(a, o), n
    assert bool((out[~fits] == 0).all()) and bool((out[fits] != 0).any(-1).all()) and not bool(torch.isnan(out).any())
    call(parts, want, 0, step)                           # something else in between
    call(kv, again, 0, B)
    assert torch.equal(out, again), "the same step gives other bits"


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("B,nsplit", [(2, 1), (2, 3), (140, 1)])
@pytest.mark.parametrize("H,KVH,D", [(2, 2, 64), (2, 2, 128), (4, 2, 64), (4, 2, 128), (20, 2, 64)])
def test_blocks_with_a_nan(ops, fmt, H, KVH, D, B, nsplit):
    """One head and several, both head sizes: a key with an infinity or a NaN makes the rows that attend it NaN, a value its
    block of 32 elements, and nothing else changes."""
    n, G = 600, H // KVH
    args, k, v, q = attention_case(ops, fmt, B, H, KVH, D, n, [n, 560] + [40] * (B - 2), nsplit)
    ops.attn_decode_mx(*args)
    clean = args[4][:B].clone()
    k[0, 411, 1, 3] = float("inf")
    v[1, 50, 0, D - 1] = float("nan")
    v[1, 333, 1, 2] = float("-inf")
    v[1, 560:, 1] = float("nan")           # behind the stream's last key
    put(ops, args[2].streams(0, 2), k[:2], v[:2], [0, 0])
    ops.attn_decode_mx(*args)
    nan = torch.zeros(B, KVH, G, D, dtype=torch.bool)
    nan[0, 1], nan[1, 0, :, D - 32:], nan[1, 1, :, :32] = True, True, True
    nan = nan.view(B, H * D).to(dev())
    got = args[4][:B]
    assert torch.equal(torch.isnan(got), nan)
    assert torch.equal(got[~nan], clean[~nan])


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("H,KVH,D,nsplit", [(2, 2, 64, 1), (2, 2, 128, 3), (4, 2, 64, 3), (4, 2, 128, 1), (20, 2, 128, 2)])
def test_new_token_with_a_nan(ops, fmt, H, KVH, D, nsplit):
    """The decode step's own key or value is not finite: its block is marked in the cache, its rows (its elements) are NaN."""
    B, L, G = 3, 700, H // KVH
    kv, qkv, (wq, wk), cs, _, _, _ = many_streams(ops, fmt, 8, H, KVH, D, L, D + H)
    kv, qkv = kv.streams(0, B), qkv[:B].clone()
    heads = qkv.view(B, H + 2 * KVH, D)
    heads[0, H + 1, 5] = float("nan")                      # (a key's norm spreads it over the head's row)
    heads[1, H + KVH, D - 1] = float("inf")
    pos = torch.tensor([650, 300, 9], dtype=torch.int32, device=dev())
    out = torch.empty(B, H * D, dtype=torch.bfloat16, device=dev())
    ws = torch.empty(max(1, ops.attn_decode_workspace(B, H, D, nsplit)), dtype=torch.float32, device=dev())
    ops.attn_decode_prep_mx(qkv, (H + 2 * KVH) * D, wq, wk, cs, pos, 1e-6, False, kv, pos + 1, out, H * D, ws, B, H, nsplit,
                            D ** -0.5)
    nan = torch.zeros(B, KVH, G, D, dtype=torch.bool, device=dev())
    nan[0, 1], nan[1, 0, :, D - 32:] = True, True
    assert torch.equal(torch.isnan(out).view_as(nan), nan)
    at = torch.arange(B, device=dev())
    ks, vs = kv.k_scale[at, :, pos.long()], kv.v_scale[at, :, pos.long()]      # [B, KVH, D / 32]
    bad_k, bad_v = torch.zeros_like(ks, dtype=torch.bool), torch.zeros_like(vs, dtype=torch.bool)
    bad_k[0, 1], bad_v[1, 0, -1] = True, True
    assert torch.equal(ks == 255, bad_k) and torch.equal(vs == 255, bad_v)
    assert bool((kv.k[at, :, pos.long()][0, 1] == 0).all())


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("H,KVH,D,nsplit", [(2, 2, 64, 1), (2, 2, 128, 1), (4, 2, 64, 1), (4, 2, 128, 2)])
def test_largest_values_whose_sums_are_finite(ops, fmt, H, KVH, D, nsplit):
    """Values of 2^119 / keys in magnitude, weights that run ahead of the maximum in use (which lags by up to 2^8): the sums of
    keys x weight x value stay below fp32's largest number."""
    n = 1500                                              # 2^119 / 1500 > 2^108
    args, k, v, q = attention_case(ops, fmt, 1, H, KVH, D, n, [n], nsplit)
    q[:] = 1.0
    k[:] = 0.4375                                         # scores up to 4.95, a weight of 2^7.2 against a score of 0
    k[:, :n // nsplit // 64 * 32] = 0.0                   # the first units of every wave
    k[:, n // nsplit:][:, :256 if nsplit > 1 else 0] = 0.0
    v[:] = 2.0 ** 108
    v[:, :, 0] *= -1
    put(ops, args[2], k, v, [0])
    args = (q.to(dev()), *args[1:])
    ops.attn_decode_mx(*args)
    check_attention(fmt, args, k, v, q)
    assert bool(torch.isfinite(args[4]).all())
