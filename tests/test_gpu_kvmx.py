"""The KV cache in 4 or 8 bits on the GPU: quantising rows as they are written (bytes equal to the oracle's), reading them
back, single-token attention over the cache (within the oracle's derived bound) and the decode step's fused form (the
bits of the launches it stands for)."""
import numpy as np
import pytest
import torch

from oracle import ref_kvmx as K

pytestmark = pytest.mark.gpu

FMT = ["mxfp4", "mxfp8"]


def dev():
    return torch.device("cuda:0")


@pytest.fixture(scope="module")
def ops():
    from mgen import ops as o
    return o


def bf16_rows(g, *shape, spread=6):
    x = torch.randn(*shape, generator=g) * torch.exp2(torch.randint(-spread, spread + 1, shape[-1:], generator=g).float())
    return x.bfloat16()


def filled(ops, B, KVH, L, D, fmt, byte=0xFF):
    """A cache whose memory holds NaN codes and NaN scales."""
    kv = ops.MXKV.empty(B, KVH, L, D, fmt, dev())
    for t in (kv.k, kv.k_scale, kv.v, kv.v_scale):
        t.fill_(byte)
    return kv


def put(ops, kv, rows_k, rows_v, pos):
    """rows [B, n, KVH, D] on the CPU into slots pos[b] ..."""
    B, n = rows_k.shape[:2]
    w = kv.KVH * kv.D
    k, v = rows_k.reshape(B * n, w).to(dev()), rows_v.reshape(B * n, w).to(dev())
    ops.kv_append_mx(k, v, w, w, kv, torch.tensor(pos, dtype=torch.int32, device=dev()), B, n)


def special_rows(D, fmt):
    """Ties, powers of two around the scale's edges, zeros of both signs, the smallest and largest numbers, non-finite."""
    e = K.EDGE[fmt]
    x = torch.zeros(14, D)
    x[0, :8] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0])
    x[1, :4] = torch.tensor([e, e * 1.0078125, -e, 1.0])
    x[2, :3] = torch.tensor([e * 1.0078125, -0.0, 0.5])
    x[3] = 0.0
    x[4] = -0.0
    x[5, ::3] = 1e-40
    x[6, 3] = 2.0 ** -126
    x[7, 5] = 3.3895e38
    x[8, 5], x[8, 6] = -3.3895e38, 1e30
    x[9, 2] = float("inf")
    x[10, D - 1] = float("nan")
    x[11, D // 2] = float("-inf")
    x[12] = torch.linspace(-8, 8, D)
    x[13, :32], x[13, 32:] = 1e-20, 1e20
    return x.bfloat16()


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("B,n,KVH,D,L,ld_extra", [(1, 1, 1, 128, 1, 0), (3, 1, 8, 64, 40, 64), (2, 17, 3, 128, 33, 8),
                                                  (4, 65, 5, 64, 100, 0), (1, 1031, 2, 128, 1031, 128), (7, 3, 1, 64, 9, 8)])
def test_write_and_read_back(ops, fmt, B, n, KVH, D, L, ld_extra):
    g = torch.Generator().manual_seed(B * 1000 + n + D)
    w = KVH * D
    rows = [bf16_rows(g, B * n, w + ld_extra) for _ in range(2)]
    sp = special_rows(D, fmt)
    for r in rows:
        at = torch.randperm(B * n, generator=g)[:14]
        for i, x in zip(at.tolist(), sp[torch.randperm(14, generator=g)]):
            r[i, :D] = x
    pos = torch.randint(0, L - n + 1, (B,), generator=g)
    kv = filled(ops, B, KVH, L, D, fmt, byte=0x5A)
    src = [r.to(dev()) for r in rows]
    ops.kv_append_mx(src[0], src[1], w + ld_extra, w + ld_extra, kv, pos.int().to(dev()), B, n)
    dst = [torch.full((B * n + 1, w + ld_extra), 7.0, dtype=torch.bfloat16, device=dev()) for _ in range(2)]
    ops.kv_read_mx(kv, pos.int().to(dev()), dst[0], dst[1], w + ld_extra, w + ld_extra, B, n)
    for r, d, codes, scales in ((rows[0], dst[0], kv.k, kv.k_scale), (rows[1], dst[1], kv.v, kv.v_scale)):
        x = r[:, :w].reshape(B, n, KVH, D).permute(0, 2, 1, 3).double().numpy()
        want, e = K.quantise(x, fmt)
        want = K.pack(want, fmt)
        codes, scales = codes.cpu().numpy(), scales.cpu().numpy()
        inside = np.zeros((B, L), bool)
        for b in range(B):
            p = int(pos[b])
            inside[b, p:p + n] = True
            assert np.array_equal(scales[b, :, p:p + n], e[b]), b
            assert np.array_equal(codes[b, :, p:p + n], want[b]), b
        assert (codes.transpose(0, 2, 1, 3)[~inside] == 0x5A).all() and (scales.transpose(0, 2, 1, 3)[~inside] == 0x5A).all()
        back = d[:B * n, :w].reshape(B, n, KVH, D).permute(0, 2, 1, 3).float().cpu().numpy()
        val = torch.from_numpy(K.values(want, e, fmt)).bfloat16().float().numpy()
        # (a value below bf16's smallest number, where the block's scale is 2^-126, may read as 0)
        ok = (back == val) | (np.isnan(back) & np.isnan(val)) | ((back == 0) & (np.abs(val) < 2.0 ** -130))
        assert ok.all()
        assert bool((d[B * n] == 7.0).all()) and bool((d[:, w:] == 7.0).all()), "wrote beside the rows"


@pytest.mark.parametrize("fmt", FMT)
def test_slots_outside_the_cache_are_left_alone(ops, fmt):
    B, n, KVH, D, L = 5, 4, 2, 64, 6
    g = torch.Generator().manual_seed(3)
    w = KVH * D
    rows = bf16_rows(g, B * n, w).to(dev())
    pos = torch.tensor([-2, 4, 6, -2 ** 31, 2 ** 31 - 1], dtype=torch.int32, device=dev())
    kv = filled(ops, B, KVH, L, D, fmt, byte=0x21)
    ops.kv_append_mx(rows, rows, w, w, kv, pos, B, n)
    used = (kv.k_scale.cpu() != 0x21).any(-1).any(1)          # [B, L]
    assert used.tolist() == [[True, True, False, False, False, False], [False] * 4 + [True, True]] + [[False] * 6] * 3
    dst = torch.full((B * n, w), 7.0, dtype=torch.bfloat16, device=dev())
    ops.kv_read_mx(kv, pos, dst, dst.clone(), w, w, B, n)
    there = (dst != 7.0).any(-1).view(B, n).tolist()
    assert there == [[False, False, True, True], [True, True, False, False]] + [[False] * 4] * 3


def attention_case(ops, fmt, B, H, KVH, D, L, lens, nsplit, seed=0, ld_extra=0, spread=2):
    """Cache filled through the append kernel behind a background of NaN, one attention call, the oracle's result."""
    g = torch.Generator().manual_seed(seed + sum(lens) + H)
    kv = filled(ops, B, KVH, L, D, fmt)
    n = max(max(lens), 1)
    k, v = bf16_rows(g, B, n, KVH, D, spread=spread), bf16_rows(g, B, n, KVH, D, spread=spread)
    for b in range(B):
        if min(lens[b], L):
            m = min(lens[b], L)
            one = kv.streams(b, b + 1)
            put(ops, one, k[b:b + 1, :m], v[b:b + 1, :m], [0])
    ld = H * D + ld_extra
    q = bf16_rows(g, B, ld, spread=spread)
    out = torch.full((B + 1, ld), 7.0, dtype=torch.bfloat16, device=dev())
    ws = torch.empty(max(1, ops.attn_decode_workspace(B, H, D, nsplit)), dtype=torch.float32, device=dev())
    kv_len = torch.tensor(lens, dtype=torch.int32, device=dev())
    args = (q.to(dev()), ld, kv, kv_len, out, ld, ws, B, H, nsplit, D ** -0.5)
    return args, k, v, q


def check_attention(fmt, args, k, v, q, streams=None):
    _, ld, kv, _, out, _, _, B, H, _, scale = args
    D, L = kv.D, kv.max_len
    lens = args[3].tolist()
    got = out.float().cpu().numpy()
    assert (got[B] == 7).all() and (got[:, H * D:] == 7).all(), "wrote beside the rows"
    worst = 0.0
    for b in (range(B) if streams is None else streams):
        m = max(0, min(lens[b], L))
        kk, vv = ((lambda x: K.values(K.pack(K.quantise(x, fmt)[0], fmt), K.quantise(x, fmt)[1], fmt))(
            t[b, :m].permute(1, 0, 2).double().numpy()) for t in (k, v))
        ref, bound = K.attend(q[b, :H * D].view(H, D).double().numpy(), kk, vv, scale)
        err = np.abs(got[b, :H * D].reshape(H, D) - ref)
        worst = max(worst, float((err / np.maximum(bound, 1e-30)).max()) if m else float(err.max()))
        assert (err <= bound).all(), (b, m, worst)
    return worst


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("B,H,KVH,D,L,lens,nsplit", [
    (1, 1, 1, 128, 1, [1], 1), (4, 2, 2, 64, 70, [0, 1, 16, 70], 1), (4, 2, 2, 128, 300, [15, 17, 255, 257], 1),
    (3, 2, 2, 128, 129, [63, 64, 65], 2), (3, 4, 2, 64, 1030, [1, 513, 1025], 3), (2, 6, 2, 128, 515, [515, 31], 2),
    (2, 8, 2, 64, 200, [129, 200], 1), (1, 8, 1, 128, 4100, [4097], 64), (2, 10, 2, 128, 90, [90, 33], 2),
    (3, 24, 24, 64, 777, [777, 3, 400], 4), (2, 3, 1, 64, 40, [40, 0], 7), (2, 2, 2, 128, 50, [-3, 60], 1),
    (2, 2, 2, 64, 50, [0, 60], 5), (1, 5, 1, 64, 33, [33], 64)])
def test_attention(ops, fmt, B, H, KVH, D, L, lens, nsplit):
    args, k, v, q = attention_case(ops, fmt, B, H, KVH, D, L, lens, nsplit)
    ops.attn_decode_mx(*args)
    check_attention(fmt, args, k, v, q)
    first = args[4].clone()
    ops.attn_decode_mx(*args)
    assert torch.equal(first, args[4]), "the same call gives other bits"


@pytest.mark.parametrize("fmt", FMT)
def test_attention_strided_rows_and_growing_maxima(ops, fmt):
    """Row strides beyond H * D; scores that grow along the keys, so that the running maximum moves many times."""
    args, k, v, q = attention_case(ops, fmt, 3, 4, 2, 128, 900, [900, 700, 512], 2, ld_extra=72)
    ops.attn_decode_mx(*args)
    check_attention(fmt, args, k, v, q)
    args, k, v, q = attention_case(ops, fmt, 1, 2, 2, 64, 1500, [1500], 1, spread=0)
    ramp = torch.linspace(0, 8, 1500).view(1, 1500, 1, 1)
    k = (q[0, :128].view(1, 1, 2, 64).float().sign() * ramp + 0.1 * k.float()).bfloat16()
    put(ops, args[2], k, v, [0])
    ops.attn_decode_mx(*args)
    check_attention(fmt, args, k, v, q)


@pytest.mark.parametrize("fmt", FMT)
def test_a_block_with_a_nan_shows(ops, fmt):
    """A key written with an infinity or a NaN makes the rows that attend it NaN (as in a bf16 cache), and no others."""
    args, k, v, q = attention_case(ops, fmt, 2, 4, 2, 128, 100, [100, 60], 1)
    k[0, 7, 1, 3] = float("inf")
    v[1, 50, 0, 99] = float("nan")
    v[1, 60:, 1] = float("nan")            # behind the second stream's last key
    put(ops, args[2], k, v, [0, 0])
    ops.attn_decode_mx(*args)
    o = args[4][:2].view(2, 4, 128)
    assert bool(torch.isnan(o[0, 2:]).all()) and not bool(torch.isnan(o[0, :2]).any())
    assert bool(torch.isnan(o[1, :2, 96:]).all()) and not bool(torch.isnan(o[1, :2, :96]).any())
    assert not bool(torch.isnan(o[1, 2:]).any())


def step_inputs(ops, fmt, B, H, KVH, D, L, lens, norm, seed=0):
    g = torch.Generator().manual_seed(seed + sum(lens) + D)
    caches = [filled(ops, B, KVH, L, D, fmt) for _ in range(2)]
    old = [bf16_rows(g, B, L, KVH, D, spread=2) for _ in range(2)]
    for kv in caches:
        for b in range(B):
            if lens[b] > 1:
                put(ops, kv.streams(b, b + 1), old[0][b:b + 1, :lens[b] - 1], old[1][b:b + 1, :lens[b] - 1], [0])
    qkv = bf16_rows(g, B, (H + 2 * KVH) * D + 16, spread=2).to(dev())
    gains = [1 + 0.3 * torch.randn(D, generator=g).to(dev()) for _ in range(2)] if norm else [None, None]
    inv = 1.0 / 10000 ** (torch.arange(0, D, 2).float() / D)
    cs = ops.rope_table(inv.to(dev()), L + 3)
    pos = torch.tensor([n - 1 for n in lens], dtype=torch.int32, device=dev())
    return caches, qkv, gains, cs, pos


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("il", [False, True])
@pytest.mark.parametrize("B,H,KVH,D,lens,nsplit,norm", [(1, 1, 1, 128, [1], 1, True), (4, 4, 4, 64, [1, 16, 17, 300], 1, False),
                                                        (3, 8, 2, 128, [513, 2, 256], 3, True),
                                                        (2, 6, 2, 64, [90, 700], 2, True), (2, 16, 2, 128, [33, 5], 2, False)])
def test_decode_step_equals_its_launches(ops, fmt, il, B, H, KVH, D, lens, nsplit, norm):
    """attn_decode_prep_mx against decode_qkv_prep (bf16 rows) -> kv_append_mx -> attn_decode_mx: outputs and caches."""
    L, ld = max(lens) + 2, (H + 2 * KVH) * D + 16
    (kv0, kv1), qkv, (wq, wk), cs, pos = step_inputs(ops, fmt, B, H, KVH, D, L, lens, norm)
    kv_len = pos + 1
    ws = torch.empty(max(1, ops.attn_decode_workspace(B, H, D, nsplit)), dtype=torch.float32, device=dev())
    o0 = torch.empty(B, H * D, dtype=torch.bfloat16, device=dev())
    o1 = torch.empty_like(o0)
    q = torch.empty_like(o0)
    kc = torch.empty(B, KVH, L, D, dtype=torch.bfloat16, device=dev())
    vc = torch.empty_like(kc)
    ops.decode_qkv_prep(qkv, ld, q.data_ptr(), H * D, kc, vc, wq, wk, cs, pos, B, H, KVH, D, L, 1e-6, il)
    at = torch.arange(B, device=dev())
    kn, vn = (t[at, :, pos.long()].reshape(B, KVH * D).contiguous() for t in (kc, vc))
    ops.kv_append_mx(kn, vn, KVH * D, KVH * D, kv0, pos, B, 1)
    ops.attn_decode_mx(q, H * D, kv0, kv_len, o0, H * D, ws, B, H, nsplit, D ** -0.5)
    ops.attn_decode_prep_mx(qkv, ld, wq, wk, cs, pos, 1e-6, il, kv1, kv_len, o1, H * D, ws, B, H, nsplit, D ** -0.5)
    for name in ("k", "k_scale", "v", "v_scale"):
        assert torch.equal(getattr(kv0, name), getattr(kv1, name)), name
    assert torch.equal(o0, o1)
    assert not bool(torch.isnan(o1).any())


@pytest.mark.parametrize("fmt", FMT)
def test_decode_step_skips_streams_that_do_not_fit(ops, fmt):
    """pos outside the cache or the rotary table, kv_len other than pos + 1: zeros, and nothing of the cache written."""
    B, H, KVH, D, L = 6, 4, 2, 64, 20
    (kv, before), qkv, (wq, wk), cs, pos = step_inputs(ops, fmt, B, H, KVH, D, L, [5] * B, True)
    pos = torch.tensor([4, -1, L, 4, 4, 18], dtype=torch.int32, device=dev())
    kv_len = torch.tensor([5, 0, L + 1, 4, 6, 19], dtype=torch.int32, device=dev())
    out = torch.full((B, H * D), 7.0, dtype=torch.bfloat16, device=dev())
    ld = (H + 2 * KVH) * D + 16
    for nsplit in (1, 3):
        ws = torch.empty(ops.attn_decode_workspace(B, H, D, 3), dtype=torch.float32, device=dev())
        ops.attn_decode_prep_mx(qkv, ld, wq, wk, cs[:18], pos, 1e-6, False, kv, kv_len, out, H * D, ws, B, H, nsplit, 0.125)
        assert bool((out[1:] == 0).all()) and not bool((out[0] == 0).all())
        for name in ("k", "k_scale", "v", "v_scale"):
            a, b = getattr(kv, name).clone(), getattr(before, name)
            a[0, :, 4] = b[0, :, 4]
            assert torch.equal(a, b), name


@pytest.mark.parametrize("fmt", FMT)
def test_slots_behind_four_gigabytes(ops, fmt):
    """The last streams of a cache whose codes are larger than 4 GiB: written, read back and attended."""
    KVH, D, L = 8, 128, 1 << 17
    B = 40 if fmt == "mxfp8" else 72
    kv = ops.MXKV.empty(B, KVH, L, D, fmt, dev())
    assert kv.k.numel() > 1 << 32
    one = kv.streams(B - 1, B)
    for t in (one.k, one.k_scale, one.v, one.v_scale):
        t.zero_()
    g = torch.Generator().manual_seed(5)
    n = 100
    k, v = bf16_rows(g, 1, n, KVH, D), bf16_rows(g, 1, n, KVH, D)
    w = KVH * D
    rows = [torch.zeros(B * n, w, dtype=torch.bfloat16, device=dev()) for _ in range(2)]
    rows[0][-n:], rows[1][-n:] = k.view(n, w).to(dev()), v.view(n, w).to(dev())
    pos = torch.full((B,), L - n, dtype=torch.int32, device=dev())
    ops.kv_append_mx(rows[0], rows[1], w, w, kv, pos, B, n)
    back = [torch.empty_like(rows[0]) for _ in range(2)]
    ops.kv_read_mx(kv, pos, back[0], back[1], w, w, B, n)
    q = bf16_rows(g, B, w).to(dev())
    out = torch.empty(B, w, dtype=torch.bfloat16, device=dev())
    kv_len = torch.zeros(B, dtype=torch.int32, device=dev())
    kv_len[-1] = L
    ws = torch.empty(ops.attn_decode_workspace(B, KVH, D, 64), dtype=torch.float32, device=dev())
    ops.attn_decode_mx(q, w, kv, kv_len, out, w, ws, B, KVH, 64, D ** -0.5)
    full = []
    for x, r in ((k, back[0]), (v, back[1])):
        c, e = K.quantise(x[0].permute(1, 0, 2).double().numpy(), fmt)
        val = K.values(K.pack(c, fmt), e, fmt)
        assert np.array_equal(r[-n:].view(n, KVH, D).permute(1, 0, 2).double().cpu().numpy(), val)
        full.append(np.concatenate([np.zeros((KVH, L - n, D)), val], 1))
    ref, bound = K.attend(q[-1].view(KVH, D).double().cpu().numpy(), full[0], full[1], D ** -0.5)
    assert (np.abs(out[-1].view(KVH, D).double().cpu().numpy() - ref) <= bound).all()
    assert bool((out[:-1] == 0).all())


def test_another_stream_and_a_replayed_graph(ops):
    """On a side stream, and captured: every replay follows the inputs of its time (two graphs share one workspace)."""
    fmt, B, H, KVH, D, L = "mxfp8", 3, 4, 2, 128, 600
    lens = [600, 333, 64]
    caches, qkv, (wq, wk), cs, pos = step_inputs(ops, fmt, B, H, KVH, D, L, lens, True)
    ld, nsplit = (H + 2 * KVH) * D + 16, 4
    ws = torch.empty(ops.attn_decode_workspace(B, H, D, nsplit), dtype=torch.float32, device=dev())
    out = [torch.empty(B, H * D, dtype=torch.bfloat16, device=dev()) for _ in range(2)]
    kv_len = pos + 1

    def step(i):
        ops.attn_decode_prep_mx(qkv, ld, wq, wk, cs, pos, 1e-6, False, caches[i], kv_len, out[i], H * D, ws, B, H, nsplit,
                                D ** -0.5)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(0)
    torch.cuda.current_stream().wait_stream(side)
    eager = out[0].clone()
    graphs = []
    for i in range(2):
        step(i)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            step(i)
        graphs.append(gr)
    for r in range(4):
        for i in (0, 1):
            graphs[i].replay()
            assert torch.equal(out[i], eager), (r, i)
        qkv.add_(0.25)
        step(0)
        fresh = out[0].clone()
        assert not torch.equal(fresh, eager)
        eager = fresh


def test_wrapper_refuses(ops):
    kv = ops.MXKV.empty(2, 2, 8, 64, "mxfp8", dev())
    rows = torch.zeros(2, 128, dtype=torch.bfloat16, device=dev())
    pos = torch.zeros(2, dtype=torch.int32, device=dev())
    ws = torch.empty(4, dtype=torch.float32, device=dev())
    att = lambda **kw: ops.attn_decode_mx(*[kw.get(k, d) for k, d in (  # noqa: E731
        ("q", rows), ("ld_q", 128), ("kv", kv), ("kv_len", pos), ("out", rows.clone()), ("ld_o", 128), ("ws", ws), ("B", 2),
        ("H", 2), ("nsplit", 1), ("scale", 0.1))])
    att()
    for bad in (dict(B=3), dict(B=0), dict(kv_len=pos.long()), dict(kv_len=pos[:1]), dict(kv_len=pos.cpu()),
                dict(q=rows.float()), dict(q=rows[:1]), dict(q=rows.cpu()), dict(ld_q=64), dict(out=rows[:, 1:]), dict(ld_o=64),
                dict(nsplit=2), dict(nsplit=2, ws=None), dict(nsplit=2, ws=torch.empty(264).double().to(dev())),
                dict(H=4)):
        with pytest.raises(ValueError):
            att(**bad)
    with pytest.raises(ValueError):
        ops.kv_append_mx(rows, rows, 128, 128, kv, pos, 2, 2)          # two tokens a stream need four rows
    with pytest.raises(ValueError):
        ops.kv_read_mx(kv, pos.float(), rows, rows, 128, 128, 2, 1)
    qkv = torch.zeros(2, 6 * 64, dtype=torch.bfloat16, device=dev())
    cs = ops.rope_table(torch.ones(32, device=dev()), 8)
    step = lambda **kw: ops.attn_decode_prep_mx(*[kw.get(k, d) for k, d in (  # noqa: E731
        ("qkv", qkv), ("ld", 384), ("wq", None), ("wk", None), ("cs", cs), ("pos", pos), ("eps", 1e-6), ("il", False),
        ("kv", kv), ("kv_len", pos + 1), ("out", rows.clone()), ("ld_o", 128), ("ws", ws), ("B", 2), ("H", 2), ("nsplit", 1),
        ("scale", 0.1))])
    step()
    for bad in (dict(pos=pos.long()), dict(cs=cs.double()), dict(ld=256), dict(wq=torch.ones(64).to(dev()).bfloat16()),
                dict(wk=torch.ones(32, device=dev()))):
        with pytest.raises(ValueError):
            step(**bad)
    from mgen._lib import MgenError
    with pytest.raises(MgenError):
        step(wq=torch.ones(64, device=dev()))


def test_more_rows_than_one_round_of_workgroups(ops):
    """A call with more rows than 2^20 workgroups hold at once: its last rows."""
    KVH, D, fmt = 8, 64, "mxfp4"
    n = (1 << 22) + 3
    w = KVH * D
    g = torch.Generator().manual_seed(11)
    tail = bf16_rows(g, 40, w)
    rows = torch.zeros(n, w, dtype=torch.bfloat16, device=dev())
    rows[-40:] = tail.to(dev())
    kv = ops.MXKV.empty(1, KVH, n, D, fmt, dev())
    for t in (kv.k, kv.k_scale, kv.v, kv.v_scale):
        t.fill_(0xFF)
    pos = torch.zeros(1, dtype=torch.int32, device=dev())
    ops.kv_append_mx(rows, rows, w, w, kv, pos, 1, n)
    code, e = K.quantise(tail.view(40, KVH, D).permute(1, 0, 2).double().numpy(), fmt)
    for c, s in ((kv.k, kv.k_scale), (kv.v, kv.v_scale)):
        assert np.array_equal(c[0, :, -40:].cpu().numpy(), K.pack(code, fmt))
        assert np.array_equal(s[0, :, -40:].cpu().numpy(), e)
        assert bool((s[0, :, :-40] == 1).all()) and bool((c[0, :, :-40] == 0).all())
    back = torch.full((n, w), 7.0, dtype=torch.bfloat16, device=dev())
    ops.kv_read_mx(kv, pos, back, rows, w, w, 1, n)
    want = torch.from_numpy(K.values(K.pack(code, fmt), e, fmt)).bfloat16().permute(1, 0, 2).reshape(40, w)
    assert torch.equal(back[-40:].cpu(), want) and torch.equal(rows[-40:], back[-40:])
    assert bool((back[:-40] == 0).all())


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("B,H,KVH,D,lens,nsplit", [
    (2, 12, 1, 128, [70, 33], 1), (1, 18, 2, 64, [700], 3),              # more query heads than one workgroup takes
    (48, 24, 8, 128, [1, 31, 32, 33, 0, 129, 200, 64], 1),               # several heads, more workgroups than CUs
    (40, 16, 4, 64, [300, 600, 31], 2), (70, 16, 16, 64, [5, 257, 520, 96], 2)])
def test_attention_of_many_workgroups(ops, fmt, B, H, KVH, D, lens, nsplit):
    lens = [lens[b % len(lens)] for b in range(B)]
    args, k, v, q = attention_case(ops, fmt, B, H, KVH, D, max(lens), lens, nsplit)
    ops.attn_decode_mx(*args)
    check_attention(fmt, args, k, v, q, streams=sorted({0, 1, 2, 3, B - 2, B - 1} & set(range(B))))
    first = args[4].clone()
    few, out = args[2].streams(0, 1), torch.empty(1, H * D, dtype=torch.bfloat16, device=dev())
    ops.attn_decode_mx(args[0], H * D, few, args[3], out, H * D, args[6], 1, H, nsplit, D ** -0.5)
    # alone, a stream may take the kernel of 8 waves: the same sums in another order, each within the bound
    check_attention(fmt, (args[0], H * D, few, args[3], torch.cat((out, first[:1] * 0 + 7)), H * D, None, 1, H, nsplit,
                          D ** -0.5), k, v, q, streams=[0])


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("il", [False, True])
@pytest.mark.parametrize("B,H,KVH,D,lens,nsplit", [(2, 18, 2, 128, [40, 700], 3), (1, 11, 1, 64, [33], 1),
                                                   (72, 8, 4, 128, [1, 17, 32, 130], 1), (36, 16, 8, 64, [64, 300, 2], 2)])
def test_decode_step_of_many_workgroups(ops, fmt, il, B, H, KVH, D, lens, nsplit):
    test_decode_step_equals_its_launches(ops, fmt, il, B, H, KVH, D, [lens[b % len(lens)] for b in range(B)], nsplit, True)


def test_workspace_on_the_cache_device(ops):
    kv = ops.MXKV.empty(1, 2, 600, 64, "mxfp8", dev())
    rows = torch.zeros(1, 128, dtype=torch.bfloat16, device=dev())
    n = torch.ones(1, dtype=torch.int32, device=dev())
    with pytest.raises(ValueError, match="workspace"):
        ops.attn_decode_mx(rows, 128, kv, n, rows.clone(), 128, torch.empty(4096), 1, 2, 2, 0.1)


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("B,H,KVH,nsplit,step", [(140, 8, 8, 1, 70), (150, 16, 8, 1, 75), (530, 8, 8, 1, 106), (645, 8, 8, 1, 100),
                                                 (90, 8, 8, 2, 40), (1100, 2, 1, 1, 550)])
def test_order_of_the_streams_does_not_show(ops, fmt, B, H, KVH, nsplit, step):
    """Streams of different lengths in a call with more workgroups than the chip holds, which takes long ones first: the bits
    of calls that take them as they are numbered; every row is written."""
    D, L = 64, 1030
    g = torch.Generator().manual_seed(B)
    kv = ops.MXKV.empty(B, KVH, L, D, fmt, dev())
    rows = bf16_rows(g, L, KVH * D, spread=1).to(dev())
    ops.kv_append_mx(rows.repeat(8, 1), rows.flip(0).repeat(8, 1), KVH * D, KVH * D, kv, torch.zeros(8, dtype=torch.int32,
                     device=dev()), 8, L)
    for t in (kv.k, kv.k_scale, kv.v, kv.v_scale):
        t[8:] = t[:1]
    lens = torch.randint(0, L + 1, (B,), generator=g, dtype=torch.int32)
    lens[::5] = 700                                      # equal ones
    lens[3::7] = torch.tensor([0, 1, L, L + 9, -2], dtype=torch.int32).repeat(B)[:lens[3::7].numel()]
    lens = lens.to(dev())
    q = bf16_rows(g, B, H * D, spread=1).to(dev())
    ws = torch.empty(ops.attn_decode_workspace(B, H, D, nsplit), dtype=torch.float32, device=dev())
    whole, parts = (torch.full((B, H * D), 7.0, dtype=torch.bfloat16, device=dev()) for _ in range(2))
    ops.attn_decode_mx(q, H * D, kv, lens, whole, H * D, ws, B, H, nsplit, D ** -0.5)
    for b in range(0, B, step):
        e = min(b + step, B)
        ops.attn_decode_mx(q[b:e], H * D, kv.streams(b, e), lens[b:e], parts[b:e], H * D, ws, e - b, H, nsplit, D ** -0.5)
    assert torch.equal(whole, parts)
    assert not bool((whole == 7.0).all(-1).any())
    assert bool((whole[lens <= 0] == 0).all())
