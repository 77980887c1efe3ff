"""Refusals of the quantised cache's entry points, without a GPU: every bad size, type, alignment or missing pointer is an
error before anything is launched."""
import pytest
import torch


def _append(**kw):
    a = dict(k=4096, v=4096, ldk=1024, ldv=1024, kc=4096, ks=4096, vc=4096, vs=4096, pos=4096, B=2, n=3, KVH=8, D=128, L=16,
             bits=8)
    a.update(kw)
    return [a[x] for x in ("k", "v", "ldk", "ldv", "kc", "ks", "vc", "vs", "pos", "B", "n", "KVH", "D", "L", "bits")] + [None]


def _read(**kw):
    a = _append(**kw)
    return a[4:9] + a[0:4] + a[9:]


def _attend(**kw):
    a = dict(q=4096, ldq=1024, kc=4096, ks=4096, vc=4096, vs=4096, n=4096, out=4096, ldo=1024, ws=4096, B=2, H=8, KVH=8,
             D=128, L=16, bits=8, split=1)
    a.update(kw)
    return [a[x] for x in ("q", "ldq", "kc", "ks", "vc", "vs", "n", "out", "ldo", "ws", "B", "H", "KVH", "D", "L", "bits",
                           "split")] + [1.0, None]


def _prep(**kw):
    a = dict(qkv=4096, ld=3 * 1024, wq=None, wk=None, cs=4096, npos=16, pos=4096, kc=4096, ks=4096, vc=4096, vs=4096, n=4096,
             out=4096, ldo=1024, ws=4096, B=2, H=8, KVH=8, D=128, L=16, bits=8, split=1)
    a.update(kw)
    return ([a[x] for x in ("qkv", "ld", "wq", "wk", "cs", "npos", "pos")] + [1e-6, 0] +
            [a[x] for x in ("kc", "ks", "vc", "vs", "n", "out", "ldo", "ws", "B", "H", "KVH", "D", "L", "bits", "split")] +
            [1.0, None])


ROWS = [dict(k=None), dict(v=None), dict(kc=None), dict(ks=None), dict(vc=None), dict(vs=None), dict(pos=None), dict(B=0),
        dict(n=0), dict(n=-1), dict(KVH=0), dict(D=96), dict(D=32), dict(L=0), dict(bits=6), dict(ldk=1020), dict(ldv=1023),
        dict(ldk=512), dict(k=4104), dict(v=4098), dict(kc=4100), dict(vc=4104), dict(B=70000, n=70000), dict(ks=4098), dict(vs=4097), dict(D=64, ks=4097)]
ATTN = [dict(kc=None), dict(ks=None), dict(vc=None), dict(vs=None), dict(n=None), dict(out=None), dict(B=0), dict(B=65536),
        dict(H=0), dict(KVH=0), dict(H=9, KVH=2, ldo=4096), dict(D=256), dict(L=0), dict(L=1 << 24), dict(bits=16),
        dict(split=0), dict(split=65), dict(split=2, ws=None), dict(ldo=1000), dict(kc=4104), dict(vc=4097), dict(ks=4098),
        dict(vs=4097), dict(D=64, vs=4097),
        dict(H=65536, KVH=65536, ldo=1 << 24)]


@pytest.mark.parametrize("fn,args", [("mgen_kv_append_mx", _append), ("mgen_kv_read_mx", _read)])
@pytest.mark.parametrize("bad", ROWS, ids=str)
def test_rows_refuse(fn, args, bad):
    from mgen._lib import MgenError, call
    with pytest.raises(MgenError, match=fn):
        call(fn, *args(**bad))


@pytest.mark.parametrize("bad", ATTN + [dict(q=None), dict(q=4104), dict(ldq=1028)], ids=str)
def test_attention_refuses(bad):
    from mgen._lib import MgenError, call
    with pytest.raises(MgenError, match="mgen_attn_decode_mx"):
        call("mgen_attn_decode_mx", *_attend(**bad))


@pytest.mark.parametrize("bad", [b for b in ATTN if "H" not in b] + [
    dict(qkv=None), dict(cs=None), dict(pos=None), dict(npos=0), dict(wq=4096), dict(wk=4096), dict(ld=3 * 1024 + 4),
    dict(ld=1024), dict(qkv=4100), dict(cs=4104)], ids=str)
def test_decode_step_refuses(bad):
    from mgen._lib import MgenError, call
    with pytest.raises(MgenError, match="mgen_attn_decode_prep_mx"):
        call("mgen_attn_decode_prep_mx", *_prep(**bad))


@pytest.mark.parametrize("B,H,KVH,D,longest", [(1, 8, 8, 128, 1), (1, 8, 8, 128, 4096), (256, 8, 8, 128, 4096),
                                               (1, 32, 1, 64, 1 << 20), (3, 24, 24, 64, 777), (65535, 1, 1, 64, 5)])
def test_suggested_splits_are_valid(B, H, KVH, D, longest):
    from mgen import ops
    n = ops.attn_decode_mx_splits(B, H, KVH, D, longest)
    assert 1 <= n <= 64 and (n == 1 or n <= longest)


def test_suggested_splits_of_nothing():
    from mgen import ops
    assert ops.attn_decode_mx_splits(0, 8, 8, 128, 100) == 1
    assert ops.attn_decode_mx_splits(1, 8, 8, 128, 0) == 1
    assert ops.attn_decode_mx_splits(1, 1, 8, 128, 5) == 1


def test_cache_object_refuses():
    from mgen import ops
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)  # noqa: E731
    good = lambda: [u8(2, 4, 10, 128), u8(2, 4, 10, 4), u8(2, 4, 10, 128), u8(2, 4, 10, 4)]  # noqa: E731
    with pytest.raises(RuntimeError, match="GPU"):
        ops.MXKV(*good())                              # shapes are fine: the device is not
    for i, bad in [(0, u8(2, 4, 10, 96)), (1, u8(2, 4, 10, 3)), (2, u8(2, 4, 10, 64)), (3, u8(2, 4, 9, 4)),
                   (0, torch.zeros(2, 4, 10, 128)), (0, u8(2, 4, 128)), (0, u8(2, 4, 128, 10).transpose(2, 3)),
                   (1, u8(3, 4, 10, 4))]:
        t = good()
        t[i] = bad
        with pytest.raises(ValueError):
            ops.MXKV(*t)
    for d, w in ((32, 32), (256, 256), (96, 48)):
        with pytest.raises(ValueError):
            ops.MXKV(u8(1, 1, 4, w), u8(1, 1, 4, d // 32), u8(1, 1, 4, w), u8(1, 1, 4, d // 32))
    with pytest.raises(ValueError, match="mxfp6"):
        ops.MXKV.empty(1, 1, 4, 64, "mxfp6", "cpu")


@pytest.mark.parametrize("B,H,KVH,D", [(1, 8, 8, 128), (3, 24, 24, 64), (16, 32, 8, 128), (24, 8, 8, 128), (28, 64, 8, 64),
                                       (31, 8, 8, 64), (32, 8, 8, 128), (200, 12, 1, 64), (255, 1, 1, 128), (300, 4, 4, 64)])
def test_suggested_splits_never_fall_with_the_length(B, H, KVH, D):
    """A workspace sized for the longest call of a run holds all of them."""
    from mgen import ops
    last = 0
    for longest in [*range(1, 3000, 37), *range(3000, 140000, 1021), 1 << 24, (1 << 31) - 1]:
        n = ops.attn_decode_mx_splits(B, H, KVH, D, longest)
        assert 1 <= n <= 64 and n >= last
        last = n


@pytest.mark.parametrize("fn,args", [("mgen_kv_append_mx", _append), ("mgen_kv_read_mx", _read)])
@pytest.mark.parametrize("big", [dict(B=1 << 30, n=1 << 30, KVH=1 << 8, ldk=1 << 15, ldv=1 << 15),
                                 dict(B=(1 << 31) - 1, n=(1 << 31) - 1, KVH=(1 << 31) - 1, ldk=1 << 40, ldv=1 << 40),
                                 dict(B=1 << 16, n=1 << 15)], ids=str)
def test_row_counts_do_not_wrap(fn, args, big):
    """2^64 rows are 0 in 64 bits: refused as too many, not launched as none."""
    from mgen._lib import MgenError, call
    with pytest.raises(MgenError, match="too many rows"):
        call(fn, *args(**big))
