"""Generation with a quantised cache at contexts of several units, waves and key splits: against the bf16 kernels over the
quantised values, the one-call layer against its launches, captured steps, parts against the whole, and the prompt's rows
read back against the oracle's quantisation of a bf16 cache's."""
import numpy as np
import pytest
import torch

from oracle import ref_kvmx as K
from test_gpu_kvmx_generate import FMT, agree, small, through_bf16

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    return small()


def prompt(B, P, seed=0):
    return torch.randint(3, 2048, (B, P), generator=torch.Generator().manual_seed(seed)).cuda()


def splits_of(model, B, lengths):
    return {model._decode_split(B, n, "mxfp8") for n in lengths}


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("kw", [{}, dict(num_attention_heads=4, num_key_value_heads=4, qk_norm=False, rope_interleaved=True)],
                         ids=["gqa", "mha"])
def test_key_splits_against_a_bf16_cache_with_the_quantised_values(fmt, kw, monkeypatch):
    """The split count changes on the way (none up to 896 keys, several beyond); the workspace is that of the longest step."""
    m = small(**kw)
    ids = prompt(2, 888)
    counts = splits_of(m, 2, range(889, 889 + 16))
    assert 1 in counts and max(counts) >= 4
    run = lambda: m.generate(ids, max_new_tokens=16, return_step_logits=True, kv_cache=fmt)  # noqa: E731
    got = run()
    from mgen import generation as G
    with monkeypatch.context() as mp:
        mp.setattr(G, "_LAYER_IN_ONE_CALL", False)
        apart = run()
    assert torch.equal(got[0], apart[0]) and torch.equal(got[1], apart[1])
    with monkeypatch.context() as mp:
        through_bf16(mp, fmt)
        want = m.generate(ids, max_new_tokens=16, return_step_logits=True)
    agree(got, want, 888)


@pytest.mark.parametrize("fmt", FMT)
def test_captured_steps_across_split_counts(model, fmt, monkeypatch):
    from mgen import generation as G
    ids = prompt(2, 890, seed=1)
    assert len(splits_of(model, 2, range(891, 891 + 24))) > 1
    run = lambda: model.generate(ids, max_new_tokens=24, do_sample=True, seed=4, kv_cache=fmt)  # noqa: E731
    eager = run()
    monkeypatch.setattr(G, "_DECODE_GRAPH", True)
    for _ in range(2):
        assert torch.equal(run(), eager)


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("B,heads", [(130, 2), (64, 4)], ids=["gqa", "mha"])
def test_parts_at_a_longer_context(B, heads, fmt, monkeypatch):
    """A batch in two parts against the whole: with several heads a kv head a part may run with other waves (other orders of
    the same sums), with one head it has the same bits."""
    m = small(num_key_value_heads=heads)
    ids = prompt(B, 300, seed=2)
    run = lambda: m.generate(ids, max_new_tokens=6, return_step_logits=True, kv_cache=fmt)  # noqa: E731
    monkeypatch.setenv("MGEN_DECODE_PARTS", "2")
    parts = run()
    monkeypatch.setenv("MGEN_DECODE_PARTS", "1")
    whole = run()
    agree(parts, whole, 300)
    if heads == 4:
        assert torch.equal(parts[0], whole[0]) and torch.equal(parts[1], whole[1])


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("kw", [{}, dict(num_attention_heads=8, num_key_value_heads=8, head_dim=64, norm_kind="layer")],
                         ids=["gqa128", "layernorm64"])
def test_prompt_rows_read_back(fmt, kw):
    """Every layer's keys and values of every prompt position: the bf16 cache's, quantised."""
    m = small(**kw)
    B, P = 3, 37
    ids = prompt(B, P, seed=3)
    m.reserve_kv_cache(B, 50)
    m.generate(ids, max_new_tokens=3)
    plain = m._kv_reserved
    m.reserve_kv_cache(B, 50, kv_cache=fmt)
    m.generate(ids, max_new_tokens=3, kv_cache=fmt)
    held = m._kv_reserved
    m.release_kv_cache()
    zero = torch.zeros(B, dtype=torch.int32, device="cuda")
    for l in range(2):
        for got, rows in zip(held.read(l, zero, P), (plain.k[l], plain.v[l])):
            x = rows[:, :, :P].double().cpu().numpy()                     # [B, KVH, P, D]
            code, e = K.quantise(x, fmt)
            want = K.values(K.pack(code, fmt), e, fmt).transpose(0, 2, 1, 3)
            assert np.array_equal(got.double().cpu().numpy(), want), l
