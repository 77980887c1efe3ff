"""Generation with a KV cache in 4 or 8 bits: the logits of a bf16 cache that holds the quantised values (another set of
kernels over the same numbers), the one-call layer against its launches, batches in two parts, padded prompts, a captured
step, reserved caches, and the models with a decode step of their own."""
import pytest
import torch

pytestmark = pytest.mark.gpu
FMT = ["mxfp4", "mxfp8"]


def small(**kw):
    from mgen import MidiLM, LMConfig
    cfg = dict(vocab_size=2048, hidden_size=512, intermediate_size=2048, num_hidden_layers=2, num_attention_heads=4,
               num_key_value_heads=2, head_dim=128)
    cfg.update(kw)
    return MidiLM(LMConfig(**cfg), device="cuda:0", seed=3)


@pytest.fixture(scope="module")
def model():
    return small()


def through_bf16(monkeypatch, fmt):
    """KVCache whose rows pass through a quantised cache on their way in: the bf16 kernels over the quantised values."""
    from mgen import generation as G, ops

    class RoundTrip(G.KVCache):
        def __init__(self, cfg, batch, max_len, device):
            super().__init__(cfg, batch, max_len, device)
            self.mx = G.MXKVCache(cfg, batch, max_len, device, fmt)
            self.heads = cfg.num_attention_heads
            self.tmp = torch.empty(batch, cfg.num_key_value_heads, max_len, cfg.head_dim, dtype=torch.bfloat16,
                                   device=device)

        def part(self, b0, b1):
            assert (b0, b1) == (0, self.batch)
            return self

        def append(self, l, k_src, v_src, ld_k, ld_v, pos0, B, n):
            self.mx.append(l, k_src, v_src, ld_k, ld_v, pos0, B, n)
            k, v = self.mx.read(l, pos0, n)
            w = k.shape[2] * k.shape[3]
            super().append(l, k.data_ptr(), v.data_ptr(), w, w, pos0, B, n)

        def attend_prep(self, l, qkv, ld_in, wq, wk, cs, pos, eps, il, kv_len, out, ld_o, ws, B, H, nsplit, scale):
            _, KVH, _, D = self.k[l].shape
            q = torch.empty(B, H * D, dtype=torch.bfloat16, device=self.device)
            tmp_v = torch.empty_like(self.tmp)
            ops.decode_qkv_prep(qkv, ld_in, q.data_ptr(), H * D, self.tmp, tmp_v, wq, wk, cs, pos, B, H, KVH, D,
                                self.max_len, eps, il)
            at = torch.arange(B, device=self.device)
            k, v = (t[at, :, pos[:B].long()].contiguous() for t in (self.tmp, tmp_v))
            self.append(l, k.data_ptr(), v.data_ptr(), KVH * D, KVH * D, pos, B, 1)
            self.attend(l, q.data_ptr(), H * D, kv_len, out, ld_o, ws, B, H, nsplit, scale)

    monkeypatch.setattr(G, "KVCache", RoundTrip)
    monkeypatch.setattr(G, "_LAYER_IN_ONE_CALL", False)
    monkeypatch.setenv("MGEN_DECODE_PARTS", "1")


def agree(a, b, P, tol=2e-2):
    """Step logits of two runs, compared for as long as both chose the same tokens (at least two steps)."""
    (ta, la), (tb, lb) = a, b
    steps = 0
    for i in range(la.shape[0]):
        err = float((la[i] - lb[i]).abs().max() / lb[i].abs().max())
        assert err < tol, (i, err)
        steps += 1
        if not torch.equal(ta[:, P + i], tb[:, P + i]):
            break
    assert steps >= 2


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("kw", [{}, dict(num_attention_heads=8, num_key_value_heads=8, head_dim=64, qk_norm=False,
                                         rope_interleaved=True, norm_kind="layer")], ids=["gqa128", "layernorm64"])
def test_logits_are_those_of_a_bf16_cache_with_the_quantised_values(fmt, kw, monkeypatch):
    m = small(**kw)
    ids = torch.randint(3, 2048, (3, 70), generator=torch.Generator().manual_seed(5)).cuda()
    got = m.generate(ids, max_new_tokens=12, return_step_logits=True, kv_cache=fmt)
    plain = m.generate(ids, max_new_tokens=12, return_step_logits=True)
    through_bf16(monkeypatch, fmt)
    want = m.generate(ids, max_new_tokens=12, return_step_logits=True)
    agree(got, want, 70)
    assert torch.equal(got[1][0], plain[1][0]), "the prompt's own attention is not quantised"
    assert not torch.equal(got[1][1], plain[1][1]), "the cache was not quantised"


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("B", [3, 64, 130])
def test_one_call_equals_launch_by_launch_and_parts_equal_the_whole(model, B, fmt, monkeypatch):
    from mgen import generation as G
    prompt = torch.randint(3, 2048, (B, 5), generator=torch.Generator().manual_seed(B)).cuda()
    run = lambda: model.generate(prompt, max_new_tokens=20, return_step_logits=True, kv_cache=fmt)  # noqa: E731
    a = run()
    monkeypatch.setattr(G, "_LAYER_IN_ONE_CALL", False)
    b = run()
    monkeypatch.setenv("MGEN_DECODE_PARTS", "1")
    c = run()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])


@pytest.mark.parametrize("fmt", FMT)
def test_left_padded_prompts(model, fmt):
    g = torch.Generator().manual_seed(9)
    lens, P = [3, 17, 11], 17
    ids = torch.randint(3, 2048, (3, P), generator=g).cuda()
    mask = torch.stack([torch.cat([torch.zeros(P - n), torch.ones(n)]) for n in lens]).long().cuda()
    both = model.generate(ids, max_new_tokens=10, attention_mask=mask, kv_cache=fmt)
    for i, n in enumerate(lens):
        alone = model.generate(ids[i:i + 1, P - n:], max_new_tokens=10, kv_cache=fmt)
        assert torch.equal(both[i, P:], alone[0, n:]), i


def test_captured_steps(model, monkeypatch):
    from mgen import generation as G
    prompt = torch.randint(3, 2048, (64, 250), generator=torch.Generator().manual_seed(1)).cuda()
    run = lambda: model.generate(prompt, max_new_tokens=30, do_sample=True, seed=4, kv_cache="mxfp8")  # noqa: E731
    eager = run()
    monkeypatch.setattr(G, "_DECODE_GRAPH", True)
    assert torch.equal(run(), eager)


def test_reserved_caches(model):
    prompt = torch.randint(3, 2048, (4, 9), generator=torch.Generator().manual_seed(2)).cuda()
    want = {f: model.generate(prompt, max_new_tokens=8, kv_cache=f) for f in ("bf16", *FMT)}
    sizes = {}
    for held in ("bf16", *FMT):
        model.reserve_kv_cache(6, 40, kv_cache=held)
        try:
            sizes[held] = model._kv_reserved.bytes_per_token()
            for f in want:            # a reserved cache of another type is not taken
                assert torch.equal(model.generate(prompt, max_new_tokens=8, kv_cache=f), want[f]), (held, f)
        finally:
            model.release_kv_cache()
    assert sizes["mxfp8"] * 64 == sizes["bf16"] * 33 and sizes["mxfp4"] * 64 == sizes["bf16"] * 17


def test_cache_reads_back_what_the_prompt_wrote(model):
    model.reserve_kv_cache(2, 30, kv_cache="mxfp8")
    try:
        ids = torch.randint(3, 2048, (2, 20), generator=torch.Generator().manual_seed(6)).cuda()
        model.generate(ids, max_new_tokens=5, kv_cache="mxfp8")
        k, v = model._kv_reserved.read(1, torch.full((2,), 10, dtype=torch.int32, device="cuda"), 25)
        assert k.shape == v.shape == (2, 25, 2, 128)
        assert bool((k[:, :14] != 0).any(-1).all()) and bool((k[:, 14:] == 0).all()) and not bool(torch.isnan(k).any())
    finally:
        model.release_kv_cache()


@pytest.mark.parametrize("fmt", FMT)
def test_gpt2(fmt, monkeypatch):
    from mgen import MidiGPT2LM, LMConfig
    cfg = LMConfig(arch="gpt2", vocab_size=1024, hidden_size=256, intermediate_size=1024, num_hidden_layers=2,
                   num_attention_heads=4, num_key_value_heads=4, head_dim=64, max_position_embeddings=256,
                   tie_word_embeddings=True, qk_norm=False)
    m = MidiGPT2LM(cfg, device="cuda:0", seed=1).eval()
    ids = torch.randint(3, 1024, (3, 33), generator=torch.Generator().manual_seed(5)).cuda()
    got = m.generate(ids, max_new_tokens=10, return_step_logits=True, kv_cache=fmt)
    through_bf16(monkeypatch, fmt)
    agree(got, m.generate(ids, max_new_tokens=10, return_step_logits=True), 33)


@pytest.mark.parametrize("fmt", FMT)
def test_generate_music(fmt, monkeypatch):
    m = small(vocab_size=1, tie_word_embeddings=False, pos4d=True, num_key_value_heads=4)
    start = torch.rand(2, 3, 4, generator=torch.Generator().manual_seed(5)).cuda() * 20
    got, p0 = m.generate_music(start, 4, return_preds=True, kv_cache=fmt)
    through_bf16(monkeypatch, fmt)
    want, p1 = m.generate_music(start, 4, return_preds=True)
    assert torch.equal(p0[:, 0], p1[:, 0])
    assert float((p0[:, 1] - p1[:, 1]).abs().max()) < 2e-2       # (unit pairs; the notes are decoded from them)


def test_refusals(model):
    from mgen import MidiLM, LMConfig
    ids = torch.full((1, 4), 5).cuda()
    with pytest.raises(ValueError, match="mxfp6"):
        model.generate(ids, max_new_tokens=2, kv_cache="mxfp6")
    with pytest.raises(ValueError, match="mxfp6"):
        model.reserve_kv_cache(1, 8, kv_cache="mxfp6")
    with pytest.raises(ValueError, match="use_cache"):
        model.generate(ids, max_new_tokens=2, kv_cache="mxfp8", use_cache=False)
    full = MidiLM(LMConfig(vocab_size=64, hidden_size=128, intermediate_size=256, num_hidden_layers=1, num_attention_heads=1,
                           num_key_value_heads=1, head_dim=128), device="cuda:0", seed=0, compute_dtype=torch.float32)
    with pytest.raises(ValueError, match="fp32"):
        full.generate(ids, max_new_tokens=2, kv_cache="mxfp8")
