"""`generate` with its options on the GPU: 8-bit caches, sampled rows that share a clip's cross-attention keys, a drafting model - the cached
operators run together through SpeechMixEED.generate / decoding.CachedDecoder."""
import math

import pytest
import torch

from tests import decode_ref as R
from tests.test_gpu_e2e import _build

pytestmark = pytest.mark.gpu

ENC = dict(model_type="wav2vec2", hidden_size=128, num_hidden_layers=1, num_attention_heads=2, intermediate_size=256, conv_dim=[64] * 7,
           conv_kernel=[10, 3, 3, 3, 3, 2, 2], conv_stride=[5, 2, 2, 2, 2, 2, 2], num_conv_pos_embeddings=16, num_conv_pos_embedding_groups=4,
           feat_extract_norm="group", do_stable_layer_norm=False, conv_bias=False, layer_norm_eps=1e-5, hidden_act="gelu")
BART = dict(model_type="bart", vocab_size=203, d_model=128, encoder_layers=1, decoder_layers=2, encoder_attention_heads=2,
            decoder_attention_heads=2, encoder_ffn_dim=256, decoder_ffn_dim=256, max_position_embeddings=64, pad_token_id=1, bos_token_id=0,
            eos_token_id=2, decoder_start_token_id=2, activation_function="gelu", scale_embedding=False)
T5 = dict(model_type="t5", vocab_size=200, d_model=128, num_layers=1, num_decoder_layers=2, num_heads=2, d_kv=64, d_ff=256,
          relative_attention_num_buckets=32, relative_attention_max_distance=128, feed_forward_proj="relu", pad_token_id=0, eos_token_id=1,
          decoder_start_token_id=0, layer_norm_epsilon=1e-6, tie_word_embeddings=True)


def _model(lm, dtype="fp32", seed=0, spread=6.0):
    """A small model whose logits differ (random-init heads give nearly equal ones): the embedding - the tied head - scaled up."""
    from speechmix_amd.model import SpeechMixEED
    m = SpeechMixEED(ENC, lm, down_scale=2, compute_dtype=dtype, init_seed=seed).eval()
    with torch.no_grad():
        emb = m.decoder_model.shared.weight if lm["model_type"] == "t5" else m.decoder_model.model.shared.weight
        emb.mul_(spread)
    m.store.invalidate()
    return m


def _wave(B, seed=0):
    return torch.randn(B, 8000, generator=torch.Generator().manual_seed(seed)) * 0.1


@pytest.mark.parametrize("case", ["eed_w2v2_bart", "eed_hubert_mbart", "eed_w2v2_t5_trainable"])
def test_the_cached_decoder_gives_the_greedy_loops_logits(case):
    """fp32: a forced continuation fed one token at a time, three at a time, and with rows at different lengths - every logit within the fp32
    criterion (1e-3) of Engine.greedy_decode's; and `generate(kv_cache="fp32")` emits generate's tokens."""
    from speechmix_amd.decoding import CachedDecoder
    model, inp, gold, m = _build(case, "fp32")
    model.eval()
    lc, eng = model.decoder_model.config, model.engine
    steps = 8
    with torch.no_grad():
        enc, B, S = model._speech_encode(inp["input_values"])
        forced = torch.randint(4, lc.vocab_size, (B, steps), generator=torch.Generator().manual_seed(3)).to(model.device)
        kept = []
        eng.greedy_decode(enc, B, S, steps, lc.decoder_start_token_id, -1, lc.pad_token_id, forced=forced, keep_logits=kept)
        want = torch.stack(kept, 1)
        fed = torch.cat([torch.full((B, 1), lc.decoder_start_token_id, dtype=torch.int64, device=model.device), forced[:, :-1]], 1)
        for cuts in ((1,) * 8, (3, 1, 4), (8,)):
            dec = CachedDecoder(eng, enc, B, S, 1, steps + 1)
            t = 0
            for n in cuts:
                lg = dec.step(fed[:, t:t + n].contiguous())
                assert (lg - want[:, t:t + n]).abs().max().item() < 1e-3
                dec.lens += n
                t += n
        # two rows per clip, the second one two tokens behind
        dec = CachedDecoder(eng, enc, B, S, 2, steps + 1)
        rows = fed.repeat_interleave(2, 0)
        dec.step(rows[:, :4].contiguous())
        dec.lens += 4
        dec.lens[1::2] -= 2
        at = dec.lens.long()
        nxt = torch.gather(rows, 1, at[:, None] + torch.arange(3, device=model.device))
        lg = dec.step(nxt)
        ref = torch.stack([want.repeat_interleave(2, 0)[i, a:a + 3] for i, a in enumerate(at.tolist())])
        assert (lg - ref).abs().max().item() < 1e-3
    eos = lc.eos_token_id
    for e in (eos, -1):
        lc.eos_token_id = e
        assert model.generate(inp["input_values"], max_length=7, kv_cache="fp32") == model.generate(inp["input_values"], max_length=7)
    lc.eos_token_id = eos


class _Plain:
    """Plain 64-bit stand-ins for the cache and attention operators: the quantisation of decode_ref and a softmax on the CPU."""

    def __init__(self, fmt):
        self.fmt, self.vals = fmt, {}

    def kv_append(self, cache, k, v, start=0):
        K, V = self.vals.setdefault(id(cache), [torch.zeros(cache.B, cache.H, cache.cap, cache.D, dtype=torch.float64) for _ in range(2)])
        st = start.tolist() if isinstance(start, torch.Tensor) else [start] * cache.B
        for dst, x in ((K, k), (V, v)):
            x = x.float().cpu().transpose(1, 2)
            val = R.values(*R.quantise(x, self.fmt), self.fmt) if self.fmt in ("e4m3", "int8") else x.to(torch.bfloat16).double()
            for b, s in enumerate(st):
                dst[b, :, s:s + x.shape[2]] = val[b]

    def attention_cached(self, q, cache, klen=None, causal=True, scale=None, rel_bias=None, prefix=None, **kw):
        K, V = self.vals[id(cache)] if cache is not None else (None, None)
        PK, PV = self.vals[id(prefix)] if prefix is not None else (None, None)
        B = q.shape[0]
        o = R.attention(q, K, V, klen.tolist() if klen is not None else None, [prefix.cap] * prefix.B if prefix is not None else None, PK, PV,
                        B // prefix.B if prefix is not None else 1, causal, scale, rel_bias)[0]
        return o.to(q.dtype).to(q.device), None


@pytest.mark.parametrize("kv", ["fp8", "int8", "bf16"])
@pytest.mark.parametrize("lm", [BART, T5], ids=["bart", "t5"])
def test_a_quantised_decoder_against_plain_operators(lm, kv, monkeypatch):
    """The whole decoder over an 8-bit (or bf16) cache, fp32 queries, against itself with the cache and the attention computed plainly in 64
    bits: logits within the fp32 criterion."""
    from speechmix_amd import decoding
    model = _model(lm, spread=1.0)
    with torch.no_grad():
        enc, B, S = model._speech_encode(_wave(2))
        g = torch.Generator().manual_seed(5)
        fed = torch.randint(4, 200, (4, 9), generator=g).to(model.device)

        def run():
            dec = decoding.CachedDecoder(model.engine, enc, B, S, 2, 12, kv)
            out = [dec.step(fed[:, :4].contiguous())]
            dec.lens += torch.tensor([4, 3, 2, 4], dtype=torch.int32, device=model.device)
            out.append(dec.step(fed[:, 4:5].contiguous()))
            dec.lens += 1
            out.append(dec.step(fed[:, 5:9].contiguous()))
            return torch.cat(out, 1).cpu(), dec
        got, dec = run()
        assert dec.fmt == {"fp8": "e4m3"}.get(kv, kv)
        plain = _Plain(dec.fmt)
        monkeypatch.setattr(decoding.ops, "kv_append", plain.kv_append)
        monkeypatch.setattr(decoding.ops, "attention_cached", plain.attention_cached)
        want, _ = run()
    err = (got - want).abs().max().item()
    print(f"[{lm['model_type']} {kv}] logits (largest {want.abs().max():.2f}) max err {err:.2e}")
    assert err < 1e-3


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("lm", [BART, T5], ids=["bart", "t5"])
def test_a_drafting_model_changes_the_steps_not_the_tokens(lm, dtype):
    """Greedy: whatever the assistant drafts, the tokens are those without it; a model that drafts for itself needs fewer steps."""
    model, other = _model(lm, dtype), _model(lm, dtype, seed=7)
    lc = model.decoder_model.config
    wave = _wave(3, seed=2)
    for eos in (lc.eos_token_id, -1):
        for m in (model, other):
            m.decoder_model.config.eos_token_id = eos
        kv = "fp32" if dtype == "fp32" else "fp8"
        want = model.generate(wave, max_length=14, kv_cache=kv)
        assert len(want) == 3
        if eos == -1:
            assert all(len(w) == 14 for w in want)
        if dtype == "fp32":          # (bf16: five tokens at a time round differently from one, a near-tie may fall the other way)
            for n in (1, 4):
                assert model.generate(wave, max_length=14, kv_cache=kv, assistant_model=other, num_assistant_tokens=n) == want
        got = model.generate(wave, max_length=14, kv_cache=kv, assistant_model=model, num_assistant_tokens=4)
        assert all(len(a) <= 14 for a in got)
        if dtype == "fp32":
            assert got == want
            if eos == -1:
                assert model.last_decode_steps == math.ceil(14 / 5)


@pytest.mark.parametrize("lm", [BART, T5], ids=["bart", "t5"])
def test_replayed_steps_equal_eager_ones(lm, monkeypatch):
    """bf16 steps are captured at their second use and replayed: the same bits as eager steps, over several replays with other work between them,
    for one and for several tokens, on rows at different lengths; and generate emits the same tokens either way."""
    from speechmix_amd.decoding import CachedDecoder
    model = _model(lm, "bf16")
    with torch.no_grad():
        enc, B, S = model._speech_encode(_wave(2))
        fed = torch.randint(4, 200, (4, 3), generator=torch.Generator().manual_seed(5)).to(model.device)
        outs = []
        for flag in ("0", "1"):
            monkeypatch.setenv("SMX_DECODE_GRAPH", flag)
            dec = CachedDecoder(model.engine, enc, B, S, 2, 40, "fp8")
            got = []
            for k in range(6):
                for ids in (fed[:, :1].contiguous(), (fed + k) % 200):
                    got.append(dec.step(ids).clone())
                    dec.lens += torch.tensor([1, 2, 1, ids.shape[1]], dtype=torch.int32, device=model.device).clamp_max(ids.shape[1])
                    torch.randn(1000, device=model.device).sum().item()
            assert bool(dec.graphs) == (flag == "1") and all(dec.graphs.values())
            outs.append(got)
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    model.decoder_model.config.eos_token_id = -1
    kw = dict(max_length=11, kv_cache="int8", do_sample=True, num_return_sequences=3, assistant_model=model, num_assistant_tokens=2)
    rows = []
    for flag in ("0", "1"):
        monkeypatch.setenv("SMX_DECODE_GRAPH", flag)
        rows.append(model.generate(_wave(2), generator=torch.Generator(device=model.device).manual_seed(4), **kw))
    assert rows[0] == rows[1]


def test_a_replayed_step_leaves_replaced_workspaces_alone():
    """A feed-forward that splits its reduction takes a scratch buffer of the engine, and a wider step replaces that buffer: the narrow step's
    graph still runs on the old one, which nothing else may be given meanwhile."""
    from speechmix_amd.decoding import CachedDecoder
    model = _model(dict(BART, decoder_ffn_dim=2048), "bf16")
    eng = model.engine
    with torch.no_grad():
        enc, B, S = model._speech_encode(_wave(2))
        eng._persist.pop("fwd_slabs", None)
        dec = CachedDecoder(eng, enc, B, S, 2, 40, "fp8")
        ids = torch.full((4, 1), 7, dtype=torch.int64, device=model.device)
        want = [dec.step(ids).clone() for _ in range(3)][-1]
        old = eng._persist["fwd_slabs"]
        size, where = old.numel(), old.data_ptr()
        del old
        dec.step(ids.expand(4, 24).contiguous())
        assert eng._persist["fwd_slabs"].data_ptr() != where
        canaries = [torch.full((size,), 3.0, device=model.device) for _ in range(16)]
        got = dec.step(ids).clone()
        assert torch.equal(got, want) and all((c == 3.0).all() for c in canaries)
        assert all(c.data_ptr() != where for c in canaries)


@pytest.mark.parametrize("kv", [None, "fp8"])
def test_sampled_rows(kv):
    """Rows per clip, seeds, temperatures."""
    model = _model(BART, "bf16", spread=2.0)
    model.decoder_model.config.eos_token_id = -1
    wave = _wave(2, seed=3)
    gen = lambda s: torch.Generator(device=model.device).manual_seed(s)
    a = model.generate(wave, max_length=9, num_return_sequences=5, do_sample=True, kv_cache=kv, generator=gen(1))
    b = model.generate(wave, max_length=9, num_return_sequences=5, do_sample=True, kv_cache=kv, generator=gen(1))
    c = model.generate(wave, max_length=9, num_return_sequences=5, do_sample=True, kv_cache=kv, generator=gen(2))
    assert len(a) == 10 and all(len(r) == 9 and all(0 <= t < 203 for t in r) for r in a)
    assert a == b and a != c and len({tuple(r) for r in a}) > 1
    cold = model.generate(wave, max_length=9, num_return_sequences=2, do_sample=True, temperature=1e-4, kv_cache=kv, generator=gen(3))
    greedy = model.generate(wave, max_length=9, kv_cache=kv or "bf16")
    assert cold[0][:1] == greedy[0][:1] and cold[2][:1] == greedy[1][:1]
    text = model.generate_from_text(torch.randint(4, 200, (2, 6)), max_length=5, num_return_sequences=3, do_sample=True, kv_cache=kv)
    assert len(text) == 6


@pytest.mark.parametrize("assistant", [False, True])
def test_the_first_token_is_drawn_from_the_models_distribution(assistant):
    """4 000 rows of one clip: the frequency of every token within five standard deviations (plus one count) of softmax(logits / T), with and
    without a drafting model whose own distribution is another."""
    model, other = _model(BART, "fp32", spread=2.0), _model(BART, "fp32", seed=7, spread=2.0)
    wave, T, N = _wave(1, seed=4), 1.7, 4000
    with torch.no_grad():
        enc, B, S = model._speech_encode(wave)
        from speechmix_amd.decoding import CachedDecoder
        lc = model.decoder_model.config
        lg = CachedDecoder(model.engine, enc, B, S, 1, 2).step(torch.full((1, 1), lc.decoder_start_token_id, dtype=torch.int64, device=model.device))
    p = torch.softmax(lg[0, 0].double() / T, 0).cpu()
    for m in (model, other):
        m.decoder_model.config.eos_token_id = -1
    rows = model.generate(wave, max_length=1, num_return_sequences=N, do_sample=True, temperature=T, kv_cache="fp32",
                          assistant_model=other if assistant else None, num_assistant_tokens=2,
                          generator=torch.Generator(device=model.device).manual_seed(11))
    f = torch.bincount(torch.tensor([r[0] for r in rows]), minlength=203).double() / N
    assert ((f - p).abs() <= 5 * (p * (1 - p) / N).sqrt() + 1 / N).all()


def test_the_memory_an_8_bit_cache_takes():
    from speechmix_amd.decoding import CachedDecoder
    model = _model(BART, "bf16")
    with torch.no_grad():
        enc, B, S = model._speech_encode(_wave(2))
        full, small = (CachedDecoder(model.engine, enc, B, S, 4, 40, kv).bytes() for kv in (None, "fp8"))
    assert small * 128 == full * 68                     # 64 codes and one 4-byte scale against 128 bytes
