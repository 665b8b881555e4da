"""The options of `generate` that are refused, on the CPU (checked before anything runs)."""
import pytest
import torch

from speechmix_amd.model import SpeechMixEED

ENC = dict(model_type="wav2vec2", hidden_size=64, num_hidden_layers=1, num_attention_heads=2, intermediate_size=64, conv_dim=[32] * 7,
           conv_kernel=[10, 3, 3, 3, 3, 2, 2], conv_stride=[5, 2, 2, 2, 2, 2, 2], num_conv_pos_embeddings=16, num_conv_pos_embedding_groups=4)
LM = dict(model_type="bart", vocab_size=50, d_model=64, encoder_layers=1, decoder_layers=1, encoder_attention_heads=2, decoder_attention_heads=2,
          encoder_ffn_dim=64, decoder_ffn_dim=64, max_position_embeddings=32)


@pytest.fixture(scope="module")
def model():
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    return SpeechMixEED(ENC, LM, down_scale=2)


@pytest.mark.parametrize("kw,err", [(dict(kv_cache="fp4"), ValueError), (dict(num_return_sequences=0), ValueError), (dict(num_return_sequences=2), ValueError),
                                    (dict(num_return_sequences=1.5, do_sample=True), ValueError), (dict(temperature=0.0, do_sample=True), ValueError),
                                    (dict(temperature=float("nan"), do_sample=True), ValueError), (dict(generator=torch.Generator()), ValueError),
                                    (dict(assistant_model="distil"), TypeError)])
def test_refused_options(model, kw, err):
    for call in (lambda: model.generate(torch.zeros(1, 8000), **kw), lambda: model.generate_from_text(torch.zeros(1, 4, dtype=torch.int64), **kw)):
        with pytest.raises(err):
            call()


@pytest.mark.parametrize("kw", [dict(max_length=0, kv_cache="fp8"), dict(max_length=-1, do_sample=True), dict(num_return_sequences=2.0, do_sample=True)])
def test_refused_lengths_and_counts(model, kw):
    for call in (lambda: model.generate(torch.zeros(1, 8000), **kw), lambda: model.generate_from_text(torch.zeros(1, 4, dtype=torch.int64), **kw)):
        with pytest.raises(ValueError, match="max_length|num_return_sequences"):
            call()


def test_refused_assistants(model):
    other = SpeechMixEED(ENC, dict(LM, vocab_size=51), down_scale=2)
    with pytest.raises(ValueError, match="vocabulary"):
        model.generate(torch.zeros(1, 8000), assistant_model=other)
    same = SpeechMixEED(ENC, LM, down_scale=2)
    with pytest.raises(ValueError, match="num_assistant_tokens"):
        model.generate(torch.zeros(1, 8000), assistant_model=same, num_assistant_tokens=2.0)
    for n in (0, 65):
        with pytest.raises(ValueError, match="num_assistant_tokens"):
            model.generate(torch.zeros(1, 8000), assistant_model=same, num_assistant_tokens=n)
    with pytest.raises(RuntimeError, match="no CPU fallback"):          # good options get as far as the missing device
        model.generate(torch.zeros(1, 8000), assistant_model=same, kv_cache="fp8")


def test_cache_formats():
    from speechmix_amd import ops
    from speechmix_amd.decoding import cache_format
    assert cache_format(None, ops.BF16) == "bf16" and cache_format(None, ops.F32) == "f32"
    assert cache_format("fp8", ops.BF16) == "e4m3" and cache_format("int8", ops.F32) == "int8"


@pytest.mark.parametrize("temperature", [1e-21, 1e-40, 5e-324, -1.0, float("inf")])
def test_temperatures_that_leave_no_numbers_are_refused(model, temperature):
    """Logits divided by a vanishing temperature are infinite, their probabilities NaN and the drawn token 0: refused."""
    for call in (lambda: model.generate(torch.zeros(1, 8000), do_sample=True, temperature=temperature),
                 lambda: model.generate_from_text(torch.zeros(1, 4, dtype=torch.int64), do_sample=True, temperature=temperature)):
        with pytest.raises(ValueError, match="temperature"):
            call()
    with pytest.raises(RuntimeError, match="no CPU fallback"):          # the lowest that is taken gets as far as the missing device
        model.generate(torch.zeros(1, 8000), do_sample=True, temperature=1e-20)
