"""Every cache format under either type of model, and generate on a stream of the caller's."""
import pytest
import torch

from tests.test_gpu_generate_options import BART, T5, _model, _wave

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lm", [BART, T5], ids=["bart", "t5"])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("kv", [None, "bf16", "fp32", "f32", "fp8", "e4m3", "int8"])
def test_every_format_under_every_model(lm, dtype, kv):
    """Logits of forced tokens, one and three at a time, against the fp32 model over its own cache.  The yardstick of a format is what its rounding of the
    keys and values does to the fp32 model (e_fmt: fp32 queries, that cache); of the type, what bf16 arithmetic does over a cache that rounds nothing (e_type: bf16
    model, f32 cache).  Both together change a logit by no more than twice their sum (their effects add to first order)."""
    from speechmix_amd.decoding import CachedDecoder
    fed = torch.randint(4, 200, (4, 7), generator=torch.Generator().manual_seed(5))

    def run(dtype, kv):
        model = _model(lm, dtype, spread=2.0)
        with torch.no_grad():
            enc, B, S = model._speech_encode(_wave(2))
            dec = CachedDecoder(model.engine, enc, B, S, 2, 9, kv)
            out = []
            for a, b in ((0, 1), (1, 2), (2, 3), (3, 6), (6, 7)):
                out.append(dec.step(fed[:, a:b].contiguous().to(model.device)).clone())
                dec.lens += b - a
        return torch.cat(out, 1), dec.fmt
    exact, _ = run("fp32", None)
    got, fmt = run(dtype, kv)
    assert fmt == {None: {"bf16": "bf16", "fp32": "f32"}[dtype], "fp32": "f32", "fp8": "e4m3"}.get(kv, kv)
    e_fmt = (run("fp32", kv)[0] - exact).abs().max().item()
    e_type = (run("bf16", "f32")[0] - exact).abs().max().item() if dtype == "bf16" else 0.0
    err = (got - exact).abs().max().item()
    print(f"[{lm['model_type']} {dtype} {kv}] err {err:.2e} format {e_fmt:.2e} type {e_type:.2e}")
    assert err <= 2 * (e_fmt + e_type)


@pytest.mark.parametrize("assistant", [False, True])
def test_generate_on_a_side_stream(assistant):
    """The same tokens on a stream of the caller's as on the default one, with captured steps on both."""
    model = _model(BART, "bf16")
    model.decoder_model.config.eos_token_id = -1
    kw = dict(max_length=9, kv_cache="fp8", do_sample=True, num_return_sequences=3, assistant_model=model if assistant else None, num_assistant_tokens=2)
    gen = lambda: torch.Generator(device=model.device).manual_seed(4)
    want = model.generate(_wave(2), generator=gen(), **kw)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = model.generate(_wave(2), generator=gen(), **kw)
    torch.cuda.current_stream().wait_stream(s)
    assert got == want and model.generate(_wave(2), generator=gen(), **kw) == want
