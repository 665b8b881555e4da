"""Assisted decoding in bf16, the type whose steps are captured: the loop against a plain re-run of it, and its steps of several tokens against steps
of one."""
import pytest
import torch

from tests.test_gpu_generate_options import BART, T5, _model, _wave

pytestmark = pytest.mark.gpu


def _prefix_logits(model, enc, B, S, cap, kv, prefixes, column):
    """Logits of `model` behind every row's prefix (rows of different lengths), from a fresh decoder fed one token at a time: each row's at its own
    last token.  Rows that are done go on with their last token."""
    from speechmix_amd.decoding import CachedDecoder
    dec = CachedDecoder(model.engine, enc, B, S, 1, cap, kv)
    out = [None] * B
    for t in range(max(len(p) for p in prefixes)):
        ids = torch.tensor([[p[min(t, len(p) - 1)]] for p in prefixes], device=model.device)
        lg = dec.step(ids)[:, 0, column:].clone()
        dec.lens += 1
        for b, p in enumerate(prefixes):
            if t == len(p) - 1:
                out[b] = lg[b]
    return out


def _rerun(model, other, enc, aenc, B, S, n, nd, start, eos, pad, kv):
    """The greedy assisted loop once more, from lists: drafts come from the whole prefix each time (no cache of the drafter survives a round), the
    verification is a comparison of numbers on the host."""
    from speechmix_amd.decoding import CachedDecoder
    cap = n + nd + 1
    dec = CachedDecoder(model.engine, enc, B, S, 1, cap, kv)
    seqs, done, steps = [[start] for _ in range(B)], [False] * B, 0
    while not all(done):
        drafted = [list(s) for s in seqs]
        for _ in range(nd):
            lg = _prefix_logits(other, aenc, B, S, cap, kv, drafted, 0)
            for b in range(B):
                drafted[b].append(int(lg[b].argmax()))
        fed = torch.tensor([d[len(s) - 1:len(s) + nd] for d, s in zip(drafted, seqs)], device=model.device)
        best = dec.step(fed).argmax(-1).tolist()
        steps += 1
        for b in range(B):
            if done[b]:
                continue
            k = 0
            while k < nd and best[b][k] == int(fed[b, k + 1]):
                k += 1
            new = fed[b, 1:k + 1].tolist() + [best[b][k]]
            dec.lens[b] += k + 1
            if eos in new:
                new = new[:new.index(eos) + 1]
            seqs[b] = (seqs[b] + new)[:n + 1]
            done[b] = eos in new or len(seqs[b]) > n
    return [s[1:s.index(eos)] if eos in s[1:] else s[1:] for s in seqs], steps


@pytest.mark.parametrize("lm", [BART, T5], ids=["bart", "t5"])
@pytest.mark.parametrize("own", [True, False], ids=["itself", "another"])
@pytest.mark.parametrize("nd", [1, 4])
@pytest.mark.parametrize("eos", [None, -1])
def test_the_assisted_loop_in_bf16_against_a_plain_rerun(lm, own, nd, eos):
    """The same widths, rows and kernels give the same logits, so the tokens and the number of steps are equal: any draft accepted wrongly, length moved
    wrongly or key missed by the drafter would show.  eos: the model's own, or none."""
    model = _model(lm, "bf16")
    other = model if own else _model(lm, "bf16", seed=7)
    lc = model.decoder_model.config
    for m in (model, other):
        m.decoder_model.config.eos_token_id = lc.eos_token_id if eos is None else eos
    wave, n = _wave(3, seed=2), 14
    got = model.generate(wave, max_length=n, kv_cache="fp8", assistant_model=other, num_assistant_tokens=nd)
    steps = model.last_decode_steps
    with torch.no_grad():
        enc, B, S = model._speech_encode(wave)
        aenc = other._speech_encode(wave)[0]
        want, wsteps = _rerun(model, other, enc, aenc, B, S, n, nd, lc.decoder_start_token_id, lc.eos_token_id, lc.pad_token_id, "fp8")
    assert got == want and steps == wsteps
    if eos == -1:
        assert all(len(r) == n for r in got)
        if own:
            assert steps < n


@pytest.mark.parametrize("lm", [BART, T5], ids=["bart", "t5"])
@pytest.mark.parametrize("own", [True, False], ids=["itself", "another"])
def test_tokens_of_the_assisted_loop_are_those_of_single_steps(lm, own):
    """Every token that the bf16 loop emits, forced through steps of one token: its logit is next to that step's largest.  How near: let l1, l5 be the
    logits of steps of one and of five tokens over the same prefix, d = max |l1 - l5|.  The token t is the largest of l5, so l1[t] >= l5[t] - d >=
    l5[best of l1] - d >= max l1 - 2 d.  And d <= e1 + e5, the distances of both from the logits of the same weights in fp32: e1 is measured, and
    e5 - the same arithmetic in another order - is held to twice that."""
    from speechmix_amd.decoding import CachedDecoder
    model, exact = _model(lm, "bf16"), _model(lm, "fp32")
    other = model if own else _model(lm, "bf16", seed=7)
    for m in (model, other, exact):
        m.decoder_model.config.eos_token_id = -1
    lc = model.decoder_model.config
    wave, n = _wave(3, seed=2), 15
    got = model.generate(wave, max_length=n, kv_cache="fp8", assistant_model=other, num_assistant_tokens=4)
    fed = torch.tensor([[lc.decoder_start_token_id] + r[:-1] for r in got], device=model.device)
    with torch.no_grad():
        logits = {}
        for name, m, width in (("one", model, 1), ("five", model, 5), ("fp32", exact, 1)):
            enc, B, S = m._speech_encode(wave)
            dec = CachedDecoder(m.engine, enc, B, S, 1, n + 5, "fp8")
            out = []
            for t in range(0, n, width):
                out.append(dec.step(fed[:, t:t + width].contiguous()).clone())
                dec.lens += width
            logits[name] = torch.cat(out, 1)
    e1, e5 = ((logits[k] - logits["fp32"]).abs().max().item() for k in ("one", "five"))
    print(f"[{lm['model_type']}] e1 {e1:.3f} e5 {e5:.3f} largest {logits['fp32'].abs().max():.1f}")
    assert e5 <= 2 * e1
    one, tok = logits["one"], torch.tensor(got, device=model.device)
    short = one.amax(-1) - one.gather(-1, tok[..., None])[..., 0]
    assert (short <= 2 * (e1 + e5)).all()
    assert (short == 0).float().mean() > 0.8                       # (a margin that any token would meet says nothing)
