"""Decoding over K/V caches: the decoder half of the LM on the cached operators (ops.kv_append, ops.attention_cached, ops.verify_draft).

`SpeechMixEED.generate` without options keeps its greedy loop (engine.Engine.greedy_decode).  The options here - an 8-bit cache, several
sampled rows per clip, a drafting model - need what that loop cannot do: rows at different lengths, more than one new token per row and
step, and cross-attention keys that the rows of a clip share (HF's `generate(num_return_sequences=, do_sample=, temperature=,
assistant_model=)`; the reference's loops are greedy, ref:train.py:18-34, and its HF twin hands generation to HF, ref:speechmix/hf_model.py:354-375).
"""
import gc
import math
import os
import warnings

import torch

from . import ops
from .engine import _act_id
from .ops import BF16, view

KV_CACHE_FORMATS = {"fp8": "e4m3", "e4m3": "e4m3", "int8": "int8", "bf16": "bf16", "fp32": "f32", "f32": "f32"}


def cache_format(kv_cache, dt):
    """The cache format behind `generate(kv_cache=...)`; None: the engine's own type, unquantised."""
    if kv_cache is None:
        return "bf16" if dt == BF16 else "f32"
    if kv_cache not in KV_CACHE_FORMATS:
        raise ValueError(f"kv_cache must be one of {sorted(KV_CACHE_FORMATS)} or None, got {kv_cache!r}")
    return KV_CACHE_FORMATS[kv_cache]


class CachedDecoder:
    """The LM decoder of `eng` over `rows_per_clip` rows of each of `clips` clips (encoder output enc [clips * S, d]).

    `step(ids)` feeds Tq new tokens to every row and returns their logits; `lens` (int32, device) holds how many tokens each row's caches
    hold, and is the caller's to move: a step writes its tokens at lens .. lens + Tq - 1 and attends over lens + Tq, so a caller that keeps fewer
    of them (rejected drafts) just advances by less.  The cross-attention keys of a clip are projected once and read by all its rows."""

    def __init__(self, eng, enc, clips, S, rows_per_clip, capacity, kv_cache=None, logit_scale=1.0):
        self.eng = eng
        lc, lp, st = eng.lc, eng.lp, eng.st
        self.t5 = lc.model_type == "t5"
        self.pre_ln = lc.model_type in ("mbart", "t5")
        self.d, self.H, self.F = lc.d_model, lc.decoder_attention_heads, lc.decoder_ffn_dim
        self.hd = lc.d_kv if self.t5 else self.d // self.H
        if self.H * self.hd != self.d:
            raise NotImplementedError("cached decoding assumes num_heads * d_kv == d_model")
        self.fmt = cache_format(kv_cache, eng.dt)
        self.clips, self.N, self.cap = clips, clips * rows_per_clip, capacity
        self.eps = lc.layer_norm_epsilon if self.t5 else 1e-5
        self.scale = 1.0 if self.t5 else self.hd ** -0.5
        self.emb = lp + ("shared.weight" if self.t5 else "model.shared.weight")
        self.escale = math.sqrt(self.d) if (lc.scale_embedding and not self.t5) else 1.0
        self.pd = lp + "model.decoder."
        self.names = [(eng._t5_layer_names if self.t5 else eng._bart_layer_names)("decoder", i) for i in range(lc.decoder_layers)]
        self.V, self.Vp = lc.vocab_size, (lc.vocab_size + 7) // 8 * 8
        self.head = lp + "lm_head.weight" if eng.has(lp + "lm_head.weight") else self.emb
        # logits / temperature come out of the head's product
        self.head_alpha = (self.d ** -0.5 if (self.t5 and lc.tie_word_embeddings) else 1.0) * logit_scale
        self.flb = st.module.get_buffer(lp + "final_logits_bias").view(-1) * logit_scale if not self.t5 else None
        self.lens = torch.zeros(self.N, dtype=torch.int32, device=eng.dev)
        self.use_graphs = eng.dev.type == "cuda" and eng.dt == BF16 and os.environ.get("SMX_DECODE_GRAPH", "1") != "0"
        self.graphs, self.warm = {}, set()
        self.rel = None
        if self.t5:            # [H, n], indexed by query - key: what the last of n queries sees.  The last bucket holds every distance from
            # relative_attention_max_distance on, and the operator clamps to the table's end: no more than that, whatever the capacity
            n = min(capacity, lc.relative_attention_max_distance + 1)
            self.rel = eng._t5_bias("decoder", 1, n, first=n - 1)[0][:, 0].flip(-1).contiguous()
        else:
            self.max_pos = st.offsets[self.pd + "embed_positions.weight"][2][0] - 1
        self.own = [ops.KVCache.empty(self.N, self.H, capacity, self.hd, self.fmt, eng.dev) for _ in self.names]
        self.cross = [self._project_cross(nm["xattn"], enc, S) for nm in self.names]

    def _cat_b(self, a, b):
        return self.eng.st.cat([a[1], b[1]], "p32") if a[1] else None

    def _project_cross(self, xa, enc, S):
        eng, d = self.eng, self.d
        kv = eng.lin(enc, eng.st.cat([xa["k"][0], xa["v"][0]]), self._cat_b(xa["k"], xa["v"]), self.clips * S, 2 * d, d)
        kv = kv.view(self.clips, S, 2, self.H, self.hd)
        if self.fmt == ("bf16" if eng.dt == BF16 else "f32"):          # read where the projection left it
            return ops.KVCache(kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2), fmt=self.fmt)
        c = ops.KVCache.empty(self.clips, self.H, S, self.hd, self.fmt, eng.dev)
        ops.kv_append(c, kv[:, :, 0], kv[:, :, 1], 0)
        return c

    def bytes(self):
        return sum(c.bytes() for c in self.own + self.cross)

    def step(self, ids):
        """ids int64 [N, Tq] -> logits fp32 [N, Tq, V] (a view of rows of Vp, valid until the next step of as many tokens).  Rows past the
        capacity (finished ones that are still fed) write nothing and give logits without meaning.

        Nothing in a step but `lens` and the ids depends on the position, and both are in device memory: the second step of a width is
        captured into a HIP graph (its kernel picks are made by then) and replayed from then on, as greedy_decode does per position
        (bf16; SMX_DECODE_GRAPH=0: off)."""
        Tq = ids.shape[1]
        g = self.graphs.get(Tq)
        if g is None and Tq in self.warm and self.use_graphs:
            g = self.graphs[Tq] = self._capture(ids)
        if not g:                                       # (False: capture was refused, this width stays eager)
            self.warm.add(Tq)
            return self._step(ids)
        graph, buf, logits, _ = g
        buf.copy_(ids)
        graph.replay()
        return logits

    def _capture(self, ids):
        graph, buf = torch.cuda.CUDAGraph(), ids.clone()
        gc_was = gc.isenabled()
        gc.disable()                                    # (no finaliser may run on a capturing thread: graphs.StepGraphs.capture)
        try:
            with torch.cuda.graph(graph, capture_error_mode=os.environ.get("SMX_CAPTURE_MODE", "thread_local")):
                logits = self._step(buf)
        except RuntimeError as e:
            warnings.warn(f"CachedDecoder: HIP graph capture failed ({e}); decoding eagerly")
            return False
        finally:
            if gc_was:
                gc.enable()
        # (the graph holds addresses: a workspace of the engine that a wider step replaces must outlive it)
        return graph, buf, logits, self.eng.workspaces()

    def _step(self, ids):
        eng, lc = self.eng, self.eng.lc
        N, Tq = ids.shape
        M, d, H, hd, eps, t5 = N * Tq, self.d, self.H, self.hd, self.eps, self.t5
        act = _act_id(lc.activation_function)
        flat = ids.reshape(-1).contiguous()
        y = eng.new(M, d)
        ops.embed_fwd(flat, eng.W(self.emb), y, M, d, self.escale, eng.dt)
        if not t5:
            pos = (self.lens[:, None] + torch.arange(2, 2 + Tq, device=eng.dev)).clamp_max(self.max_pos).reshape(-1).long()
            pe, xs = eng.new(M, d), eng.new(M, d)
            ops.embed_fwd(pos, eng.W(self.pd + "embed_positions.weight"), pe, M, d, 1.0, eng.dt)
            ops.add(y, pe, xs, M * d, eng.dt)
            y, _ = eng.ln_fwd(xs, self.pd + "layernorm_embedding.weight", self.pd + "layernorm_embedding.bias", M, d, eps)
        total = (self.lens + Tq).clamp_max(self.cap)
        for li, nm in enumerate(self.names):
            a, xa = nm["attn"], nm["xattn"]
            x0 = y
            xin = eng.ln_fwd(x0, nm["ln1"][0], nm["ln1"][1], M, d, eps, rms=t5)[0] if self.pre_ln else x0
            q = eng.lin(xin, eng.W(a["q"][0]), eng._b(a["q"][1]), M, d, d)
            kv = eng.lin(xin, eng.st.cat([a["k"][0], a["v"][0]]), self._cat_b(a["k"], a["v"]), M, 2 * d, d).view(N, Tq, 2, H, hd)
            ops.kv_append(self.own[li], kv[:, :, 0], kv[:, :, 1], self.lens)
            o, _ = ops.attention_cached(q.view(N, Tq, H, hd), self.own[li], total, scale=self.scale, rel_bias=self.rel)
            s1 = eng.lin(o, eng.W(a["o"][0]), eng._b(a["o"][1]), M, d, d, resid=x0)
            if self.pre_ln:
                h = s1
                xin2 = eng.ln_fwd(h, nm["lnx"][0], nm["lnx"][1], M, d, eps, rms=t5)[0]
            else:
                h = xin2 = eng.ln_fwd(s1, nm["ln1"][0], nm["ln1"][1], M, d, eps)[0]
            q = eng.lin(xin2, eng.W(xa["q"][0]), eng._b(xa["q"][1]), M, d, d)
            o, _ = ops.attention_cached(q.view(N, Tq, H, hd), None, scale=self.scale, prefix=self.cross[li])
            s2 = eng.lin(o, eng.W(xa["o"][0]), eng._b(xa["o"][1]), M, d, d, resid=h)
            if self.pre_ln:
                n2 = eng.ln_fwd(s2, nm["ln2"][0], nm["ln2"][1], M, d, eps, rms=t5)[0]
                y, _ = eng._ffn_fwd(n2, M, d, self.F, nm["fc1"], nm["fc2"], act, s2)
            else:
                h2 = eng.ln_fwd(s2, nm["lnx"][0], nm["lnx"][1], M, d, eps)[0]
                s3, _ = eng._ffn_fwd(h2, M, d, self.F, nm["fc1"], nm["fc2"], act, h2)
                y = eng.ln_fwd(s3, nm["ln2"][0], nm["ln2"][1], M, d, eps)[0]
            if eng.lm_adapters:
                y, _ = eng.adapter_fwd(y, lc.encoder_layers + li, M, d)
        if t5:
            y = eng.ln_fwd(y, eng.lp + "decoder.final_layer_norm.weight", None, M, d, eps, rms=True)[0]
        elif self.pre_ln:
            y = eng.ln_fwd(y, self.pd + "layer_norm.weight", self.pd + "layer_norm.bias", M, d, eps)[0]
        logits = eng.new(M, self.Vp, dt=torch.float32)
        ops.gemm(y, eng.W(self.head), logits, M, self.V, d, eng.dt, cv=view(self.Vp), bias=self.flb, out_f32=True, alpha=self.head_alpha)
        return logits.view(N, Tq, self.Vp)[..., :self.V]

    def probabilities(self, logits):
        """softmax of `step`'s logits, in place -> fp32 [N, Tq, V]."""
        N, Tq, V = logits.shape
        full = logits.as_strided((N * Tq, self.Vp), (self.Vp, 1))
        if self.Vp != V:
            full[:, V:] = -math.inf
        ops.softmax_rows(full, N * Tq, self.Vp)
        return logits


def decode(dec, max_new_tokens, start_id, eos_id, pad_id, sample=False, generator=None, draft=None, num_draft=4):
    """Generate up to max_new_tokens for every row of `dec` (a CachedDecoder; `draft`: a second, cheaper one over the same rows that proposes
    num_draft tokens a step).  sample: draw from the (temperature-scaled) probabilities, with uniforms from `generator`; otherwise greedy.
    With a draft the result is what `dec` alone would give: the same tokens when greedy, the same distribution when sampled.
    -> (int64 [N, <= max_new_tokens] ids, padded with pad_id behind eos, and the number of times `dec` ran)."""
    dev, N = dec.eng.dev, dec.N
    n = num_draft if draft is not None else 0
    out = torch.full((N, max_new_tokens + n + 1), pad_id, dtype=torch.int64, device=dev)
    count = torch.zeros(N, dtype=torch.int64, device=dev)
    done = torch.zeros(N, dtype=torch.bool, device=dev)
    tok = torch.full((N, 1), start_id, dtype=torch.int64, device=dev)
    cols = torch.arange(n + 1, device=dev)

    def uniforms(k):
        return torch.rand(N, k, device=dev, generator=generator) if sample else None
    none = torch.empty(N, 0, dtype=torch.int64, device=dev)
    q = torch.empty(N, n, dec.V, device=dev) if sample and n else None
    steps = 0
    while True:
        ids = [tok]
        for i in range(n):
            lg = draft.step(ids[-1])
            pr = draft.probabilities(lg) if sample else lg
            nxt = ops.verify_draft(pr, none, None, uniforms(1))[1]            # (nothing drafted: a plain draw / arg max)
            draft.lens += 1
            ids.append(nxt[:, None])
            if sample:
                q[:, i] = pr[:, 0]
        if n:                                                                 # the last draft's keys, in case it is accepted
            draft.step(ids[-1])
        fed = torch.cat(ids, 1)
        lg = dec.step(fed)
        pr = dec.probabilities(lg) if sample else lg
        acc, nxt = ops.verify_draft(pr, fed[:, 1:], q, uniforms(n + 1))
        steps += 1
        # accepted drafts, then the next token; what stands behind it is overwritten by the next step
        acc = acc.long()
        new = torch.where(cols < acc[:, None], torch.cat([fed[:, 1:], nxt[:, None]], 1), nxt[:, None])
        new = torch.where(cols <= acc[:, None], new, torch.full_like(new, pad_id))
        stop = (new == eos_id) & (cols <= acc[:, None])
        new = torch.where(stop.long().cumsum(1) - stop.long() > 0, torch.full_like(new, pad_id), new)     # behind an accepted eos
        new = torch.where(done[:, None], torch.full_like(new, pad_id), new)
        out.scatter_(1, (count[:, None] + cols).clamp_max(out.shape[1] - 1), new)
        count = torch.where(done, count, count + acc + 1)
        done = done | stop.any(1) | (count >= max_new_tokens)
        count = count.clamp_max(max_new_tokens)
        moved = torch.where(done, dec.lens, dec.lens + acc.to(torch.int32) + 1)
        dec.lens.copy_(moved)
        if draft is not None:
            draft.lens.copy_(moved)
        tok = nxt[:, None]
        if bool(done.all()):
            break
    return out[:, :min(int(count.max()), max_new_tokens)].clone(), steps
