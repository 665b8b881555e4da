"""Cases of the decoding operators: writing and reading an 8-bit K/V cache, attention of new tokens over such a cache, the same with a
prefix that several rows share, and the verification of drafted tokens.

`run` computes the plain form with elementary torch operations (`own` false) or calls the package's operators (`own` true).
"""
import math

import torch

own = False

E4M3, INT8, BF16 = "e4m3", "int8", "bf16"
_DT = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---- cases -------------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one decoding step of a batch of clips writes one token per clip and layer (heads of the base models)
        dict(name="cache_step", kind="cache", B=32, T=1, H=12, D=64, cap=128, fmt=E4M3, dt="bf16"),
        # the cross-attention K/V of a batch of 30 s clips before length adapters, large model's heads, written at once
        dict(name="cache_prompt", kind="cache", B=48, T=1499, H=16, D=64, cap=1500, fmt=INT8, dt="bf16"),
        # latency: one clip, base model, a caption's length
        dict(name="decode_one", kind="decode", B=1, Tq=1, H=12, Hkv=12, D=64, cap=64, lo=37, hi=37, fmt=E4M3, dt="bf16",
             causal=True, nrel=0),
        # a decoding step of a batch, ragged, up to the position limit of the LM; some rows have nothing yet
        dict(name="decode_batch", kind="decode", B=64, Tq=1, H=16, Hkv=16, D=64, cap=1024, lo=0, hi=1024, fmt=E4M3, dt="bf16",
             causal=True, nrel=0),
        # long context with grouped heads, the largest call
        dict(name="decode_long", kind="decode", B=8, Tq=1, H=32, Hkv=8, D=128, cap=32768, lo=30001, hi=32768, fmt=E4M3, dt="bf16",
             causal=True, nrel=0),
        # the pass that checks four drafted tokens, relative-position bias, int8 cache
        dict(name="decode_draft", kind="decode", B=32, Tq=5, H=16, Hkv=16, D=64, cap=777, lo=5, hi=777, fmt=INT8, dt="bf16",
             causal=True, nrel=130),
        # single precision queries, unaligned length, one row over a long cache: the split over keys
        dict(name="decode_f32", kind="decode", B=1, Tq=1, H=12, Hkv=12, D=64, cap=8191, lo=8191, hi=8191, fmt=INT8, dt="f32",
             causal=True, nrel=0),
        # cross-attention of sampled transcriptions: eight rows of each clip read one set of bf16 keys
        dict(name="prefix_cross", kind="prefix", NG=16, R=8, Tq=1, H=12, Hkv=12, D=64, P=499, plo=62, cap=0, lo=0, hi=0, fmt=BF16,
             dt="bf16", nrel=0),
        # a batch behind one long common prompt, each row with its own tokens after it
        dict(name="prefix_prompt", kind="prefix", NG=1, R=64, Tq=1, H=32, Hkv=8, D=128, P=8192, plo=8192, cap=512, lo=0, hi=512,
             fmt=E4M3, dt="bf16", nrel=0),
        # one clip, greedy check of four drafts
        dict(name="verify_greedy", kind="verify", B=1, n=4, V=32128, mode="greedy"),
        # a serving batch, sampled
        dict(name="verify_sampled", kind="verify", B=64, n=4, V=50265, mode="sampled"),
        # plain sampling of many rows: nothing drafted
        dict(name="verify_none", kind="verify", B=256, n=0, V=50265, mode="sampled"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["cache", "decode", "decode", "prefix", "verify"])
    while True:
        if kind == "cache":
            T = _log(rng, 1, 1500)
            c = dict(kind=kind, B=_log(rng, 1, 64), T=T, H=rng.choice([4, 8, 12, 16]), D=rng.choice([64, 64, 128]),
                     cap=T + rng.randint(0, 100), fmt=rng.choice([E4M3, INT8]), dt=rng.choice(["bf16", "bf16", "f32"]))
        elif kind == "decode":
            Hkv = rng.choice([2, 4, 8, 12, 16])
            Tq = rng.choice([1, 1, 1, 2, 3, 5, 8, 17])
            cap = max(_log(rng, 1, 32768), Tq)
            hi = rng.randint(max(1, cap // 2), cap)
            c = dict(kind=kind, B=_log(rng, 1, 64), Tq=Tq, H=Hkv * rng.choice([1, 1, 2, 4, 8]), Hkv=Hkv, D=rng.choice([64, 64, 128]),
                     cap=cap, lo=rng.randint(0, hi), hi=hi, fmt=rng.choice([E4M3, INT8, BF16]),
                     dt=rng.choice(["bf16", "bf16", "f32"]), causal=rng.random() < 0.8, nrel=rng.choice([0, 0, 0, 130]))
        elif kind == "prefix":
            Hkv = rng.choice([4, 8, 12, 16])
            P = _log(rng, 16, 8192)
            cap = rng.choice([0, _log(rng, 1, 512)])
            hi = rng.randint(cap // 2, cap)
            c = dict(kind=kind, NG=rng.choice([1, 1, 2, 5, 16]), R=rng.choice([2, 3, 8, 16, 33, 64]), Tq=rng.choice([1, 1, 4]),
                     H=Hkv * rng.choice([1, 1, 4]), Hkv=Hkv, D=rng.choice([64, 64, 128]), P=P, plo=rng.randint(0, P), cap=cap,
                     lo=rng.randint(0, hi), hi=hi, fmt=rng.choice([E4M3, INT8, BF16]), dt=rng.choice(["bf16", "bf16", "f32"]),
                     nrel=rng.choice([0, 0, 130]))
        else:
            c = dict(kind=kind, B=_log(rng, 1, 256), n=rng.randint(0, 8), V=_log(rng, 1000, 50265),
                     mode=rng.choice(["greedy", "sampled", "sampled", "onehot"]))
        w, big = work(c), work(next(x for x in listed() if x["name"] == "decode_long"))
        dense = c.get("B", c.get("NG", 1)) * max(c.get("cap", 0), c.get("P", 0)) * c.get("H", 0) * c.get("D", 0) * c.get("Tq", 1)
        held = 8 * c["B"] * (c["n"] + 1) * c["V"] if kind == "verify" else 0
        if w["bytes"] <= big["bytes"] and w["flops"] <= big["flops"] and dense <= 8 * 32768 * 32 * 128 and held <= 1 << 30:
            return c


def _mean_len(c):
    return (c["lo"] + c["hi"]) / 2


def work(case):
    c = case
    if c["kind"] == "cache":
        es = _DT[c["dt"]].itemsize
        n = c["B"] * c["T"] * c["H"]
        return {"bytes": 2 * n * (2 * c["D"] * es + 2 * (c["D"] + 4)), "flops": 2 * n * c["D"] * 6}
    if c["kind"] == "verify":
        if c["mode"] == "greedy":
            n = c["B"] * (c["n"] + 1) * c["V"]
            return {"bytes": 4 * n, "flops": n}
        rows = 2 if (c["mode"] == "sampled" and c["n"]) else 1
        return {"bytes": 4 * rows * c["B"] * c["V"], "flops": 3 * c["B"] * c["V"]}
    es = _DT[c["dt"]].itemsize
    row = 2 * (c["D"] * 2 if c["fmt"] == BF16 else c["D"] + 4) * c["Hkv"]
    rows = c["B"] if c["kind"] == "decode" else c["NG"] * c["R"]
    keys = rows * _mean_len(c)
    qo = 2 * rows * c["Tq"] * c["H"] * c["D"] * es + 4 * rows * c["Tq"] * c["H"]
    shared, pairs = 0, keys
    if c["kind"] == "prefix":
        shared = c["NG"] * (c["plo"] + c["P"]) / 2
        pairs += shared * c["R"]
    return {"bytes": int((keys + shared) * row + qo), "flops": int(4 * pairs * c["Tq"] * c["H"] * c["D"])}


# ---- inputs ------------------------------------------------------------------------------------------------------------------

def _quantise(x, fmt):
    """Codes and scales of rows x [..., D] (fp32), one scale a row."""
    a = x.abs().amax(-1)
    if fmt == E4M3:
        m, e = torch.frexp(a)
        # the smallest power of two s with a / s <= 448 = 0.875 * 2^9
        e = torch.where(m <= 0.875, e - 9, e - 8).clamp_min(-126)
        s = torch.where(a > 0, torch.ldexp(torch.ones_like(a), e), torch.ones_like(a))
        return (x / s[..., None]).to(torch.float8_e4m3fn).view(torch.uint8), s
    s = (a / 127.0).clamp_min(2.0 ** -126)
    s = torch.where(a > 0, s, torch.ones_like(a))
    return torch.round(x / s[..., None]).clamp(-127, 127).to(torch.int8).view(torch.uint8), s


def _values(codes, scales, fmt):
    if fmt == BF16:
        return codes.float()
    c = codes.view(torch.float8_e4m3fn if fmt == E4M3 else torch.int8).float()
    return c * scales[..., None]


def _make_cache(N, H, cap, D, fmt, g):
    """K/V as they stand in a user's cache: [N, H, cap, D] codes and [N, H, cap] scales; keys with a common direction, as trained keys
    have, so that the scores of a row differ by several units."""
    out = []
    for which in range(2):
        x = torch.randn(N, H, cap, D, device="cuda", generator=g)
        if which == 0:
            x += torch.randn(N, H, 1, D, device="cuda", generator=g)
        if fmt == BF16:
            out += [x.to(torch.bfloat16), None]
        else:
            out += list(_quantise(x, fmt))
        del x
    k, ks, v, vs = out
    return dict(k=k, v=v, ks=ks, vs=vs, fmt=fmt)


def _handle(c):
    from speechmix_amd import ops
    return ops.KVCache(c["k"], c["v"], c["ks"], c["vs"], fmt=c["fmt"])


def _lengths(n, lo, hi, g):
    """Ragged lengths in [lo, hi], both ends among them where there is room."""
    t = torch.randint(lo, hi + 1, (n,), device="cuda", generator=g).to(torch.int32)
    if n > 1:
        t[0], t[1] = hi, lo
    return t


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    if c["kind"] == "cache":
        dt = _DT[c["dt"]]
        shape = (c["B"], c["T"], c["H"], c["D"])
        # K | V side by side, as one projection writes them
        kv = torch.randn(c["B"], c["T"], 2, c["H"], c["D"], device="cuda", generator=g) * 2
        kv = kv.to(dt)
        cache = dict(k=torch.zeros(c["B"], c["H"], c["cap"], c["D"], dtype=torch.uint8, device="cuda"), fmt=c["fmt"])
        cache["v"] = torch.zeros_like(cache["k"])
        cache["ks"] = torch.ones(c["B"], c["H"], c["cap"], device="cuda")
        cache["vs"] = torch.ones(c["B"], c["H"], c["cap"], device="cuda")
        st = dict(case=c, kv=kv, cache=cache, start=_lengths(c["B"], 0, c["cap"] - c["T"], g),
                  out=(torch.empty(shape, dtype=dt, device="cuda"), torch.empty(shape, dtype=dt, device="cuda")))
        if own:
            st["handle"] = _handle(cache)
        return st
    if c["kind"] == "verify":
        B, n, V = c["B"], c["n"], c["V"]
        logits = torch.randn(B, n + 1, V, device="cuda", generator=g) * 3
        if c["mode"] == "greedy":
            ids = logits[:, :n].argmax(-1)
            # a good draft model: four of five tokens agree with the target
            wrong = torch.rand(B, n, device="cuda", generator=g) < 0.2
            ids = torch.where(wrong, torch.randint(0, V, (B, n), device="cuda", generator=g), ids)
            return dict(case=c, p=logits, q=None, ids=ids, u=None)
        p = torch.softmax(logits, -1)
        noisy = logits[:, :n] + torch.randn(B, n, V, device="cuda", generator=g)
        q = torch.softmax(noisy, -1)
        del logits, noisy
        pick = torch.rand(B, n, 1, device="cuda", generator=g, dtype=torch.float64)
        ids = torch.searchsorted(q.double().cumsum(-1), pick).squeeze(-1).clamp_max(V - 1) if n else \
            torch.empty(B, 0, dtype=torch.int64, device="cuda")
        if c["mode"] == "onehot":
            q = None
        u = torch.rand(B, n + 1, device="cuda", generator=g)
        return dict(case=c, p=p, q=q, ids=ids, u=u)
    rows = c["B"] if c["kind"] == "decode" else c["NG"] * c["R"]
    st = dict(case=c)
    st["q"] = (torch.randn(rows, c["Tq"], c["H"], c["D"], device="cuda", generator=g) * 1.5).to(_DT[c["dt"]])
    st["scale"] = c["D"] ** -0.5
    st["rel"] = torch.randn(c["H"], c["nrel"], device="cuda", generator=g) if c["nrel"] else None
    st["cache"], st["klen"] = None, None
    if c["cap"]:
        st["cache"] = _make_cache(rows, c["Hkv"], c["cap"], c["D"], c["fmt"], g)
        st["klen"] = _lengths(rows, c["lo"], c["hi"], g)
    if c["kind"] == "prefix":
        st["prefix"] = _make_cache(c["NG"], c["Hkv"], c["P"], c["D"], c["fmt"], g)
        st["plen"] = _lengths(c["NG"], c["plo"], c["P"], g)
    if own:
        st["handle"] = _handle(st["cache"]) if c["cap"] else None
        if c["kind"] == "prefix":
            st["prefix_handle"] = _handle(st["prefix"])
    return st


# ---- one pass ----------------------------------------------------------------------------------------------------------------

def run(state):
    c = state["case"]
    if c["kind"] == "cache":
        return _run_cache(state)
    if c["kind"] == "verify":
        return _run_verify(state)
    return _run_attention(state)


def _run_cache(st):
    c, cache, (ko, vo) = st["case"], st["cache"], st["out"]
    k, v = st["kv"][:, :, 0], st["kv"][:, :, 1]
    if own:
        from speechmix_amd import ops
        ops.kv_append(st["handle"], k, v, st["start"])
        ops.kv_read(st["handle"], st["start"], ko, vo)
        return [ko, vo]
    b = torch.arange(c["B"], device="cuda")[:, None]
    t = st["start"].long()[:, None] + torch.arange(c["T"], device="cuda")
    for x, code, scale, o in ((k, "k", "ks", ko), (v, "v", "vs", vo)):
        q, s = _quantise(x.float(), c["fmt"])
        cache[code][b, :, t] = q
        cache[scale][b, :, t] = s
        o.copy_(_values(cache[code][b, :, t], cache[scale][b, :, t], c["fmt"]))
    return [ko, vo]


def _run_attention(st):
    c = st["case"]
    prefix = c["kind"] == "prefix"
    causal = c.get("causal", True)
    if own:
        from speechmix_amd import ops
        return list(ops.attention_cached(st["q"], st["handle"], st["klen"], causal=causal, scale=st["scale"], rel_bias=st["rel"],
                                         prefix=st["prefix_handle"] if prefix else None,
                                         prefix_len=st["plen"] if prefix else None, want_lse=True))
    q = st["q"].float()
    N, Tq, H, D = q.shape
    Hkv, G = c["Hkv"], H // c["Hkv"]
    q = q.view(N, Tq, Hkv, G, D).permute(0, 2, 3, 1, 4)                       # [N, Hkv, G, Tq, D]
    dev = q.device
    plen = st["plen"].long().repeat_interleave(c["R"]) if prefix else torch.zeros(N, dtype=torch.long, device=dev)
    klen = st["klen"].long() if c["cap"] else torch.zeros(N, dtype=torch.long, device=dev)
    qpos = (plen + klen - Tq)[:, None] + torch.arange(Tq, device=dev)         # [N, Tq]
    scores, values = [], []

    def part(cache, NG, pos0, length, cut):
        K, V = _values(cache["k"], cache["ks"], c["fmt"]), _values(cache["v"], cache["vs"], c["fmt"])
        T = K.shape[2]
        R = N // NG
        # rows of one group side by side: one product with the group's keys
        qq = q.view(NG, R, Hkv, G, Tq, D).transpose(1, 2).reshape(NG, Hkv, R * G * Tq, D)
        s = torch.matmul(qq, K.transpose(-1, -2).contiguous()).view(NG, Hkv, R, G, Tq, T).transpose(1, 2)
        s = s.reshape(N, Hkv, G, Tq, T) * st["scale"]
        j = torch.arange(T, device=dev)
        if st["rel"] is not None:
            dist = (qpos[:, :, None] - (pos0[:, None] + j)[:, None, :]).clamp(0, c["nrel"] - 1)
            s = s + st["rel"][:, dist].view(Hkv, G, N, Tq, T).permute(2, 0, 1, 3, 4)
        ok = (j < length[:, None])[:, None, :].expand(N, Tq, T)
        if cut:
            ok = ok & ((pos0[:, None] + j)[:, None, :] <= qpos[:, :, None])
        scores.append(s.masked_fill(~ok[:, None, None], float("-inf")))
        values.append(V)

    if prefix:
        part(st["prefix"], c["NG"], torch.zeros_like(plen), plen, False)
    if c["cap"]:
        part(st["cache"], N, plen, klen, causal)
    m = torch.stack([s.amax(-1) for s in scores]).amax(0)
    m0 = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    total, acc = 0, 0
    for s, V in zip(scores, values):
        p = torch.exp(s - m0[..., None])
        total = total + p.sum(-1)
        NG, T = V.shape[0], V.shape[2]
        R = N // NG
        pp = p.view(NG, R, Hkv, G, Tq, T).transpose(1, 2).reshape(NG, Hkv, R * G * Tq, T)
        acc = acc + torch.matmul(pp, V).view(NG, Hkv, R, G, Tq, D).transpose(1, 2).reshape(N, Hkv, G, Tq, D)
    out = torch.where(total[..., None] > 0, acc / total[..., None], torch.zeros_like(acc))
    lse = m0 + torch.log(total)
    return [out.permute(0, 3, 1, 2, 4).reshape(N, Tq, H, D).to(st["q"].dtype), lse.reshape(N, H, Tq)]


def _run_verify(st):
    c, p, q, ids, u = st["case"], st["p"], st["q"], st["ids"], st["u"]
    if own:
        from speechmix_amd import ops
        return list(ops.verify_draft(p, ids, q, u))
    B, n = ids.shape
    rows = torch.arange(B, device=p.device)
    if c["mode"] == "greedy":
        best = p.argmax(-1)
        ok = best[:, :n] == ids
        acc = ok.long().cumprod(1).sum(1)
        return [acc.to(torch.int32), best[rows, acc]]
    px = p[:, :n].gather(2, ids[..., None])[..., 0].double()
    qx = q.gather(2, ids[..., None])[..., 0].double() if q is not None else torch.ones_like(px)
    acc = (u[:, :n].double() * qx < px).long().cumprod(1).sum(1)
    w = p[rows, acc].double()
    if n:
        rejected = (acc < n)[:, None]
        r = acc.clamp_max(n - 1)
        if q is not None:
            w = torch.where(rejected, (w - q[rows, r].double()).clamp_min(0), w)
        else:
            w[rows, ids[rows, r]] = torch.where(rejected[:, 0], 0.0, w[rows, ids[rows, r]])
    cum = w.cumsum(1)
    token = (cum <= (u[:, n].double() * cum[:, -1])[:, None]).sum(1)
    last = (w > 0).long().mul(torch.arange(c["V"], device=p.device)).amax(1)
    return [acc.to(torch.int32), torch.minimum(token, last)]


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------------

def _exact_row(x, fmt):
    """Value of each element after storage, from the definition of the nearest code (x: fp64 [..., D], values of the input type)."""
    a = x.abs().amax(-1, keepdim=True)
    if fmt == INT8:
        s = (a.float() / 127).double()                         # the scale itself is a single precision number
        s = torch.where(a > 0, s, torch.ones_like(s))
        y = (x.float() / s.float()).double()                   # and so is the quotient that is rounded
        return torch.sign(y) * torch.where((y.abs() % 1) == 0.5, 2 * torch.round(y.abs() / 2), torch.floor(y.abs() + 0.5)) * s
    s = torch.exp2(torch.ceil(torch.log2(a / 448)))
    # log2 may be off by an ulp next to a border
    s = torch.where(a / s > 448, 2 * s, s)
    s = torch.where(2 * a / s <= 448, s / 2, s)
    s = torch.where(a > 0, s, torch.ones_like(s))
    y = x / s
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)     # three bits behind the leading one, 2^-9 at least
    r = y / step
    f = torch.floor(r)
    d = r - f
    up = (d > 0.5) | ((d == 0.5) & (f % 2 != 0))
    return (f + up) * step * s


def exact(case, seed):
    c = case
    st = prepare(c, seed)
    if c["kind"] == "cache":
        return [_exact_row(st["kv"][:, :, i].double(), c["fmt"]) for i in range(2)]
    if c["kind"] == "verify":
        acc, tok = [], []
        for b in range(c["B"]):
            p = st["p"][b].double()
            k, done = 0, False
            ids = st["ids"][b].tolist()
            w = None
            for i, x in enumerate(ids):
                if c["mode"] == "greedy":
                    if int(p[i].argmax()) != x:
                        break
                else:
                    qx = float(st["q"][b, i, x]) if st["q"] is not None else 1.0
                    if not float(st["u"][b, i]) * qx < float(p[i, x]):
                        if st["q"] is not None:
                            w = torch.relu(p[i] - st["q"][b, i].double())
                        else:
                            w = p[i].clone()
                            w[x] = 0
                        break
                k += 1
            acc.append(k)
            if c["mode"] == "greedy":
                tok.append(int(p[k].argmax()))
                continue
            if w is None:
                w = p[k]
            cum = torch.cumsum(w, 0)
            hit = torch.nonzero(cum > float(st["u"][b, c["n"]]) * float(cum[-1]))
            tok.append(int(hit[0]) if len(hit) else int(torch.nonzero(w > 0)[-1]))
        return [torch.tensor(acc, dtype=torch.int32), torch.tensor(tok, dtype=torch.int64)]
    q = st["q"].double()
    N, Tq, H, D = q.shape
    G = H // c["Hkv"]
    out = torch.zeros(N, Tq, H, D, dtype=torch.float64, device="cuda")
    lse = torch.full((N, H, Tq), float("-inf"), dtype=torch.float64, device="cuda")

    def load(cache, i, n):
        r = []
        for code, scale in (("k", "ks"), ("v", "vs")):
            x = cache[code][i, :, :n]
            if c["fmt"] != BF16:
                x = x.view(torch.float8_e4m3fn if c["fmt"] == E4M3 else torch.int8).float().double() * cache[scale][i, :, :n, None].double()
            r.append(x.double())
        return r                                                # [Hkv, n, D]

    for b in range(N):
        P = int(st["plen"][b // c["R"]]) if c["kind"] == "prefix" else 0
        L = int(st["klen"][b]) if c["cap"] else 0
        ks, vs = [], []
        if P:
            k, v = load(st["prefix"], b // c["R"], P)
            ks.append(k)
            vs.append(v)
        if L:
            k, v = load(st["cache"], b, L)
            ks.append(k)
            vs.append(v)
        if not ks:
            continue
        K, V = torch.cat(ks, 1), torch.cat(vs, 1)
        for t in range(Tq):
            qpos = P + L - Tq + t
            n = P + L
            if c.get("causal", True) and c["cap"]:
                n = max(P, min(n, qpos + 1))
            if n == 0:
                continue
            qh = q[b, t].view(c["Hkv"], G, D)
            s = torch.bmm(qh, K[:, :n].transpose(1, 2).contiguous()) * st["scale"]      # [Hkv, G, n]
            if st["rel"] is not None:
                dist = (qpos - torch.arange(n, device="cuda")).clamp(0, c["nrel"] - 1)
                s = s + st["rel"].double()[:, dist].view(c["Hkv"], G, n)
            z = torch.logsumexp(s, -1)
            out[b, t] = torch.bmm(torch.exp(s - z[..., None]), V[:, :n].contiguous()).view(H, D)
            lse[b, :, t] = z.view(H)
    return [out, lse]
