"""The decoding operators on the GPU against plain 64-bit references (tests/decode_ref.py): the K/V cache in its formats, attention over it with
and without a shared prefix, the verification of drafted tokens.  Codes, scales, accepted counts and tokens are compared exactly; attention within
the bounds derived in decode_ref.attention_bounds."""
import numpy as np
import pytest
import torch

from tests import decode_ref as R

pytestmark = pytest.mark.gpu
FMTS = ["e4m3", "int8", "bf16", "f32"]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _filled(B, H, cap, D, fmt, seed, scale=1.0):
    from speechmix_amd import ops
    g = _gen(seed)
    c = ops.KVCache.empty(B, H, cap, D, fmt, "cuda")
    k = torch.randn(B, cap, H, D, device="cuda", generator=g) * scale + torch.randn(1, 1, H, D, device="cuda", generator=g)
    v = torch.randn(B, cap, H, D, device="cuda", generator=g) * scale
    ops.kv_append(c, k, v, 0)
    return c


def _vals(c):
    return R.values(c.k, c.ks, c.fmt), R.values(c.v, c.vs, c.fmt)


# ---- cache ----

@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,T,H,D,cap", [(1, 1, 1, 64, 1), (3, 1, 12, 64, 9), (2, 7, 2, 128, 20), (2, 37, 3, 16, 37), (1, 5, 2, 24, 8), (2, 4, 1, 256, 6),
                                         (1, 130, 2, 8, 200), (1, 3, 1, 40, 3)])
def test_append_and_read(fmt, dtype, B, T, H, D, cap):
    from speechmix_amd import ops
    g = _gen(B * 1000 + T)
    c = ops.KVCache.empty(B, H, cap, D, fmt, "cuda")
    for t in (c.k, c.v):
        t.view(torch.uint8).fill_(0x5a)
    before = [t.clone() for t in (c.k, c.v, c.ks, c.vs) if t is not None]
    kv = (torch.randn(B, T, 2, H, D, device="cuda", generator=g) * 3).to(dtype)          # K | V side by side: strided rows
    kv[0, 0, 0, 0] = 0                                                                     # a row of zeros
    kv[-1, -1, 1, -1] *= 1e-38                                                             # magnitudes next to the smallest normal number
    kv[0, T // 2, 1, 0, 0] = 3e38
    start = torch.randint(0, cap - T + 1, (B,), device="cuda", generator=g).to(torch.int32)
    ops.kv_append(c, kv[:, :, 0], kv[:, :, 1], start)
    st = start.tolist()
    for i, (code, scale) in enumerate(((c.k, c.ks), (c.v, c.vs))):
        x = kv[:, :, i].float().cpu()
        for b in range(B):
            got = code[b, :, st[b]:st[b] + T].transpose(0, 1).cpu()
            if fmt in ("e4m3", "int8"):
                wc, ws = R.quantise(x[b], fmt)
                assert torch.equal(scale[b, :, st[b]:st[b] + T].t().cpu(), ws)
                assert torch.equal(got.contiguous().view(torch.uint8), wc)
            else:
                assert torch.equal(got, x[b].to(got.dtype))
            # what lies outside the written range is as it was
            ref = before[i]
            keep = torch.ones(cap, dtype=torch.bool)
            keep[st[b]:st[b] + T] = False
            assert torch.equal(code[b].view(torch.uint8)[:, keep], ref[b].view(torch.uint8)[:, keep])
            if scale is not None:
                assert torch.equal(scale[b][:, keep], torch.ones_like(scale[b][:, keep]))
    for odt in (torch.bfloat16, torch.float32):
        ko, vo = (torch.full((B, T, H, D), 7.0, dtype=odt, device="cuda") for _ in range(2))
        ops.kv_read(c, start, ko, vo)
        for o, x in zip((ko, vo), _vals(c)):
            for b in range(B):
                want = x[b, :, st[b]:st[b] + T].transpose(0, 1)
                # code * scale: one rounding to fp32, one to the output's type (double rounding: the fp32 one is 2^-24 of the value).
                # Below 2^-126 both types step evenly, fp32 by 2^-149 and bf16 (seven mantissa bits) by 2^-133: half of that, absolutely.
                tol = want.abs() * (2.0 ** -24 if odt == torch.float32 else 2.0 ** -8 + 2.0 ** -24) + (2.0 ** -150 if odt == torch.float32 else 2.0 ** -134)
                assert ((o[b].double().cpu() - want).abs() <= tol).all()


def test_append_outside_the_capacity_is_dropped_and_read_leaves_rows_alone():
    from speechmix_amd import ops
    B, T, H, D, cap = 4, 6, 2, 64, 8
    for fmt in ("e4m3", "bf16"):
        c = ops.KVCache.empty(B, H, cap, D, fmt, "cuda")
        x = torch.randn(B, T, H, D, device="cuda", generator=_gen(1))
        start = torch.tensor([-3, 5, 2147483647, -2147483648], dtype=torch.int32, device="cuda")
        ops.kv_append(c, x, x, start)
        k, _ = _vals(c)
        assert (k[0, :, 3:] == 0).all() and (k[1, :, :5] == 0).all() and (k[2:] == 0).all()
        assert (k[0, :, :3].abs().sum(-1) > 0).all() and (k[1, :, 5:].abs().sum(-1) > 0).all()
        o, o2 = torch.full((2, B, T, H, D), 7.0, device="cuda")
        ops.kv_read(c, start, o, o2)
        assert (o[0, :3] == 7).all() and (o[1, 3:] == 7).all() and (o[2:] == 7).all() and torch.equal(o[0, 3:].cpu().double(), k[0, :, :3].transpose(0, 1))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_a_row_that_is_not_finite(fmt, bad):
    from speechmix_amd import ops
    c = ops.KVCache.empty(1, 2, 4, 64, fmt, "cuda")
    x = torch.randn(1, 4, 2, 64, device="cuda", generator=_gen(3))
    x[0, 2, 1, 17] = bad
    ops.kv_append(c, x, x, 0)
    assert (c.k[0, 1, 2] == 0).all() and torch.isnan(c.ks[0, 1, 2])
    assert torch.isfinite(c.ks).sum() == 7
    o, o2 = torch.zeros(2, 1, 4, 2, 64, device="cuda")
    ops.kv_read(c, 0, o, o2)
    assert torch.isnan(o[0, 2, 1]).all() and torch.isfinite(o).sum() == 7 * 64


def test_cache_beyond_32_bit_offsets():
    """Heads that start behind 2^31 elements: written, read and attended like the first."""
    from speechmix_amd import ops
    H, cap, D = 17, 1 << 20, 128
    c = ops.KVCache.empty(1, H, cap, D, "int8", "cuda")
    x = torch.randn(1, 40, H, D, device="cuda", generator=_gen(5))
    far = cap - 40
    for st in (0, far):
        ops.kv_append(c, x, x, st)
        o, o2 = torch.zeros(2, 1, 40, H, D, device="cuda")
        ops.kv_read(c, st, o, o2)
        wc, ws = R.quantise(x.cpu(), "int8")
        assert torch.equal(o.cpu().double(), (R.values(wc, ws, "int8").float()).double())
    q = torch.randn(1, 1, H, D, device="cuda", generator=_gen(6)).to(torch.bfloat16)
    _check(q, c, [40], causal=True)


# ---- attention ----

def _check(q, c, klen, causal=True, rel=None, pre=None, plen=None, scale=None, out=None):
    from speechmix_amd import ops
    B, Tq, H, D = q.shape
    kl = torch.tensor(klen, dtype=torch.int32, device="cuda") if klen is not None else None
    pl = torch.tensor(plen, dtype=torch.int32, device="cuda") if plen is not None else None
    o, lse = ops.attention_cached(q, c, kl, out=out, causal=causal, scale=scale, rel_bias=rel, prefix=pre, prefix_len=pl, want_lse=True)
    K = V = PK = PV = None

    def cut(cc, n):          # (only the valid rows travel to the CPU)
        n = max(1, min(max(n), cc.cap))
        return [R.values(t[:, :, :n], s[:, :, :n] if s is not None else None, cc.fmt) for t, s in ((cc.k, cc.ks), (cc.v, cc.vs))]
    if c is not None:
        klen = [min(max(x, 0), c.cap) for x in klen] if klen is not None else [c.cap] * B
        K, V = cut(c, klen)
    if pre is not None:
        plen = [min(max(x, 0), pre.cap) for x in plen] if plen is not None else [pre.cap] * pre.B
        PK, PV = cut(pre, plen)
    ref = R.attention(q, K, V, klen, plen, PK, PV, B // pre.B if pre is not None else 1, causal, D ** -0.5 if scale is None else scale, rel)
    tol_o, tol_l = R.attention_bounds(*ref, D, q.dtype)
    err = (o.double().cpu() - ref[0]).abs()
    assert (err <= tol_o).all(), (err - tol_o).max()
    empty = torch.isinf(ref[1])
    assert torch.equal(torch.isinf(lse.cpu()) & (lse.cpu() < 0), empty)
    assert ((lse.double().cpu() - ref[1]).abs()[~empty] <= tol_l[~empty]).all()
    return o, lse


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128, 32])
def test_attention_ragged_lengths(fmt, dtype, D):
    """Lengths around every border of a 16 / 32 / 64-key tile, nothing at all, one key, the whole capacity, more than it."""
    klen = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 200, 201, 999, -5]
    B, H = len(klen), 2
    c = _filled(B, H, 201, D, fmt, 11)
    q = torch.randn(B, 1, H, D, device="cuda", generator=_gen(12)).to(dtype)
    o, lse = _check(q, c, klen)
    assert (o[0] == 0).all() and (o[-1] == 0).all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("D,H,Hkv,Tq", [(64, 4, 4, 5), (128, 8, 1, 1), (64, 12, 4, 3), (128, 4, 2, 17), (64, 8, 2, 33), (16, 4, 2, 3), (64, 70, 1, 2)])
def test_attention_heads_queries_and_causality(fmt, D, H, Hkv, Tq):
    klen = [Tq, Tq + 1, 77, 40, Tq - 1, 1]
    B = len(klen)
    c = _filled(B, Hkv, 80, D, fmt, 21)
    q = torch.randn(B, Tq, H, D, device="cuda", generator=_gen(22)).to(torch.bfloat16)
    for causal in (True, False):
        _check(q, c, klen, causal=causal)


@pytest.mark.parametrize("fmt", ["e4m3", "bf16", "f32"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 24])
def test_attention_distance_bias(fmt, dtype, D):
    c = _filled(3, 4, 150, D, fmt, 31)
    q = torch.randn(3, 4, 4, D, device="cuda", generator=_gen(32)).to(dtype)
    for n in (1, 7, 130):
        rel = torch.randn(4, n, device="cuda", generator=_gen(33)) * 2
        _check(q, c, [4, 150, 67], rel=rel, scale=1.0 if n == 7 else None)
        pre = _filled(1, 4, 45, D, fmt, 34)
        _check(q, c, [4, 150, 2], rel=rel, pre=pre, plen=[45])


@pytest.mark.parametrize("fmt", ["e4m3", "bf16", "f32"])
@pytest.mark.parametrize("D", [64, 16])
def test_attention_bias_that_masks(fmt, D):
    """Distances masked with the type's lowest value or with -inf count as nothing next to others; where every key has the lowest value, all count
    alike (the scores vanish beside it); where every key has -inf, nothing is seen."""
    from speechmix_amd import ops
    c = _filled(2, 2, 100, D, fmt, 35)
    q = torch.randn(2, 1, 2, D, device="cuda", generator=_gen(36)).to(torch.bfloat16)
    kl = torch.tensor([100, 37], dtype=torch.int32, device="cuda")
    low = torch.finfo(torch.float32).min
    for m in (low, -float("inf")):
        rel = torch.full((2, 101), m, device="cuda")
        rel[:, :5] = 0.25                              # the last five keys are seen
        o, lse = ops.attention_cached(q, c, kl, rel_bias=rel, want_lse=True)
        for b, n in enumerate((100, 37)):
            K, V = (R.values(t[b:b + 1, :, n - 5:n], s[b:b + 1, :, n - 5:n] if s is not None else None, fmt) for t, s in ((c.k, c.ks), (c.v, c.vs)))
            ref = R.attention(q[b:b + 1], K, V, [5], None, None, None, 1, True, D ** -0.5, torch.full((2, 5), 0.25))
            tol_o, tol_l = R.attention_bounds(*ref, D, q.dtype)
            assert ((o[b:b + 1].double().cpu() - ref[0]).abs() <= tol_o).all() and ((lse[b:b + 1].double().cpu() - ref[1]).abs() <= tol_l).all()
        o, lse = ops.attention_cached(q, c, kl, rel_bias=torch.full((2, 7), m, device="cuda"), want_lse=True)
        if m == low:
            flat, _ = ops.attention_cached(torch.zeros_like(q), c, kl)
            assert (o.double() - flat.double()).abs().max() <= 2.0 ** -7 * flat.double().abs().max() and (lse == low).all()
        else:
            assert (o == 0).all() and (lse == m).all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("NG,R_,H,Hkv,D,P,Tq", [(1, 2, 2, 2, 64, 100, 1), (2, 3, 4, 2, 128, 65, 2), (3, 8, 2, 2, 64, 33, 1), (1, 33, 4, 1, 64, 70, 1),
                                                (2, 17, 2, 2, 64, 257, 1), (2, 2, 4, 2, 40, 30, 3)])
def test_attention_shared_prefix(fmt, dtype, NG, R_, H, Hkv, D, P, Tq):
    B = NG * R_
    pre = _filled(NG, Hkv, P, D, fmt, 41)
    q = torch.randn(B, Tq, H, D, device="cuda", generator=_gen(42)).to(dtype)
    plen = [P - 3, 0, 1][:NG]
    _check(q, None, None, pre=pre, plen=plen)                       # the prefix alone (a group with nothing in it gives zeros)
    _check(q, None, None, pre=pre)                                  # its whole capacity
    c = _filled(B, Hkv, 20, D, fmt, 43)
    klen = [(7 * b) % 21 for b in range(B)]
    _check(q, c, klen, pre=pre, plen=plen)


@pytest.mark.parametrize("fmt", ["e4m3", "int8", "bf16"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,Tq", [(64, 1), (128, 2)])
def test_attention_many_short_rows(fmt, dtype, D, Tq):
    """More rows and heads than the chip holds workgroups, few keys each, alone and behind a prefix."""
    B, H = 93, 6
    klen = [(11 * b) % 48 for b in range(B)]
    c = _filled(B, H, 47, D, fmt, 45)
    q = torch.randn(B, Tq, H, D, device="cuda", generator=_gen(46)).to(dtype)
    _check(q, c, klen)
    pre = _filled(3, H, 20, D, fmt, 47)
    _check(q, c, klen, pre=pre, plen=[20, 0, 7])


@pytest.mark.parametrize("fmt", ["e4m3", "int8", "bf16"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,R_,cap,P", [(64, 49, 0, 70), (64, 64, 0, 33), (128, 21, 0, 70), (64, 18, 0, 40), (64, 49, 260, 3500), (64, 49, 40, 600),
                                        (128, 21, 260, 5000), (128, 30, 40, 1300), (64, 17, 33, 700)])
def test_attention_many_rows_of_many_prefixes(fmt, dtype, D, R_, cap, P):
    """Enough groups that an item takes 32 or 64 rows of a prefix (a few rows are left over), without own keys, with long ones and with short
    ones: the first, a middle and the last group against the reference."""
    NG, H = 32, 8
    B = NG * R_
    pre = _filled(NG, H, P, D, fmt, 61)
    q = torch.randn(B, 1, H, D, device="cuda", generator=_gen(62)).to(dtype)
    plen = [(13 * g) % 70 for g in range(NG - 1)] + [min(P, 70)]
    c = _filled(B, H, cap, D, fmt, 63) if cap else None
    klen = [(7 * b) % 38 for b in range(B)] if cap else None
    rel = torch.randn(H, 50, device="cuda", generator=_gen(64)) if R_ == 49 else None
    from speechmix_amd import ops
    kl, pl = (torch.tensor(x, dtype=torch.int32, device="cuda") if x is not None else None for x in (klen, plen))
    o, lse = ops.attention_cached(q, c, kl, rel_bias=rel, prefix=pre, prefix_len=pl, want_lse=True)
    for g in (0, 17, NG - 1):
        rows = slice(g * R_, (g + 1) * R_)
        vals = []
        for cc, sl, n in ((c, rows, 38), (pre, slice(g, g + 1), 70)):
            vals += [R.values(t[sl, :, :n], s[sl, :, :n] if s is not None else None, cc.fmt) for t, s in ((cc.k, cc.ks), (cc.v, cc.vs))] if cc is not None else [None, None]
        ref = R.attention(q[rows], vals[0], vals[1], klen[rows] if cap else None, [plen[g]], vals[2], vals[3], R_, True, D ** -0.5, rel)
        tol_o, tol_l = R.attention_bounds(*ref, D, dtype)
        assert ((o[rows].double().cpu() - ref[0]).abs() <= tol_o).all(), g
        empty = torch.isinf(ref[1])
        assert torch.equal(torch.isinf(lse[rows].cpu()), empty) and ((lse[rows].double().cpu() - ref[1]).abs()[~empty] <= tol_l[~empty]).all(), g


@pytest.mark.parametrize("fmt", ["e4m3", "int8", "bf16"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,NG,R_,Hkv,G,Tq,cap,P", [(64, 43, 24, 8, 1, 1, 20, 300), (128, 43, 24, 8, 2, 2, 20, 300), (64, 9, 115, 8, 1, 3, 33, 40), (64, 17, 61, 16, 1, 1, 0, 90),
                                                    (128, 17, 61, 16, 1, 1, 0, 90), (64, 17, 21, 16, 2, 2, 0, 250)])
def test_attention_an_item_per_wave(fmt, dtype, D, NG, R_, Hkv, G, Tq, cap, P):
    """So many rows that every wave works for itself, prefixes included, and a row has one partial result of each part: groups without a prefix,
    rows without a key of their own, rows with neither."""
    from speechmix_amd import ops
    B, H = NG * R_, Hkv * G
    pre = _filled(NG, Hkv, P, D, fmt, 71)
    q = torch.randn(B, Tq, H, D, device="cuda", generator=_gen(72)).to(dtype)
    plen = [P] + [(29 * g) % (P + 1) for g in range(1, NG - 1)] + [0]
    c = _filled(B, Hkv, cap, D, fmt, 73) if cap else None
    klen = [(7 * b) % (cap + 1) for b in range(B)] if cap else None
    rel = torch.randn(H, 9, device="cuda", generator=_gen(74)) if G == 2 else None
    kl, pl = (torch.tensor(x, dtype=torch.int32, device="cuda") if x is not None else None for x in (klen, plen))
    o, lse = ops.attention_cached(q, c, kl, rel_bias=rel, prefix=pre, prefix_len=pl, want_lse=True)
    for g in (0, NG // 2, NG - 1):
        rows = slice(g * R_, (g + 1) * R_)
        vals = []
        for cc, sl in ((c, rows), (pre, slice(g, g + 1))):
            vals += [R.values(t[sl], s[sl] if s is not None else None, cc.fmt) for t, s in ((cc.k, cc.ks), (cc.v, cc.vs))] if cc is not None else [None, None]
        ref = R.attention(q[rows], vals[0], vals[1], klen[rows] if cap else None, [plen[g]], vals[2], vals[3], R_, True, D ** -0.5, rel)
        tol_o, tol_l = R.attention_bounds(*ref, D, dtype)
        assert ((o[rows].double().cpu() - ref[0]).abs() <= tol_o).all(), g
        empty = torch.isinf(ref[1])
        assert torch.equal(torch.isinf(lse[rows].cpu()), empty) and ((lse[rows].double().cpu() - ref[1]).abs()[~empty] <= tol_l[~empty]).all(), g


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
def test_attention_many_queries_of_many_rows(fmt):
    """64 and more rows a KV head out of queries and grouped heads, causal, in items of several tiles."""
    B, Tq, Hkv, G = 40, 33, 8, 2
    c = _filled(B, Hkv, 70, 64, fmt, 65)
    q = torch.randn(B, Tq, Hkv * G, 64, device="cuda", generator=_gen(66)).to(torch.bfloat16)
    klen = [(9 * b) % 71 for b in range(B)]
    from speechmix_amd import ops
    o, _ = ops.attention_cached(q, c, torch.tensor(klen, dtype=torch.int32, device="cuda"))
    for b in (0, 7, 39):
        ref = R.attention(q[b:b + 1], *(R.values(t[b:b + 1], s[b:b + 1] if s is not None else None, fmt) for t, s in ((c.k, c.ks), (c.v, c.vs))), klen[b:b + 1], None,
                          None, None, 1, True, 64 ** -0.5, None)
        tol_o, _ = R.attention_bounds(*ref, 64, q.dtype)
        assert ((o[b:b + 1].double().cpu() - ref[0]).abs() <= tol_o).all(), b


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_long_cache_is_split_and_joined(fmt, dtype):
    c = _filled(2, 2, 5000, 64, fmt, 51)
    q = torch.randn(2, 1, 2, 64, device="cuda", generator=_gen(52)).to(dtype)
    o, lse = _check(q, c, [4999, 130])
    for _ in range(3):                                              # the same bits every time
        from speechmix_amd import ops
        o2, l2 = ops.attention_cached(q, c, torch.tensor([4999, 130], dtype=torch.int32, device="cuda"), want_lse=True)
        assert torch.equal(o, o2) and torch.equal(lse, l2)


@pytest.mark.parametrize("fmt", ["e4m3", "int8", "bf16", "f32"])
@pytest.mark.parametrize("D", [64, 16])
def test_what_lies_behind_the_last_token_never_counts(fmt, D):
    """NaN scales, NaN codes and infinities behind a row's length, and in tokens that causality hides from a query, change nothing."""
    from speechmix_amd import ops
    B, H, cap, Tq = 2, 2, 100, 3
    c = _filled(B, H, cap, D, fmt, 61)
    q = torch.randn(B, Tq, H, D, device="cuda", generator=_gen(62)).to(torch.bfloat16)
    klen = torch.tensor([41, 70], dtype=torch.int32, device="cuda")
    want, wl = ops.attention_cached(q, c, klen, want_lse=True)
    for b, n in enumerate((41, 70)):
        for t in (c.k, c.v):
            if fmt in ("e4m3", "int8"):
                t[b, :, n:] = 0x7f
            else:
                t[b, :, n:] = float("nan")
                t[b, :, n + 1] = float("inf")
        for s in (c.ks, c.vs):
            if s is not None:
                s[b, :, n:] = float("nan")
                s[b, :, n + 2] = float("inf")
    got, gl = ops.attention_cached(q, c, klen, want_lse=True)
    assert torch.equal(want, got) and torch.equal(wl, gl)
    # the newest token of row 0 turns bad: only its own query sees it
    bad = torch.full((B, 1, H, D), float("nan"), device="cuda")
    bad[1] = float("inf")
    ops.kv_append(c, bad, bad, klen - 1)
    got, gl = ops.attention_cached(q, c, klen, want_lse=True)
    assert torch.equal(want[:, :2], got[:, :2]) and torch.equal(wl[..., :2], gl[..., :2])
    assert torch.isnan(got[0, 2]).all()


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
def test_hidden_tokens_in_items_of_several_tiles(fmt, D):
    """What causality hides from a query may hold NaN and infinities, also where a wave has 32 or 64 rows."""
    from speechmix_amd import ops
    B, Tq, H, cap = 80, 40, 8, 64
    c = _filled(B, H, cap, D, fmt, 67)
    q = torch.randn(B, Tq, H, D, device="cuda", generator=_gen(68)).to(torch.bfloat16)
    klen = torch.full((B,), 60, dtype=torch.int32, device="cuda")
    want, _ = ops.attention_cached(q, c, klen)
    bad = torch.full((B, 1, H, D), float("nan"), device="cuda")
    bad[::2] = float("inf")
    ops.kv_append(c, bad, bad, klen - 3)
    got, _ = ops.attention_cached(q, c, klen)
    assert torch.equal(want[:, :Tq - 3], got[:, :Tq - 3])
    assert not torch.isfinite(got[:, Tq - 3:]).any()


def test_attention_over_the_decoder_own_interleaved_cache():
    """The bf16 cache layout of greedy_decode ([B, L, K | V], heads side by side) is read in place; q and out are strided views."""
    from speechmix_amd import ops
    B, L, H, D = 3, 50, 4, 64
    d = H * D
    buf = torch.randn(B, L, 2 * d, device="cuda", generator=_gen(71)).to(torch.bfloat16)
    kv = buf.view(B, L, 2, H, D)
    c = ops.KVCache(kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2), fmt="bf16")
    qbuf = torch.randn(B, 2, 3 * d, device="cuda", generator=_gen(72)).to(torch.bfloat16)
    q = qbuf.view(B, 2, 3, H, D)[:, :, 1]
    out = torch.full((B, 2, H, 2 * D), 5.0, device="cuda", dtype=torch.bfloat16)
    _check(q, c, [50, 2, 31], out=out[..., :D])
    assert (out[..., D:] == 5).all()


def test_attention_large_scores():
    """Scores of several hundreds: one key takes all; and a common offset of that size."""
    for fmt, dtype in (("e4m3", torch.bfloat16), ("int8", torch.float32), ("bf16", torch.bfloat16)):
        c = _filled(2, 2, 90, 64, fmt, 81, scale=20.0)
        q = (torch.randn(2, 1, 2, 64, device="cuda", generator=_gen(82)) * 10).to(dtype)
        _check(q, c, [90, 47])


def test_attention_in_a_graph_on_a_side_stream_two_at_once():
    """Two captured calls, replayed at once on two streams, with eager work between the replays: each replay equals the eager result."""
    from speechmix_amd import ops
    cs = [_filled(4, 2, 3000, 64, "e4m3", 91 + i) for i in range(2)]
    qs = [torch.randn(4, 1, 2, 64, device="cuda", generator=_gen(95 + i)).to(torch.bfloat16) for i in range(2)]
    kl = [torch.full((4,), 3000 - i, dtype=torch.int32, device="cuda") for i in range(2)]
    want = [ops.attention_cached(qs[i], cs[i], kl[i])[0].clone() for i in range(2)]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, capture_error_mode="thread_local"):
            outs.append(ops.attention_cached(qs[i], cs[i], kl[i])[0])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for rep in range(4):
        for o in outs:
            o.zero_()
        if rep == 2:                                   # new inputs in the same buffers
            for i in range(2):
                qs[i].mul_(0.5)
                kl[i].sub_(17)
            want = [ops.attention_cached(qs[i], cs[i], kl[i])[0].clone() for i in range(2)]
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(outs[i], want[i]) for i in range(2)), rep


# ---- verification ----

def _probs(B, n, V, seed, noise=1.0):
    g = _gen(seed)
    lp = torch.randn(B, n + 1, V, device="cuda", generator=g) * 2
    lq = lp[:, :n] + noise * torch.randn(B, n, V, device="cuda", generator=g)
    p, q = torch.softmax(lp, -1), torch.softmax(lq, -1)
    ids = torch.multinomial(q.reshape(-1, V), 1, generator=g).view(B, n) if n else torch.empty(B, 0, dtype=torch.int64, device="cuda")
    return p, q, ids, torch.rand(B, n + 1, device="cuda", generator=g)


def _verify(p, ids, q, u):
    from speechmix_amd import ops
    acc, tok = ops.verify_draft(p, ids, q, u)
    wa, wt = R.verify(p.cpu().numpy(), ids.cpu().numpy(), q.cpu().numpy() if q is not None else None, u.cpu().numpy() if u is not None else None)
    assert acc.tolist() == wa and tok.tolist() == wt
    return wa, wt


@pytest.mark.parametrize("mode", ["sampled", "picked", "greedy"])
@pytest.mark.parametrize("B,n,V", [(1, 0, 1), (5, 0, 2048), (3, 1, 2047), (4, 4, 2049), (16, 7, 50265), (2, 64, 300), (40, 3, 5), (300, 2, 4097), (1, 4, 32128), (2, 15, 9000), (2, 16, 9001), (2, 3, 250027)])
def test_verify(mode, B, n, V):
    p, q, ids, u = _probs(B, n, V, B + V)
    if mode == "greedy":
        best = p.argmax(-1)[:, :n]
        ids = torch.where(torch.rand(B, n, device="cuda", generator=_gen(7)) < 0.7, best, ids)
    _verify(p, ids, q if mode == "sampled" else None, None if mode == "greedy" else u)


def test_verify_borders():
    """Uniforms of 0 and next to 1, ids outside the vocabulary, a draft equal to the target, a target that excludes the draft, zero mass."""
    from speechmix_amd import ops
    B, n, V = 8, 3, 3001
    p, q, ids, u = _probs(B, n, V, 5)
    u[0] = 0.0
    u[1] = 1.0 - 2.0 ** -24
    ids[2, 0], ids[3, 1], ids[4, 2] = -1, V, 1 << 40
    p[5, :n] = q[5]                                    # every draft is as likely: all accepted
    p[6, 0, ids[6, 0]] = 0.0                           # impossible under the target: rejected at once
    p[7, 0] = 0.5 * q[7, 0]                            # p < q everywhere: rejected or not, what is left has no mass but p itself
    u[7, 0] = 0.75
    acc, _ = _verify(p, ids, q, u)
    assert acc[5] == n and acc[6] == 0 and acc[7] == 0 and acc[2] == 0
    acc, tok = _verify(p, ids, None, u)
    assert acc[2] == 0
    # rows of zeros: token 0, nothing out of range
    z = torch.zeros(2, 2, 77, device="cuda")
    a, t = ops.verify_draft(z, torch.zeros(2, 1, dtype=torch.int64, device="cuda"), None, torch.rand(2, 2, device="cuda"))
    assert a.tolist() == [0, 0] and t.tolist() == [0, 0]
    # a last weight of zero and a uniform that rounds up to the total: the last index with mass
    w = torch.zeros(1, 1, 5000, device="cuda")
    w[0, 0, 10] = w[0, 0, 4000] = 0.5
    a, t = ops.verify_draft(w, torch.zeros(1, 0, dtype=torch.int64, device="cuda"), None, torch.full((1, 1), 1.0, device="cuda"))
    assert t.item() == 4000


def test_verify_greedy_ties_logits_and_strides():
    from speechmix_amd import ops
    B, n, V = 3, 2, 5000
    buf = torch.randn(B, n + 1, V + 56, device="cuda", generator=_gen(9)) - 50
    t = buf[..., :V]
    t[..., [4990, 17, 2500]] = 1.0                     # ties: the lowest index
    buf[..., V:] = 1e9                                 # the padding of the rows does not count
    ids = torch.tensor([[17, 17], [17, 2500], [4990, 17]], device="cuda")
    a, tok = ops.verify_draft(t, ids)
    assert a.tolist() == [2, 1, 0] and tok.tolist() == [17, 17, 17]
    t[0, 0] = float("-inf")
    t[1, 0] = float("nan")
    a, tok = ops.verify_draft(t, ids)
    assert a.tolist()[:2] == [0, 0] and tok.tolist()[:2] == [0, 0]


def test_verify_greedy_ties_over_workgroups():
    """The same where several workgroups share the rows: ties far apart, a row without a number, a row of the lowest values."""
    from speechmix_amd import ops
    V = 90001
    t = torch.randn(3, 3, V, device="cuda", generator=_gen(10)) - 50
    t[..., [90000, 45001, 30007]] = 1.0
    ids = torch.tensor([[30007, 30007], [30007, 90000], [45001, 30007]], device="cuda")
    a, tok = ops.verify_draft(t, ids)
    assert a.tolist() == [2, 1, 0] and tok.tolist() == [30007, 30007, 30007]
    t[0, 0] = float("-inf")
    t[1, 0] = float("nan")
    t[2, 0] = torch.finfo(torch.float32).min
    t[2, 0, 70000] = -1e38
    a, tok = ops.verify_draft(t, ids)
    assert a.tolist() == [0, 0, 0] and tok.tolist() == [0, 0, 70000]


def test_verify_distribution():
    """What comes out is distributed as the target whatever the draft: 60 000 draws of a five-token vocabulary, each frequency within five
    standard deviations."""
    from speechmix_amd import ops
    V, N = 5, 60000
    p = torch.tensor([0.05, 0.3, 0.1, 0.35, 0.2], device="cuda")
    q = torch.tensor([0.5, 0.1, 0.2, 0.1, 0.1], device="cuda")
    g = _gen(17)
    ids = torch.multinomial(q, N, replacement=True, generator=g).view(N, 1)
    acc, tok = ops.verify_draft(p.expand(N, 2, V), ids, q.expand(N, 1, V), torch.rand(N, 2, device="cuda", generator=g))
    first = torch.where(acc == 1, ids[:, 0], tok)
    freq = torch.bincount(first, minlength=V).double() / N
    sd = (p.double() * (1 - p.double()) / N).sqrt()
    assert ((freq - p.double()).abs() <= 5 * sd).all()


def test_refusals_on_gpu_tensors():
    from speechmix_amd import ops
    c = ops.KVCache.empty(2, 4, 8, 64, "e4m3", "cuda")
    x = torch.zeros(2, 1, 4, 64, device="cuda")
    i64 = torch.zeros(2, dtype=torch.int64, device="cuda")
    bad = [
        lambda: ops.KVCache(c.k, c.v, fmt="e4m3"), lambda: ops.KVCache(c.k, c.v, c.ks, c.vs, fmt="bf16"), lambda: ops.KVCache(c.k, c.v[:, :2], c.ks, c.vs),
        lambda: ops.KVCache(c.k[:, :1].expand(2, 4, 8, 64), c.v[:, :1].expand(2, 4, 8, 64), c.ks, c.vs), lambda: ops.KVCache(c.k, c.v, c.ks.half(), c.vs.half()),
        lambda: ops.kv_append(c, x[:, :, :3], x[:, :, :3]), lambda: ops.kv_append(c, x.half(), x.half()), lambda: ops.kv_append(c, x, x.bfloat16()),
        lambda: ops.kv_append(c, x, x, i64), lambda: ops.kv_append(c, x, x, 1 << 40), lambda: ops.kv_append(c, x.transpose(2, 3).contiguous().transpose(2, 3), x),
        lambda: ops.kv_read(c, 0, x[:, :, :1].expand(2, 1, 4, 64), x), lambda: ops.kv_append(c, x.cpu(), x.cpu()),
        lambda: ops.attention_cached(x[..., :32], c), lambda: ops.attention_cached(x[:1], c), lambda: ops.attention_cached(x[:, :, :3], c),
        lambda: ops.attention_cached(x, c, i64), lambda: ops.attention_cached(x, c, torch.zeros(3, dtype=torch.int32, device="cuda")),
        lambda: ops.attention_cached(x, None), lambda: ops.attention_cached(x, c, out=x.bfloat16()), lambda: ops.attention_cached(x, c, rel_bias=x),
        lambda: ops.attention_cached(x, c, prefix=ops.KVCache.empty(1, 4, 8, 64, "int8", "cuda")),
        lambda: ops.attention_cached(x, c, prefix=ops.KVCache.empty(3, 4, 8, 64, "e4m3", "cuda")), lambda: ops.attention_cached(x[:, :0], c),
        lambda: ops.attention_cached(x.cpu(), c), lambda: ops.attention_cached(x, c, prefix_len=torch.zeros(1, dtype=torch.int32, device="cuda")),
        lambda: ops.verify_draft(x[0].half(), i64[:, None]), lambda: ops.verify_draft(x[:, 0], i64[:, None]), lambda: ops.verify_draft(x[:, 0], i64[:, None].int()),
        lambda: ops.verify_draft(torch.zeros(2, 2, 9, device="cuda"), i64[:, None], torch.zeros(2, 1, 9, device="cuda")),
        lambda: ops.verify_draft(torch.zeros(2, 2, 9, device="cuda"), i64[:, None], None, torch.zeros(2, 1, device="cuda")),
        lambda: ops.verify_draft(torch.zeros(2, 66, 9, device="cuda"), torch.zeros(2, 65, dtype=torch.int64, device="cuda")),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            raise AssertionError(f"call {i} was not refused")
