"""Numbers at the edges of their range in the decoding operators: rows that are NaN, values near the largest and the smallest of the type."""
import pytest
import torch

from tests import decode_ref as R

pytestmark = pytest.mark.gpu
FMTS = ["e4m3", "int8", "bf16", "f32"]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(B, H, cap, D, fmt, seed):
    from speechmix_amd import ops
    g = _gen(seed)
    c = ops.KVCache.empty(B, H, cap, D, fmt, "cuda")
    ops.kv_append(c, *(torch.randn(B, cap, H, D, device="cuda", generator=g) for _ in range(2)), 0)
    return c


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128, 32])
# one workgroup a row; heads of 64 by eight waves; keys split and joined; a wave a row; behind prefixes, also with one result of each part; prefixes only
@pytest.mark.parametrize("B,H,cap,P", [(6, 2, 40, 0), (6, 2, 300, 0), (6, 2, 5000, 0), (96, 6, 47, 0), (6, 2, 40, 30), (6, 2, 600, 700), (96, 6, 47, 20), (6, 2, 0, 700)])
def test_a_row_that_is_nan_has_no_log_sum_exp(fmt, dtype, D, B, H, cap, P):
    """A query of NaN, and rows whose only token is stored as not finite: output and log-sum-exp are NaN, and no other row notices."""
    from speechmix_amd import ops
    c = _rows(B, H, cap, D, fmt, 1) if cap else None
    pre = _rows(B // 3, H, P, D, fmt, 2) if P else None
    q = torch.randn(B, 1, H, D, device="cuda", generator=_gen(3)).to(dtype)
    klen = torch.tensor([max(cap // 2, 1), 1, 1, 3, 0, 7] * (B // 6), dtype=torch.int32, device="cuda") if cap else None
    plen = torch.tensor([0, 5] * (B // 6), dtype=torch.int32, device="cuda") if P else None
    if not cap:
        plen = torch.tensor([P, P // 2] * (B // 6), dtype=torch.int32, device="cuda")
    want, wl = ops.attention_cached(q, c, klen, prefix=pre, prefix_len=plen, want_lse=True)
    assert torch.isfinite(want).all()
    q[0::6] = float("nan")
    nan = [0]
    if cap:
        bad = torch.zeros(B, 1, H, D, device="cuda")
        bad[1::6], bad[2::6] = float("nan"), float("inf")
        start = torch.full((B,), cap, dtype=torch.int32, device="cuda")              # (the other rows: dropped)
        start[1::6] = start[2::6] = 0
        ops.kv_append(c, bad, bad, start)
        nan = [0, 1, 2]
    got, gl = ops.attention_cached(q, c, klen, prefix=pre, prefix_len=plen, want_lse=True)
    for i in range(6):
        if i in nan:
            assert torch.isnan(got[i::6]).all() and torch.isnan(gl[i::6]).all(), i
        else:
            assert torch.equal(got[i::6], want[i::6]) and torch.equal(gl[i::6], wl[i::6]), i


def _values_case(fmt, dtype, D, B, H, cap, P, mag, seed=11):
    """Caches whose later half has keys of one direction that a row's query gives scores some 15 log-2 units above the first half's, and values of
    magnitude `mag`."""
    from speechmix_amd import ops
    g = _gen(seed)
    q = torch.randn(B, 1, H, D, device="cuda", generator=g).to(dtype)
    out = [q]
    for n, N in ((cap, B), (P, B // 3)):
        if not n:
            out.append(None)
            continue
        c = ops.KVCache.empty(N, H, n, D, fmt, "cuda")
        k = torch.randn(N, n, H, D, device="cuda", generator=g) * 0.02
        qq = q[:, 0].float()[::B // N]                                             # (a prefix: its first row's query)
        k[:, n // 2:] += (10.4 * D ** 0.5 * qq / (qq * qq).sum(-1, keepdim=True))[:, None]
        ops.kv_append(c, k, torch.randn(N, n, H, D, device="cuda", generator=g) * mag, 0)
        out.append(c)
    return out


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128, 32])
@pytest.mark.parametrize("B,H,cap,P", [(6, 2, 260, 0), (3, 1, 600, 0), (6, 2, 5000, 0), (96, 6, 250, 0), (6, 2, 270, 300), (96, 6, 100, 200), (6, 2, 0, 700)])
@pytest.mark.parametrize("mag", [1e36, 1e-36, 1e-18])
def test_values_near_the_ends_of_the_range(fmt, dtype, D, B, H, cap, P, mag):
    """Finite caches give finite, right outputs whatever the values' magnitude: probabilities far above the reference times large values do not
    overflow, small ones keep their bits.

    Beside attention_bounds (which is relative) the smallest steps count: fp32 numbers below 2^-126 step by 2^-149, so each of the products and sums
    of a row - one per key in the general kernel, one per split or wave where results meet - may be off by half of that; a bf16 output below
    2^-126 steps by 2^-133."""
    from speechmix_amd import ops
    q, c, pre = _values_case(fmt, dtype, D, B, H, cap, P, mag)
    klen = torch.tensor(([cap, cap - 1, cap // 2 + 40] * (B // 3)), dtype=torch.int32, device="cuda") if cap else None
    plen = torch.tensor([P, P - 3] * (B // 6), dtype=torch.int32, device="cuda") if P else None
    o, lse = ops.attention_cached(q, c, klen, prefix=pre, prefix_len=plen, want_lse=True)
    rows = slice(0, 6) if B > 6 else slice(0, B)
    K, V, PK, PV = None, None, None, None
    if cap:
        K, V = (R.values(t[rows], s[rows] if s is not None else None, fmt) for t, s in ((c.k, c.ks), (c.v, c.vs)))
    if P:
        PK, PV = (R.values(t[:2], s[:2] if s is not None else None, fmt) for t, s in ((pre.k, pre.ks), (pre.v, pre.vs)))
    ref = R.attention(q[rows], K, V, klen[rows].tolist() if cap else None, plen[:2].tolist() if P else None, PK, PV, 3, True, D ** -0.5, None)
    tol_o, tol_l = R.attention_bounds(*ref, D, dtype)
    tol_o = tol_o + (ref[4] + 64).transpose(1, 2)[..., None] * 2.0 ** -150 + (2.0 ** -134 if dtype == torch.bfloat16 else 0.0)
    assert torch.isfinite(o).all() and torch.isfinite(lse).all()
    err = (o[rows].double().cpu() - ref[0]).abs()
    assert (err <= tol_o).all(), ((err - tol_o).max(), (err / tol_o).max())
    assert ((lse[rows].double().cpu() - ref[1]).abs() <= tol_l).all()


@pytest.mark.parametrize("fmt", FMTS)
def test_large_and_small_values_side_by_side(fmt):
    """Head elements that cancel exactly beside small ones, tokens of huge values that nothing looks at, values of zero."""
    from speechmix_amd import ops
    c = ops.KVCache.empty(3, 1, 64, 64, fmt, "cuda")
    k = torch.zeros(3, 64, 1, 64, device="cuda")
    v = torch.randn(3, 64, 1, 64, device="cuda", generator=_gen(5)) * 1e-13
    v[0, ::2, 0, 0], v[0, 1::2, 0, 0] = 1e20, -1e20              # (all scores alike: the first element's sum is zero)
    k[1, 7, 0] = -1000.0                                         # row 1: a token of no weight ...
    v[1, 7] = 3e38                                               # ... and huge values
    v[2] = 0
    ops.kv_append(c, k, v, 0)
    q = torch.ones(3, 1, 1, 64, device="cuda")
    o, lse = ops.attention_cached(q, c, want_lse=True)
    ref = R.attention(q, R.values(c.k, c.ks, fmt), R.values(c.v, c.vs, fmt), [64] * 3, None, None, None, 1, True, 0.125, None)
    tol_o, _ = R.attention_bounds(*ref, 64, torch.float32)
    assert ((o.double().cpu() - ref[0]).abs() <= tol_o).all()
    assert (o[2] == 0).all() and torch.isfinite(lse).all()


@pytest.mark.parametrize("fmt", FMTS)
def test_large_values_under_a_bias_that_masks(fmt):
    """Every distance biased by the type's lowest value: the scores vanish beside it and all keys count alike, also where only some of the blocks
    hold large values.  The mean of 300 values: 300 products and sums of the cache's own numbers, and a probability of 1 has no rounding."""
    from speechmix_amd import ops
    c = ops.KVCache.empty(1, 2, 300, 64, fmt, "cuda")
    x = torch.randn(1, 300, 2, 64, device="cuda", generator=_gen(6))
    v = x.clone()
    v[:, 200:230] *= 1e35
    ops.kv_append(c, x, v, 0)
    low = torch.finfo(torch.float32).min
    o, lse = ops.attention_cached(x[:, :1].clone(), c, rel_bias=torch.full((2, 3), low, device="cuda"), want_lse=True)
    V = R.values(c.v, c.vs, fmt)[0]
    tol = (300 + 64) * 2.0 ** -24 * V.abs().mean(1) + 2.0 ** -24 * V.mean(1).abs()
    assert ((o[0, 0].double().cpu() - V.mean(1)).abs() <= tol).all() and (lse == low).all()


@pytest.mark.parametrize("fmt", ["bf16", "f32"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128, 32])
@pytest.mark.parametrize("B,H,cap,P,Tq,causal", [(3, 2, 1, 0, 1, False), (3, 2, 40, 0, 1, False), (3, 2, 300, 0, 1, True), (3, 2, 5000, 0, 1, True), (3, 2, 40, 0, 4, True), (3, 2, 40, 0, 33, False),
                                                 (93, 6, 47, 0, 1, True), (6, 2, 40, 30, 2, True), (96, 6, 47, 20, 1, True), (6, 2, 0, 700, 1, False), (96, 8, 0, 60, 1, False)])
def test_visible_values_that_are_not_finite(fmt, dtype, D, B, H, cap, P, Tq, causal):
    """Caches that hold the values themselves may hold infinities and NaN: where a query sees one, that element of its output - and no other - is
    the infinity or NaN that a positive probability makes of it."""
    from speechmix_amd import ops
    q = torch.randn(B, Tq, H, D, device="cuda", generator=_gen(3)).to(dtype)
    kl = torch.tensor([max(cap - i, 1) for i in range(3)] * (B // 3), dtype=torch.int32, device="cuda") if cap else None
    c = _rows(B, H, cap, D, fmt, 1) if cap else None
    pre = _rows(B // 3, H, P, D, fmt, 2) if P else None
    want, wl = ops.attention_cached(q, c, kl, causal=causal, prefix=pre, want_lse=True)
    main, other = (c, pre) if cap else (pre, None)
    main.v[0, 0, 0, 3], main.v[0, 0, 0, 4], main.v[0, 1, 0, 5] = float("inf"), -float("inf"), float("nan")
    if main.cap > 6:
        main.v[0, 0, 6, 3], main.v[0, 0, 5, 4] = float("inf"), float("inf")               # inf twice, inf and -inf
    if other is not None:
        other.v[0, 1, 7, 9] = float("inf")
    got, gl = ops.attention_cached(q, c, kl, causal=causal, prefix=pre, want_lse=True)
    assert torch.equal(gl, wl)
    expect = want.clone().float()
    for r in range(1 if cap else 3):                       # (a prefix: the rows of its first group)
        for t in range(Tq):
            seen = main.cap if not cap else int(kl[0]) if not causal else int(kl[0]) - Tq + t + 1
            if seen > 0:
                expect[r, t, 0, 3], expect[r, t, 0, 4], expect[r, t, 1, 5] = float("inf"), -float("inf") if seen <= 5 else float("nan"), float("nan")
    if other is not None:
        expect[:3, :, 1, 9] = float("inf")
    same = torch.isfinite(expect)
    assert torch.equal(got.float().nan_to_num(nan=7e30, posinf=8e30, neginf=9e30)[~same], expect.nan_to_num(nan=7e30, posinf=8e30, neginf=9e30)[~same])
    assert torch.equal(got[same], want[same])
