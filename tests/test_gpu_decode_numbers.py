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
