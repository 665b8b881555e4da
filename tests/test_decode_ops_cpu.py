"""CPU checks of the decoding operators' boundary: what the C entries and the Python wrappers refuse, and the struct mirrors.  No kernel runs."""
import ctypes as C

import pytest
import torch

from speechmix_amd import _lib as L
from tests import decode_ref as R


@pytest.fixture(scope="module")
def lib():
    import os
    if not os.path.exists(L.LIB_PATH):
        import __graft_entry__ as g
        g.build()
    l = L.lib()
    l.smx_attention_cached_ws_bytes.restype = C.c_longlong
    l.smx_verify_draft_ws_bytes.restype = C.c_longlong
    return l


def _cache(B=2, H=4, cap=16, D=64, fmt=L.KV_E4M3):
    d = L.KVCacheDesc()
    d.k, d.v = 4096, 8192
    if fmt <= L.KV_INT8:
        d.ks, d.vs = 16384, 32768
    d.bs, d.hs, d.ts = H * cap * D, cap * D, D
    d.sbs, d.shs = H * cap, cap
    d.B, d.H, d.cap, d.D, d.fmt = B, H, cap, D, fmt
    return d


def test_struct_mirrors(lib):
    for name, st in (("SmxKVCache", L.KVCacheDesc), ("SmxKVRowsParams", L.KVRowsParams), ("SmxCachedAttnParams", L.CachedAttnParams),
                     ("SmxVerifyParams", L.VerifyParams)):
        assert getattr(lib, "smx_sizeof_" + name)() == C.sizeof(st), name


@pytest.mark.parametrize("change", [dict(k=0), dict(v=0), dict(ks=0), dict(B=0), dict(H=-1), dict(cap=0), dict(D=0), dict(D=63), dict(D=264), dict(fmt=4),
                                    dict(fmt=-1), dict(fmt=L.KV_BF16), dict(k=4097), dict(bs=4100), dict(hs=4), dict(ts=65)])
def test_a_cache_the_kernels_cannot_address_is_refused(lib, change):
    c = _cache()
    for k, v in change.items():
        setattr(c, k, v)
    rows = L.KVRowsParams(c=c, k=4096, v=4096, k_bs=256, k_ts=256, k_hs=64, v_bs=256, v_ts=256, v_hs=64, T=1)
    assert lib.smx_kv_append(C.byref(rows), 1, None) == -22
    assert lib.smx_kv_read(C.byref(rows), 1, None) == -22
    p = L.CachedAttnParams(q=4096, o=4096, own=c, B=2, Tq=1, H=4, scale=1.0)
    assert lib.smx_attention_cached(C.byref(p), 1, None) == -22
    if change.get("k", 1) != 0:                        # (k == NULL: no prefix)
        p = L.CachedAttnParams(q=4096, o=4096, own=_cache(), pre=c, B=2, Tq=1, H=4, scale=1.0)
        assert lib.smx_attention_cached(C.byref(p), 1, None) == -22


@pytest.mark.parametrize("change", [dict(k=None), dict(k=4104), dict(k_bs=4), dict(v_hs=3), dict(T=-1)])
def test_rows_refused(lib, change):
    rows = L.KVRowsParams(c=_cache(), k=4096, v=4096, k_bs=256, k_ts=256, k_hs=64, v_bs=256, v_ts=256, v_hs=64, T=1)
    for k, v in change.items():
        setattr(rows, k, v)
    assert lib.smx_kv_append(C.byref(rows), 1, None) == -22
    rows.T = 1 if "T" not in change else -1
    assert lib.smx_kv_read(C.byref(rows), 1, None) == -22
    assert lib.smx_kv_append(C.byref(L.KVRowsParams(c=_cache(), k=4096, v=4096, T=1)), 2, None) == -22        # unknown dtype


@pytest.mark.parametrize("change", [dict(q=None), dict(o=None), dict(B=0), dict(B=3), dict(Tq=0), dict(H=6), dict(H=0), dict(q=4100), dict(q_hs=4),
                                    dict(rel_bias=4096, nrel=0), dict(pre=_cache(B=3)), dict(pre=_cache(H=2)), dict(pre=_cache(D=128)),
                                    dict(pre=_cache(fmt=L.KV_INT8)), dict(own=_cache(B=4))])
def test_attention_refused(lib, change):
    p = L.CachedAttnParams(q=4096, o=4096, own=_cache(), B=2, Tq=1, H=4, scale=1.0)
    for k, v in change.items():
        setattr(p, k, v)
    assert lib.smx_attention_cached_ws_bytes(C.byref(p), 1) == -22
    assert lib.smx_attention_cached(C.byref(p), 1, None) == -22
    p = L.CachedAttnParams(q=4096, o=4096, B=2, Tq=1, H=4, scale=1.0)
    assert lib.smx_attention_cached(C.byref(p), 1, None) == -22               # neither a cache nor a prefix
    p = L.CachedAttnParams(q=4096, o=4096, own=_cache(), B=2, Tq=1, H=4, scale=1.0)
    assert lib.smx_attention_cached(C.byref(p), 3, None) == -22


def test_attention_refuses_a_workspace_that_is_too_small(lib):
    p = L.CachedAttnParams(q=4096, o=4096, own=_cache(B=1, H=1, cap=1 << 20), B=1, Tq=1, H=1, scale=1.0)
    n = lib.smx_attention_cached_ws_bytes(C.byref(p), 1)
    if n:                                              # (this call splits its keys)
        p.ws, p.ws_bytes = 4096, n - 1
        assert lib.smx_attention_cached(C.byref(p), 1, None) == -22
        p.ws, p.ws_bytes = 4104, n
        assert lib.smx_attention_cached(C.byref(p), 1, None) == -22
        p.ws = None
        assert lib.smx_attention_cached(C.byref(p), 1, None) == -22


@pytest.mark.parametrize("change", [dict(target=None), dict(accepted=None), dict(token=None), dict(B=0), dict(B=65536), dict(n=-1), dict(n=65), dict(V=0),
                                    dict(ids=None), dict(u=None, draft=4096), dict(ws=None), dict(ws=4097), dict(ws_bytes=8),
                                    dict(u=None, ws=None), dict(u=None, ws_bytes=8)])
def test_verify_refused(lib, change):
    # (two rows of 250 027: several workgroups a row, which need the workspace; so does the greedy form)
    p = L.VerifyParams(target=4096, u=4096, ids=4096, accepted=4096, token=4096, ws=4096, ws_bytes=1 << 20, B=2, n=3, V=250027)
    for k, v in change.items():
        setattr(p, k, v)
    assert lib.smx_verify_draft(C.byref(p), None) == -22


def test_wrappers_refuse_cpu_tensors():
    from speechmix_amd import ops
    z = torch.zeros(1, 1, 8, 64)
    for call in (lambda: ops.KVCache(z, z, fmt="f32"), lambda: ops.verify_draft(torch.zeros(1, 1, 5), torch.zeros(1, 0, dtype=torch.int64)),
                 lambda: ops.attention_cached(torch.zeros(1, 1, 1, 64), None)):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(RuntimeError, match="format"):
        ops.KVCache(z, z, fmt="fp4")


def test_reference_quantisation_against_torch():
    """The oracle's own rounding agrees with torch's conversion to float8_e4m3fn on every representable border."""
    v = torch.tensor(R.E4M3_VALUES)
    mids = (v[1:] + v[:-1]) / 2
    x = torch.cat([v, mids, mids * (1 + 2.0 ** -20), mids * (1 - 2.0 ** -20), torch.tensor([448.0])]).float()
    code, s = R.quantise(x[None], "e4m3")
    assert s.item() == 1.0
    assert torch.equal(code[0].view(torch.uint8), x.to(torch.float8_e4m3fn).view(torch.uint8))
    assert torch.equal(R.values(code, s, "e4m3")[0], x.to(torch.float8_e4m3fn).double())


def test_a_split_call_needs_its_workspace(lib):
    """A row of 2^20 keys is split in every format that is split at all: it has a workspace, and none, a short or an unaligned one is refused."""
    for fmt in (L.KV_E4M3, L.KV_INT8, L.KV_BF16):
        p = L.CachedAttnParams(q=4096, o=4096, own=_cache(B=1, H=1, cap=1 << 20, fmt=fmt), B=1, Tq=1, H=1, scale=1.0)
        n = lib.smx_attention_cached_ws_bytes(C.byref(p), 1)
        assert n >= 2 * (64 + 2) * 4                   # at least two partial rows of 64 numbers, a maximum and a sum
        for ws, size in ((4096, n - 1), (4104, n), (None, n), (4096, 0)):
            p.ws, p.ws_bytes = ws, size
            assert lib.smx_attention_cached(C.byref(p), 1, None) == -22
