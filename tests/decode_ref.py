"""Plain 64-bit references of the decoding operators (CPU, numpy / torch float64), and the error bounds the tests hold them to."""
import math

import numpy as np
import torch


def quantise(x, fmt):
    """x fp32 [..., D] -> (codes uint8, scales fp32), from the definition: the nearest code, ties to the even one."""
    x = x.detach().cpu().numpy().astype(np.float32)
    finite = np.isfinite(x).all(-1)
    a = np.abs(np.where(finite[..., None], x, 0)).max(-1)
    if fmt == "e4m3":
        m, e = np.frexp(a)                                       # 448 = 0.875 * 2^9
        s = np.ldexp(np.float32(1), np.maximum(np.where(m <= 0.875, e - 9, e - 8), -126)).astype(np.float32)
        s = np.where(a > 0, s, np.float32(1))
        vals = np.array(E4M3_VALUES)                             # codes 0 .. 126
        y = np.where(finite[..., None], x, 0).astype(np.float64) / s[..., None].astype(np.float64)
        mag = np.abs(y)
        hi = np.clip(np.searchsorted(vals, mag), 1, 126)
        lo = hi - 1
        dl, dh = mag - vals[lo], vals[hi] - mag
        code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi).astype(np.uint8)
        code |= np.where(np.signbit(y), 128, 0).astype(np.uint8)
    else:
        s = np.maximum(a / np.float32(127), np.float32(2.0 ** -126)).astype(np.float32)
        s = np.where(a > 0, s, np.float32(1))
        y = np.where(finite[..., None], x, 0).astype(np.float32) / s[..., None]
        code = np.clip(np.rint(y), -127, 127).astype(np.int8).view(np.uint8)
    s = np.where(finite, s, np.float32("nan"))
    return torch.from_numpy(code), torch.from_numpy(s.astype(np.float32))


E4M3_VALUES = [(c & 7) * 2.0 ** -9 if c < 8 else (8 + (c & 7)) * 2.0 ** ((c >> 3) - 10) for c in range(127)]


def values(code, scale, fmt):
    """fp64 values of a cache tensor (CPU)."""
    if fmt in ("bf16", "f32"):
        return code.detach().cpu().double()
    c = code.detach().cpu().view(torch.uint8)
    if fmt == "int8":
        v = c.view(torch.int8).double()
    else:
        table = torch.tensor(E4M3_VALUES + [float("nan")] + [-x for x in E4M3_VALUES] + [float("nan")], dtype=torch.float64)
        v = table[c.long()]
    return v * scale.detach().cpu().double()[..., None]


def attention(q, K, V, klen, plen, PK, PV, R, causal, scale, rel):
    """q [B, Tq, H, D]; K, V [B, Hkv, cap, D] or None; PK, PV [groups, Hkv, P, D] or None (all fp64, CPU).  klen, plen: lists.
    -> out, lse, and for the bounds: mean |v| under the probabilities, the largest sum of |q k| behind a row's scores, the number of keys, the largest |v|."""
    q = q.detach().cpu().double()
    B, Tq, H, D = q.shape
    Hkv = (K if K is not None else PK).shape[1]
    G = H // Hkv
    out = torch.zeros(B, Tq, H, D, dtype=torch.float64)
    mag = torch.zeros_like(out)
    lse = torch.full((B, H, Tq), -math.inf, dtype=torch.float64)
    sabs = torch.zeros(B, H, Tq, dtype=torch.float64)
    nk = torch.zeros(B, H, Tq, dtype=torch.float64)
    vmax = torch.zeros(B, H, Tq, dtype=torch.float64)
    for b in range(B):
        P = plen[b // R] if PK is not None else 0
        L = klen[b] if K is not None else 0
        for t in range(Tq):
            vis = L if not causal else max(0, min(L, L - Tq + t + 1))
            qpos = P + L - Tq + t
            pos = torch.cat([torch.arange(P), P + torch.arange(vis)])
            if pos.numel() == 0:
                continue
            for h in range(H):
                kk, vv = [], []
                if P:
                    kk.append(PK[b // R, h // G, :P])
                    vv.append(PV[b // R, h // G, :P])
                if vis:
                    kk.append(K[b, h // G, :vis])
                    vv.append(V[b, h // G, :vis])
                kk, vv = torch.cat(kk), torch.cat(vv)
                s = (kk @ q[b, t, h]) * scale
                bound = (kk.abs() @ q[b, t, h].abs()) * abs(scale)
                if rel is not None:
                    r = rel.detach().cpu().double()[h, (qpos - pos).clamp(0, rel.shape[1] - 1)]
                    s, bound = s + r, bound + r.abs()
                z = torch.logsumexp(s, 0)
                pr = torch.exp(s - z)
                out[b, t, h] = pr @ vv
                mag[b, t, h] = pr @ vv.abs()
                lse[b, h, t], sabs[b, h, t], nk[b, h, t], vmax[b, h, t] = z, bound.max(), pos.numel(), vv.abs().max()
    return out, lse, mag, sabs, nk, vmax


def attention_bounds(out, lse, mag, sabs, nk, vmax, D, dtype):
    """Largest error a 32-bit evaluation may make.  A score: D products and sums, the scales and the bias, each half an ulp of numbers up to
    sabs, and the exponent's argument another rounding: es = (D + 8) 2^-24 sabs.  A probability carries es twice (its own, the sum's) and
    the sum over n keys n + 64 roundings (64: joining splits).  bf16 outputs round once (2^-8 of the value) and hold probabilities as the sum
    of two bf16 numbers (2^-16); fp32 outputs as the sum of three (2^-22).  A probability below 2^-126, the smallest normal number, may count as nothing: n 2^-126 of the
    largest |v|."""
    es = (D + 8) * 2.0 ** -24 * sabs
    common = 2 * es + (nk + 64) * 2.0 ** -24
    split, rnd = (2.0 ** -16, 2.0 ** -8) if dtype == torch.bfloat16 else (2.0 ** -22, 2.0 ** -24)
    tol_o = out.abs() * rnd + mag * (common + split).transpose(1, 2)[..., None] + (nk * 2.0 ** -126 * vmax).transpose(1, 2)[..., None]
    tol_l = common + lse.abs().nan_to_num(posinf=0.0) * 2.0 ** -23
    return tol_o, tol_l


def verify(p, ids, q, u):
    """p [B, n + 1, V], q [B, n, V] or None, u [B, n + 1] or None (numpy); -> accepted, token lists."""
    acc, tok = [], []
    B, n1, V = p.shape
    for b in range(B):
        k, w = 0, None
        while k < n1 - 1:
            x = int(ids[b, k])
            if x < 0 or x >= V:
                break
            if u is None:
                if int(np.argmax(p[b, k])) != x:
                    break
            else:
                qx = float(q[b, k, x]) if q is not None else 1.0
                if not float(u[b, k]) * qx < float(p[b, k, x]):
                    if q is not None:
                        w = np.maximum(p[b, k].astype(np.float64) - q[b, k].astype(np.float64), 0)
                    else:
                        w = p[b, k].astype(np.float64)
                        w[x] = 0
                    break
            k += 1
        acc.append(k)
        if u is None:
            tok.append(int(np.argmax(p[b, k])))
            continue
        if w is None or not w.sum() > 0:
            w = p[b, k].astype(np.float64)
        cum = np.cumsum(w)
        hit = np.nonzero(cum > float(u[b, n1 - 1]) * cum[-1])[0]
        tok.append(int(hit[0]) if len(hit) else (int(np.nonzero(w > 0)[0][-1]) if (w > 0).any() else 0))
    return acc, tok
