// Matrix-core form of the cached attention (head widths 64 and 128; e4m3, int8 and bf16 caches; bf16 and fp32 queries).
//
// The rows of one KV head - Tq x G of a batch entry's own keys, R x Tq x G of a prefix - are the columns of S^T = K Q^T tiles (16 keys x 16 rows),
// so a lane owns one row (i = lane & 15) and four keys (4 g + r, g = lane >> 4) of each tile, and the exponentiated tile already is the
// B operand of O^T = V^T P^T: no pass through LDS.  8-bit codes are exact in bf16, so the products are exact up to the 32-bit accumulation; fp32
// queries are held as three bf16 numbers (24 bits) and probabilities as two (bf16 queries) or three: one rounding to bf16 would cost as much
// as the rounding of the output.
//   K operand: a lane's 16 contiguous bytes of one key ARE eight k-indices of two (one for bf16) products; Q is loaded in the same order.
//   V operand: a lane takes DPL = D / 16 neighbouring elements of each of its eight keys; one byte permute per register pairs two keys.
// Softmax: every wave keeps its own reference m per row and moves it only when a score passes m + 16 (a wave-wide test): probabilities stay
// below 2^24, and most blocks need no rescaling and no cross-lane maximum.  Four waves take every fourth block of BK keys, and meet in LDS;
// long caches are split over workgroups as well, whose unnormalised (m, l, O) a second kernel joins in a fixed order.
#pragma once
#include "kv_common.h"

#define CA_WAVES 4
#define CA_LOG2E 1.44269504088896340736f
#define CA_SLACK 16.f             // a score may pass the reference by this much (natural units) before it moves

struct CaPlan {
    int G, Hkv, R;                // query heads per KV head; rows per prefix
    int mbo, mbp;                 // blocks of 16 * MT rows per (entry, KV head): own, prefix
    int nso, nsp;                 // key splits: own, prefix
    int items_p;                  // workgroups of the prefix part (they come first)
    int join;                     // partial results to po / pml instead of the output
    float *po, *pml;              // [item][16 MT][D], [item][16 MT][2]
};

template <int FMT> struct CaFmt;
template <> struct CaFmt<SMX_KV_E4M3> { enum { ES = 1 }; };
template <> struct CaFmt<SMX_KV_INT8> { enum { ES = 1 }; };
template <> struct CaFmt<SMX_KV_BF16> { enum { ES = 2 }; };

struct __attribute__((packed, aligned(4))) CaF4 { float v[4]; };

__device__ __forceinline__ f32x4_t ca_mfma(const unsigned a[4], const unsigned b[4], f32x4_t c) {
    union { unsigned u[4]; bf16x8_t v; } x, y;
#pragma unroll
    for (int e = 0; e < 4; ++e) { x.u[e] = a[e]; y.u[e] = b[e]; }
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.v, y.v, c, 0, 0, 0);
}
// four codes -> two registers of bf16 pairs
template <int FMT>
__device__ __forceinline__ void ca_cvt4(unsigned u, unsigned& lo, unsigned& hi) {
    if (FMT == SMX_KV_E4M3) {
        union { smx_bf16x2_t b; unsigned u; } a, b;
        a.b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u, 1.0f, false);
        b.b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u, 1.0f, true);
        lo = a.u;
        hi = b.u;
    } else {
        lo = pack_bf2((float)(signed char)u, (float)(signed char)(u >> 8));
        hi = pack_bf2((float)(signed char)(u >> 16), (float)(signed char)(u >> 24));
    }
}
__device__ __forceinline__ float ca_exp(float x) { return __builtin_amdgcn_exp2f(x * CA_LOG2E); }

// one wave's block of BK keys in flight
template <int FMT, int D, int NB>
struct CaBlock {
    enum { ES = CaFmt<FMT>::ES, KC = D * ES / 64, VW = D * ES / 64 };      // 16-byte K chunks, V registers per key
    uint4 k[2 * NB][KC];
    unsigned v[2 * NB][4][VW];
    CaF4 ks[2 * NB], vs[2 * NB];
};

template <int FMT, int D, int NB, bool TAIL>
__device__ __forceinline__ void ca_load(CaBlock<FMT, D, NB>& x, const SmxKVCache& c, long long base, long long sbase, int j0, int nmax) {
    typedef CaBlock<FMT, D, NB> B;
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const char* kb = (const char*)c.k + (base + (long long)j0 * c.ts) * B::ES;
    const char* vb = (const char*)c.v + (base + (long long)j0 * c.ts) * B::ES;
    const int tsb = (int)c.ts * B::ES, last = nmax - 1 - j0;       // (TAIL: keys past the last visible one read the last one)
#pragma unroll
    for (int a = 0; a < 2 * NB; ++a) {
        const int tk = TAIL ? min(16 * a + i, last) : i;
        const char* p = kb + (TAIL ? 0ll : 16ll * a * tsb);
        const unsigned off = (unsigned)(tk * tsb + 16 * g);
#pragma unroll
        for (int q = 0; q < B::KC; ++q) x.k[a][q] = *reinterpret_cast<const uint4*>(p + off + 64 * q);
    }
#pragma unroll
    for (int a = 0; a < 2 * NB; ++a)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int tk = TAIL ? min(16 * a + 4 * g + r, last) : 4 * g;
            const char* p = vb + (TAIL ? 0ll : (16ll * a + r) * tsb);
            const unsigned off = (unsigned)(tk * tsb + 4 * B::VW * i);
            if (B::VW == 1) x.v[a][r][0] = *reinterpret_cast<const unsigned*>(p + off);
            else if (B::VW == 2) {
                const uint2 u = *reinterpret_cast<const uint2*>(p + off);
                x.v[a][r][0] = u.x;
                x.v[a][r][B::VW > 1 ? 1 : 0] = u.y;
            } else {
                const uint4 u = *reinterpret_cast<const uint4*>(p + off);
                x.v[a][r][0] = u.x;
                x.v[a][r][B::VW > 1 ? 1 : 0] = u.y;
                x.v[a][r][B::VW > 2 ? 2 : 0] = u.z;
                x.v[a][r][B::VW > 2 ? 3 : 0] = u.w;
            }
        }
    if (FMT <= SMX_KV_INT8) {
        const float *ks = c.ks + sbase + j0, *vs = c.vs + sbase + j0;
#pragma unroll
        for (int a = 0; a < 2 * NB; ++a) {
            if (TAIL) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int tk = min(16 * a + 4 * g + r, last);
                    x.ks[a].v[r] = ks[tk];
                    x.vs[a].v[r] = vs[tk];
                }
            } else {
                x.ks[a] = *reinterpret_cast<const CaF4*>(ks + 16 * a + 4 * g);
                x.vs[a] = *reinterpret_cast<const CaF4*>(vs + 16 * a + 4 * g);
            }
        }
    }
}

template <int FMT, int D, int MT, typename T>
__global__ __launch_bounds__(256, 2) void attn_cached_mfma(SmxCachedAttnParams p, CaPlan pl) {
    enum { ES = CaFmt<FMT>::ES, NB = (ES * D == 64 && MT <= 2) ? 2 : 1, BK = 32 * NB, KF = D / 32, DT = D / 16,
           NQ = sizeof(T) == 4 ? 3 : 1, NP = sizeof(T) == 4 ? 3 : 2 };
    typedef CaBlock<FMT, D, NB> Blk;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    // ---- which rows, which keys
    int id = blockIdx.x;
    const bool pre = id < pl.items_p;
    if (!pre) id -= pl.items_p;
    const SmxKVCache& c = pre ? p.pre : p.own;
    const int ns = pre ? pl.nsp : pl.nso;
    const int s = id % ns;
    id /= ns;
    const int hk = id % pl.Hkv;
    id /= pl.Hkv;
    const int b = id % c.B, row0 = id / c.B * (16 * MT);
    const int per = p.Tq * pl.G, nrows = (pre ? pl.R : 1) * per, b0 = pre ? b * pl.R : b;
    int np = 0, nk = 0;
    if (p.pre.k) np = p.plen ? min(max(p.plen[b0 / pl.R], 0), p.pre.cap) : p.pre.cap;
    if (p.own.k && !pre) nk = p.klen ? min(max(p.klen[b], 0), p.own.cap) : p.own.cap;
    const bool causal = p.causal && !pre;
    const int rlast = min(nrows, row0 + 16 * MT) - 1;
    // keys that the block's first row sees (all rows see them) and that its last row sees
    const int nmax = pre ? np : causal ? max(min(nk, nk - p.Tq + rlast / pl.G + 1), 0) : nk;
    const int nall = causal ? max(nk - p.Tq + row0 / pl.G + 1, 0) : nmax;
    const int nblk = (nmax + BK - 1) / BK, bps = (nblk + ns - 1) / ns;
    const int blk_end = min(nblk, (s + 1) * bps);
    const long long base = (long long)b * c.bs + (long long)hk * c.hs, sbase = (long long)b * c.sbs + (long long)hk * c.shs;
    // ---- this lane's rows
    int lim[MT], qpos[MT], hq[MT];
    unsigned qf[MT][NQ][KF][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int r = row0 + 16 * mt + i;
        const int rr = min(r, nrows - 1), bb = b0 + rr / per, t = rr % per / pl.G;
        hq[mt] = hk * pl.G + rr % pl.G;
        int own = nk;                                   // (a prefix row's own length: for its position only)
        if (pre) own = !p.own.k ? 0 : p.klen ? min(max(p.klen[bb], 0), p.own.cap) : p.own.cap;
        qpos[mt] = np + own - p.Tq + t;
        lim[mt] = causal ? max(min(nk, nk - p.Tq + t + 1), 0) : nmax;
        const T* q = reinterpret_cast<const T*>(p.q) + bb * p.q_bs + t * p.q_ts + hq[mt] * p.q_hs;
#pragma unroll
        for (int f = 0; f < KF; ++f) {
            const int d = ES == 1 ? 64 * (f >> 1) + 16 * g + 8 * (f & 1) : 32 * f + 8 * g;
            float x[8];
            load8(q + d, x);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float u = r < nrows ? x[2 * e] : 0.f, v = r < nrows ? x[2 * e + 1] : 0.f;
#pragma unroll
                for (int n = 0; n < NQ; ++n) {          // the part of the value that n earlier bf16 numbers leave over
                    const unsigned h = pack_bf2(u, v);
                    qf[mt][n][f][e] = h;
                    // (the first part of an infinity or NaN holds it all)
                    u = n == 0 && !(fabsf(u) < INFINITY) ? 0.f : u - __uint_as_float(h << 16);
                    v = n == 0 && !(fabsf(v) < INFINITY) ? 0.f : v - __uint_as_float(h & 0xffff0000u);
                }
            }
        }
    }
    f32x4_t acc[MT][DT];
    float m[MT], l[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        m[mt] = -INFINITY;
        l[mt] = 0.f;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[mt][d] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    }
    __shared__ float sm[CA_WAVES][16], sl[CA_WAVES][16];
    __shared__ __attribute__((aligned(16))) float so[CA_WAVES][16][D + 4];

    Blk x, y;
    int blk = s * bps + w;
    if (blk < blk_end) {
        if (blk * BK + BK <= nmax) ca_load<FMT, D, NB, false>(x, c, base, sbase, blk * BK, nmax);
        else ca_load<FMT, D, NB, true>(x, c, base, sbase, blk * BK, nmax);
    }
    for (; blk < blk_end; blk += CA_WAVES) {
        const int j0 = blk * BK, jn = j0 + CA_WAVES * BK;
        if (blk + CA_WAVES < blk_end) {
            if (jn + BK <= nmax) ca_load<FMT, D, NB, false>(y, c, base, sbase, jn, nmax);
            else ca_load<FMT, D, NB, true>(y, c, base, sbase, jn, nmax);
        }
        const bool masked = j0 + BK > nall;
        // ---- scores
        f32x4_t sc[MT][2 * NB];
#pragma unroll
        for (int a = 0; a < 2 * NB; ++a) {
            unsigned kf[KF][4];
#pragma unroll
            for (int q = 0; q < Blk::KC; ++q) {
                const unsigned u[4] = {x.k[a][q].x, x.k[a][q].y, x.k[a][q].z, x.k[a][q].w};
                if (ES == 2) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) kf[q % KF][e] = u[e];
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) ca_cvt4<FMT>(u[e], kf[(2 * q + (e >> 1)) % KF][2 * (e & 1)], kf[(2 * q + (e >> 1)) % KF][2 * (e & 1) + 1]);
                }
            }
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                sc[mt][a] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int n = NQ - 1; n >= 0; --n)       // small parts first
#pragma unroll
                    for (int f = 0; f < KF; ++f) sc[mt][a] = ca_mfma(kf[f], qf[mt][n][f], sc[mt][a]);
#pragma unroll
                for (int r = 0; r < 4; ++r) sc[mt][a][r] *= FMT <= SMX_KV_INT8 ? x.ks[a].v[r] * p.scale : p.scale;
                if (p.rel_bias) {
                    const float* rb = p.rel_bias + (long long)hq[mt] * p.nrel;
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        sc[mt][a][r] += rb[min(max(qpos[mt] - (pre ? 0 : np) - (j0 + 16 * a + 4 * g + r), 0), p.nrel - 1)];
                }
                if (masked)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (j0 + 16 * a + 4 * g + r >= lim[mt]) sc[mt][a][r] = -INFINITY;
            }
        }
        // ---- reference
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            float mx = sc[mt][0][0];
#pragma unroll
            for (int a = 0; a < 2 * NB; ++a)
#pragma unroll
                for (int r = 0; r < 4; ++r) mx = fmaxf(mx, sc[mt][a][r]);
            if (__ballot(mx > m[mt] + CA_SLACK)) {
                mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
                mx = fmaxf(fmaxf(mx, __shfl_xor(mx, 32, 64)), m[mt]);
                const float al = mx == m[mt] ? 1.f : ca_exp(m[mt] - mx);        // (equal also while both are -inf)
                m[mt] = mx;
                l[mt] *= al;
#pragma unroll
                for (int d = 0; d < DT; ++d) acc[mt][d] *= al;
            }
        }
        // ---- probabilities and the second product, 32 keys at a time
        bool odd = false;                               // bf16: a value that is not finite among keys that some row must not see
        if (FMT == SMX_KV_BF16 && masked) {
            if (j0 + BK > nmax) {
#pragma unroll
                for (int a = 0; a < 2 * NB; ++a)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (j0 + 16 * a + 4 * g + r >= nmax)
#pragma unroll
                            for (int q = 0; q < Blk::VW; ++q) x.v[a][r][q] = 0u;
            }
            bool bad = false;
#pragma unroll
            for (int a = 0; a < 2 * NB; ++a)
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int q = 0; q < Blk::VW; ++q)
                        bad |= (x.v[a][r][q] & 0x7f80u) == 0x7f80u || (x.v[a][r][q] & 0x7f800000u) == 0x7f800000u;
            odd = __ballot(bad) != 0;
        }
#pragma unroll
        for (int st = 0; st < NB; ++st) {
            unsigned pf[MT][NP][4];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                const float ref = m[mt] == -INFINITY ? 0.f : m[mt];
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                    float pr[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        pr[r] = ca_exp(sc[mt][2 * st + a][r] - ref);
                        l[mt] += pr[r];
                        if (FMT <= SMX_KV_INT8) {
                            pr[r] *= x.vs[2 * st + a].v[r];
                            if (masked && j0 + 32 * st + 16 * a + 4 * g + r >= lim[mt]) pr[r] = 0.f;
                        }
                    }
                    if (FMT == SMX_KV_BF16 && odd) {
                        // rare: key by key, so that a zero probability never meets an infinity
                        for (int k = 0; k < 16; ++k) {
                            const int src = (k >> 2) * 16 + i, j = j0 + 32 * st + 16 * a + k;
                            const float p0 = __shfl(pr[0], src, 64), p1 = __shfl(pr[1], src, 64), p2 = __shfl(pr[2], src, 64), p3 = __shfl(pr[3], src, 64);
                            const float pk = (k & 2) ? ((k & 1) ? p3 : p2) : ((k & 1) ? p1 : p0);
                            if (j < lim[mt]) {
                                const bf16_t* v = reinterpret_cast<const bf16_t*>(c.v) + base + (long long)j * c.ts;
#pragma unroll
                                for (int d = 0; d < DT; ++d)
#pragma unroll
                                    for (int r = 0; r < 4; ++r) acc[mt][d][r] = fmaf(pk, bf2f(v[DT * (4 * g + r) + d]), acc[mt][d][r]);
                            }
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NP; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const unsigned h = pack_bf2(pr[2 * e], pr[2 * e + 1]);
                            pf[mt][n][2 * a + e] = h;
                            pr[2 * e] -= __uint_as_float(h << 16);
                            pr[2 * e + 1] -= __uint_as_float(h & 0xffff0000u);
                        }
                }
            }
            if (FMT == SMX_KV_BF16 && odd) continue;
            // V: registers of DPL elements per key -> per d-tile registers of two keys
            unsigned vx[8][DT / 2];
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int q = 0; q < Blk::VW; ++q) {
                    const unsigned u = x.v[2 * st + (e >> 2)][e & 3][q];
                    if (ES == 2) vx[e][q % (DT / 2)] = u;
                    else ca_cvt4<FMT>(u, vx[e][(2 * q) % (DT / 2)], vx[e][(2 * q + 1) % (DT / 2)]);
                }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                unsigned vf[4];
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    vf[q] = __builtin_amdgcn_perm(vx[2 * q + 1][d >> 1], vx[2 * q][d >> 1], (d & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int n = NP - 1; n >= 0; --n) acc[mt][d] = ca_mfma(vf, pf[mt][n], acc[mt][d]);
            }
        }
        x = y;
    }

    // ---- the four waves meet: rows of 16, one tile at a time
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        l[mt] += __shfl_xor(l[mt], 16, 64);
        l[mt] += __shfl_xor(l[mt], 32, 64);
        if (mt) __syncthreads();
        if (g == 0) {
            sm[w][i] = m[mt];
            sl[w][i] = l[mt];
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int d = 0; d < DT; d += 4)
                *reinterpret_cast<float4*>(&so[w][i][DT * (4 * g + r) + d]) =
                    make_float4(acc[mt][d][r], acc[mt][d + 1][r], acc[mt][d + 2][r], acc[mt][d + 3][r]);
        __syncthreads();
        const int row = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * DT, r = row0 + 16 * mt + row;
        float M = -INFINITY, L = 0.f, o[DT];
#pragma unroll
        for (int v = 0; v < CA_WAVES; ++v) M = fmaxf(M, sm[v][row]);
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] = 0.f;
#pragma unroll
        for (int v = 0; v < CA_WAVES; ++v) {
            const float mv = sm[v][row], f = mv == M ? 1.f : ca_exp(mv - M);
            L = fmaf(sl[v][row], f, L);
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] = fmaf(so[v][row][d0 + d], f, o[d]);
        }
        if (pl.join) {
            const long long pr = (long long)blockIdx.x * (16 * MT) + 16 * mt + row;
            if (r < nrows) {
                if (d0 == 0) {
                    pl.pml[2 * pr] = M;
                    pl.pml[2 * pr + 1] = L;
                }
#pragma unroll
                for (int d = 0; d < DT; d += 4) *reinterpret_cast<float4*>(pl.po + pr * D + d0 + d) = make_float4(o[d], o[d + 1], o[d + 2], o[d + 3]);
            }
        } else if (r < nrows) {
            const int bb = b0 + r / per, t = r % per / pl.G, h = hk * pl.G + r % pl.G;
            const float inv = L == 0.f ? 0.f : 1.f / L;
            T* out = reinterpret_cast<T*>(p.o) + bb * p.o_bs + t * p.o_ts + h * p.o_hs + d0;
#pragma unroll
            for (int d = 0; d < DT; ++d) Cvt<T>::st(out + d, L == 0.f ? 0.f : o[d] * inv);
            if (p.lse && d0 == 0) p.lse[((long long)bb * p.H + h) * p.Tq + t] = L == 0.f ? -INFINITY : M + logf(L);
        }
    }
}

// O = sum over the splits of both parts, in order.  One wave per (row, head, query).
template <int D, typename T>
__global__ __launch_bounds__(256) void attn_cached_join(SmxCachedAttnParams p, CaPlan pl, int mt16) {
    const long long id = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (id >= (long long)p.B * p.H * p.Tq) return;
    const int t = (int)(id % p.Tq), h = (int)(id / p.Tq % p.H), b = (int)(id / ((long long)p.Tq * p.H)), hk = h / pl.G;
    float m = -INFINITY, l = 0.f, o[D / 64];
#pragma unroll
    for (int d = 0; d < D / 64; ++d) o[d] = 0.f;
    for (int part = 0; part < 2; ++part) {
        const SmxKVCache& c = part ? p.own : p.pre;
        if (!c.k) continue;
        const int ns = part ? pl.nso : pl.nsp, e = part ? b : b / pl.R;
        const int r = (part ? 0 : b % pl.R * p.Tq * pl.G) + t * pl.G + h % pl.G;
        const long long it = (part ? pl.items_p : 0) + (((long long)(r / mt16) * c.B + e) * pl.Hkv + hk) * ns;
        // at most 64 splits: a lane holds one's maximum and sum
        float ms = -INFINITY, ls = 0.f;
        if (lane < ns) {
            const float* q = pl.pml + 2 * ((it + lane) * mt16 + r % mt16);
            ms = q[0];
            ls = q[1];
        }
        const float M = fmaxf(m, wave_max(ms));
        const float f0 = m == M ? 1.f : ca_exp(m - M), fs = ls == 0.f ? 0.f : ca_exp(ms - M);
        l = l * f0 + wave_sum(ls * fs);
        m = M;
#pragma unroll
        for (int d = 0; d < D / 64; ++d) o[d] *= f0;
        for (int s = 0; s < ns; ++s) {
            const float f = __shfl(fs, s, 64);
            if (f == 0.f) continue;                      // (nothing there, or too little to count)
            const float* q = pl.po + ((it + s) * mt16 + r % mt16) * D;
#pragma unroll
            for (int d = 0; d < D / 64; ++d) o[d] = fmaf(q[lane + 64 * d], f, o[d]);
        }
    }
    T* out = reinterpret_cast<T*>(p.o) + b * p.o_bs + t * p.o_ts + h * p.o_hs;
    const float inv = 1.f / l;
#pragma unroll
    for (int d = 0; d < D / 64; ++d) Cvt<T>::st(out + lane + 64 * d, l == 0.f ? 0.f : o[d] * inv);
    if (p.lse && lane == 0) p.lse[id / p.Tq * p.Tq + t] = l == 0.f ? -INFINITY : m + logf(l);
}
