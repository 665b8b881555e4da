// Matrix-core form of the cached attention (head widths 64 and 128; e4m3, int8 and bf16 caches; bf16 and fp32 queries).
//
// The rows of one KV head - Tq x G of a batch entry's own keys, R x Tq x G of a prefix - are the columns of S^T = K Q^T tiles (16 keys x 16 rows),
// so a lane owns one row (i = lane & 15) and four keys (4 g + r, g = lane >> 4) of each tile, and the exponentiated tile already is the
// B operand of O^T = V^T P^T: no pass through LDS.  8-bit codes are exact in bf16, so the products are exact up to the 32-bit accumulation; fp32
// queries are held as three bf16 numbers (24 bits) and probabilities as two (bf16 queries) or three: one rounding to bf16 would cost as much
// as the rounding of the output.
//   K operand: a lane's 16 contiguous bytes of one key ARE eight k-indices of two (one for bf16) products; Q is loaded in the same order.
//   V operand: a lane takes DPL = D / 16 neighbouring elements of each of its eight keys; one byte permute per register pairs two keys.
// Softmax in units of log 2: every wave keeps its own reference m per row and moves it only when a probability passes 2^16 (a wave-wide test): most
// blocks need no rescaling and no cross-lane maximum.  Four waves take every fourth block of BK keys, and meet in LDS;
// long caches are split over workgroups as well, whose unnormalised (m, l, O) a second kernel joins in a fixed order.
//
// Bounds.  Up to 16 rows a KV head: HBM - 8 rows x 8 heads of 128 x 30 - 33 000 e4m3 keys 100 us (5.3 TB/s), 256 heads x 8 192 x 64 int8 keys 52 us
// (5.5 TB/s), bf16 96 us (5.6 TB/s).  Short caches: the chain length -> keys -> products -> LDS -> store, 4 - 5 us.  Many rows: the vector instructions of
// the softmax and of the conversions, about 6.5 a score (256 rows x 8 heads x 65 536 keys of 64: 90 us, 380 TF): why a score costs one fused
// product and difference, one exponential, and the splitting of probabilities one dot product each.
#pragma once
#include "kv_common.h"

#define CA_BK 32                  // keys per block and wave (64: more registers than they save instructions; two blocks ahead: spills)
#define CA_LOG2E 1.44269504088896340736f
#define CA_LN2 0.69314718055994530942f
#define CA_BIG 65536.f            // a probability may pass 1 by this factor before the reference moves
// Range: sums of probabilities (of up to 2^16) times values shall overflow no sooner than those of the values themselves.
//   8 bit: a probability times the scale keeps 16 (24) bits as two (three) bf16 numbers down to 2^-110, the smallest scale is 2^-126, and 2^16 times
//   the largest does not fit.  Scales enter times CA_LIFT, from the first one past CA_LARGE on times CA_DROP; neither costs an ordinary one a bit.
//   bf16: in a block with large values (told by the sum of a lane's squares) the reference moves at 1.
// (Together 0.1 us a launch: 64 x 16 heads x 0 - 1 024 keys 17.0 -> 17.2 us, 16 x 33 queries x 16 x 700 keys 18.9 -> 19.4; a second pass over the keys where
// the sums got large, in place of this, cost twice that.)
#define CA_LIFT 0x1p32f
#define CA_DROP 0x1p-30f
#define CA_LARGE 0x1p28f
#define CA_LARGE_SQ 0x1p120f
#define CA_LOWEST (-3.402823466e38f)

// waves per SIMD the registers are held to
constexpr int ca_occ(int es, int d, int mt, int qsize) { return qsize == 4 || (es == 2 && d == 128) || mt > 2 || (mt == 2 && d == 128) ? 2 : mt == 2 || d == 128 ? 3 : 4; }

// Division of 0 <= r < 2^31 by a number known to the host: k = ceil(log2 d), m = ceil(2^(31 + k) / d) < 2^32, and 2 r m / 2^(32 + k) falls short of
// nothing, since m d - 2^(31 + k) < 2^k.  (The compiler's division is some thirty instructions, a few of them per row: a cold kernel waits for
// every line of its code.)
struct CaDiv { unsigned m; int k, d; };
__device__ __forceinline__ int ca_div(const CaDiv& v, int r) { return (int)(__umulhi((unsigned)r << 1, v.m) >> v.k); }

struct CaPlan {
    CaDiv per, g;                 // by Tq * G, by G
    CaDiv nso_, nsp_, hkv_, bo_, bp_, r_; // by nso, nsp, Hkv, the entries of either part, R
    int G, Hkv, R;                // query heads per KV head; rows per prefix
    int mbo, mbp;                 // blocks of 16 * MT rows per (entry, KV head): own, prefix
    int nso, nsp;                 // key splits: own, prefix
    int items_p;                  // work items = workgroups of the prefix part (they come first)
    int items_o;                  // work items of the own part
    int single;                   // a wave per item, four items per workgroup (short caches, many rows): 1 own items, 2 all items
    int join;                     // partial results to po / pml instead of the output
    int sp, so, mtl;              // partial rows of an item of either part: 2^mtl = 16 MT, or all its rows where those are fewer
    float *po, *pml;              // [partial row][D], [partial row][2]: the prefix's items, then the others
};

template <int FMT> struct CaFmt;
template <> struct CaFmt<SMX_KV_E4M3> { enum { ES = 1 }; };
template <> struct CaFmt<SMX_KV_INT8> { enum { ES = 1 }; };
template <> struct CaFmt<SMX_KV_BF16> { enum { ES = 2 }; };

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
__device__ __forceinline__ float ca_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
// bf16 pair product a . b + c
__device__ __forceinline__ float ca_dot2(unsigned a, unsigned b, float c) {
    union { unsigned u; smx_bf16x2_t v; } x, y;
    x.u = a;
    y.u = b;
    return __builtin_amdgcn_fdot2_f32_bf16(x.v, y.v, c, false);
}
// a bias in log 2 units (the type's lowest value times log2 e is no longer finite; -inf and NaN stay)
__device__ __forceinline__ float ca_bias2(float b) {
    const float v = b * CA_LOG2E;
    return v < CA_LOWEST && b >= CA_LOWEST ? CA_LOWEST : v;
}
// log-sum-exp in natural units from a reference in log 2 units (a bias of the type's lowest value stays what it is).  A NaN never moves the
// reference from where it starts, the lowest value: such a row is told by its sum.
__device__ __forceinline__ float ca_lse(float m, float l) {
    return l == 0.f ? -INFINITY : m == CA_LOWEST && l == l ? CA_LOWEST : fmaf(m, CA_LN2, logf(l));
}

typedef __attribute__((ext_vector_type(4))) unsigned ca_u4;
typedef __attribute__((ext_vector_type(2))) unsigned ca_u2;
// One wave's block of BK keys in flight.  K (with its scales) is asked for again as soon as the scores are out, V as soon as the second product is:
// each is on its way while the other is worked on, out of one set of registers.  All loads go through buffer descriptors that end behind the
// last visible key: what lies past it comes back as zeros, and there is one code path for whole and partial blocks.
template <int FMT, int D>
struct CaBlock {
    enum { ES = CaFmt<FMT>::ES, KC = D * ES / 64, VW = D * ES / 64 };      // 16-byte K chunks, V registers per key
    ca_u4 k[2][KC];
    unsigned v[2][4][VW];
    unsigned ks, vs;        // lane (g, i), i < 8: the scale of key 16 (i >> 2) + 4 g + (i & 3); DPP row broadcasts hand it to the other lanes of g
};
struct CaView {             // one head of a cache
    const char *k, *v;
    const float *ks, *vs;
    int tsb;                // bytes between tokens
    int nmax;
    int koff, voff, soff;   // this lane's offsets within a block
};
__device__ __forceinline__ __amdgpu_buffer_rsrc_t ca_rsrc(const void* base, long long bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)(bytes < 0x7ffffff0ll ? bytes : 0x7ffffff0ll), 0x00020000);
}
template <int FMT, int D>
__device__ __forceinline__ unsigned ca_load_scales(const float* s, const CaView& c, int j0) {
    return __builtin_amdgcn_raw_buffer_load_b32(ca_rsrc(s + j0, (c.nmax - j0) * 4ll), c.soff, 0, 0);
}
template <int FMT, int D>
__device__ __forceinline__ void ca_load_k(CaBlock<FMT, D>& x, const CaView& c, int j0) {
    typedef CaBlock<FMT, D> B;
    int off = c.koff;
    asm volatile("" : "+v"(off));       // (a sum per load: offsets kept from block to block would cost the registers of a tile)
    const __amdgpu_buffer_rsrc_t rs = ca_rsrc(c.k + (long long)j0 * c.tsb, (long long)(c.nmax - 1 - j0) * c.tsb + D * B::ES);
    if (FMT <= SMX_KV_INT8) x.ks = ca_load_scales<FMT, D>(c.ks, c, j0);
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int q = 0; q < B::KC; ++q) x.k[a][q] = __builtin_amdgcn_raw_buffer_load_b128(rs, off + 16 * a * c.tsb + 64 * q, 0, 0);
}
template <int FMT, int D>
__device__ __forceinline__ void ca_load_v(CaBlock<FMT, D>& x, const CaView& c, int j0) {
    typedef CaBlock<FMT, D> B;
    int off = c.voff;
    asm volatile("" : "+v"(off));
    const __amdgpu_buffer_rsrc_t rs = ca_rsrc(c.v + (long long)j0 * c.tsb, (long long)(c.nmax - 1 - j0) * c.tsb + D * B::ES);
    if (FMT <= SMX_KV_INT8) x.vs = ca_load_scales<FMT, D>(c.vs, c, j0);
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int o = off + (16 * a + r) * c.tsb;
            if (B::VW == 1) x.v[a][r][0] = __builtin_amdgcn_raw_buffer_load_b32(rs, o, 0, 0);
            else if (B::VW == 2) {
                const ca_u2 u = __builtin_amdgcn_raw_buffer_load_b64(rs, o, 0, 0);
                x.v[a][r][0] = u[0];
                x.v[a][r][B::VW > 1 ? 1 : 0] = u[1];
            } else {
                const ca_u4 u = __builtin_amdgcn_raw_buffer_load_b128(rs, o, 0, 0);
                x.v[a][r][0] = u[0];
                x.v[a][r][B::VW > 1 ? 1 : 0] = u[1];
                x.v[a][r][B::VW > 2 ? 2 : 0] = u[2];
                x.v[a][r][B::VW > 2 ? 3 : 0] = u[3];
            }
        }
}
// the scale of key 16 a + 4 g + r of the block, from the lane of this row of 16 that holds it
template <int K>
__device__ __forceinline__ float ca_bcast(unsigned v) {
    return __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x150 + K, 0xf, 0xf, true));
}
__device__ __forceinline__ float ca_scale(unsigned v, int a, int r) {         // (a, r: constants once unrolled)
    switch (4 * a + r) {
        case 0: return ca_bcast<0>(v);
        case 1: return ca_bcast<1>(v);
        case 2: return ca_bcast<2>(v);
        case 3: return ca_bcast<3>(v);
        case 4: return ca_bcast<4>(v);
        case 5: return ca_bcast<5>(v);
        case 6: return ca_bcast<6>(v);
        case 7: return ca_bcast<7>(v);
        case 8: return ca_bcast<8>(v);
        case 9: return ca_bcast<9>(v);
        case 10: return ca_bcast<10>(v);
        case 11: return ca_bcast<11>(v);
        case 12: return ca_bcast<12>(v);
        case 13: return ca_bcast<13>(v);
        case 14: return ca_bcast<14>(v);
        default: return ca_bcast<15>(v);
    }
}

// four outputs side by side (offsets are multiples of 4 elements of a row whose base is 16-byte aligned)
__device__ __forceinline__ void ca_store4(float* p, const float v[4]) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void ca_store4(bf16_t* p, const float v[4]) { *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3])); }

template <int D, int WV> struct CaShared {       // where the waves meet
    float m[WV][16], l[WV][16];
    __attribute__((aligned(16))) float o[WV][16][D + 4];
};
struct CaItem { bool pre; int s, hk, b, row0; long long prow; };      // key split, KV head, batch entry, first row; first partial row

// One work item: 16 * MT rows (as many as there are of the kernel's 16 * MTB) over one split of the keys, by the workgroup's WV = 4 or 8 waves or by one
template <int FMT, int D, int MT, int MTB, int WV, int SW, typename T>
__device__ __forceinline__ void ca_body(const SmxCachedAttnParams& p, const CaPlan& pl, const CaItem& it, CaShared<D, SW>& sh) {
    static_assert(WV < 8 || MT == 1, "eight waves: one tile of rows");
    enum { ES = CaFmt<FMT>::ES, BK = CA_BK, KF = D / 32, DT = D / 16,
           NQ = sizeof(T) == 4 ? 3 : 1, NP = sizeof(T) == 4 ? 3 : 2 };
    typedef CaBlock<FMT, D> Blk;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const bool pre = it.pre;
    const int s = it.s, hk = it.hk, b = it.b, row0 = it.row0;
    const SmxKVCache& c = pre ? p.pre : p.own;
    const int ns = pre ? pl.nsp : pl.nso;
    const int per = p.Tq * pl.G, nrows = (pre ? pl.R : 1) * per, b0 = pre ? b * pl.R : b;
    int np = 0, nk = 0;
    if (p.pre.k) np = p.plen ? min(max(p.plen[pre ? b : b / pl.R], 0), p.pre.cap) : p.pre.cap;
    if (p.own.k && !pre) nk = p.klen ? min(max(p.klen[b], 0), p.own.cap) : p.own.cap;
    const bool causal = p.causal && !pre;
    const int rlast = min(nrows, row0 + 16 * MT) - 1;
    // keys that the block's first row sees (all rows see them) and that its last row sees
    const int nmax = pre ? np : causal ? max(min(nk, nk - p.Tq + ca_div(pl.g, rlast) + 1), 0) : nk;
    const int nall = causal ? max(nk - p.Tq + ca_div(pl.g, row0) + 1, 0) : nmax;
    const int nblk = (nmax + BK - 1) / BK, bps = ca_div(pre ? pl.nsp_ : pl.nso_, nblk + ns - 1);
    const int blk_end = min(nblk, (s + 1) * bps);
    const long long base = (long long)b * c.bs + (long long)hk * c.hs, sbase = (long long)b * c.sbs + (long long)hk * c.shs;
    const CaView cv = {(const char*)c.k + base * ES, (const char*)c.v + base * ES, c.ks + sbase, c.vs + sbase, (int)c.ts * ES, nmax,
                       i * (int)c.ts * ES + 16 * g, 4 * g * (int)c.ts * ES + 4 * Blk::VW * i, 4 * (16 * ((i >> 2) & 1) + 4 * g + (i & 3))};
    Blk x;
    int blk = s * bps + (WV == 1 ? 0 : w);
    if (blk < blk_end) {
        ca_load_k<FMT, D>(x, cv, blk * BK);
        ca_load_v<FMT, D>(x, cv, blk * BK);
    }
    // ---- this lane's rows
    const int kpos0 = pre ? 0 : np;                     // position of key 0
    int lim[MT], qpos[MT], hq[MT];
    unsigned qf[MT][NQ][KF][4];
    const float scale2 = p.scale * CA_LOG2E;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int r = row0 + 16 * mt + i;
        const int rr = min(r, nrows - 1), br = pre ? ca_div(pl.per, rr) : 0, bb = b0 + br, rt = rr - br * per, t = ca_div(pl.g, rt);
        hq[mt] = hk * pl.G + rt - t * pl.G;
        int own = nk;                                   // (a prefix row's own length: for its position only)
        if (pre) own = !p.own.k ? 0 : p.klen ? min(max(p.klen[bb], 0), p.own.cap) : p.own.cap;
        qpos[mt] = np + own - p.Tq + t;
        lim[mt] = causal ? max(min(nk, nk - p.Tq + t + 1), 0) : nmax;
        const T* q = reinterpret_cast<const T*>(p.q) + bb * p.q_bs + t * p.q_ts + hq[mt] * p.q_hs;
#pragma unroll
        for (int f = 0; f < KF; ++f) {
            const int d = ES == 1 ? 64 * (f >> 1) + 16 * g + 8 * (f & 1) : 32 * f + 8 * g;
            if (NQ == 1) {
                const uint4 u = r < nrows ? *reinterpret_cast<const uint4*>(q + d) : make_uint4(0u, 0u, 0u, 0u);
                qf[mt][0][f][0] = u.x; qf[mt][0][f][1] = u.y; qf[mt][0][f][2] = u.z; qf[mt][0][f][3] = u.w;
            } else {
                float x[8];
                load8(q + d, x);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float u = r < nrows ? x[2 * e] : 0.f, v = r < nrows ? x[2 * e + 1] : 0.f;
#pragma unroll
                    for (int n = 0; n < NQ; ++n) {      // the part of the value that n earlier bf16 numbers leave over
                        const unsigned h = pack_bf2(u, v);
                        qf[mt][n][f][e] = h;
                        // (the first part of an infinity or NaN holds it all)
                        u = n == 0 && !(fabsf(u) < INFINITY) ? 0.f : u - __uint_as_float(h << 16);
                        v = n == 0 && !(fabsf(v) < INFINITY) ? 0.f : v - __uint_as_float(h & 0xffff0000u);
                    }
                }
            }
        }
    }
    unsigned one_lo = 0x0000bf80u, one_hi = 0xbf800000u;          // (-1, 0), (0, -1)
    asm("" : "+v"(one_lo), "+v"(one_hi));                       // (in registers: not every form of these constants means a pair)
    f32x4_t acc[MT][DT];
    float m[MT], l[MT], lift = CA_LIFT;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        m[mt] = CA_LOWEST;
        l[mt] = 0.f;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[mt][d] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    }
    for (; blk < blk_end; blk += WV) {
        const int j0 = blk * BK;
        const bool more = blk + WV < blk_end;
        const bool masked = j0 + BK > nall;
        // ---- scores
        f32x4_t sc[MT][2];                         // q . codes; times ksc it is the score in log 2 units
        float ksc[2][4];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            unsigned kf[KF][4];
#pragma unroll
            for (int q = 0; q < Blk::KC; ++q) {
                const unsigned u[4] = {x.k[a][q][0], x.k[a][q][1], x.k[a][q][2], x.k[a][q][3]};
                if (ES == 2) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) kf[q % KF][e] = u[e];
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) ca_cvt4<FMT>(u[e], kf[(2 * q + (e >> 1)) % KF][2 * (e & 1)], kf[(2 * q + (e >> 1)) % KF][2 * (e & 1) + 1]);
                }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) ksc[a][r] = FMT <= SMX_KV_INT8 ? ca_scale(x.ks, a, r) * scale2 : scale2;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                sc[mt][a] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int n = NQ - 1; n >= 0; --n)       // small parts first
#pragma unroll
                    for (int f = 0; f < KF; ++f) sc[mt][a] = ca_mfma(kf[f], qf[mt][n][f], sc[mt][a]);
                if (masked || p.rel_bias) {             // (uniform; sc is the score itself from here on: its factor becomes 1 below)
                    if (p.rel_bias) {
                        const float* rb = p.rel_bias + (long long)hq[mt] * p.nrel;
                        // keys so far back that every distance of the tile is beyond the table: its last value, without the gathers
                        if (__ballot(qpos[mt] - kpos0 - (j0 + 16 * a + 15) < p.nrel - 1) == 0) {
                            const float end = ca_bias2(rb[p.nrel - 1]);
#pragma unroll
                            for (int r = 0; r < 4; ++r) sc[mt][a][r] = fmaf(sc[mt][a][r], ksc[a][r], end);
                        } else {
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const float bias = rb[min(max(qpos[mt] - kpos0 - (j0 + 16 * a + 4 * g + r), 0), p.nrel - 1)];
                                sc[mt][a][r] = fmaf(sc[mt][a][r], ksc[a][r], ca_bias2(bias));
                            }
                        }
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; ++r) sc[mt][a][r] *= ksc[a][r];
                    }
                    if (masked)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (j0 + 16 * a + 4 * g + r >= lim[mt]) sc[mt][a][r] = -INFINITY;
                }
            }
            if (masked || p.rel_bias)
#pragma unroll
                for (int r = 0; r < 4; ++r) ksc[a][r] = 1.f;
        }
        if (more) ca_load_k<FMT, D>(x, cv, j0 + WV * BK);
        // bf16: large values in the block; some that are not finite
        bool large = false, odd = false;
        if (FMT == SMX_KV_BF16) {
            const auto squares = [&x]() {               // of this lane's values
                float sq = 0.f;
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int q = 0; q < Blk::VW; ++q) sq = ca_dot2(x.v[a][r][q], x.v[a][r][q], sq);
                return sq;
            };
            large = __ballot(!(squares() < CA_LARGE_SQ)) != 0;
            if (__builtin_expect(large, 0)) {
                // The product leaves those that are not finite out (a hidden one, or the zero that a probability's second part may be, would make NaN of
                // them); the rows that see them get them below.
                bool bad = false;
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int q = 0; q < Blk::VW; ++q) {
                            unsigned& u = x.v[a][r][q];
                            if ((u & 0x7f80u) == 0x7f80u) { u &= 0xffff0000u; bad = true; }
                            if ((u & 0x7f800000u) == 0x7f800000u) { u &= 0xffffu; bad = true; }
                        }
                odd = __ballot(bad) != 0;
                large = __ballot(!(squares() < CA_LARGE_SQ)) != 0;
            }
        }
        unsigned vs = 0;
        if (FMT <= SMX_KV_INT8) {
            if (__builtin_expect(__ballot(__uint_as_float(x.vs) > CA_LARGE) != 0 && lift == CA_LIFT, 0)) {
                lift = CA_DROP;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int d = 0; d < DT; ++d) acc[mt][d] *= CA_DROP / CA_LIFT;
            }
            vs = __float_as_uint(__uint_as_float(x.vs) * lift);
        }
        float vsc[2][4];
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int r = 0; r < 4; ++r) vsc[a][r] = FMT <= SMX_KV_INT8 ? ca_scale(vs, a, r) : 1.f;
        // ---- probabilities: one fused product and difference, one exponential.  A probability above 2^16 (also the first ever: the reference
        // starts at the lowest value) sends the row's wave back to the scores for a new reference.
        unsigned pf[MT][NP][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            f32x4_t pr[2];
            float big = 0.f;
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    pr[a][r] = ca_exp2(fmaf(sc[mt][a][r], ksc[a][r], -m[mt]));
                    big = fmaxf(big, pr[a][r]);
                }
            if (__ballot(big > (large ? 1.f : CA_BIG))) {
                float mx = m[mt];
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int r = 0; r < 4; ++r) mx = fmaxf(mx, sc[mt][a][r] * ksc[a][r]);
                mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
                mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
                const float al = mx == m[mt] ? 1.f : ca_exp2(m[mt] - mx);
                m[mt] = mx;
                l[mt] *= al;
#pragma unroll
                for (int d = 0; d < DT; ++d) acc[mt][d] *= al;
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int r = 0; r < 4; ++r) pr[a][r] = ca_exp2(fmaf(sc[mt][a][r], ksc[a][r], -mx));
            }
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                l[mt] += (pr[a][0] + pr[a][1]) + (pr[a][2] + pr[a][3]);
                if (FMT <= SMX_KV_INT8) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) pr[a][r] *= vsc[a][r];
                    if (masked)                         // (a hidden key's scale may be anything)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (j0 + 16 * a + 4 * g + r >= lim[mt]) pr[a][r] = 0.f;
                }
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int n = 0; n < NP; ++n) {
                        const unsigned h = pack_bf2(pr[a][2 * e], pr[a][2 * e + 1]);
                        pf[mt][n][2 * a + e] = h;
                        if (n + 1 < NP) {               // what h leaves over: -1 * its half + the number, one instruction
                            pr[a][2 * e] = ca_dot2(h, one_lo, pr[a][2 * e]);
                            pr[a][2 * e + 1] = ca_dot2(h, one_hi, pr[a][2 * e + 1]);
                        }
                    }
            }
        }
        // ---- the second product.  V, register by register of the keys: 4 (bf16: 2) d-tiles of two keys per register
        enum { DR = 4 / ES };
#pragma unroll
        for (int q = 0; q < Blk::VW; ++q) {
            unsigned vx[8][DR / 2];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const unsigned u = x.v[e >> 2][e & 3][q];
                if (ES == 2) vx[e][0] = u;
                else ca_cvt4<FMT>(u, vx[e][0], vx[e][DR / 2 - 1]);
            }
#pragma unroll
            for (int d = 0; d < DR; ++d) {
                unsigned vf[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) vf[k] = __builtin_amdgcn_perm(vx[2 * k + 1][d >> 1], vx[2 * k][d >> 1], (d & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int n = NP - 1; n >= 0; --n) acc[mt][DR * q + d] = ca_mfma(vf, pf[mt][n], acc[mt][DR * q + d]);
            }
        }
        if (FMT == SMX_KV_BF16 && odd) {
            for (int k = 0; k < BK; ++k) {              // rare: key by key, the elements that are not finite, for the rows that see the key
                const int j = j0 + k, src = ((k >> 2) & 3) * 16 + i, wd = 2 * ((k >> 4) & 1) + ((k >> 1) & 1);
                const bf16_t* v = reinterpret_cast<const bf16_t*>(c.v) + base + (long long)min(j, nmax - 1) * c.ts;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const unsigned w0 = pf[mt][0][0], w1 = pf[mt][0][1], w2 = pf[mt][0][2], w3 = pf[mt][0][3];
                    const unsigned u01 = wd & 1 ? w1 : w0, u23 = wd & 1 ? w3 : w2, u = (unsigned)__shfl((int)(wd & 2 ? u23 : u01), src, 64);
                    const float pk = __uint_as_float(k & 1 ? u & 0xffff0000u : u << 16);
                    if (j < lim[mt])
#pragma unroll
                        for (int d = 0; d < DT; ++d)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const float f = bf2f(v[DT * (4 * g + r) + d]);
                                if (!(fabsf(f) < INFINITY)) acc[mt][d][r] = fmaf(pk, f, acc[mt][d][r]);
                            }
                }
            }
        }
        if (more) ca_load_v<FMT, D>(x, cv, j0 + WV * BK);
    }
    if (FMT <= SMX_KV_INT8) {
        // (large values: what the reference lags behind is taken out of the sums as well, 1 / CA_DROP alone might not fit)
        const bool low = lift != CA_LIFT;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            float f = 1.f / CA_LIFT;
            if (low) {
                const bool lag = m[mt] != CA_LOWEST;    // (at the lowest value: none, and nothing to add to it)
                f = lag ? 0x1p-16f / CA_DROP : 1.f / CA_DROP;
                l[mt] *= lag ? 0x1p-16f : 1.f;
                m[mt] += lag ? 16.f : 0.f;
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) acc[mt][d] *= f;
        }
    }

    if (WV == 1) {                                      // a wave has all of its rows: out of the registers
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            float L = l[mt];
            L += __shfl_xor(L, 16, 64);
            L += __shfl_xor(L, 32, 64);
            const int r = row0 + 16 * mt + i;
            if (r >= nrows) continue;
            if (pl.join) {
                const long long pr = it.prow + 16 * mt + i;
                if (g == 0) *reinterpret_cast<float2*>(pl.pml + 2 * pr) = make_float2(m[mt], L);
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int d = 0; d < DT; d += 4)
                        *reinterpret_cast<float4*>(pl.po + pr * D + DT * (4 * g + q) + d) = make_float4(acc[mt][d][q], acc[mt][d + 1][q], acc[mt][d + 2][q], acc[mt][d + 3][q]);
            } else {
                const int br = pre ? ca_div(pl.per, r) : 0, bb = b0 + br, rt = r - br * per, t = ca_div(pl.g, rt), h = hk * pl.G + rt - t * pl.G;
                const float inv = 1.f / L;
                T* out = reinterpret_cast<T*>(p.o) + bb * p.o_bs + t * p.o_ts + h * p.o_hs;
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int d = 0; d < DT; d += 4) {
                        float v[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = L == 0.f ? 0.f : acc[mt][d + e][q] * inv;
                        ca_store4(out + DT * (4 * g + q) + d, v);
                    }
                if (p.lse && g == 0) p.lse[((long long)bb * p.H + h) * p.Tq + t] = ca_lse(m[mt], L);
            }
        }
        return;
    }
    // ---- the waves meet: rows of 16, one tile at a time
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        l[mt] += __shfl_xor(l[mt], 16, 64);
        l[mt] += __shfl_xor(l[mt], 32, 64);
        if (mt) __syncthreads();
        if (g == 0) {
            sh.m[w][i] = m[mt];
            sh.l[w][i] = l[mt];
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int d = 0; d < DT; d += 4)
                *reinterpret_cast<float4*>(&sh.o[w][i][DT * (4 * g + r) + d]) =
                    make_float4(acc[mt][d][r], acc[mt][d + 1][r], acc[mt][d + 2][r], acc[mt][d + 3][r]);
        __syncthreads();
        if (WV == 8 && threadIdx.x >= 256) return;
        const int row = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * DT, r = row0 + 16 * mt + row;
        float M = CA_LOWEST, L = 0.f, o[DT];
#pragma unroll
        for (int v = 0; v < WV; ++v) M = fmaxf(M, sh.m[v][row]);
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] = 0.f;
#pragma unroll
        for (int v = 0; v < WV; ++v) {
            const float mv = sh.m[v][row], f = mv == M ? 1.f : ca_exp2(mv - M);
            L = fmaf(sh.l[v][row], f, L);
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] = fmaf(sh.o[v][row][d0 + d], f, o[d]);
        }
        if (pl.join) {
            const long long pr = it.prow + 16 * mt + row;
            if (r < nrows) {
                if (d0 == 0) {
                    pl.pml[2 * pr] = M;
                    pl.pml[2 * pr + 1] = L;
                }
#pragma unroll
                for (int d = 0; d < DT; d += 4) *reinterpret_cast<float4*>(pl.po + pr * D + d0 + d) = make_float4(o[d], o[d + 1], o[d + 2], o[d + 3]);
            }
        } else if (r < nrows) {
            const int br = pre ? ca_div(pl.per, r) : 0, bb = b0 + br, rt = r - br * per, t = ca_div(pl.g, rt), h = hk * pl.G + rt - t * pl.G;
            const float inv = L == 0.f ? 0.f : 1.f / L;
            T* out = reinterpret_cast<T*>(p.o) + bb * p.o_bs + t * p.o_ts + h * p.o_hs + d0;
#pragma unroll
            for (int d = 0; d < DT; d += 4) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = L == 0.f ? 0.f : o[d + e] * inv;
                ca_store4(out + d, v);
            }
            if (p.lse && d0 == 0) p.lse[((long long)bb * p.H + h) * p.Tq + t] = ca_lse(M, L);
        }
    }
}

// What a launch's items look like.  Each combination is a kernel of its own: a second body beside the one that runs costs 1.4 us a launch (its
// instructions lie between those that run), as much as a short cache takes.
enum {
    CA_PLAIN = 0,       // every item: 16 * MT rows by four waves
    CA_SINGLE = 1,      // a wave per item of 16 rows, four items per workgroup
    CA_SMALL = 2,       // prefix items as in CA_PLAIN, own items of up to 16 rows by four waves
    CA_MIXED = 3,       // prefix items as in CA_PLAIN, own items by a wave each
    CA_EIGHT = 4        // CA_PLAIN with eight waves
};
template <int FMT, int D, int MT, int MODE, typename T>
__global__ __launch_bounds__(MODE == CA_EIGHT ? 512 : 256, ca_occ(CaFmt<FMT>::ES, D, MT, sizeof(T))) void attn_cached_mfma(SmxCachedAttnParams p, CaPlan pl) {
    enum { WV = MODE == CA_EIGHT ? 8 : 4 };
    __shared__ CaShared<D, WV> sh;
    CaItem it;
    int id = blockIdx.x;
    if (MODE == CA_SINGLE) id = 4 * id + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (MODE == CA_SINGLE && id >= pl.items_p + pl.items_o) return;      // (the last workgroup's spare waves; no barrier in that form)
    it.pre = id < pl.items_p;
    if (!it.pre) id -= pl.items_p;
    if (MODE == CA_MIXED && !it.pre) id = 4 * id + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (MODE == CA_MIXED && !it.pre && id >= pl.items_o) return;
    it.prow = it.pre ? (long long)id * pl.sp : (long long)pl.items_p * pl.sp + (long long)id * pl.so;
    const CaDiv &dns = it.pre ? pl.nsp_ : pl.nso_, &dcb = it.pre ? pl.bp_ : pl.bo_;
    const int q1 = ca_div(dns, id), q2 = ca_div(pl.hkv_, q1), q3 = ca_div(dcb, q2);      // key split fastest, then KV head, entry, block of rows
    it.s = id - q1 * dns.d;
    it.hk = q1 - q2 * pl.Hkv;
    it.b = q2 - q3 * dcb.d;
    it.row0 = q3 * (16 * MT);
    if (MODE == CA_SINGLE) ca_body<FMT, D, 1, MT, 1, WV, T>(p, pl, it, sh);
    else if (MODE == CA_MIXED && !it.pre) ca_body<FMT, D, 1, MT, 1, WV, T>(p, pl, it, sh);
    else if (MODE == CA_SMALL && !it.pre) ca_body<FMT, D, 1, MT, 4, WV, T>(p, pl, it, sh);
    else ca_body<FMT, D, MT, MT, WV, WV, T>(p, pl, it, sh);
}

// The id-th of a join's rows: ids go by (entry, KV head, query, head of the group), the order of the partial rows.
struct CaJoinRow { int b, hk, h, t, r, e, rp; };        // r of its entry's rows; entry e of the prefix and the row of those
__device__ __forceinline__ CaJoinRow ca_join_row(const SmxCachedAttnParams& p, const CaPlan& pl, int id) {
    CaJoinRow w;
    const int u = ca_div(pl.per, id);
    w.r = id - u * pl.per.d;
    w.b = ca_div(pl.hkv_, u);
    w.hk = u - w.b * pl.Hkv;
    w.t = ca_div(pl.g, w.r);
    w.h = w.hk * pl.G + w.r - w.t * pl.G;
    w.e = ca_div(pl.r_, w.b);
    w.rp = (w.b - w.e * pl.R) * pl.per.d + w.r;
    return w;
}
// where row r of entry e (of B) and KV head hk has its partial result of the first of ns splits
__device__ __forceinline__ long long ca_prow(const CaPlan& pl, int own, int r, int B, int e, int hk, int ns) {
    const int blk = r >> pl.mtl;
    const long long it = (((long long)blk * B + e) * pl.Hkv + hk) * ns;
    return (own ? (long long)pl.items_p * pl.sp + it * pl.so : it * pl.sp) + (r - (blk << pl.mtl));
}
template <int D, typename T>
__device__ __forceinline__ void ca_join_store(const SmxCachedAttnParams& p, const CaJoinRow& w, int dl, float m, float l, float o[4]) {
    T* out = reinterpret_cast<T*>(p.o) + w.b * p.o_bs + w.t * p.o_ts + w.h * p.o_hs + dl;
    const float inv = 1.f / l;
#pragma unroll
    for (int d = 0; d < 4; ++d) o[d] = l == 0.f ? 0.f : o[d] * inv;
    ca_store4(out, o);
    if (p.lse && dl == 0) p.lse[((long long)w.b * p.H + w.h) * p.Tq + w.t] = ca_lse(m, l);
}

// O = sum over the splits of both parts, in a fixed order: JW waves per (row, head, query), D / 4 lanes per split.  A lane's loads depend on nothing but
// the weights, and with four waves even 64 splits are four (D = 128: eight) of them.
template <int D, int JW, typename T>
__global__ __launch_bounds__(256) void attn_cached_join(SmxCachedAttnParams p, CaPlan pl) {
    enum { LD = D / 4, NG = 64 / LD * JW };
    const int lane = threadIdx.x & 63, tid = JW == 4 ? threadIdx.x : lane;
    const int id = JW == 4 ? blockIdx.x : blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (id >= p.B * p.H * p.Tq) return;
    const CaJoinRow w = ca_join_row(p, pl, id);
    const int grp = tid / LD, dl = tid % LD * 4;
    float m = CA_LOWEST, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int part = 0; part < 2; ++part) {
        const SmxKVCache& c = part ? p.own : p.pre;
        if (!c.k) continue;
        const int ns = part ? pl.nso : pl.nsp, e = part ? w.b : w.e, r = part ? w.r : w.rp;
        const int step = part ? pl.so : pl.sp;                  // partial rows from one split to the next
        const long long r0 = ca_prow(pl, part, r, c.B, e, w.hk, ns);
        const float* po = pl.po + r0 * D + dl;
        // at most 64 splits: a lane holds one's maximum and sum
        float ms = CA_LOWEST, ls = 0.f;
        if (lane < ns) {
            const float2 q = *reinterpret_cast<const float2*>(pl.pml + 2 * (r0 + (long long)lane * step));
            ms = q.x;
            ls = q.y;
        }
        const float M = fmaxf(m, wave_max(ms));
        const float f0 = m == M ? 1.f : ca_exp2(m - M), fs = ls == 0.f ? 0.f : ca_exp2(ms - M);
        l = l * f0 + wave_sum(ls * fs);
        m = M;
#pragma unroll
        for (int d = 0; d < 4; ++d) o[d] *= f0;
        for (int s0 = 0; s0 < ns; s0 += 4 * NG) {
            float4 q[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) q[u] = *reinterpret_cast<const float4*>(po + (long long)min(s0 + NG * u + grp, ns - 1) * step * D);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int s = s0 + NG * u + grp;
                const float f = __shfl(fs, s & 63, 64);
                if (s < ns) {                           // (an infinity times a weight of zero is not nothing)
                    o[0] = fmaf(q[u].x, f, o[0]);
                    o[1] = fmaf(q[u].y, f, o[1]);
                    o[2] = fmaf(q[u].z, f, o[2]);
                    o[3] = fmaf(q[u].w, f, o[3]);
                }
            }
        }
    }
#pragma unroll
    for (int k = LD; k < 64; k <<= 1)
#pragma unroll
        for (int d = 0; d < 4; ++d) o[d] += __shfl_xor(o[d], k, 64);
    if (JW == 4) {
        __shared__ __attribute__((aligned(16))) float so[JW][D];
        if (lane < LD) *reinterpret_cast<float4*>(&so[threadIdx.x >> 6][dl]) = make_float4(o[0], o[1], o[2], o[3]);
        __syncthreads();
#pragma unroll
        for (int d = 0; d < 4; ++d) o[d] = (so[0][dl + d] + so[1][dl + d]) + (so[2][dl + d] + so[3][dl + d]);
    }
    if (grp == 0) ca_join_store<D, T>(p, w, dl, m, l, o);
}

// The same where each part has one split (prefixes and own keys that are both short): D / 4 lanes per row and nothing to pass between them.
template <int D, typename T>
__global__ __launch_bounds__(256) void attn_cached_join2(SmxCachedAttnParams p, CaPlan pl) {
    enum { LD = D / 4 };
    const int id = blockIdx.x * (256 / LD) + threadIdx.x / LD, dl = threadIdx.x % LD * 4;
    if (id >= p.B * p.H * p.Tq) return;
    const CaJoinRow w = ca_join_row(p, pl, id);
    const long long ia = ca_prow(pl, 0, w.rp, p.pre.B, w.e, w.hk, 1), ib = ca_prow(pl, 1, w.r, p.own.B, w.b, w.hk, 1);
    const float2 qa = *reinterpret_cast<const float2*>(pl.pml + 2 * ia), qb = *reinterpret_cast<const float2*>(pl.pml + 2 * ib);
    const float4 a = *reinterpret_cast<const float4*>(pl.po + ia * D + dl), c = *reinterpret_cast<const float4*>(pl.po + ib * D + dl);
    const float m = fmaxf(qa.x, qb.x);
    const float fa = qa.y == 0.f ? 0.f : ca_exp2(qa.x - m), fb = qb.y == 0.f ? 0.f : ca_exp2(qb.x - m);
    float o[4] = {fmaf(c.x, fb, a.x * fa), fmaf(c.y, fb, a.y * fa), fmaf(c.z, fb, a.z * fa), fmaf(c.w, fb, a.w * fa)};
    ca_join_store<D, T>(p, w, dl, m, fmaf(qb.y, fb, qa.y * fa), o);
}
