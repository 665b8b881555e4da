// Attention of Tq >= 1 new tokens per row over a K/V cache, optionally behind a prefix that the rows of a group share.
//   S[t, j] = scale * k_scale[j] * (q_t . k_code[j]) + rel_bias[h, clamp(qpos - kpos, 0, nrel - 1)]
//   O_t = sum_j p_j v_scale[j] v_code[j] / sum_j p_j,  p_j = exp(S - max),  lse = max + log(sum_j p_j)
// over the plen[g] prefix keys (all visible; positions 0 .. plen - 1) and the klen[b] own keys (positions plen + j).  The Tq queries are the
// last Tq own positions: query t sits at plen + klen - Tq + t, and with `causal` sees own keys up to itself.  No visible key: O = 0, lse = -inf.
#include <algorithm>
#include "kv_common.h"

__device__ __forceinline__ int ca_len(const int* len, int i, int cap) { return len ? min(max(len[i], 0), cap) : cap; }

// ---- general kernel (head widths other than 64 / 128, fp32 caches): one wave per (row, head, query) --------------------------------------
// 64 keys at a time: a lane takes one key's score, the wave shares maximum and sum, then a lane owns output elements d = lane + 64 i.
template <int FMT, typename T>
__global__ __launch_bounds__(256) void attn_cached_simple(SmxCachedAttnParams p) {
    __shared__ float sq[4][SMX_KV_MAXD];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const long long id = (long long)blockIdx.x * 4 + w;
    if (id >= (long long)p.B * p.H * p.Tq) return;            // (whole waves; no barrier below)
    const int t = (int)(id % p.Tq), h = (int)(id / p.Tq % p.H), b = (int)(id / ((long long)p.Tq * p.H));
    const int D = p.own.k ? p.own.D : p.pre.D, Hkv = p.own.k ? p.own.H : p.pre.H, hk = h / (p.H / Hkv);
    const T* q = reinterpret_cast<const T*>(p.q) + b * p.q_bs + t * p.q_ts + h * p.q_hs;
    for (int d = lane; d < D; d += 64) sq[w][d] = Cvt<T>::ld(q + d);
    __builtin_amdgcn_wave_barrier();
    const int g = p.pre.k ? b / (p.B / p.pre.B) : 0;
    const int np = p.pre.k ? ca_len(p.plen, g, p.pre.cap) : 0, nk = p.own.k ? ca_len(p.klen, b, p.own.cap) : 0;
    const int qpos = np + nk - p.Tq + t;
    float m = -INFINITY, l = 0.f, o[SMX_KV_MAXD / 64] = {0.f, 0.f, 0.f, 0.f};
    for (int part = 0; part < 2; ++part) {
        const SmxKVCache& c = part ? p.own : p.pre;
        const int n = part ? (p.causal ? min(nk, max(nk - p.Tq + t + 1, 0)) : nk) : np;
        const int pos0 = part ? np : 0, cb = part ? b : g;
        const long long base = cb * c.bs + hk * c.hs, sbase = cb * c.sbs + hk * c.shs;
        for (int j0 = 0; j0 < n; j0 += 64) {
            const int j = j0 + lane;
            float s = -INFINITY, vscale = 1.f;
            if (j < n) {
                float a = 0.f;
                for (int d = 0; d < D; d += 8) {
                    float kv[8];
                    kv_load8<FMT>(c.k, base + j * c.ts + d, kv);
#pragma unroll
                    for (int e = 0; e < 8; ++e) a = fmaf(sq[w][d + e], kv[e], a);
                }
                if (FMT <= SMX_KV_INT8) {
                    a *= c.ks[sbase + j];
                    vscale = c.vs[sbase + j];
                }
                s = a * p.scale;
                if (p.rel_bias) s += p.rel_bias[(long long)h * p.nrel + min(max(qpos - pos0 - j, 0), p.nrel - 1)];
            }
            const float mn = fmaxf(m, wave_max(s));
            const float ref = mn == -INFINITY ? 0.f : mn;
            const float alpha = expf(m - ref), e = j < n ? expf(s - ref) : 0.f;
            l = l * alpha + wave_sum(e);
            m = mn;
            const float ev = j < n ? e * vscale : 0.f;
#pragma unroll
            for (int i = 0; i < SMX_KV_MAXD / 64; ++i) o[i] *= alpha;
            const int cnt = min(64, n - j0);
            for (int tt = 0; tt < cnt; ++tt) {
                const float pt = __shfl(ev, tt, 64);
#pragma unroll
                for (int i = 0; i < SMX_KV_MAXD / 64; ++i)
                    if (lane + 64 * i < D) o[i] = fmaf(pt, kv_load1<FMT>(c.v, base + (j0 + tt) * c.ts + lane + 64 * i), o[i]);
            }
        }
    }
    T* out = reinterpret_cast<T*>(p.o) + b * p.o_bs + t * p.o_ts + h * p.o_hs;
#pragma unroll
    for (int i = 0; i < SMX_KV_MAXD / 64; ++i)
        if (lane + 64 * i < D) Cvt<T>::st(out + lane + 64 * i, l == 0.f ? 0.f : o[i] / l);
    if (p.lse && lane == 0) p.lse[((long long)b * p.H + h) * p.Tq + t] = l == 0.f ? -INFINITY : m + logf(l);
}

// The call as the kernels take it: the token stride of a cache of one token means nothing, but blocks of keys are addressed by it (what lies past the last
// key must lie past the end of the buffer).
static SmxCachedAttnParams ca_params(SmxCachedAttnParams p) {
    for (SmxKVCache* c : {&p.own, &p.pre})
        if (c->k && c->cap == 1) c->ts = c->D;
    return p;
}
static int ca_check(const SmxCachedAttnParams& p, int dtype) {
    if (!p.q || !p.o || p.B <= 0 || p.Tq <= 0 || p.H <= 0 || (dtype != SMX_F32 && dtype != SMX_BF16)) return SMX_EINVAL;
    if (!p.own.k && !p.pre.k) return SMX_EINVAL;
    for (const SmxKVCache* c : {&p.own, &p.pre})
        if (c->k && kv_cache_check(*c)) return SMX_EINVAL;
    if (p.own.k && p.own.B != p.B) return SMX_EINVAL;
    if (p.pre.k && p.B % p.pre.B) return SMX_EINVAL;
    if (p.own.k && p.pre.k && (p.own.D != p.pre.D || p.own.H != p.pre.H || p.own.fmt != p.pre.fmt)) return SMX_EINVAL;
    if (p.H % (p.own.k ? p.own.H : p.pre.H)) return SMX_EINVAL;
    if (p.rel_bias && p.nrel <= 0) return SMX_EINVAL;
    if ((((size_t)p.q | (size_t)p.o) & 15) || ((p.q_bs | p.q_ts | p.q_hs | p.o_bs | p.o_ts | p.o_hs) & 7)) return SMX_EINVAL;
    if ((long long)p.B * p.H * p.Tq > 0x7fff0000ll) return SMX_EINVAL;
    // positions and key counts are 32-bit
    if ((long long)(p.own.k ? p.own.cap : 0) + (p.pre.k ? p.pre.cap : 0) + p.Tq > 0x7fff0000ll) return SMX_EINVAL;
    return SMX_OK;
}

#include "attention_cached_mfma.h"

// ---- host ----
// The matrix-core kernel takes head widths 64 and 128 and every format but f32, where a 16-byte piece of a key is aligned and the offsets of 64
// keys fit 31 bits.
static bool ca_mfma_ok(const SmxCachedAttnParams& p) {
    const SmxKVCache& m = p.own.k ? p.own : p.pre;
    if (m.fmt == SMX_KV_F32 || (m.D != 64 && m.D != 128)) return false;
    for (const SmxKVCache* c : {&p.own, &p.pre})
        if (c->k) {
            const int es = kv_es(c->fmt);
            if (((c->bs | c->hs | c->ts) * es) & 15) return false;
            if (c->ts < 0 || c->ts * es > (1ll << 24)) return false;
        }
    return true;
}
static int ca_cdiv(long long a, long long b) { return (int)((a + b - 1) / b); }
#define CA_SHORT 256          // keys of a cache that one wave takes
// Splits of `cap` keys for `base` workgroups: up to `want` workgroups.  A split costs the second launch (4 us) and its partial rows, so it has to take
// at least 512 keys (256 where few workgroups share the chip), and 2 048 where the rows alone already give it a workgroup per CU (32 x 16 heads x 777 keys: one launch 13 us,
// two splits 14 + 4; 16 x 16 heads x 8 192 int8 keys: 84 us unsplit, 52 in four).  Up to `one` keys are not split at all.
static int ca_splits(long long base, int cap, long long want, int one) {
    if (cap <= one) return 1;
    const long long n = want / base, most = ca_cdiv(cap, base >= 256 ? 2048 : base >= 64 ? 512 : 256);
    const long long m = n < most ? n : most;
    return (int)(m < 1 ? 1 : m > 64 ? 64 : m);
}
static CaDiv ca_divisor(int d) {
    CaDiv v = {0u, 0, d};
    while ((1ll << v.k) < d) ++v.k;
    v.m = (unsigned)(((1ull << (31 + v.k)) + d - 1) / d);
    return v;
}
static void ca_plan_mt(const SmxCachedAttnParams& p, int mt, bool all1, CaPlan& pl, long long& items) {
    const SmxKVCache& m = p.own.k ? p.own : p.pre;
    const long long ro = p.own.k ? (long long)p.Tq * pl.G : 0, rp = p.pre.k ? (long long)pl.R * p.Tq * pl.G : 0;
    pl.mbo = ca_cdiv(ro, 16 * mt);
    pl.mbp = ca_cdiv(rp, 16 * mt);
    const long long bo = (long long)pl.mbo * p.own.B * pl.Hkv, bp = (long long)pl.mbp * p.pre.B * pl.Hkv;
    // what is resident at once: four workgroups per CU of the small form, two or three of the others; a prefix gets what its rows' own keys leave
    const long long want = mt == 1 && m.D == 64 ? 1024 : 512;
    // a wave per item where there are many items of few keys: a workgroup's other three waves would have nothing to do (16 384 rows and heads of
    // 43 keys behind prefixes: 151 us with a workgroup each, 55 so)
    // What a single launch gets through sooner than two, one tile of rows per item (16 heads of 64, 300 keys: 4.9 us for 7.4, 777: 7.2 for 7.5,
    // 1 000: 8.2 for 7.6; 192 of them, 1 000 keys: 9.3 for 11.8; 16 heads of 128, 500 keys: 8.2 for 8.6, 777: 11.4 for 8.6; 192, 1 000 keys: 15.2
    // for 16.0); two parts are joined in any case, but sooner where each has one result (8 rows x 12 heads of 64, 30 keys behind 300 and 500: 6.9 and 7.8
    // us for 8.8 and 8.8; heads of 128, 500 keys: 10.2 for 10.0; in items of 64 rows 15.6 for 14.2).
    const long long b1 = p.own.k ? bo : bp;
    const int one = mt > 1 ? 0 : p.own.k && p.pre.k ? (m.D == 64 ? 512 : 0) : m.D == 64 ? (b1 >= 64 ? 1024 : 768) : b1 >= 128 ? 1024 : 512;
    pl.single = all1 ? 2 : p.own.k && ro <= 16 && p.own.cap <= CA_SHORT && bo > 512;
    pl.nso = !p.own.k ? 0 : pl.single ? 1 : ca_splits(bo, p.own.cap, want, one);
    const long long left = want - (pl.single ? 0 : bo * pl.nso);        // (those of short caches are soon gone)
    pl.nsp = !p.pre.k ? 0 : all1 ? 1 : ca_splits(bp, p.pre.cap, left > want / 2 ? left : want / 2, one);
    pl.nso_ = ca_divisor(pl.nso > 0 ? pl.nso : 1);
    pl.nsp_ = ca_divisor(pl.nsp > 0 ? pl.nsp : 1);
    pl.items_p = (int)(bp * pl.nsp);
    pl.items_o = (int)(bo * pl.nso);
    items = bp * pl.nsp + bo * pl.nso;
    pl.join = pl.nso + pl.nsp > 1;
    pl.mtl = mt == 1 ? 4 : mt == 2 ? 5 : 6;
    pl.so = pl.mbo == 1 ? (int)ro : 16 * mt;
    pl.sp = pl.mbp == 1 ? (int)rp : 16 * mt;
}
static int ca_plan(const SmxCachedAttnParams& p, int dtype, CaPlan& pl, long long& items) {
    const SmxKVCache& m = p.own.k ? p.own : p.pre;
    pl.Hkv = m.H;
    pl.G = p.H / m.H;
    pl.R = p.pre.k ? p.B / p.pre.B : 1;
    pl.r_ = ca_divisor(pl.R);
    pl.per = ca_divisor(p.Tq * pl.G);
    pl.g = ca_divisor(pl.G);
    pl.hkv_ = ca_divisor(pl.Hkv);
    pl.bo_ = ca_divisor(p.own.k ? p.own.B : 1);
    pl.bp_ = ca_divisor(p.pre.k ? p.pre.B : 1);
    const long long ro = p.own.k ? (long long)p.Tq * pl.G : 0, rp = p.pre.k ? (long long)pl.R * p.Tq * pl.G : 0, rmax = ro > rp ? ro : rp;
    int mt = dtype == SMX_F32 || rmax <= 16 ? 1 : rmax <= 32 || m.D == 128 ? 2 : 4;
    // (own keys that outweigh the prefix's decide: more of their small items are resident beside a small form)
    if (p.own.k && p.pre.k && ro <= 16 && (long long)p.own.B * p.own.cap > (rp + 15) / 16 * p.pre.B * (long long)p.pre.cap) mt = 1;
    // Every item to a wave of its own, 16 rows each: a prefix's keys are converted again for every 16 of its rows, but no waves have to meet.  With
    // own keys where those are many and short and the prefix is not long (16 384 rows and heads of 17 keys behind 16 prefixes of 450, D 64: 39.2 us
    // in items of 64 rows, 29.6 so; of 100: 27.1 and 25.1; 4 096 of them: no gain); a prefix alone where the rows are many, but not the keys, of
    // bf16 of 64 or fp32 of 128 (16 prefixes x 16 heads x 64 rows, bf16, D 64, 60 keys: 9.3 and 7.0, 250: 11.3 and 10.4, 500: 15.0 and 19.8; fp32,
    // D 128, 30 keys: 14.1 and 9.6, 250: 20.4 and 19.3; against it bf16, D 128, 200 keys: 11.9 and 14.5, and fp32, D 64, 60 keys: 7.8 and 8.3).
    const bool all1 = p.own.k && p.pre.k ? ro <= 16 && (long long)p.own.B * pl.Hkv >= 8192 && p.own.cap <= CA_SHORT && p.pre.cap <= 2 * CA_SHORT
                    : p.pre.k && rp > 16 && (rp + 15) / 16 * p.pre.B * pl.Hkv >= 1024 && p.pre.cap <= CA_SHORT && (m.D == 64) == (dtype == SMX_BF16);
    if (all1) {
        ca_plan_mt(p, 1, true, pl, items);
        return 1;
    }
    ca_plan_mt(p, mt, false, pl, items);
    // Fewer rows per item while that leaves CUs idle: a block of keys takes 2.5 us for 64 rows and 0.9 for 16 (33 rows x 171 keys x 12 heads: 11.0 us
    // in 12 workgroups, 5.7 in 36).
    while (mt > 1 && items < 256) {
        mt >>= 1;
        ca_plan_mt(p, mt, false, pl, items);
    }
    return mt;
}

static long long ca_prows(const CaPlan& pl) { return (long long)pl.items_p * pl.sp + (long long)pl.items_o * pl.so; }

// bytes of workspace smx_attention_cached needs for these sizes (0: none)
extern "C" long long smx_attention_cached_ws_bytes(const SmxCachedAttnParams* pp, int dtype) {
    if (ca_check(*pp, dtype)) return SMX_EINVAL;
    const SmxCachedAttnParams p = ca_params(*pp);
    if (!ca_mfma_ok(p)) return 0;
    CaPlan pl;
    long long items;
    ca_plan(p, dtype, pl, items);
    return pl.join ? ca_prows(pl) * ((p.own.k ? p.own.D : p.pre.D) + 2) * 4 : 0;
}

#define CA_SIMPLE(FMT)                                                                                                                \
    do {                                                                                                                              \
        const unsigned n = (unsigned)(((long long)p.B * p.H * p.Tq + 3) / 4);                                                         \
        if (dtype == SMX_BF16) hipLaunchKernelGGL((attn_cached_simple<FMT, bf16_t>), dim3(n), dim3(256), 0, stream, p);               \
        else hipLaunchKernelGGL((attn_cached_simple<FMT, float>), dim3(n), dim3(256), 0, stream, p);                                  \
    } while (0)
#define CA_GO(FMT, D, MT, MODE, T) hipLaunchKernelGGL((attn_cached_mfma<FMT, D, MT, MODE, T>), grid, dim3(mode == CA_EIGHT ? 512 : 256), 0, stream, p, pl)
#define CA_MODE1(FMT, D, T)                                           \
    do {                                                              \
        if (mode == CA_SINGLE) CA_GO(FMT, D, 1, CA_SINGLE, T);        \
        else if (mode == CA_MIXED) CA_GO(FMT, D, 1, CA_MIXED, T);     \
        else if (D == 64 && mode == CA_EIGHT) CA_GO(FMT, 64, 1, CA_EIGHT, T); \
        else CA_GO(FMT, D, 1, CA_PLAIN, T);                           \
    } while (0)
#define CA_MODEN(FMT, D, MT, T)                                       \
    do {                                                              \
        if (mode == CA_SMALL) CA_GO(FMT, D, MT, CA_SMALL, T);         \
        else if (mode == CA_MIXED) CA_GO(FMT, D, MT, CA_MIXED, T);    \
        else CA_GO(FMT, D, MT, CA_PLAIN, T);                          \
    } while (0)
#define CA_MFMA_D(FMT, D)                                             \
    do {                                                              \
        if (dtype == SMX_F32) CA_MODE1(FMT, D, float);                \
        else if (mt == 1) CA_MODE1(FMT, D, bf16_t);                   \
        else if (mt == 2) CA_MODEN(FMT, D, 2, bf16_t);                \
        else CA_MODEN(FMT, D, (D == 64 ? 4 : 2), bf16_t);             \
    } while (0)
#define CA_MFMA(FMT)                           \
    do {                                       \
        if (D == 64) CA_MFMA_D(FMT, 64);       \
        else CA_MFMA_D(FMT, 128);              \
    } while (0)

#define CA_JOIN_T(D, T)                                                                                                               \
    do {                                                                                                                              \
        if (pair) hipLaunchKernelGGL((attn_cached_join2<D, T>), jg, dim3(256), 0, stream, p, pl);                            \
        else if (wide) hipLaunchKernelGGL((attn_cached_join<D, 4, T>), jg, dim3(256), 0, stream, p, pl);                          \
        else hipLaunchKernelGGL((attn_cached_join<D, 1, T>), jg, dim3(256), 0, stream, p, pl);                               \
    } while (0)
#define CA_JOIN(D)                                 \
    do {                                           \
        if (dtype == SMX_F32) CA_JOIN_T(D, float); \
        else CA_JOIN_T(D, bf16_t);                 \
    } while (0)

extern "C" int smx_attention_cached(const SmxCachedAttnParams* pp, int dtype, hipStream_t stream) {
    (void)hipGetLastError();
    const int rc = ca_check(*pp, dtype);
    if (rc) return rc;
    const SmxCachedAttnParams p = ca_params(*pp);
    const int fmt = p.own.k ? p.own.fmt : p.pre.fmt, D = p.own.k ? p.own.D : p.pre.D;
    if (ca_mfma_ok(p)) {
        CaPlan pl;
        long long items;
        const int mt = ca_plan(p, dtype, pl, items);
        if (items > 0x7fffffffll) return SMX_EINVAL;
        if (pl.join) {
            const long long rows = ca_prows(pl);
            if (!p.ws || ((size_t)p.ws & 15) || p.ws_bytes < rows * (D + 2) * 4) return SMX_EINVAL;
            pl.po = (float*)p.ws;
            pl.pml = pl.po + rows * D;
        }
        const bool few = p.own.k && p.pre.k && (long long)p.Tq * pl.G <= 16;
        // keys a workgroup may have to go through; eight waves halve that where the chip has room for them (32 x 16 heads x 777 keys, five queries:
        // 13.5 -> 12.2 us; heads of 128 have no room: 64 x 8 x 512 11.6 -> 14.3)
        const int keys = std::max(p.own.k ? p.own.cap / pl.nso : 0, p.pre.k ? p.pre.cap / pl.nsp : 0);
        const int mode = pl.single ? (p.pre.k && pl.single == 1 ? CA_MIXED : CA_SINGLE) : mt > 1 && few ? CA_SMALL : mt == 1 && D == 64 && items <= 512 && keys >= 256 ? CA_EIGHT : CA_PLAIN;
        const dim3 grid((unsigned)(mode == CA_SINGLE ? (items + 3) / 4 : pl.items_p + (pl.single ? (pl.items_o + 3) / 4 : pl.items_o)));
        if (fmt == SMX_KV_E4M3) CA_MFMA(SMX_KV_E4M3);
        else if (fmt == SMX_KV_INT8) CA_MFMA(SMX_KV_INT8);
        else CA_MFMA(SMX_KV_BF16);
        if (pl.join) {
            const long long rows = (long long)p.B * p.H * p.Tq;
            // a workgroup per row where there are many splits to add (64 splits of 128 wide: 7.7 us by a wave, 5.3 by four)
            const bool wide = pl.nso > 8 || pl.nsp > 8;
            // (16 384 rows, D 64, of one split each: 17.0 us with a wave per row, 5.0 so)
            const bool pair = pl.nso == 1 && pl.nsp == 1;
            const int per = pair ? 1024 / D : wide ? 1 : 4;
            const dim3 jg((unsigned)((rows + per - 1) / per));
            if (D == 64) CA_JOIN(64);
            else CA_JOIN(128);
        }
    } else {
        switch (fmt) {
            case SMX_KV_E4M3: CA_SIMPLE(SMX_KV_E4M3); break;
            case SMX_KV_INT8: CA_SIMPLE(SMX_KV_INT8); break;
            case SMX_KV_BF16: CA_SIMPLE(SMX_KV_BF16); break;
            default: CA_SIMPLE(SMX_KV_F32);
        }
    }
    SMX_CHECK_LAUNCH();
}
extern "C" int smx_sizeof_SmxCachedAttnParams(void) { return (int)sizeof(SmxCachedAttnParams); }
