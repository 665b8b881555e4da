// Attention of Tq >= 1 new tokens per row over a K/V cache, optionally behind a prefix that the rows of a group share.
//   S[t, j] = scale * k_scale[j] * (q_t . k_code[j]) + rel_bias[h, clamp(qpos - kpos, 0, nrel - 1)]
//   O_t = sum_j p_j v_scale[j] v_code[j] / sum_j p_j,  p_j = exp(S - max),  lse = max + log(sum_j p_j)
// over the plen[g] prefix keys (all visible; positions 0 .. plen - 1) and the klen[b] own keys (positions plen + j).  The Tq queries are the
// last Tq own positions: query t sits at plen + klen - Tq + t, and with `causal` sees own keys up to itself.  No visible key: O = 0, lse = -inf.
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
    if ((long long)p.B * p.H * p.Tq > 0x7fffffffll) return SMX_EINVAL;
    // positions and key counts are 32-bit
    if ((long long)(p.own.k ? p.own.cap : 0) + (p.pre.k ? p.pre.cap : 0) + p.Tq > 0x7fffffffll) return SMX_EINVAL;
    return SMX_OK;
}

#define CA_SIMPLE(FMT)                                                                                                                \
    do {                                                                                                                              \
        const unsigned n = (unsigned)(((long long)p.B * p.H * p.Tq + 3) / 4);                                                         \
        if (dtype == SMX_BF16) hipLaunchKernelGGL((attn_cached_simple<FMT, bf16_t>), dim3(n), dim3(256), 0, stream, p);               \
        else hipLaunchKernelGGL((attn_cached_simple<FMT, float>), dim3(n), dim3(256), 0, stream, p);                                  \
    } while (0)

// bytes of fp32 workspace smx_attention_cached needs for these sizes (0: none)
extern "C" long long smx_attention_cached_ws_bytes(const SmxCachedAttnParams* pp, int dtype) { return ca_check(*pp, dtype) ? SMX_EINVAL : 0; }

extern "C" int smx_attention_cached(const SmxCachedAttnParams* pp, int dtype, hipStream_t stream) {
    (void)hipGetLastError();
    const SmxCachedAttnParams p = *pp;
    const int rc = ca_check(p, dtype);
    if (rc) return rc;
    switch (p.own.k ? p.own.fmt : p.pre.fmt) {
        case SMX_KV_E4M3: CA_SIMPLE(SMX_KV_E4M3); break;
        case SMX_KV_INT8: CA_SIMPLE(SMX_KV_INT8); break;
        case SMX_KV_BF16: CA_SIMPLE(SMX_KV_BF16); break;
        default: CA_SIMPLE(SMX_KV_F32);
    }
    SMX_CHECK_LAUNCH();
}
extern "C" int smx_sizeof_SmxCachedAttnParams(void) { return (int)sizeof(SmxCachedAttnParams); }
