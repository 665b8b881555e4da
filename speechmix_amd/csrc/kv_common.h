// K/V cache of the decoding operators (kvcache.hip, attention_cached.hip): parameter blocks and the element formats.
//   e4m3 / int8: one byte per element ("codes") and one fp32 scale per (row, head, token); value = code * scale.  Codes are always finite: a
//   row that held a non-finite element is stored as zeros under a NaN scale, so that a masked token can never put a NaN into a product.
//   bf16 / f32: the values themselves, no scales.
#pragma once
#include "smx_common.h"

enum { SMX_KV_E4M3 = 0, SMX_KV_INT8 = 1, SMX_KV_BF16 = 2, SMX_KV_F32 = 3 };
#define SMX_KV_MAXD 256

struct SmxKVCache {
    void* k; void* v;          // codes / values: element (b, h, t, d) at b * bs + h * hs + t * ts + d
    float* ks; float* vs;      // scales (8-bit formats): (b, h, t) at b * sbs + h * shs + t
    long long bs, hs, ts, sbs, shs;
    int B, H, cap, D, fmt, _pad;
};
struct SmxKVRowsParams {
    SmxKVCache c;
    void* k; void* v;          // T new rows per batch entry (append: read; read: written); strides in elements, D contiguous
    const int* start;          // [B] position of the first of the T rows, or null: start0 for every entry
    long long k_bs, k_ts, k_hs, v_bs, v_ts, v_hs;
    int T, start0;
};
struct SmxCachedAttnParams {
    const void* q; void* o; float* lse;     // q, o: [B, Tq, H, D] through strides; lse [B, H, Tq] fp32 or null
    SmxKVCache own, pre;                    // k == null: absent.  pre.B groups of B / pre.B consecutive rows each
    const int *klen, *plen;                 // [B], [pre.B] valid tokens (null: the capacity)
    const float* rel_bias;                  // [H, nrel]: score += rel_bias[h, clamp(qpos - kpos, 0, nrel - 1)]
    long long q_bs, q_ts, q_hs, o_bs, o_ts, o_hs;
    void* ws; long long ws_bytes;
    int B, Tq, H, causal, nrel; float scale;
};

__host__ __device__ __forceinline__ int kv_es(int fmt) { return fmt == SMX_KV_F32 ? 4 : fmt == SMX_KV_BF16 ? 2 : 1; }

// 4 consecutive codes -> floats (without the scale)
template <int FMT>
__device__ __forceinline__ void kv_unpack4(unsigned u, float o[4]) {
    if (FMT == SMX_KV_E4M3) {
        const smx_f32x2_t a = __builtin_amdgcn_cvt_pk_f32_fp8((int)u, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)u, true);
        o[0] = a[0]; o[1] = a[1]; o[2] = b[0]; o[3] = b[1];
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (float)(signed char)(u >> (8 * e));
    }
}
// 8 consecutive elements at element offset `off` (a multiple of 8; the base is 16-byte aligned)
template <int FMT>
__device__ __forceinline__ void kv_load8(const void* base, long long off, float o[8]) {
    if (FMT == SMX_KV_F32) {
        load8(reinterpret_cast<const float*>(base) + off, o);
    } else if (FMT == SMX_KV_BF16) {
        load8(reinterpret_cast<const bf16_t*>(base) + off, o);
    } else {
        const uint2 u = *reinterpret_cast<const uint2*>(reinterpret_cast<const unsigned char*>(base) + off);
        kv_unpack4<FMT>(u.x, o);
        kv_unpack4<FMT>(u.y, o + 4);
    }
}
template <int FMT>
__device__ __forceinline__ float kv_load1(const void* base, long long off) {
    if (FMT == SMX_KV_F32) return reinterpret_cast<const float*>(base)[off];
    if (FMT == SMX_KV_BF16) return bf2f(reinterpret_cast<const bf16_t*>(base)[off]);
    const unsigned char c = reinterpret_cast<const unsigned char*>(base)[off];
    if (FMT == SMX_KV_INT8) return (float)(signed char)c;
    return __builtin_amdgcn_cvt_f32_fp8((int)c, 0);
}

// host: is this a cache the kernels can address?  (16-byte vector accesses: bases and strides in 8-element units)
static inline int kv_cache_check(const SmxKVCache& c) {
    if (!c.k || !c.v || c.B <= 0 || c.H <= 0 || c.cap <= 0 || c.D <= 0 || (c.D & 7) || c.D > SMX_KV_MAXD) return SMX_EINVAL;
    if (c.fmt < SMX_KV_E4M3 || c.fmt > SMX_KV_F32) return SMX_EINVAL;
    if ((c.fmt <= SMX_KV_INT8) != (c.ks && c.vs)) return SMX_EINVAL;
    if (((size_t)c.k | (size_t)c.v) & 15) return SMX_EINVAL;
    if ((c.bs | c.hs | c.ts) & 7) return SMX_EINVAL;
    return SMX_OK;
}
