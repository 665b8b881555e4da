// Writing K/V rows into an (8-bit) cache and reading them back.
//   x: the D elements of one token and head, a = max |x|
//   e4m3: scale = the smallest power of two with a / scale <= 448 (at least 2^-126; 1 for a = 0), code = nearest-even e4m3 of x / scale.  A
//         power of two divides exactly, so the code's 3 mantissa bits are the only rounding, and code * scale is exact in bf16.
//   int8: scale = max(a / 127, 2^-126) (1 for a = 0), code = nearest-even integer of x / scale, both quotients correctly rounded fp32.
// Both run at the HBM rate on long prompts (48 x 1 499 tokens x 16 heads of 64, bf16 -> int8: append 103 us = 4.4 TB/s, read 80 us = 5.6 TB/s; append has
// some eight vector instructions per element beside its loads) and in 3 - 4 us for a decoding step's token.
#include "kv_common.h"

// A row takes LPR = 2^lsh lanes of 8 elements; t runs fastest over the rows of a workgroup: a run of cache rows is contiguous (T x D elements), and
// a source row of a 64-wide bf16 head is one full 128-byte line.  A thread takes KV_ROWS rows, 256 / LPR apart: their loads are on the way
// together and the addressing is paid for once (one row each: 48 x 1 499 x 16 heads of 64, bf16 -> int8: 144 us, now 103).
#define KV_ROWS 4
struct KvWork { int b, h, t0, pos0, which, d0; };      // t0: the thread's first row; pos0: where row 0 of the entry goes
__device__ __forceinline__ KvWork kv_work(const SmxKVRowsParams& p, int lsh) {
    const int rpb = KV_ROWS << (8 - lsh);
    const unsigned tb = (p.T + rpb - 1) / rpb;
    unsigned id = blockIdx.x;                           // (uniform: scalar arithmetic)
    KvWork k;
    k.t0 = (int)(id % tb) * rpb + (threadIdx.x >> lsh);
    id /= tb;
    k.which = id & 1;
    id >>= 1;
    k.h = id % p.c.H;
    k.b = id / p.c.H;
    k.d0 = (threadIdx.x & ((1 << lsh) - 1)) * 8;
    k.pos0 = p.start ? p.start[k.b] : p.start0;
    return k;
}
// is row t there, and its position in the cache?  (outside: the row is dropped (append) / left alone (read))
__device__ __forceinline__ bool kv_has(const SmxKVRowsParams& p, const KvWork& k, int t) {
    const long long ps = (long long)k.pos0 + t;
    return t < p.T && ps >= 0 && ps < p.c.cap && k.d0 < p.c.D;
}

// 8 source elements as they come, their values, and the largest magnitude's bits (integer order is the order of the floats, and infinities / NaN,
// >= 0x7f800000, stay on top)
template <typename T> struct KvRaw;
template <> struct KvRaw<bf16_t> {
    uint4 u;
    __device__ __forceinline__ void load(const bf16_t* p) { u = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void zero() { u = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void values(float x[8]) const {
        const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) { x[2 * e] = __uint_as_float(w[e] << 16); x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u); }
    }
    __device__ __forceinline__ unsigned amax() const {
        typedef __attribute__((ext_vector_type(2))) unsigned short us2;
        union { unsigned u; us2 v; } a[4] = {{u.x & 0x7fff7fffu}, {u.y & 0x7fff7fffu}, {u.z & 0x7fff7fffu}, {u.w & 0x7fff7fffu}};
        a[0].v = __builtin_elementwise_max(__builtin_elementwise_max(a[0].v, a[1].v), __builtin_elementwise_max(a[2].v, a[3].v));
        return max(a[0].u << 16, a[0].u & 0xffff0000u);
    }
};
template <> struct KvRaw<float> {
    float x_[8];
    __device__ __forceinline__ void load(const float* p) { load8(p, x_); }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int e = 0; e < 8; ++e) x_[e] = 0.f;
    }
    __device__ __forceinline__ void values(float x[8]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = x_[e];
    }
    __device__ __forceinline__ unsigned amax() const {
        unsigned a = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) a = max(a, __float_as_uint(x_[e]) & 0x7fffffffu);
        return a;
    }
};
// maximum over the 2^lsh lanes of a row (DPP: neighbours, pairs, halves of 8, halves of 16; wider rows through LDS)
__device__ __forceinline__ unsigned kv_row_max(unsigned a, int lsh) {
    if (lsh > 0) a = max(a, (unsigned)__builtin_amdgcn_update_dpp(0, (int)a, 0xB1, 0xf, 0xf, true));
    if (lsh > 1) a = max(a, (unsigned)__builtin_amdgcn_update_dpp(0, (int)a, 0x4E, 0xf, 0xf, true));
    if (lsh > 2) a = max(a, (unsigned)__builtin_amdgcn_update_dpp(0, (int)a, 0x141, 0xf, 0xf, true));
    if (lsh > 3) a = max(a, (unsigned)__builtin_amdgcn_update_dpp(0, (int)a, 0x140, 0xf, 0xf, true));
    if (lsh > 4) a = max(a, (unsigned)__shfl_xor((int)a, 16, 64));
    return a;
}

template <int FMT, typename T>
__global__ __launch_bounds__(256) void kv_append_kernel(SmxKVRowsParams p, int lsh) {
    const KvWork k = kv_work(p, lsh);
    const int step = 256 >> lsh;
    const T* src = k.which ? reinterpret_cast<const T*>(p.v) + k.b * p.v_bs + k.h * p.v_hs : reinterpret_cast<const T*>(p.k) + k.b * p.k_bs + k.h * p.k_hs;
    const long long ts = k.which ? p.v_ts : p.k_ts;
    void* dst = k.which ? p.c.v : p.c.k;
    float* sc = k.which ? p.c.vs : p.c.ks;
    const long long base = (long long)k.b * p.c.bs + (long long)k.h * p.c.hs + k.d0;
    KvRaw<T> raw[KV_ROWS];
#pragma unroll
    for (int u = 0; u < KV_ROWS; ++u) {
        raw[u].zero();
        if (k.t0 + u * step < p.T && k.d0 < p.c.D) raw[u].load(src + (k.t0 + u * step) * ts + k.d0);
    }
#pragma unroll
    for (int u = 0; u < KV_ROWS; ++u) {
        const int t = k.t0 + u * step;
        const bool ok = kv_has(p, k, t);
        const long long pos = (long long)k.pos0 + t, off = base + pos * p.c.ts;
        float x[8];
        raw[u].values(x);
        if (FMT == SMX_KV_F32) {
            if (ok) store8(reinterpret_cast<float*>(dst) + off, x);
            continue;
        }
        if (FMT == SMX_KV_BF16) {
            if (ok) store8(reinterpret_cast<bf16_t*>(dst) + off, x);
            continue;
        }
        const unsigned a = kv_row_max(raw[u].amax(), lsh);
        const bool finite = a < 0x7f800000u;
        if (!finite)
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = 0.f;
        float scale;
        unsigned lo, hi;
        if (FMT == SMX_KV_E4M3) {
            // 448 = 1.75 * 2^8: exponent of a, one higher when its mantissa exceeds 1.75
            int e = (int)(a >> 23) - 8 + ((a & 0x7fffffu) > 0x600000u);
            e = max(e, 1);
            scale = a == 0 ? 1.f : __uint_as_float((unsigned)e << 23);
            const float inv = a == 0 ? 1.f : __uint_as_float((unsigned)(254 - e) << 23);     // 1 / scale, exact (e <= 247)
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] *= inv;
            int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
            lo = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], w, true);
            w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4], x[5], 0, false);
            hi = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x[6], x[7], w, true);
        } else {
            // The code is the nearest-even integer of the correctly rounded quotient x / scale, at most 127 in magnitude (a / scale <= 127 (1 +
            // 2^-23)).  x * (1 / scale) is within 127 * 2^-22 of that quotient, so both round to the same integer unless the product lies within
            // 2^-14 of a half: only then is the division carried out.  Adding 1.5 * 2^23 rounds, and leaves the integer in the low byte.
            const float magic = 12582912.f;
            scale = a == 0 ? 1.f : fmaxf(__fdiv_rn(__uint_as_float(a), 127.f), 0x1p-126f);
            const float inv = __builtin_amdgcn_rcpf(scale);
            float far = scale < 0x1p125f ? 0.f : 1.f;        // (a reciprocal that may be subnormal: always divide)
            unsigned c[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float q = x[i] * inv, r = __fadd_rn(q, magic);
                c[i] = __float_as_uint(r);
                far = fmaxf(far, fabsf(q - __fsub_rn(r, magic)));
            }
            if (!(far < 0.5f - 0x1p-14f))
#pragma unroll
                for (int i = 0; i < 8; ++i) c[i] = __float_as_uint(__fadd_rn(__fdiv_rn(x[i], scale), magic));
            lo = __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[3], c[2], 0x00000400u), __builtin_amdgcn_perm(c[1], c[0], 0x00000400u), 0x05040100u);
            hi = __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[7], c[6], 0x00000400u), __builtin_amdgcn_perm(c[5], c[4], 0x00000400u), 0x05040100u);
        }
        if (ok) {
            *reinterpret_cast<uint2*>(reinterpret_cast<unsigned char*>(dst) + off) = make_uint2(lo, hi);
            if (k.d0 == 0) sc[k.b * p.c.sbs + k.h * p.c.shs + pos] = finite ? scale : __uint_as_float(0x7fc00000u);
        }
    }
}

template <int FMT, typename T>
__global__ __launch_bounds__(256) void kv_read_kernel(SmxKVRowsParams p, int lsh) {
    const KvWork k = kv_work(p, lsh);
    const int step = 256 >> lsh;
    T* dst = k.which ? reinterpret_cast<T*>(p.v) + k.b * p.v_bs + k.h * p.v_hs : reinterpret_cast<T*>(p.k) + k.b * p.k_bs + k.h * p.k_hs;
    const long long ts = k.which ? p.v_ts : p.k_ts;
    const void* src = k.which ? p.c.v : p.c.k;
    const float* sc = (k.which ? p.c.vs : p.c.ks) + (FMT <= SMX_KV_INT8 ? k.b * p.c.sbs + k.h * p.c.shs : 0);
    const long long base = (long long)k.b * p.c.bs + (long long)k.h * p.c.hs + k.d0;
    float x[KV_ROWS][8], s[KV_ROWS];
    bool ok[KV_ROWS];
#pragma unroll
    for (int u = 0; u < KV_ROWS; ++u) {
        ok[u] = kv_has(p, k, k.t0 + u * step);
        const long long pos = (long long)k.pos0 + k.t0 + u * step;
        if (ok[u]) {
            kv_load8<FMT>(src, base + pos * p.c.ts, x[u]);
            if (FMT <= SMX_KV_INT8) s[u] = sc[pos];
        }
    }
#pragma unroll
    for (int u = 0; u < KV_ROWS; ++u)
        if (ok[u]) {
            if (FMT <= SMX_KV_INT8)
#pragma unroll
                for (int e = 0; e < 8; ++e) x[u][e] *= s[u];
            store8(dst + (k.t0 + u * step) * ts + k.d0, x[u]);
        }
}

static int kv_rows_check(const SmxKVRowsParams& p, int dtype, int& lsh, unsigned& blocks) {
    int rc = kv_cache_check(p.c);
    if (rc) return rc;
    if (!p.k || !p.v || p.T < 0 || (dtype != SMX_F32 && dtype != SMX_BF16)) return SMX_EINVAL;
    if ((((size_t)p.k | (size_t)p.v) & 15) || ((p.k_bs | p.k_ts | p.k_hs | p.v_bs | p.v_ts | p.v_hs) & 7)) return SMX_EINVAL;
    for (lsh = 0; (8 << lsh) < p.c.D; ++lsh) {}
    const int rpb = KV_ROWS << (8 - lsh);
    const long long n = 2ll * p.c.B * p.c.H * ((p.T + rpb - 1) / rpb);
    if (n > 0x7fffffffll) return SMX_EINVAL;
    blocks = (unsigned)n;
    return SMX_OK;
}

#define KV_LAUNCH(KERNEL, FMT)                                                                                           \
    do {                                                                                                                 \
        if (dtype == SMX_BF16) hipLaunchKernelGGL((KERNEL<FMT, bf16_t>), dim3(blocks), dim3(256), 0, stream, *pp, lsh);  \
        else hipLaunchKernelGGL((KERNEL<FMT, float>), dim3(blocks), dim3(256), 0, stream, *pp, lsh);                     \
    } while (0)
#define KV_DISPATCH(KERNEL)                                                     \
    (void)hipGetLastError();                                                    \
    int lsh;                                                                    \
    unsigned blocks;                                                            \
    const int rc = kv_rows_check(*pp, dtype, lsh, blocks);                      \
    if (rc || blocks == 0) return rc;                                           \
    switch (pp->c.fmt) {                                                        \
        case SMX_KV_E4M3: KV_LAUNCH(KERNEL, SMX_KV_E4M3); break;                \
        case SMX_KV_INT8: KV_LAUNCH(KERNEL, SMX_KV_INT8); break;                \
        case SMX_KV_BF16: KV_LAUNCH(KERNEL, SMX_KV_BF16); break;                \
        default: KV_LAUNCH(KERNEL, SMX_KV_F32);                                 \
    }                                                                           \
    SMX_CHECK_LAUNCH()

extern "C" int smx_kv_append(const SmxKVRowsParams* pp, int dtype, hipStream_t stream) { KV_DISPATCH(kv_append_kernel); }
extern "C" int smx_kv_read(const SmxKVRowsParams* pp, int dtype, hipStream_t stream) { KV_DISPATCH(kv_read_kernel); }
extern "C" int smx_sizeof_SmxKVCache(void) { return (int)sizeof(SmxKVCache); }
extern "C" int smx_sizeof_SmxKVRowsParams(void) { return (int)sizeof(SmxKVRowsParams); }
