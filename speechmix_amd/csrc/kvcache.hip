// Writing K/V rows into an (8-bit) cache and reading them back.
//   x: the D elements of one token and head, a = max |x|
//   e4m3: scale = the smallest power of two with a / scale <= 448 (at least 2^-126; 1 for a = 0), code = nearest-even e4m3 of x / scale.  A
//         power of two divides exactly, so the code's 3 mantissa bits are the only rounding, and code * scale is exact in bf16.
//   int8: scale = max(a / 127, 2^-126) (1 for a = 0), code = nearest-even integer of x / scale, both quotients correctly rounded fp32.
#include "kv_common.h"

// LPR lanes per row, 8 elements per lane; t runs fastest over the rows of a wave: a cache row run is contiguous (T x D bytes), and a source row
// of a 64-wide bf16 head is one full 128-byte line.
__device__ __forceinline__ bool kv_row(const SmxKVRowsParams& p, int lpr, int& b, int& h, int& t, int& which, int& pos, int& d0) {
    const int rpb = 256 / lpr;
    const int tblocks = (p.T + rpb - 1) / rpb;
    unsigned id = blockIdx.x;
    t = (int)(id % tblocks) * rpb + threadIdx.x / lpr;
    id /= tblocks;
    which = id & 1;
    id >>= 1;
    h = id % p.c.H;
    b = id / p.c.H;
    d0 = (threadIdx.x % lpr) * 8;
    if (t >= p.T) return false;
    const long long ps = (long long)(p.start ? p.start[b] : p.start0) + t;
    if (ps < 0 || ps >= p.c.cap) return false;         // a position outside the cache: the row is dropped (append) / left alone (read)
    pos = (int)ps;
    return true;
}

template <int FMT, typename T>
__global__ __launch_bounds__(256) void kv_append_kernel(SmxKVRowsParams p, int lpr) {
    int b, h, t, which, pos = 0, d0;
    const bool ok = kv_row(p, lpr, b, h, t, which, pos, d0) && d0 < p.c.D;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (ok) {
        const T* src = which ? reinterpret_cast<const T*>(p.v) + b * p.v_bs + t * p.v_ts + h * p.v_hs
                             : reinterpret_cast<const T*>(p.k) + b * p.k_bs + t * p.k_ts + h * p.k_hs;
        load8(src + d0, x);
    }
    const long long off = (long long)b * p.c.bs + (long long)h * p.c.hs + (long long)pos * p.c.ts + d0;
    void* dst = which ? p.c.v : p.c.k;
    if (FMT == SMX_KV_F32) {
        if (ok) store8(reinterpret_cast<float*>(dst) + off, x);
        return;
    }
    if (FMT == SMX_KV_BF16) {
        if (ok) store8(reinterpret_cast<bf16_t*>(dst) + off, x);
        return;
    }
    // integer maximum of the magnitude bits: the order of the floats, and infinities / NaN (>= 0x7f800000) stay on top
    unsigned a = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) a = max(a, __float_as_uint(x[e]) & 0x7fffffffu);
    for (int o = 1; o < lpr; o <<= 1) a = max(a, (unsigned)__shfl_xor((int)a, o, 64));
    const bool finite = a < 0x7f800000u;
    float scale;
    unsigned lo, hi;
    if (FMT == SMX_KV_E4M3) {
        // 448 = 1.75 * 2^8: exponent of a, one higher when its mantissa exceeds 1.75
        int e = (int)(a >> 23) - 8 + ((a & 0x7fffffu) > 0x600000u);
        e = max(e, 1);
        scale = a == 0 ? 1.f : __uint_as_float((unsigned)e << 23);
        const float inv = a == 0 ? 1.f : __uint_as_float((unsigned)(254 - e) << 23);     // 1 / scale, exact (e <= 247)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = finite ? x[i] * inv : 0.f;
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
        lo = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], w, true);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4], x[5], 0, false);
        hi = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x[6], x[7], w, true);
    } else {
        scale = a == 0 ? 1.f : fmaxf(__fdiv_rn(__uint_as_float(a), 127.f), 0x1p-126f);
        unsigned c[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float r = finite ? rintf(__fdiv_rn(x[i], scale)) : 0.f;
            c[i] = (unsigned)(int)fminf(fmaxf(r, -127.f), 127.f) & 0xffu;
        }
        lo = c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
        hi = c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24;
    }
    if (ok) {
        *reinterpret_cast<uint2*>(reinterpret_cast<unsigned char*>(dst) + off) = make_uint2(lo, hi);
        if (d0 == 0) (which ? p.c.vs : p.c.ks)[b * p.c.sbs + h * p.c.shs + pos] = finite ? scale : __uint_as_float(0x7fc00000u);
    }
}

template <int FMT, typename T>
__global__ __launch_bounds__(256) void kv_read_kernel(SmxKVRowsParams p, int lpr) {
    int b, h, t, which, pos = 0, d0;
    if (!kv_row(p, lpr, b, h, t, which, pos, d0) || d0 >= p.c.D) return;
    float x[8];
    kv_load8<FMT>(which ? p.c.v : p.c.k, (long long)b * p.c.bs + (long long)h * p.c.hs + (long long)pos * p.c.ts + d0, x);
    if (FMT <= SMX_KV_INT8) {
        const float s = (which ? p.c.vs : p.c.ks)[b * p.c.sbs + h * p.c.shs + pos];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= s;
    }
    T* dst = which ? reinterpret_cast<T*>(p.v) + b * p.v_bs + t * p.v_ts + h * p.v_hs
                   : reinterpret_cast<T*>(p.k) + b * p.k_bs + t * p.k_ts + h * p.k_hs;
    store8(dst + d0, x);
}

static int kv_rows_check(const SmxKVRowsParams& p, int dtype, int& lpr, unsigned& blocks) {
    int rc = kv_cache_check(p.c);
    if (rc) return rc;
    if (!p.k || !p.v || p.T < 0 || (dtype != SMX_F32 && dtype != SMX_BF16)) return SMX_EINVAL;
    if ((((size_t)p.k | (size_t)p.v) & 15) || ((p.k_bs | p.k_ts | p.k_hs | p.v_bs | p.v_ts | p.v_hs) & 7)) return SMX_EINVAL;
    for (lpr = 1; lpr * 8 < p.c.D; lpr <<= 1) {}
    const int rpb = 256 / lpr;
    const long long n = 2ll * p.c.B * p.c.H * ((p.T + rpb - 1) / rpb);
    if (n > 0x7fffffffll) return SMX_EINVAL;
    blocks = (unsigned)n;
    return SMX_OK;
}

#define KV_LAUNCH(KERNEL, FMT)                                                                                           \
    do {                                                                                                                 \
        if (dtype == SMX_BF16) hipLaunchKernelGGL((KERNEL<FMT, bf16_t>), dim3(blocks), dim3(256), 0, stream, *pp, lpr);  \
        else hipLaunchKernelGGL((KERNEL<FMT, float>), dim3(blocks), dim3(256), 0, stream, *pp, lpr);                     \
    } while (0)
#define KV_DISPATCH(KERNEL)                                                     \
    (void)hipGetLastError();                                                    \
    int lpr;                                                                    \
    unsigned blocks;                                                            \
    const int rc = kv_rows_check(*pp, dtype, lpr, blocks);                      \
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
