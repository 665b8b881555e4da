// Verification of drafted tokens against the target's probabilities, from given uniform numbers.
//   draft i of a row is accepted while  u_i * q_i(x_i) < p_i(x_i)  (an exact product in 64 bits); q = null: the drafts were picked, not drawn
//   (q_i is 1 at x_i).  At the first rejected draft r the next token is drawn from max(p_r - q_r, 0); when all n are accepted, or at an id
//   outside the vocabulary (the end of a shorter draft), from p itself.  Drawing: the smallest index whose running sum exceeds u_n * (the sum of
//   all weights); sums in 64 bits - the borders of 50 000 intervals lie closer than 32-bit sums are sure of.
//   u = null: greedy - draft i is accepted while it equals arg max p_i (ties: the lowest index; target may then hold logits).
#include "smx_common.h"

struct SmxVerifyParams {
    const float *target, *draft, *u;       // [B, n + 1, V], [B, n, V] or null, [B, n + 1] or null
    const long long* ids;                  // [B, n]
    int* accepted; long long* token;       // [B], [B]
    void* ws; long long ws_bytes;
    long long t_bs, t_ts, d_bs, d_ts, ids_bs, u_bs;      // element strides (vocabulary contiguous)
    int B, n, V, _pad;
};
#define VF_CHUNK 2048        // weights per workgroup: 256 threads x 8
#define VF_MAXN 64           // drafts per row: one wave decides them all

struct VfRow { const float *p, *q; int r, x; };     // weights of the next token: p - q clamped (q null: p, without index x)

__device__ __forceinline__ double vf_w(const VfRow& f, int i) {
    const double p = (double)f.p[i];
    if (i == f.x) return 0.0;
    return f.q ? fmax(p - (double)f.q[i], 0.0) : fmax(p, 0.0);        // (fmax: a NaN weighs nothing)
}
// number of accepted drafts of row b and the weights that follow; every thread of every wave calls it
__device__ __forceinline__ VfRow vf_accept(const SmxVerifyParams& p, int b) {
    const int i = threadIdx.x & 63;
    bool acc = false, valid = false;
    if (i < p.n) {
        const long long x = p.ids[b * p.ids_bs + i];
        valid = x >= 0 && x < p.V;
        if (valid) {
            const double pt = (double)p.target[b * p.t_bs + i * p.t_ts + x];
            const double qd = p.draft ? (double)p.draft[b * p.d_bs + i * p.d_ts + x] : 1.0;
            acc = (double)p.u[b * p.u_bs + i] * qd < pt;
        }
    }
    const unsigned long long no = ~__ballot(acc);
    VfRow f;
    f.r = no ? min(__ffsll((long long)no) - 1, p.n) : p.n;
    const bool rejected = f.r < p.n && ((__ballot(valid) >> f.r) & 1);
    f.p = p.target + b * p.t_bs + f.r * p.t_ts;
    f.q = rejected && p.draft ? p.draft + b * p.d_bs + f.r * p.d_ts : nullptr;
    f.x = rejected && !p.draft ? (int)p.ids[b * p.ids_bs + f.r] : -1;
    return f;
}
__device__ __forceinline__ double vf_wave_scan(double v) {             // inclusive, fixed order
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double u = __shfl_up(v, o, 64);
        if ((int)(threadIdx.x & 63) >= o) v += u;
    }
    return v;
}
// sum of the chunk's weights before this thread's eight (exclusive) and of all of them; sh: 4 doubles
__device__ __forceinline__ double vf_block_scan(double mine, double* sh, double& total) {
    const double inc = vf_wave_scan(mine);
    const int w = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 63) sh[w] = inc;
    __syncthreads();
    double base = 0.0;
    total = 0.0;
    for (int i = 0; i < 4; ++i) {
        if (i < w) base += sh[i];
        total += sh[i];
    }
    return base + inc - mine;
}
__device__ __forceinline__ double vf_chunk8(const VfRow& f, int c, int V, double w[8]) {
    double s = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int i = c * VF_CHUNK + threadIdx.x * 8 + e;
        w[e] = i < V ? vf_w(f, i) : 0.0;
        s += w[e];
    }
    return s;
}

__global__ __launch_bounds__(256) void verify_sums_kernel(SmxVerifyParams p, int nchunk, double* sums) {
    __shared__ double sh[4];
    const int c = blockIdx.x, b = blockIdx.y;
    const VfRow f = vf_accept(p, b);
    double w[8], total;
    vf_block_scan(vf_chunk8(f, c, p.V, w), sh, total);
    if (threadIdx.x == 0) sums[(long long)b * nchunk + c] = total;
}

__global__ __launch_bounds__(256) void verify_pick_kernel(SmxVerifyParams p, int nchunk, const double* sums) {
    __shared__ double sh[4];
    __shared__ int found, last;
    const int b = blockIdx.x, tid = threadIdx.x;
    VfRow f = vf_accept(p, b);
    double total = 0.0;
    for (int c = 0; c < nchunk; ++c) total += sums[(long long)b * nchunk + c];
    const bool none = !(total > 0.0);          // p <= q everywhere (rounding of their normalisation): the target's own weights
    if (none) {
        f.q = nullptr;
        f.x = -1;
        total = 0.0;
        for (int c = 0; c < nchunk; ++c) {
            double w[8], t;
            vf_block_scan(vf_chunk8(f, c, p.V, w), sh, t);
            total += t;
        }
    }
    const double goal = (double)p.u[b * p.u_bs + p.n] * total;
    if (tid == 0) { found = p.V; last = -1; }
    __syncthreads();
    double before = 0.0;
    for (int c = 0; c < nchunk; ++c) {
        if (!none) {
            const double s = sums[(long long)b * nchunk + c];
            if (before + s <= goal && c + 1 < nchunk) { before += s; continue; }
        }
        double w[8], t;
        double run = before + vf_block_scan(vf_chunk8(f, c, p.V, w), sh, t);
        for (int e = 0; e < 8; ++e) {
            const int i = c * VF_CHUNK + tid * 8 + e;
            run += w[e];
            if (w[e] > 0.0) {
                atomicMax(&last, i);
                if (run > goal) { atomicMin(&found, i); break; }
            }
        }
        __syncthreads();
        if (found < p.V) break;
        before += t;
    }
    if (found == p.V) {                        // u_n * total rounded up to the total: the last index that weighs anything
        for (int c = nchunk - 1; c >= 0 && last < 0; --c) {
            double w[8];
            vf_chunk8(f, c, p.V, w);
            __syncthreads();
            for (int e = 0; e < 8; ++e)
                if (w[e] > 0.0) atomicMax(&last, c * VF_CHUNK + tid * 8 + e);
            __syncthreads();
        }
    }
    if (tid == 0) {
        p.accepted[b] = f.r;
        p.token[b] = found < p.V ? found : max(last, 0);
    }
}

// ---- greedy ----
struct VfBest { float v; int i; };
__device__ __forceinline__ void vf_better(VfBest& a, float v, int i) {
    if (v > a.v || (v == a.v && i < a.i)) { a.v = v; a.i = i; }
}
__device__ __forceinline__ VfBest vf_wave_best(VfBest a) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) vf_better(a, __shfl_xor(a.v, o, 64), __shfl_xor(a.i, o, 64));
    return a;
}
__global__ __launch_bounds__(256) void verify_best_kernel(SmxVerifyParams p, int nchunk, VfBest* best) {
    __shared__ VfBest sh[4];
    const int c = blockIdx.x, i = blockIdx.y, b = blockIdx.z;
    const float* row = p.target + b * p.t_bs + i * p.t_ts;
    VfBest a = {-INFINITY, c * VF_CHUNK};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int j = c * VF_CHUNK + e * 256 + threadIdx.x;
        if (j < p.V) vf_better(a, row[j], j);
    }
    a = vf_wave_best(a);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = a;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 4; ++w) vf_better(a, sh[w].v, sh[w].i);
        best[((long long)b * (p.n + 1) + i) * nchunk + c] = a;
    }
}
__global__ __launch_bounds__(64) void verify_greedy_kernel(SmxVerifyParams p, int nchunk, const VfBest* best) {
    const int b = blockIdx.x, lane = threadIdx.x;
    for (int i = 0; i <= p.n; ++i) {
        const VfBest* row = best + ((long long)b * (p.n + 1) + i) * nchunk;
        VfBest a = {-INFINITY, 0};
        if (lane < nchunk) a = row[lane];
        for (int c = lane + 64; c < nchunk; c += 64) vf_better(a, row[c].v, row[c].i);
        if (lane >= nchunk) a.i = 0x7fffffff;
        a = vf_wave_best(a);
        if (i == p.n || p.ids[b * p.ids_bs + i] != a.i) {
            if (lane == 0) {
                p.accepted[b] = i;
                p.token[b] = a.i;
            }
            return;
        }
    }
}

static int vf_check(const SmxVerifyParams& p) {
    if (!p.target || !p.accepted || !p.token || p.B <= 0 || p.n < 0 || p.n > VF_MAXN || p.V <= 0) return SMX_EINVAL;
    if (p.n > 0 && !p.ids) return SMX_EINVAL;
    if (p.draft && !p.u) return SMX_EINVAL;
    if (p.B > 65535 || p.V > 0x7fffffff - VF_CHUNK) return SMX_EINVAL;
    return SMX_OK;
}
static int vf_chunks(const SmxVerifyParams& p) { return (p.V + VF_CHUNK - 1) / VF_CHUNK; }

extern "C" long long smx_verify_draft_ws_bytes(const SmxVerifyParams* p) {
    if (vf_check(*p)) return SMX_EINVAL;
    return 8ll * p->B * vf_chunks(*p) * (p->u ? 1 : p->n + 1);
}
extern "C" int smx_verify_draft(const SmxVerifyParams* pp, hipStream_t stream) {
    (void)hipGetLastError();
    const SmxVerifyParams p = *pp;
    const int rc = vf_check(p);
    if (rc) return rc;
    if (!p.ws || ((size_t)p.ws & 7) || p.ws_bytes < smx_verify_draft_ws_bytes(pp)) return SMX_EINVAL;
    const int nc = vf_chunks(p);
    if (p.u) {
        hipLaunchKernelGGL(verify_sums_kernel, dim3(nc, p.B), dim3(256), 0, stream, p, nc, (double*)p.ws);
        hipLaunchKernelGGL(verify_pick_kernel, dim3(p.B), dim3(256), 0, stream, p, nc, (const double*)p.ws);
    } else {
        hipLaunchKernelGGL(verify_best_kernel, dim3(nc, p.n + 1, p.B), dim3(256), 0, stream, p, nc, (VfBest*)p.ws);
        hipLaunchKernelGGL(verify_greedy_kernel, dim3(p.B), dim3(64), 0, stream, p, nc, (const VfBest*)p.ws);
    }
    SMX_CHECK_LAUNCH();
}
extern "C" int smx_sizeof_SmxVerifyParams(void) { return (int)sizeof(SmxVerifyParams); }
