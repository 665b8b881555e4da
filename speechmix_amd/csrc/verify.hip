// Verification of drafted tokens against the target's probabilities, from given uniform numbers.
//   draft i of a row is accepted while  u_i * q_i(x_i) < p_i(x_i)  (an exact product in 64 bits); q = null: the drafts were picked, not drawn
//   (q_i is 1 at x_i).  At the first rejected draft r the next token is drawn from max(p_r - q_r, 0); when all n are accepted, or at an id
//   outside the vocabulary (the end of a shorter draft), from p itself.  Drawing: the smallest index whose running sum exceeds u_n * (the sum of
//   all weights); sums in 64 bits - the borders of 50 000 intervals lie closer than 32-bit sums are sure of.
// Bounds: a chain of dependent loads and scans, 5.4 us whatever the size (ids -> probabilities at the ids -> the row -> its sums -> the chosen segment
// again), and what one CU reads (100 GB/s) of the one or two rows that count: 64 rows of 50 265 with four drafts 11 us, 256 rows without drafts 13 us.
//   u = null: greedy - draft i is accepted while it equals arg max p_i (ties: the lowest index; target may then hold logits; a NaN is below
//   everything - a step whose logits broke draws the best of what is left, or 0).
#include "smx_common.h"

struct SmxVerifyParams {
    const float *target, *draft, *u;       // [B, n + 1, V], [B, n, V] or null, [B, n + 1] or null
    const long long* ids;                  // [B, n]
    int* accepted; long long* token;       // [B], [B]
    void* ws; long long ws_bytes;
    long long t_bs, t_ts, d_bs, d_ts, ids_bs, u_bs;      // element strides (vocabulary contiguous)
    int B, n, V, _pad;
};
#define VF_MAXN 64           // drafts per row: one wave decides them all
#define VF_WAVES 16          // a workgroup of 1 024 threads per row (or per piece of one)
#define VF_MAXC 64           // workgroups per row

struct VfRow { const float *p, *q; int r, x; float u; };     // weights of the next token: p - q clamped (q null: p, without index x); its uniform

__device__ __forceinline__ double vf_w(const VfRow& f, int i) {
    const double p = (double)f.p[i];
    if (i == f.x) return 0.0;
    return f.q ? fmax(p - (double)f.q[i], 0.0) : fmax(p, 0.0);        // (fmax: a NaN weighs nothing)
}
// number of accepted drafts of row b and the weights that follow; every thread of every wave calls it
__device__ __forceinline__ VfRow vf_accept(const SmxVerifyParams& p, int b) {
    const int i = threadIdx.x & 63;
    bool acc = false, valid = false;
    const float u_last = p.u[b * p.u_bs + p.n];        // (asked for here: its latency passes under the others')
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
    f.u = u_last;
    f.r = no ? min(__ffsll((long long)no) - 1, p.n) : p.n;
    const bool rejected = f.r < p.n && ((__ballot(valid) >> f.r) & 1);
    f.p = p.target + b * p.t_bs + f.r * p.t_ts;
    f.q = rejected && p.draft ? p.draft + b * p.d_bs + f.r * p.d_ts : nullptr;
    f.x = rejected && !p.draft ? (int)p.ids[b * p.ids_bs + f.r] : -1;
    return f;
}
// One step of a wave's scan: v + (v of another lane, or nothing), both halves of the number by DPP (a shuffle through LDS and its wait per step:
// a row of 64 weights took 7.5 us, now 5.4)
template <int CTRL, int ROWS>
__device__ __forceinline__ double vf_dpp_add(double v) {
    union { double d; int i[2]; } a = {v}, b;
    b.i[0] = __builtin_amdgcn_update_dpp(0, a.i[0], CTRL, ROWS, 0xf, true);
    b.i[1] = __builtin_amdgcn_update_dpp(0, a.i[1], CTRL, ROWS, 0xf, true);
    return v + b.d;
}
// inclusive, fixed order: within rows of 16 lanes (shifts by 1, 2, 4, 8), then row 0's end to row 1 and row 2's to row 3, then lane 31 to both upper rows
__device__ __forceinline__ double vf_wave_scan(double v) {
    v = vf_dpp_add<0x111, 0xf>(v);
    v = vf_dpp_add<0x112, 0xf>(v);
    v = vf_dpp_add<0x114, 0xf>(v);
    v = vf_dpp_add<0x118, 0xf>(v);
    v = vf_dpp_add<0x142, 0xa>(v);
    return vf_dpp_add<0x143, 0xc>(v);
}
__device__ __forceinline__ double vf_lane(double v, int lane) {        // (lane: the same for the whole wave)
    union { double d; int i[2]; } a = {v};
    a.i[0] = __builtin_amdgcn_readlane(a.i[0], lane);
    a.i[1] = __builtin_amdgcn_readlane(a.i[1], lane);
    return a.d;
}
// inclusive sum over the workgroup's threads; sh: VF_WAVES doubles
__device__ __forceinline__ double vf_block_scan(double v, double* sh) {
    const double inc = vf_wave_scan(v);
    const int w = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 63) sh[w] = inc;
    __syncthreads();
    // (every wave scans the sixteen totals in its lanes: a loop over them is sixteen dependent LDS reads)
    const double t = vf_wave_scan((threadIdx.x & 63) < VF_WAVES ? sh[threadIdx.x & 63] : 0.0);
    const double base = vf_lane(t, __builtin_amdgcn_readfirstlane(w ? w - 1 : 0));
    return w ? base + inc : inc;
}
struct __attribute__((packed, aligned(4))) VfF4 { float v[4]; };       // (rows of an odd vocabulary start at any multiple of 4 bytes)
__device__ __forceinline__ void vf_load4(const VfRow& f, int i, int hi, double w[4]) {
    if (i + 4 <= hi) {
        const VfF4 p = *reinterpret_cast<const VfF4*>(f.p + i);
        VfF4 q = {{0.f, 0.f, 0.f, 0.f}};
        if (f.q) q = *reinterpret_cast<const VfF4*>(f.q + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = i + e == f.x ? 0.0 : fmax((double)p.v[e] - (double)q.v[e], 0.0);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = i + e < hi ? vf_w(f, i + e) : 0.0;
    }
}
// sum of the weights lo .. hi - 1 by one wave.  Four pieces of each operand on the way: the loads stand before any of their uses, without a
// branch between them (with a check per load 64 rows of 50 265 took 31 us, now 13).
template <bool Q>
__device__ __forceinline__ double vf_wave_sum_(const VfRow& f, int lo, int hi) {
    const int lane = threadIdx.x & 63;
    double s = 0.0;
    int i = lo + 4 * lane;
    for (; i + 3 * 256 + 4 <= hi; i += 4 * 256) {
        VfF4 p[4], q[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) p[u] = *reinterpret_cast<const VfF4*>(f.p + i + 256 * u);
        if (Q)
#pragma unroll
            for (int u = 0; u < 4; ++u) q[u] = *reinterpret_cast<const VfF4*>(f.q + i + 256 * u);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            double w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                w[e] = Q ? fmax((double)p[u].v[e] - (double)q[u].v[e], 0.0) : (double)fmaxf(p[u].v[e], 0.f);
                if (!Q && i + 256 * u + e == f.x) w[e] = 0.0;
            }
            s += (w[0] + w[1]) + (w[2] + w[3]);
        }
    }
    for (; i < hi; i += 256) {
        double w[4];
        vf_load4(f, i, hi, w);
        s += (w[0] + w[1]) + (w[2] + w[3]);
    }
    return vf_lane(vf_wave_scan(s), 63);
}
__device__ __forceinline__ double vf_wave_sum(const VfRow& f, int lo, int hi) { return f.q ? vf_wave_sum_<true>(f, lo, hi) : vf_wave_sum_<false>(f, lo, hi); }
struct VfShared { double sh[VF_WAVES], before; int seg, lastseg, found, last; };
// *first = the lowest lane's a among those with `isa`, *last = the highest lane's z among those with `isz`, over the workgroup (a and z ascend
// with the lane).  One LDS atomic per wave: a thousand of them on one word took 7 us.
__device__ __forceinline__ void vf_first_last(bool isa, bool isz, int a, int z, int* first, int* last) {
    const unsigned long long ma = __ballot(isa), mz = __ballot(isz);
    const int fa = __shfl(a, ma ? __ffsll((long long)ma) - 1 : 0, 64), lz = __shfl(z, mz ? 63 - __clzll((long long)mz) : 0, 64);
    if ((threadIdx.x & 63) == 0) {
        if (ma) atomicMin(first, fa);
        if (mz) atomicMax(last, lz);
    }
}
// The segments' sums -> accepted, token.  mine: the sum of segment threadIdx.x (0 beyond the last of the S segments of `len` weights).
__device__ __forceinline__ void vf_pick(const SmxVerifyParams& p, int b, VfRow f, double mine, int S, int len, double* sums, VfShared& m) {
    const int tid = threadIdx.x, w = tid >> 6;
    double inc = vf_block_scan(mine, m.sh), total = 0.0;
    __syncthreads();
    if (tid == (int)blockDim.x - 1) m.before = inc;
    __syncthreads();
    total = m.before;
    if (!(total > 0.0) && (f.q || f.x >= 0)) {       // p <= q everywhere (rounding of their normalisation): the target's own weights
        f.q = nullptr;
        f.x = -1;
        for (int s = w; s < S; s += VF_WAVES) {
            const double t = vf_wave_sum(f, min(s * len, p.V), min((s + 1) * len, p.V));
            if ((tid & 63) == 0) sums[s] = t;
        }
        __syncthreads();
        mine = tid < S ? sums[tid] : 0.0;
        inc = vf_block_scan(mine, m.sh);
        __syncthreads();
        if (tid == (int)blockDim.x - 1) m.before = inc;
        __syncthreads();
        total = m.before;
    }
    const double goal = (double)f.u * total;
    if (tid == 0) {
        m.seg = 0x7fffffff;
        m.lastseg = 0;
        m.found = 0x7fffffff;
        m.last = 0;
    }
    __syncthreads();
    vf_first_last(mine > 0.0 && inc > goal, mine > 0.0, tid, tid, &m.seg, &m.lastseg);
    __syncthreads();
    const int seg = min(m.seg, m.lastseg);           // (u_n * total rounded up to the total: the last segment that weighs anything)
    if (tid == seg) m.before = inc - mine;
    __syncthreads();
    double before = m.before;
    const int hi = min((seg + 1) * len, p.V);
    for (int lo = seg * len; lo < hi; lo += 4 * 64 * VF_WAVES) {
        double x[4];
        const int i = lo + 4 * tid;
        if (i < hi) vf_load4(f, i, hi, x);
        else x[0] = x[1] = x[2] = x[3] = 0.0;
        const double own = (x[0] + x[1]) + (x[2] + x[3]), in2 = vf_block_scan(own, m.sh);
        double run = before + (in2 - own);
        int first = -1, lastw = -1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            run += x[e];
            if (x[e] > 0.0) {
                lastw = i + e;
                if (run > goal && first < 0) first = i + e;
            }
        }
        vf_first_last(first >= 0, lastw >= 0, first, lastw, &m.found, &m.last);
        __syncthreads();
        if (m.found != 0x7fffffff) break;
        if (tid == (int)blockDim.x - 1) m.before = before + in2;
        __syncthreads();
        before = m.before;
    }
    if (tid == 0) {
        p.accepted[b] = f.r;
        p.token[b] = min(m.found, m.last);           // (nothing above the goal in the segment: its last index with a weight)
    }
}

// One workgroup per row: accept, sum (a wave per sixteenth of the vocabulary), pick.
__global__ __launch_bounds__(1024) void verify_row_kernel(SmxVerifyParams p, int len) {
    __shared__ VfShared m;
    __shared__ double sums[VF_WAVES];
    const int b = blockIdx.x, w = threadIdx.x >> 6;
    const VfRow f = vf_accept(p, b);
    const double t = vf_wave_sum(f, min(w * len, p.V), min((w + 1) * len, p.V));
    if ((threadIdx.x & 63) == 0) sums[w] = t;
    __syncthreads();
    vf_pick(p, b, f, threadIdx.x < VF_WAVES ? sums[threadIdx.x] : 0.0, VF_WAVES, len, sums, m);
}
// Few rows: several workgroups sum one row's segments, a second launch picks.
__global__ __launch_bounds__(1024) void verify_sums_kernel(SmxVerifyParams p, int len, double* sums) {
    const int b = blockIdx.y, s = blockIdx.x * VF_WAVES + (threadIdx.x >> 6);
    const VfRow f = vf_accept(p, b);
    const double t = vf_wave_sum(f, min(s * len, p.V), min((s + 1) * len, p.V));
    if ((threadIdx.x & 63) == 0) sums[(long long)b * gridDim.x * VF_WAVES + s] = t;
}
__global__ __launch_bounds__(1024) void verify_pick_kernel(SmxVerifyParams p, int S, int len, double* sums) {
    __shared__ VfShared m;
    const int b = blockIdx.x;
    sums += (long long)b * S;
    vf_pick(p, b, vf_accept(p, b), threadIdx.x < S ? sums[threadIdx.x] : 0.0, S, len, sums, m);
}

// ---- greedy ----
struct VfBest { float v; int i; };
__device__ __forceinline__ void vf_better(VfBest& a, float v, int i) {
    if (v > a.v || (v == a.v && i < a.i)) { a.v = v; a.i = i; }
}
template <int CTRL, int ROWS>
__device__ __forceinline__ void vf_dpp_best(VfBest& a) {
    const float v = __uint_as_float((unsigned)__builtin_amdgcn_update_dpp((int)0xff800000, (int)__float_as_uint(a.v), CTRL, ROWS, 0xf, false));
    vf_better(a, v, __builtin_amdgcn_update_dpp(0x7fffffff, a.i, CTRL, ROWS, 0xf, false));       // (no such lane: -inf at the last index)
}
// the best of the wave, in every lane
__device__ __forceinline__ VfBest vf_wave_best(VfBest a) {
    vf_dpp_best<0x111, 0xf>(a);
    vf_dpp_best<0x112, 0xf>(a);
    vf_dpp_best<0x114, 0xf>(a);
    vf_dpp_best<0x118, 0xf>(a);
    vf_dpp_best<0x142, 0xa>(a);
    vf_dpp_best<0x143, 0xc>(a);
    a.v = __uint_as_float((unsigned)__builtin_amdgcn_readlane((int)__float_as_uint(a.v), 63));
    a.i = __builtin_amdgcn_readlane(a.i, 63);
    return a;
}
// The best of lo .. hi - 1 of a row by one wave, eight loads on the way (a lane's indices ascend: the first of equals stays)
__device__ __forceinline__ VfBest vf_wave_argmax(const float* row, int lo, int hi) {
    VfBest a = {-INFINITY, 0x7fffffff};
    int j = lo + 4 * (threadIdx.x & 63);
    for (; j + 7 * 256 + 4 <= hi; j += 8 * 256) {
        VfF4 x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) x[u] = *reinterpret_cast<const VfF4*>(row + j + 256 * u);
#pragma unroll
        for (int u = 0; u < 8; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (x[u].v[e] > a.v) { a.v = x[u].v[e]; a.i = j + 256 * u + e; }
    }
    for (; j < hi; j += 256)
        for (int e = 0; e < 4; ++e)
            if (j + e < hi && row[j + e] > a.v) { a.v = row[j + e]; a.i = j + e; }
    return vf_wave_best(a);
}
// All rows of one batch entry in one workgroup: each of the n + 1 rows by 16 / (n + 1) waves (more than 16 rows: one wave each, in turns)
__global__ __launch_bounds__(1024) void verify_greedy_row_kernel(SmxVerifyParams p) {
    __shared__ VfBest sh[VF_MAXN + 1][VF_WAVES];
    const int b = blockIdx.x, w = threadIdx.x >> 6, lane = threadIdx.x & 63, rows = p.n + 1;
    const int parts = rows > VF_WAVES ? 1 : VF_WAVES / rows, len = ((p.V + parts - 1) / parts + 3) & ~3;
    const long long id = lane < p.n ? p.ids[b * p.ids_bs + lane] : -1;
    for (int k = w; k < rows * parts; k += VF_WAVES) {
        const int i = k % rows, part = k / rows;
        const VfBest a = vf_wave_argmax(p.target + b * p.t_bs + i * p.t_ts, min(part * len, p.V), min((part + 1) * len, p.V));
        if (lane == 0) sh[i][part] = a;
    }
    __syncthreads();
    if (w) return;
    int best = 0, last = 0;                           // of row `lane`, and of row n (64 drafts: the 65th row)
    for (int r = 0; r < 2; ++r) {
        const int i = r ? p.n : min(lane, p.n);
        VfBest a = sh[i][0];
        for (int q = 1; q < parts; ++q) vf_better(a, sh[i][q].v, sh[i][q].i);
        (r ? last : best) = a.i == 0x7fffffff ? 0 : a.i;              // (nothing above -inf)
    }
    const unsigned long long no = ~__ballot(lane < p.n && id == best);
    const int r = no ? min(__ffsll((long long)no) - 1, p.n) : p.n;
    const int tok = __shfl(best, min(r, 63), 64);
    if (lane == 0) {
        p.accepted[b] = r;
        p.token[b] = r < p.n ? tok : last;
    }
}
// Long rows: a workgroup per row, then a second launch
__global__ __launch_bounds__(1024) void verify_best_kernel(SmxVerifyParams p, VfBest* best) {
    __shared__ VfBest sh[VF_WAVES];
    const int i = blockIdx.x, b = blockIdx.y;
    const float* row = p.target + b * p.t_bs + i * p.t_ts;
    VfBest a = {-INFINITY, 0x7fffffff};
    int j = 4 * threadIdx.x;
    for (; j + 3 * 4096 + 4 <= p.V; j += 4 * 4096) {
        VfF4 x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) x[u] = *reinterpret_cast<const VfF4*>(row + j + 4096 * u);
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (x[u].v[e] > a.v) { a.v = x[u].v[e]; a.i = j + 4096 * u + e; }       // (a thread's indices ascend: the first of equals stays)
    }
    for (; j < p.V; j += 4096)
        for (int e = 0; e < 4; ++e)
            if (j + e < p.V && row[j + e] > a.v) { a.v = row[j + e]; a.i = j + e; }
    a = vf_wave_best(a);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = a;
    __syncthreads();
    if (threadIdx.x < 64) {
        a = threadIdx.x < VF_WAVES ? sh[threadIdx.x] : VfBest{-INFINITY, 0x7fffffff};
        a = vf_wave_best(a);
        if (a.i == 0x7fffffff) a.i = 0;               // nothing above -inf
        if (threadIdx.x == 0) best[(long long)b * (p.n + 1) + i] = a;
    }
}
__global__ __launch_bounds__(64) void verify_greedy_kernel(SmxVerifyParams p, const VfBest* best) {
    const int b = blockIdx.x, lane = threadIdx.x;
    best += (long long)b * (p.n + 1);
    const bool ok = lane < p.n && p.ids[b * p.ids_bs + lane] == best[lane].i;
    const unsigned long long no = ~__ballot(ok);
    const int r = no ? min(__ffsll((long long)no) - 1, p.n) : p.n;
    if (lane == 0) {
        p.accepted[b] = r;
        p.token[b] = best[r].i;
    }
}

static int vf_check(const SmxVerifyParams& p) {
    if (!p.target || !p.accepted || !p.token || p.B <= 0 || p.n < 0 || p.n > VF_MAXN || p.V <= 0) return SMX_EINVAL;
    if (p.n > 0 && !p.ids) return SMX_EINVAL;
    if (p.draft && !p.u) return SMX_EINVAL;
    if (p.B > 65535 || p.V > 0x7fffffff - 65536) return SMX_EINVAL;
    return SMX_OK;
}
// Workgroups per row of the sampled form (1: the one-launch kernel)
static int vf_pieces(const SmxVerifyParams& p) {
    // A workgroup gets through 50 000 weights in about 7 us beside 7 us of latency (ids, probabilities of the drafts, row, scans); a second
    // launch costs 6.  250 027 weights: one workgroup 30 us, pieces of 32 768 and up 5 + 6 us.
    const int most = p.V / (VF_WAVES * 2048), want = 256 / p.B;
    const int c = most < want ? most : want;
    return c < 2 ? 1 : c > VF_MAXC ? VF_MAXC : c;
}

// One launch for the greedy form of little work: two are always sooner on the GPU, but cost the caller 3 us of host time.  One set of 5 rows x 32 128:
// 8.7 us by one workgroup (100 GB/s), 9.1 a call; 6.1 in two launches, 12.3 a call.  5 x 50 265: 11.5 and 5.7; 8 x 36 398: 17.0 and 5.9; 1 x 128 000:
// 12.9 and 8.9; 64 sets of 8 x 36 398: 24.2 and 15.4.
static bool vf_greedy_one(const SmxVerifyParams& p) { return p.V <= 65536 && (long long)(p.n + 1) * p.V <= 200000; }

extern "C" long long smx_verify_draft_ws_bytes(const SmxVerifyParams* p) {
    if (vf_check(*p)) return SMX_EINVAL;
    if (!p->u) return vf_greedy_one(*p) ? 0 : 8ll * p->B * (p->n + 1);
    const int c = vf_pieces(*p);
    return c == 1 ? 0 : 8ll * p->B * c * VF_WAVES;
}
extern "C" int smx_verify_draft(const SmxVerifyParams* pp, hipStream_t stream) {
    (void)hipGetLastError();
    const SmxVerifyParams p = *pp;
    const int rc = vf_check(p);
    if (rc) return rc;
    const long long need = smx_verify_draft_ws_bytes(pp);
    if (need && (!p.ws || ((size_t)p.ws & 7) || p.ws_bytes < need)) return SMX_EINVAL;
    if (p.u) {
        const int c = vf_pieces(p), S = c * VF_WAVES, len = ((p.V + S - 1) / S + 3) & ~3;
        if (c == 1) {
            hipLaunchKernelGGL(verify_row_kernel, dim3(p.B), dim3(1024), 0, stream, p, len);
        } else {
            hipLaunchKernelGGL(verify_sums_kernel, dim3(c, p.B), dim3(1024), 0, stream, p, len, (double*)p.ws);
            hipLaunchKernelGGL(verify_pick_kernel, dim3(p.B), dim3(1024), 0, stream, p, S, len, (double*)p.ws);
        }
    } else if (vf_greedy_one(p)) {
        hipLaunchKernelGGL(verify_greedy_row_kernel, dim3(p.B), dim3(1024), 0, stream, p);
    } else {
        hipLaunchKernelGGL(verify_best_kernel, dim3(p.n + 1, p.B), dim3(1024), 0, stream, p, (VfBest*)p.ws);
        hipLaunchKernelGGL(verify_greedy_kernel, dim3(p.B), dim3(64), 0, stream, p, (const VfBest*)p.ws);
    }
    SMX_CHECK_LAUNCH();
}
extern "C" int smx_sizeof_SmxVerifyParams(void) { return (int)sizeof(SmxVerifyParams); }
