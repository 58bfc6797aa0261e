// Layer norm over the features of [n, d] activations, in either storage layout, forward and backward:
//   mu_n = mean_d x,  r_n = 1 / sqrt(mean_d (x - mu)^2 + eps),  h = (x - mu) r,  y = h w + b
//   t = gy w,  gx = r (t - mean_d t - h mean_d (t h)),  gw = sum_n gy h,  gb = sum_n gy
// Statistics and sums are held in the arithmetic type (fp32; fp64 for fp64 activations); outputs and gx are rounded once.
// The variance is a second pass over values that are on the chip, or joined from exact parts (mean, sum of squared
// differences): no sum of squares about a guessed centre, which one outlying feature would spoil.
//
// Forms: rows contiguous, up to 8 blocks of a cluster a row (norm_line_*); samples contiguous (norm_strip_*); wider rows and
// fp64 (norm_rows_*, norm_cols_*, norm_weight_*), which read their operands up to three times.
// Measured on a B200 (6.45 TB/s copy rate): bf16 8192 x 4096, forward 37 us (134 MB) and backward 55 us (201 MB and the
// weight's gradients); fp32 8192 x 4096 forward 55 us (268 MB, 75 %); fp32 16384 features x 512 samples, samples contiguous,
// both passes 56 us (168 MB at least).  What bounds the 16-bit rows is waiting: 15 instructions an entry fill 44 % of the issue
// slots and 30 % of the DRAM's rate in the forward pass, 31 an entry 62 % and 40 % in the backward pass, while 16 warps an SM
// wait for shared memory, for weight and bias, and for one another at two barriers a row.  What bounds the strips is that each
// pass reads its operands twice, and six launches.  Rows wider than the forward plan (40960 fp32, 81920 16-bit entries) are
// read three times: fp32 1024 x 65536 forward 406 us (537 MB).
#include <cuda_runtime.h>

#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "vec.cuh"

namespace clb {

namespace {

template <typename A> struct NormArgs {
    int64_t n, d, sn, sd;  // element (i, j) of x is x[i * sn + j * sd]
    int64_t gn, gd;        // the same for the second operand (y or gy)
    int64_t on, od;        // and for gx
    const A* weight;
    const A* bias;
    A eps;
    A* mean;
    A* rstd;
};

// Sum over the threads of a block; every thread gets it.
template <typename A> __device__ A block_sum(A v, A* sh) {
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    A t = 0;
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) t += sh[i];
    return t;
}

// Any width and type, rows contiguous: one block per row.
template <typename T>
__global__ void __launch_bounds__(256) norm_rows_kernel(const T* __restrict__ x, T* __restrict__ y,
                                                        NormArgs<typename Acc<T>::type> a) {
    using A = typename Acc<T>::type;
    __shared__ A sh[8];
    for (int64_t i = blockIdx.x; i < a.n; i += gridDim.x) {
        const T* p = x + i * a.sn;
        A s = 0;
        for (int64_t j = threadIdx.x; j < a.d; j += blockDim.x) s += to_acc(p[j * a.sd]);
        const A mu = block_sum(s, sh) / (A)a.d;
        A q = 0;
        for (int64_t j = threadIdx.x; j < a.d; j += blockDim.x) {
            const A c = to_acc(p[j * a.sd]) - mu;
            q += c * c;
        }
        const A r = (A)1 / sqrt(block_sum(q, sh) / (A)a.d + a.eps);
        for (int64_t j = threadIdx.x; j < a.d; j += blockDim.x) {
            A v = (to_acc(p[j * a.sd]) - mu) * r;
            if (a.weight != nullptr) v *= a.weight[j];
            if (a.bias != nullptr) v += a.bias[j];
            y[i * a.gn + j * a.gd] = from_acc<T>(v);
        }
        if (threadIdx.x == 0) {
            if (a.mean != nullptr) a.mean[i] = mu;
            if (a.rstd != nullptr) a.rstd[i] = r;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(256) norm_rows_grad_kernel(const T* __restrict__ x, const T* __restrict__ gy,
                                                             T* __restrict__ gx, NormArgs<typename Acc<T>::type> a) {
    using A = typename Acc<T>::type;
    __shared__ A sh[8];
    for (int64_t i = blockIdx.x; i < a.n; i += gridDim.x) {
        const A mu = a.mean[i], r = a.rstd[i];
        A s1 = 0, s2 = 0;
        for (int64_t j = threadIdx.x; j < a.d; j += blockDim.x) {
            const A t = to_acc(gy[i * a.gn + j * a.gd]) * (a.weight != nullptr ? a.weight[j] : (A)1);
            s1 += t;
            s2 += t * ((to_acc(x[i * a.sn + j * a.sd]) - mu) * r);
        }
        s1 = block_sum(s1, sh) / (A)a.d;
        s2 = block_sum(s2, sh) / (A)a.d;
        for (int64_t j = threadIdx.x; j < a.d; j += blockDim.x) {
            const A t = to_acc(gy[i * a.gn + j * a.gd]) * (a.weight != nullptr ? a.weight[j] : (A)1);
            const A h = (to_acc(x[i * a.sn + j * a.sd]) - mu) * r;
            gx[i * a.on + j * a.od] = from_acc<T>(r * (t - s1 - h * s2));
        }
    }
}

// Samples contiguous (fp64): a block of 32 x 8 threads per 32 samples, the lanes along the samples.
template <typename A> __device__ A column_sum(A v, A (*sh)[33]) {
    __syncthreads();
    sh[threadIdx.y][threadIdx.x] = v;
    __syncthreads();
    A t = 0;
    for (int i = 0; i < (int)blockDim.y; ++i) t += sh[i][threadIdx.x];
    return t;
}

template <typename T>
__global__ void __launch_bounds__(256) norm_cols_kernel(const T* __restrict__ x, T* __restrict__ y,
                                                        NormArgs<typename Acc<T>::type> a) {
    using A = typename Acc<T>::type;
    __shared__ A sh[8][33];
    const int64_t i = (int64_t)blockIdx.x * 32 + threadIdx.x;
    const bool in = i < a.n;
    const T* p = x + (in ? i : 0);
    A s = 0;
    for (int64_t j = threadIdx.y; j < a.d; j += blockDim.y) s += to_acc(p[j * a.sd]);
    const A mu = column_sum(s, sh) / (A)a.d;
    A q = 0;
    for (int64_t j = threadIdx.y; j < a.d; j += blockDim.y) {
        const A c = to_acc(p[j * a.sd]) - mu;
        q += c * c;
    }
    const A r = (A)1 / sqrt(column_sum(q, sh) / (A)a.d + a.eps);
    if (!in) return;
    for (int64_t j = threadIdx.y; j < a.d; j += blockDim.y) {
        A v = (to_acc(p[j * a.sd]) - mu) * r;
        if (a.weight != nullptr) v *= a.weight[j];
        if (a.bias != nullptr) v += a.bias[j];
        y[i + j * a.gd] = from_acc<T>(v);
    }
    if (threadIdx.y == 0) {
        if (a.mean != nullptr) a.mean[i] = mu;
        if (a.rstd != nullptr) a.rstd[i] = r;
    }
}

template <typename T>
__global__ void __launch_bounds__(256) norm_cols_grad_kernel(const T* __restrict__ x, const T* __restrict__ gy,
                                                             T* __restrict__ gx, NormArgs<typename Acc<T>::type> a) {
    using A = typename Acc<T>::type;
    __shared__ A sh[8][33];
    const int64_t i = (int64_t)blockIdx.x * 32 + threadIdx.x;
    const bool in = i < a.n;
    const int64_t k = in ? i : 0;
    const A mu = a.mean[k], r = a.rstd[k];
    A s1 = 0, s2 = 0;
    for (int64_t j = threadIdx.y; j < a.d; j += blockDim.y) {
        const A t = to_acc(gy[k + j * a.gd]) * (a.weight != nullptr ? a.weight[j] : (A)1);
        s1 += t;
        s2 += t * ((to_acc(x[k + j * a.sd]) - mu) * r);
    }
    s1 = column_sum(s1, sh) / (A)a.d;
    s2 = column_sum(s2, sh) / (A)a.d;
    if (!in) return;
    for (int64_t j = threadIdx.y; j < a.d; j += blockDim.y) {
        const A t = to_acc(gy[i + j * a.gd]) * (a.weight != nullptr ? a.weight[j] : (A)1);
        const A h = (to_acc(x[i + j * a.sd]) - mu) * r;
        gx[i + j * a.od] = from_acc<T>(r * (t - s1 - h * s2));
    }
}

// gw, gb: lanes along the features when they are contiguous (each block sums all rows of 32 features) ...
template <typename T>
__global__ void __launch_bounds__(256) norm_weight_rows_kernel(const T* __restrict__ x, const T* __restrict__ gy,
                                                               NormArgs<typename Acc<T>::type> a,
                                                               typename Acc<T>::type* gw, typename Acc<T>::type* gb) {
    using A = typename Acc<T>::type;
    __shared__ A sh[8][33];
    const int64_t j = (int64_t)blockIdx.x * 32 + threadIdx.x;
    const int64_t k = j < a.d ? j : 0;
    A s1 = 0, s2 = 0;
    for (int64_t i = threadIdx.y; i < a.n; i += blockDim.y) {
        const A g = to_acc(gy[i * a.gn + k]);
        s1 += g * ((to_acc(x[i * a.sn + k]) - a.mean[i]) * a.rstd[i]);
        s2 += g;
    }
    s1 = column_sum(s1, sh);
    s2 = column_sum(s2, sh);
    if (threadIdx.y != 0 || j >= a.d) return;
    if (gw != nullptr) gw[j] = s1;
    if (gb != nullptr) gb[j] = s2;
}

// ... and one block per feature when the samples are (fp64).
template <typename T>
__global__ void __launch_bounds__(256) norm_weight_cols_kernel(const T* __restrict__ x, const T* __restrict__ gy,
                                                               NormArgs<typename Acc<T>::type> a,
                                                               typename Acc<T>::type* gw, typename Acc<T>::type* gb) {
    using A = typename Acc<T>::type;
    __shared__ A sh[8];
    for (int64_t j = blockIdx.x; j < a.d; j += gridDim.x) {
        A s1 = 0, s2 = 0;
        for (int64_t i = threadIdx.x; i < a.n; i += blockDim.x) {
            const A g = to_acc(gy[i + j * a.gd]);
            s1 += g * ((to_acc(x[i + j * a.sd]) - a.mean[i]) * a.rstd[i]);
            s2 += g;
        }
        s1 = block_sum(s1, sh);
        s2 = block_sum(s2, sh);
        if (threadIdx.x == 0) {
            if (gw != nullptr) gw[j] = s1;
            if (gb != nullptr) gb[j] = s2;
        }
    }
}

// ---- rows in 16-byte windows (fp32 / bf16 / fp16) ----
// G threads own a row (of `parts` blocks of a cluster: a contiguous share of it), NP windows a thread: a warp has 32 NP
// neighbouring windows, lane l those at l, l + 32, ..., so that a thread's windows are constant distances apart.  A row that
// does not start on 16 bytes is cut from the last boundary before it, `shift` entries back.  What is known of the windows
// picks the kernels' form: each is part of the row as a whole (kFull), as a whole or not at all (kWhole: rows start on 16
// bytes and end with a window), or may be so in part (kShifted).
//
// The groups walk down the rows.  The next rows' whole windows travel to shared memory meanwhile (Ring), each thread fetching
// its own, so that no barrier stands between a copy and its use.  A thread's rows are a multiple of a whole pack's entries
// apart, so that their shift is the same and its columns do not move.

template <typename T> __device__ __forceinline__ int shift_of(const T* p) {
    return (int)((reinterpret_cast<uintptr_t>(p) / sizeof(T)) % (16 / sizeof(T)));
}

enum Windows { kFull, kWhole, kShifted };
// Rows of a group in shared memory or on their way there: the one at work and the next.  A third would take shared memory
// from the L1 cache that holds weight and bias (bf16 8192 x 4096, both passes: 101 us with two, 108 with three).
constexpr int kStages = 2;

template <typename T, int NP, Windows M> struct Line {
    static constexpr int VEC = 16 / sizeof(T), STEP = 32 * VEC;

    // whether the window at column c lies in the row, or at least a part of it does
    static __device__ __forceinline__ bool whole(int c, int d) {
        return M == kFull || (M == kWhole ? c < d : c >= 0 && c + VEC <= d);
    }
    static __device__ __forceinline__ bool any(int c, int d) {
        return M == kFull || (M == kWhole ? c < d : c < d && c + VEC > 0);
    }
    // a window that is not whole in the row, or not in memory (at: its first entry)
    static __device__ __forceinline__ Pack<T, VEC> edge(const T* __restrict__ at, int c, int d) {
        Pack<T, VEC> q = {};
        if (M == kShifted) {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if ((unsigned)(c + j) < (unsigned)d) q.raw(j, at[j]);
        }
        return q;
    }
    // wide: windows are whole 16-byte words of this row's memory too
    static __device__ __forceinline__ void store(T* __restrict__ at, int c, int d, bool wide, const float (&f)[VEC]) {
        Pack<T, VEC> q;
        q.put(f);
        if (M != kShifted || (wide && whole(c, d))) {
            q.store(at);
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if ((unsigned)(c + j) < (unsigned)d) at[j] = q.raw(j);
        }
    }
};

// A thread's slots in shared memory: OPS operands of NP windows, STAGES times; a warp's lie together.
template <int NP, int OPS, int STAGES> struct Ring {
    static constexpr int kStage = OPS * NP * 32;  // 16-byte words of a warp
    uint4* slots;
    uint32_t at;
    int put = 0, got = 0;

    __device__ __forceinline__ Ring(uint4* shared) {
        slots = shared + (threadIdx.x >> 5) * STAGES * kStage + (threadIdx.x & 31);
        at = (uint32_t)__cvta_generic_to_shared(slots);
    }
    __device__ __forceinline__ void fetch(int op, int u, const void* from) const {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at + 16 * (put * kStage + (op * NP + u) * 32)), "l"(from)
                     : "memory");
    }
    __device__ __forceinline__ void sent() {
        asm volatile("cp.async.commit_group;" ::: "memory");
        put = put + 1 == STAGES ? 0 : put + 1;
    }
    // waits for the oldest stage
    __device__ __forceinline__ const uint4* next() {
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        const uint4* p = slots + got * kStage;
        got = got + 1 == STAGES ? 0 : got + 1;
        return p;
    }
    template <typename P> static __device__ __forceinline__ P window(const uint4* stage, int op, int u) {
        const uint4 w = stage[(op * NP + u) * 32];
        P q;
        q.w[0] = w.x, q.w[1] = w.y, q.w[2] = w.z, q.w[3] = w.w;
        return q;
    }
};

// Entries [c, c + N) of a parameter vector of d entries (on 16 bytes, or 32 for N = 8, unless `loose`); `past` outside it or
// without one.  Where c is not a multiple of 4 they are cut out of aligned words.
template <int N, Windows M>
__device__ __forceinline__ void parameter(const float* __restrict__ v, int c, int d, bool loose, float past, float (&f)[N]) {
    if (v == nullptr) {
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = past;
    } else if (M != kShifted && N == 8) {
        // One 32-byte access a lane: two of 16 bytes, 32 apart from lane to lane, take twice the L1 cycles.  Volatile: a plain
        // asm statement is arithmetic to the compiler, which may carry it out before the checks that it stands behind.
        asm volatile("ld.global.nc.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3]), "=f"(f[4 % N]), "=f"(f[5 % N]), "=f"(f[6 % N]), "=f"(f[7 % N])
                     : "l"(v + c));
    } else if (M != kShifted) {
#pragma unroll
        for (int k = 0; k < N; k += 4) {
            const float4 q = __ldg(reinterpret_cast<const float4*>(v + c + k));
            f[k] = q.x, f[k + 1] = q.y, f[k + 2] = q.z, f[k + 3] = q.w;
        }
    } else if (!loose && c >= 0 && c + N + 4 <= d) {
        const int o = c & 3;
        float w[N + 4];
#pragma unroll
        for (int k = 0; k < N + 4; k += 4) {
            const float4 q = __ldg(reinterpret_cast<const float4*>(v + (c - o) + k));
            w[k] = q.x, w[k + 1] = q.y, w[k + 2] = q.z, w[k + 3] = q.w;
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float lo = o & 1 ? w[j + 1] : w[j], hi = o & 1 ? w[j + 3] : w[j + 2];
            f[j] = o & 2 ? hi : lo;
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = (unsigned)(c + j) < (unsigned)d ? v[c + j] : past;
    }
}

constexpr int kMostParts = 8;  // blocks of a row

// Threads of a block; the forward kernel has two blocks an SM, the gradient kernel one.  More threads leave each fewer
// registers (512 in the forward kernel spill).  Forward pass with 320, 384 and 512: fp16 3001 x 5001 28.8, 29.9 and 32.2 us, but
// bf16 8192 x 4096 37.0, 31.4 and 34.2, fp32 8192 x 4096 56.4, 51.8 and 49.4.  Forward and gradients of bf16 8192 x 4096: 96 us
// with gradient blocks of 640 threads of two windows, 103 with 512 of four (before the parameters were read in 32 bytes); wider
// rows need four.
constexpr int kLineThreads = 320;
template <int NP> constexpr int kGradThreads = NP <= 2 ? 640 : 512;

struct RowPlan {
    int g, rows, parts;  // threads a row and block, rows a block at a time, blocks a row
    bool loose;          // weight or bias not on the boundary of a window's entries
};

// Barrier of the G threads of a row in a block (every thread of the block where it has one row).
__device__ __forceinline__ void group_barrier(const RowPlan& plan, int group) {
    asm volatile("barrier.sync %0, %1;" ::"r"(group + 1), "r"(plan.g) : "memory");
}

// Sums of two values over the G threads of a row within a block, through `sh` (one entry a warp, another `sh` in the next
// call).
__device__ __forceinline__ float2 group_sum(float2 v, float2* sh, const RowPlan& plan, int group) {
    v.x = warp_sum(v.x);
    v.y = warp_sum(v.y);
    if (plan.g == 32) return v;
    const int w = plan.g >> 5, lane = threadIdx.x & 31;
    if (lane == 0) sh[threadIdx.x >> 5] = v;
    group_barrier(plan, group);
    v = lane < w ? sh[group * w + lane] : make_float2(0.f, 0.f);
    return make_float2(warp_sum(v.x), warp_sum(v.y));
}
__device__ __forceinline__ float group_sum(float v, float* sh, const RowPlan& plan, int group) {
    v = warp_sum(v);
    if (plan.g == 32) return v;
    const int w = plan.g >> 5, lane = threadIdx.x & 31;
    if (lane == 0) sh[threadIdx.x >> 5] = v;
    group_barrier(plan, group);
    return warp_sum(lane < w ? sh[group * w + lane] : 0.f);
}

// One value pair of every block of the cluster, in every block; `slots` of [kMostParts], another one in the next call.
__device__ __forceinline__ void cluster_share(float2* slots, float2 v, int rank, int parts) {
    if (threadIdx.x < parts) {
        uint32_t local = (uint32_t)__cvta_generic_to_shared(slots + rank), remote;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(threadIdx.x));
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(remote), "f"(v.x), "f"(v.y) : "memory");
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// 1 / sqrt(v): the hardware's estimate and one Newton step.
__device__ __forceinline__ float inverse_root(float v) {
    const float r = rsqrtf(v);
    return v > 0.f && v < INFINITY ? r * fmaf(-0.5f * v * r, r, 1.5f) : r;
}

template <typename T, int NP, Windows M>
__global__ void __launch_bounds__(kLineThreads, 2)
    norm_line_kernel(const T* __restrict__ x, T* __restrict__ y, NormArgs<float> a, RowPlan plan) {
    using L = Line<T, NP, M>;
    using P = Pack<T, L::VEC>;
    constexpr int VEC = L::VEC;
    extern __shared__ uint4 shared[];
    __shared__ float sums[kLineThreads / 32], squares[kLineThreads / 32];
    __shared__ float2 shares[2][kMostParts];
    const int g = plan.g, group = threadIdx.x / g, t = threadIdx.x - group * g;
    const int rank = (int)(blockIdx.x % (unsigned)plan.parts), share = g * NP * VEC, d = (int)a.d;
    if (plan.parts > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    const int64_t step = (int64_t)(gridDim.x / (unsigned)plan.parts) * plan.rows;
    int64_t i = (int64_t)(blockIdx.x / (unsigned)plan.parts) * plan.rows + group;
    const int shift = M == kShifted ? shift_of(x + i * a.sn) : 0;
    const int c0 = rank * share + ((t >> 5) * NP * 32 + (t & 31)) * VEC - shift;
    const bool same = M != kShifted || shift_of(y + i * a.gn) == shift;
    // entries of the row in block k's share
    auto count = [&](int k) { return min(max(d + shift - k * share, 0), share) - (k == 0 ? shift : 0); };
    const float per = 1.f / (float)d, mine = plan.parts > 1 ? 1.f / (float)max(count(rank), 1) : per;
    int turns = i < a.n ? (int)((a.n - 1 - i) / step) + 1 : 0, left = turns;
    const T *ahead = x + i * a.sn + c0, *row = ahead;
    T* out = y + i * a.gn + c0;
    const int64_t down = step * a.sn, down_out = step * a.gn;
    Ring<NP, 1, kStages> ring(shared);
    auto fetch = [&]() {
        if (left > 0) {
#pragma unroll
            for (int u = 0; u < NP; ++u)
                if (L::whole(c0 + u * L::STEP, d)) ring.fetch(0, u, ahead + u * L::STEP);
        }
        ring.sent();
        ahead += down;
        --left;
    };
#pragma unroll
    for (int k = 0; k + 1 < kStages; ++k) fetch();
    if (plan.parts > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    for (; turns > 0; --turns, i += step, row += down, out += down_out) {
        __syncwarp();  // the stage that is filled now was read in the turn before
        fetch();
        const uint4* stage = ring.next();
        P p[NP];
        float s[2] = {};
#pragma unroll
        for (int u = 0; u < NP; ++u) {
            const int c = c0 + u * L::STEP;
            p[u] = L::whole(c, d) ? ring.template window<P>(stage, 0, u) : L::edge(row + u * L::STEP, c, d);
            float f[VEC];
            p[u].get(f);
#pragma unroll
            for (int j = 0; j < VEC; ++j) s[j & 1] += f[j];
        }
        float mu = group_sum(s[0] + s[1], sums, plan, group) * mine;
        float q[2] = {};
#pragma unroll
        for (int u = 0; u < NP; ++u) {
            const int c = c0 + u * L::STEP;
            float f[VEC];
            p[u].get(f);
            if (L::whole(c, d)) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) q[j & 1] = fmaf(f[j] - mu, f[j] - mu, q[j & 1]);
            } else if (M == kShifted) {
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if ((unsigned)(c + j) < (unsigned)d) q[j & 1] = fmaf(f[j] - mu, f[j] - mu, q[j & 1]);
            }
        }
        float m2 = group_sum(q[0] + q[1], squares, plan, group);
        if (plan.parts > 1) {
            float2* slots = shares[turns & 1];
            cluster_share(slots, make_float2(mu, m2), rank, plan.parts);
            mu = m2 = 0;
            for (int k = 0; k < plan.parts; ++k) mu = fmaf(slots[k].x, (float)count(k) * per, mu);
            for (int k = 0; k < plan.parts; ++k) {
                const float c = slots[k].x - mu;
                m2 += fmaf(c * c, (float)count(k), slots[k].y);
            }
        }
        const float r = inverse_root(fmaf(m2, per, a.eps));
        if (t == 0 && rank == 0) {
            if (a.mean != nullptr) a.mean[i] = mu;
            if (a.rstd != nullptr) a.rstd[i] = r;
        }
#pragma unroll
        for (int u = 0; u < NP; ++u) {
            const int c = c0 + u * L::STEP;
            if (!L::any(c, d)) continue;
            float f[VEC], w[VEC], b[VEC];
            p[u].get(f);
            parameter<VEC, M>(a.weight, c, d, plan.loose, 1.f, w);
            parameter<VEC, M>(a.bias, c, d, plan.loose, 0.f, b);
#pragma unroll
            for (int j = 0; j < VEC; ++j) f[j] = fmaf((f[j] - mu) * r, w[j], b[j]);
            L::store(out + u * L::STEP, c, d, same, f);
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

// The weight's gradients of a thread's columns stay in its registers all the way down; in the end the groups of a block add
// theirs up.  part: [2, gridDim.x / parts, d] sums of gy h and of gy (null: not wanted).  gx null: not wanted.
template <typename T, int NP, Windows M>
__global__ void __launch_bounds__(kGradThreads<NP>, 1) norm_line_grad_kernel(const T* __restrict__ x, const T* __restrict__ gy,
                                                                         T* __restrict__ gx, NormArgs<float> a, RowPlan plan,
                                                                         float* __restrict__ part) {
    using L = Line<T, NP, M>;
    using P = Pack<T, L::VEC>;
    constexpr int VEC = L::VEC;
    extern __shared__ uint4 shared[];  // the ring; in the end [d] floats
    __shared__ float2 sums[2][kGradThreads<NP> / 32];
    __shared__ float2 shares[2][kMostParts];
    const int g = plan.g, group = threadIdx.x / g, t = threadIdx.x - group * g;
    const int rank = (int)(blockIdx.x % (unsigned)plan.parts), share = g * NP * VEC, d = (int)a.d;
    if (plan.parts > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    const int64_t step = (int64_t)(gridDim.x / (unsigned)plan.parts) * plan.rows;
    const int64_t i = (int64_t)(blockIdx.x / (unsigned)plan.parts) * plan.rows + group;
    const int shift = M == kShifted ? shift_of(x + i * a.sn) : 0;
    const int c0 = rank * share + ((t >> 5) * NP * 32 + (t & 31)) * VEC - shift;
    const bool wide = M != kShifted || shift_of(gy + i * a.gn) == shift;
    const bool same = gx != nullptr && (M != kShifted || shift_of(gx + i * a.on) == shift);
    float gw[NP][VEC] = {}, gb[NP][VEC] = {};
    const float per = 1.f / (float)d;
    int turns = i < a.n ? (int)((a.n - 1 - i) / step) + 1 : 0, left = turns;
    const T *ax = x + i * a.sn + c0, *ag = gy + i * a.gn + c0, *px = ax, *pg = ag;
    T* out = gx + i * a.on + c0;
    const float *pm = a.mean + i, *pr = a.rstd + i;
    const int64_t down_x = step * a.sn, down_g = step * a.gn, down_out = step * a.on;
    Ring<NP, 2, kStages> ring(shared);
    auto fetch = [&]() {
        if (left > 0) {
#pragma unroll
            for (int u = 0; u < NP; ++u)
                if (L::whole(c0 + u * L::STEP, d)) {
                    ring.fetch(0, u, ax + u * L::STEP);
                    if (wide) ring.fetch(1, u, ag + u * L::STEP);
                }
        }
        ring.sent();
        ax += down_x;
        ag += down_g;
        --left;
    };
#pragma unroll
    for (int k = 0; k + 1 < kStages; ++k) fetch();
    if (plan.parts > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    float mun = turns > 0 ? *pm : 0.f, rn = turns > 0 ? *pr : 0.f;
    for (; turns > 0; --turns, px += down_x, pg += down_g, out += down_out) {
        const float mu = mun, r = rn;
        if (turns > 1) {
            mun = *(pm += step);
            rn = *(pr += step);
        }
        __syncwarp();  // the stage that is filled now was read in the turn before
        fetch();
        const uint4* stage = ring.next();
        auto windows = [&](int u, float(&h)[VEC], float(&f)[VEC]) {
            const int c = c0 + u * L::STEP;
            const P p = L::whole(c, d) ? ring.template window<P>(stage, 0, u) : L::edge(px + u * L::STEP, c, d);
            const P q = L::whole(c, d) && wide ? ring.template window<P>(stage, 1, u) : L::edge(pg + u * L::STEP, c, d);
            p.get(h);
            q.get(f);
        };
        float s1[2] = {}, s2[2] = {};
#pragma unroll
        for (int u = 0; u < NP; ++u) {  // entries past the row have gy = 0
            const int c = c0 + u * L::STEP;
            if (!L::any(c, d)) continue;
            float h[VEC], f[VEC], w[VEC];
            windows(u, h, f);
            parameter<VEC, M>(a.weight, c, d, plan.loose, 1.f, w);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                h[j] = (h[j] - mu) * r;
                gw[u][j] = fmaf(f[j], h[j], gw[u][j]);
                gb[u][j] += f[j];
                f[j] *= w[j];
                s1[j & 1] += f[j];
                s2[j & 1] = fmaf(f[j], h[j], s2[j & 1]);
            }
        }
        if (gx == nullptr) continue;
        float2 s = group_sum(make_float2(s1[0] + s1[1], s2[0] + s2[1]), sums[turns & 1], plan, group);
        if (plan.parts > 1) {
            float2* slots = shares[turns & 1];
            cluster_share(slots, s, rank, plan.parts);
            s = make_float2(0.f, 0.f);
            for (int k = 0; k < plan.parts; ++k) {
                s.x += slots[k].x;
                s.y += slots[k].y;
            }
        }
        s.x *= per;
        s.y *= per;
#pragma unroll
        for (int u = 0; u < NP; ++u) {
            const int c = c0 + u * L::STEP;
            if (!L::any(c, d)) continue;
            float h[VEC], f[VEC], w[VEC];
            windows(u, h, f);
            parameter<VEC, M>(a.weight, c, d, plan.loose, 1.f, w);
#pragma unroll
            for (int j = 0; j < VEC; ++j) f[j] = r * fmaf((h[j] - mu) * r, -s.y, fmaf(f[j], w[j], -s.x));
            L::store(out + u * L::STEP, c, d, same, f);
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (part == nullptr) return;
    const int64_t blocks = gridDim.x / (unsigned)plan.parts;
    float* at = part + (int64_t)(blockIdx.x / (unsigned)plan.parts) * d;
    if (plan.rows == 1) {
#pragma unroll
        for (int u = 0; u < NP; ++u)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const int c = c0 + u * L::STEP + j;
                if ((unsigned)c < (unsigned)d) {
                    at[c] = gw[u][j];
                    at[blocks * d + c] = gb[u][j];
                }
            }
        return;
    }
    // group after group adds its sums, by column: the groups' shifts differ
    float* fold = reinterpret_cast<float*>(shared);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        for (int k = 0; k < plan.rows; ++k) {
            __syncthreads();
            if (group != k) continue;
#pragma unroll
            for (int u = 0; u < NP; ++u)
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const int c = c0 + u * L::STEP + j;
                    const float v = which == 0 ? gw[u][j] : gb[u][j];
                    if ((unsigned)c < (unsigned)d) fold[c] = k == 0 ? v : fold[c] + v;
                }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < d; c += blockDim.x) at[which * blocks * d + c] = fold[c];
    }
}

// Two sums over the same rows: out[k][j] = sum over p < groups of part[(k groups + p) ld + j], j < d, k = 0, 1 (null: not
// wanted).
struct Fold {
    const float* part;
    int64_t groups, ld, d;
    float *out0, *out1;
};

// Up to two of them in one launch, in a fixed order: 32 columns x 8 shares of the rows a block, blockIdx.y picks the sum.
__global__ void __launch_bounds__(256) norm_fold_kernel(Fold a, Fold b) {
    __shared__ float sh[8][32];
    const Fold f = blockIdx.y < 2 ? a : b;
    const int k = blockIdx.y & 1, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float* out = k == 0 ? f.out0 : f.out1;
    const int64_t j = (int64_t)blockIdx.x * 32 + lane;
    if (out == nullptr || (int64_t)blockIdx.x * 32 >= f.d) return;
    const float* part = f.part + k * f.groups * f.ld + j;
    float s[4] = {};
    if (j < f.d) {
        int64_t p = warp;
        for (; p + 24 < f.groups; p += 32) {
#pragma unroll
            for (int u = 0; u < 4; ++u) s[u] += part[(p + 8 * u) * f.ld];
        }
        for (; p < f.groups; p += 8) s[0] += part[p * f.ld];
    }
    sh[warp][lane] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    if (warp != 0 || j >= f.d) return;
    float t = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) t += sh[w][lane];
    out[j] = t;
}

cudaError_t launch_fold(const Fold& a, const Fold& b, cudaStream_t s) {
    const int64_t d = a.d > b.d ? a.d : b.d;
    norm_fold_kernel<<<dim3((unsigned)ceil_div64(d, 32), b.part != nullptr ? 4 : 2), 256, 0, s>>>(a, b);
    count_launches(1);
    return cudaGetLastError();
}

// How a width is split; np = 0: too wide.
struct LinePlan {
    RowPlan plan;
    int np;          // windows a thread
    int64_t blocks;  // of the grid, a cluster counted as one
};

LinePlan line_plan(int64_t n, int64_t d, int vec, bool shifted, bool backward) {
    LinePlan p{};
    auto threads = [&](int np) { return !backward ? kLineThreads : np <= 2 ? kGradThreads<1> : kGradThreads<4>; };
    const int64_t w = ceil_div64(d + (shifted ? vec - 1 : 0), vec);  // windows, with room for the furthest shift
    const int most = backward && w <= 2 * threads(2) * kMostParts ? 2 : 4;
    p.np = 1;
    while (p.np < most && w > 32 * p.np) p.np *= 2;
    // few rows: more threads a row, as long as they leave the SMs' places empty (bf16 200 x 4096: 3.5 us, else 3.9)
    while (!backward && p.np > 1 && n * ceil_div64(w, p.np) < (int64_t)gpu_sms() * 512) p.np /= 2;
    int64_t g = ceil_div64(w, 32 * p.np) * 32;
    while (g > threads(p.np) && p.np < most) {
        p.np *= 2;
        g = ceil_div64(w, 32 * p.np) * 32;
    }
    p.plan.parts = 1;
    while (g > threads(p.np) && p.plan.parts < kMostParts) {
        p.plan.parts *= 2;
        g = ceil_div64(w, (int64_t)32 * p.np * p.plan.parts) * 32;
    }
    if (g > threads(p.np)) return {};
    p.plan.g = (int)g;
    // Blocks that are resident at once: the gradient kernel takes up to 128 registers a thread, the forward one 64; fewer
    // rows a block rather than fewer blocks
    // (clusters: SMs come in groups of 16 or 18, which a cluster does not cross)
    const int64_t places = p.plan.parts == 1 ? gpu_sms() : gpu_sms() / 18 * (16 / p.plan.parts);
    const int64_t resident = places * (backward ? 1 : 2), spread = ceil_div64(n, resident);
    p.plan.rows = (int)(threads(p.np) / g < spread ? threads(p.np) / g : spread);
    if (p.plan.parts > 1 || p.plan.rows < 1) p.plan.rows = 1;
    if (resident * p.plan.rows >= n) {
        p.blocks = ceil_div64(n, p.plan.rows);
    } else {
        // rows of one thread a multiple of a pack's entries apart
        p.blocks = resident;
        while (shifted && p.blocks > 1 && p.blocks * p.plan.rows % vec != 0) --p.blocks;
        if (shifted && p.blocks * p.plan.rows % vec != 0) p.blocks = vec;
    }
    return p;
}

template <typename P> struct Same { using type = P; };  // a parameter that is not deduced

template <typename... P> cudaError_t launch_lines(void (*kernel)(P...), const LinePlan& p, size_t shared, cudaStream_t s,
                                                  typename Same<P>::type... args) {
    if (p.blocks * p.plan.parts > 0x7FFFFFFF) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[1];
    cfg.gridDim = dim3((unsigned)(p.blocks * p.plan.parts));
    cfg.blockDim = dim3((unsigned)(p.plan.g * p.plan.rows));
    cfg.dynamicSmemBytes = shared;
    cfg.stream = s;
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)p.plan.parts;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = p.plan.parts > 1 ? 1 : 0;
    count_launches(1);
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

unsigned blocks(int64_t n) { return (unsigned)(n < (1 << 30) ? n : (1 << 30)); }

// ---- samples contiguous (fp32 / bf16 / fp16) ----
// The statistics run down the strided axis, the weight's gradients along the contiguous one.  First pass: a warp owns a
// strip of 32 V samples (V a 16-byte pack, or 1 where rows do not start on 16 bytes) and walks down features 8 at a time,
// all 8 loads in flight; the blocks of `chunk` features leave partial results, which a small kernel folds.  Second pass:
// elementwise, reading the operands again, out of the L2 cache where they fit.  (Running both passes over one slab of samples
// after the other, each small enough to stay there, was slower: fp32 64000 x 1024 forward 267 us, in one go
// 156, and 139 since three blocks an SM are resident.)

constexpr int kColThreads = 256, kBatch = 8;

// V consecutive samples of one feature as floats; `left` of them exist.
template <typename T, int V> struct Strip {
    uint32_t w[V * sizeof(T) >= 4 ? V * sizeof(T) / 4 : 1];
    __device__ __forceinline__ void load(const T* __restrict__ p, int left) {
        if constexpr (V == 1) {
            T v = left > 0 ? *p : T(0.f);
            if constexpr (sizeof(T) == 2)
                w[0] = *reinterpret_cast<const unsigned short*>(&v);
            else
                w[0] = *reinterpret_cast<const uint32_t*>(&v);
        } else {
            Pack<T, V> q = {};
            if (left >= V) {
                q.load(p);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (j < left) q.raw(j, p[j]);
            }
#pragma unroll
            for (int k = 0; k < Pack<T, V>::kWords; ++k) w[k] = q.w[k];
        }
    }
    __device__ __forceinline__ void get(float (&f)[V]) const {
        if constexpr (V == 1) {
            if constexpr (sizeof(T) == 2) {
                const unsigned short h = (unsigned short)w[0];
                f[0] = to_acc(*reinterpret_cast<const T*>(&h));
            } else {
                f[0] = *reinterpret_cast<const float*>(&w[0]);
            }
        } else {
            Pack<T, V> q;
#pragma unroll
            for (int k = 0; k < Pack<T, V>::kWords; ++k) q.w[k] = w[k];
            q.get(f);
        }
    }
    static __device__ __forceinline__ void store(T* __restrict__ p, int left, const float (&f)[V]) {
        if constexpr (V == 1) {
            if (left > 0) *p = from_acc<T>(f[0]);
        } else {
            Pack<T, V> q;
            q.put(f);
            if (left >= V) {
                q.store(p);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (j < left) p[j] = q.raw(j);
            }
        }
    }
};

// mean and sum of squared differences of n more values (m, q) joined to those of n0
__device__ __forceinline__ void join(float& mean, float& m2, float m, float q, float part, float both) {
    const float c = m - mean;            // part = n / (n0 + n), both = n0 n / (n0 + n)
    mean = fmaf(c, part, mean);
    m2 = fmaf(c * c, both, m2 + q);
}

// stats [2, chunks, n]: mean and sum of squared differences of each chunk's features.
template <typename T, int V>
__global__ void __launch_bounds__(kColThreads, 3)
    norm_strip_stats_kernel(const T* __restrict__ x, NormArgs<float> a, int64_t chunk, float* __restrict__ stats) {
    constexpr int W = kColThreads / 32;
    __shared__ float sh[W][2][32 * V];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t i = ((int64_t)blockIdx.x * 32 + lane) * V, j0 = blockIdx.y * chunk;
    const int left = (int)(a.n - i < V ? (a.n > i ? a.n - i : 0) : V);
    const int64_t end = j0 + chunk < a.d ? j0 + chunk : a.d;
    float mean[V] = {}, m2[V] = {};
    int64_t n = 0;
    for (int64_t j = j0 + warp * kBatch; j < end; j += W * kBatch) {
        const int k = (int)(end - j < kBatch ? end - j : kBatch);
        Strip<T, V> v[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
            if (u < k) v[u].load(x + (j + u) * a.sd + i, left);
        const float per = 1.f / (float)k, part = (float)k / (float)(n + k), both = (float)n * part;
        float m[V] = {}, q[V] = {};
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
            if (u < k) {
                float f[V];
                v[u].get(f);
#pragma unroll
                for (int c = 0; c < V; ++c) m[c] += f[c];
            }
#pragma unroll
        for (int c = 0; c < V; ++c) m[c] *= per;
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
            if (u < k) {
                float f[V];
                v[u].get(f);
#pragma unroll
                for (int c = 0; c < V; ++c) q[c] = fmaf(f[c] - m[c], f[c] - m[c], q[c]);
            }
#pragma unroll
        for (int c = 0; c < V; ++c) join(mean[c], m2[c], m[c], q[c], part, both);
        n += k;
    }
#pragma unroll
    for (int c = 0; c < V; ++c) {
        sh[warp][0][c * 32 + lane] = mean[c];
        sh[warp][1][c * 32 + lane] = m2[c];
    }
    __syncthreads();
    // features warp k has walked over: whole batches from its first on, W batches apart
    for (int c = threadIdx.x; c < 32 * V; c += kColThreads) {
        const int64_t at = (int64_t)blockIdx.x * 32 * V + (c % 32) * V + c / 32;
        float m = 0, q = 0;
        int64_t n0 = 0;
        for (int k = 0; k < W; ++k) {
            int64_t nk = 0;
            for (int64_t j = j0 + k * kBatch; j < end; j += W * kBatch) nk += end - j < kBatch ? end - j : kBatch;
            if (nk == 0) break;
            const float part = (float)nk / (float)(n0 + nk);
            join(m, q, sh[k][0][c], sh[k][1][c], part, (float)n0 * part);
            n0 += nk;
        }
        if (at < a.n) {
            stats[blockIdx.y * a.n + at] = m;
            stats[(gridDim.y + blockIdx.y) * a.n + at] = q;
        }
    }
}

// mean and rstd from the chunks: 32 samples x 32 shares of the chunks a block, joined pairwise
__global__ void __launch_bounds__(1024) norm_strip_fold_kernel(const float* __restrict__ stats, int64_t n, int64_t d,
                                                               int64_t chunk, int chunks, float eps, float* mean, float* rstd) {
    __shared__ float sh[3][32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t i = (int64_t)blockIdx.x * 32 + lane;
    float m = 0, q = 0, n0 = 0;
    if (i < n)
        for (int k = warp; k < chunks; k += 32) {
            const float nk = (float)(d - k * chunk < chunk ? d - k * chunk : chunk), part = nk / (n0 + nk);
            join(m, q, stats[k * n + i], stats[(chunks + k) * n + i], part, n0 * part);
            n0 += nk;
        }
    sh[0][warp][lane] = m;
    sh[1][warp][lane] = q;
    sh[2][warp][lane] = n0;
    __syncthreads();
    // warp w joins the shares of sample w
    m = sh[0][lane][warp];
    q = sh[1][lane][warp];
    n0 = sh[2][lane][warp];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const float m1 = __shfl_xor_sync(0xffffffffu, m, o), q1 = __shfl_xor_sync(0xffffffffu, q, o),
                    n1 = __shfl_xor_sync(0xffffffffu, n0, o);
        // both lanes of a pair join in the same order
        float a = lane & o ? m1 : m, b = lane & o ? q1 : q;
        const float na = lane & o ? n1 : n0, nb = lane & o ? n0 : n1;
        const float part = nb > 0.f ? nb / (na + nb) : 0.f;
        join(a, b, lane & o ? m : m1, lane & o ? q : q1, part, na * part);
        m = a;
        q = b;
        n0 = na + nb;
    }
    const int64_t at = (int64_t)blockIdx.x * 32 + warp;
    if (lane != 0 || at >= n) return;
    mean[at] = m;
    rstd[at] = inverse_root(fmaf(q, 1.f / (float)d, eps));
}

// y from x, mean and rstd; or gx from x, gy, and the folded sums c1, c2 (GRAD)
template <typename T, int V, bool GRAD>
__global__ void __launch_bounds__(kColThreads, GRAD ? 2 : 3)
    norm_strip_apply_kernel(const T* __restrict__ x, const T* __restrict__ gy, T* __restrict__ y, NormArgs<float> a,
                            int64_t chunk, const float* mean, const float* rstd, const float* c1, const float* c2) {
    constexpr int W = kColThreads / 32, B = 4;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t i = ((int64_t)blockIdx.x * 32 + lane) * V, j0 = blockIdx.y * chunk;
    const int left = (int)(a.n - i < V ? (a.n > i ? a.n - i : 0) : V);
    const int64_t end = j0 + chunk < a.d ? j0 + chunk : a.d, ld = GRAD ? a.od : a.gd;
    if (left == 0) return;
    float mu[V], r[V], k1[V], k2[V];
    const float per = 1.f / (float)a.d;
#pragma unroll
    for (int c = 0; c < V; ++c) {
        const int64_t at = c < left ? i + c : i;
        mu[c] = mean[at];
        r[c] = rstd[at];
        if (GRAD) {
            k1[c] = c1[at] * per;
            k2[c] = c2[at] * per;
        }
    }
    for (int64_t j = j0 + warp * B; j < end; j += W * B) {
        Strip<T, V> v[B], g[GRAD ? B : 1];
#pragma unroll
        for (int u = 0; u < B; ++u)
            if (j + u < end) {
                v[u].load(x + (j + u) * a.sd + i, left);
                if (GRAD) g[u].load(gy + (j + u) * a.gd + i, left);
            }
#pragma unroll
        for (int u = 0; u < B; ++u)
            if (j + u < end) {
                float f[V], t[V];
                v[u].get(f);
                const float w = a.weight != nullptr ? a.weight[j + u] : 1.f;
                if constexpr (GRAD) {
                    g[u].get(t);
#pragma unroll
                    for (int c = 0; c < V; ++c)
                        t[c] = r[c] * (fmaf(t[c], w, -k1[c]) - (f[c] - mu[c]) * r[c] * k2[c]);
                } else {
                    const float b = a.bias != nullptr ? a.bias[j + u] : 0.f;
#pragma unroll
                    for (int c = 0; c < V; ++c) t[c] = fmaf((f[c] - mu[c]) * r[c], w, b);
                }
                Strip<T, V>::store(y + (j + u) * ld + i, left, t);
            }
    }
}

// sums [2, chunks, n]: sum of t and of t h over each chunk's features (t = gy w), by sample; and part [2, strips, d]: sums
// of gy h and of gy over each strip's samples, by feature (null: not wanted).
template <typename T, int V>
__global__ void __launch_bounds__(kColThreads, 2) norm_strip_sums_kernel(const T* __restrict__ x, const T* __restrict__ gy,
                                                                      NormArgs<float> a, int64_t chunk,
                                                                         float* __restrict__ sums,
                                                                      float* __restrict__ part) {
    constexpr int W = kColThreads / 32, B = 4;  // 2 B sums over the lanes at once
    __shared__ float sh[W][2][32 * V];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t i = ((int64_t)blockIdx.x * 32 + lane) * V, j0 = blockIdx.y * chunk;
    const int left = (int)(a.n - i < V ? (a.n > i ? a.n - i : 0) : V);
    const int64_t end = j0 + chunk < a.d ? j0 + chunk : a.d;
    float mu[V], r[V], s1[V] = {}, s2[V] = {};
#pragma unroll
    for (int c = 0; c < V; ++c) {
        mu[c] = c < left ? a.mean[i + c] : 0.f;
        r[c] = c < left ? a.rstd[i + c] : 0.f;
    }
    for (int64_t j = j0 + warp * B; j < end; j += W * B) {
        Strip<T, V> v[B], g[B];
#pragma unroll
        for (int u = 0; u < B; ++u) {
            const int have = j + u < end ? left : 0;
            v[u].load(x + (j + u) * a.sd + i, have);
            g[u].load(gy + (j + u) * a.gd + i, have);
        }
        float both[2 * B];
#pragma unroll
        for (int u = 0; u < B; ++u) {
            float f[V], t[V], p = 0, q = 0;
            v[u].get(f);
            g[u].get(t);
            const float w = a.weight != nullptr && j + u < end ? a.weight[j + u] : 1.f;
#pragma unroll
            for (int c = 0; c < V; ++c) {  // samples and features past the end have gy = h = 0
                const float h = (f[c] - mu[c]) * r[c], th = t[c] * h;
                p += th;
                q += t[c];
                s1[c] = fmaf(t[c], w, s1[c]);
                s2[c] = fmaf(th, w, s2[c]);
            }
            both[u] = p;
            both[B + u] = q;
        }
        if (part != nullptr) {
            // at each step a lane keeps half of its sums and hands over the rest, until one is left
#pragma unroll
            for (int o = 16, k = B; k >= 1; o >>= 1, k >>= 1) {
                const bool up = lane & o;
#pragma unroll
                for (int u = 0; u < k; ++u) {
                    const float keep = up ? both[u + k] : both[u], give = up ? both[u] : both[u + k];
                    both[u] = keep + __shfl_xor_sync(0xffffffffu, give, o);
                }
            }
            constexpr int SAME = 32 / (2 * B);  // neighbouring lanes that hold the same one of the 2 B sums
            float total = both[0];
#pragma unroll
            for (int o = SAME / 2; o >= 1; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
            const int u = lane / SAME;
            const int64_t f = j + (u & (B - 1));
            if (lane % SAME == 0 && f < end) part[((u >= B ? gridDim.x : 0) + (int64_t)blockIdx.x) * a.d + f] = total;
        }
    }
#pragma unroll
    for (int c = 0; c < V; ++c) {
        sh[warp][0][c * 32 + lane] = s1[c];
        sh[warp][1][c * 32 + lane] = s2[c];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 32 * V; c += kColThreads) {
        const int64_t at = (int64_t)blockIdx.x * 32 * V + (c % 32) * V + c / 32;
        float p = 0, q = 0;
        for (int k = 0; k < W; ++k) {
            p += sh[k][0][c];
            q += sh[k][1][c];
        }
        if (at < a.n) {
            sums[blockIdx.y * a.n + at] = p;
            sums[(gridDim.y + blockIdx.y) * a.n + at] = q;
        }
    }
}

struct ColPlan {
    int v;           // samples a thread owns
    int64_t strips;  // of 32 v samples
    int64_t chunk;   // features of a block
    int chunks;
};

ColPlan col_plan(int64_t n, int64_t d, int elem, bool wide, bool backward) {
    ColPlan p{};
    p.v = wide ? 16 / elem : 1;
    p.strips = ceil_div64(n, 32 * p.v);
    // as many blocks as are resident at once (or more strips than that)
    const int64_t resident = (int64_t)gpu_sms() * (backward ? 2 : 3), unit = kColThreads / 32 * kBatch;
    const int64_t wanted = resident > p.strips ? resident / p.strips : 1;
    p.chunk = ceil_div64(ceil_div64(d, wanted), unit) * unit;
    p.chunks = (int)ceil_div64(d, p.chunk);
    return p;
}

template <typename T> struct Norm {
    using A = typename Acc<T>::type;
    static constexpr int VEC = 16 / sizeof(T);

    // rows (of the strided axis) that all start on 16 bytes
    static bool wide(const void* p, int64_t ld, int64_t rows) {
        return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (rows <= 1 || ld % VEC == 0);
    }

    template <auto K> struct Kernel { static constexpr auto value = K; };

    // Lets a kernel's blocks take more shared memory than the default allows: once a kernel and device.
    template <auto K, int BYTES> static cudaError_t allow() {
        static std::atomic<uint64_t> done[2];  // a bit a device
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        if (dev < 128 && (done[dev / 64] >> (dev % 64) & 1)) return cudaSuccess;
        e = cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, BYTES);
        if (e == cudaSuccess && dev < 128) done[dev / 64] |= uint64_t(1) << (dev % 64);
        return e;
    }

    // pick() with the form of the windows
    template <typename F> static cudaError_t form(const LinePlan& p, int64_t d, bool shifted, F pick) {
        if (shifted) return pick(std::integral_constant<Windows, kShifted>());
        if ((int64_t)p.plan.g * p.plan.parts * p.np * VEC == d) return pick(std::integral_constant<Windows, kFull>());
        return pick(std::integral_constant<Windows, kWhole>());
    }

    // weight or bias off the boundary of a window's entries (16 or 32 bytes)
    static bool loose(const NormArgs<A>& a) {
        return (reinterpret_cast<uintptr_t>(a.weight) | reinterpret_cast<uintptr_t>(a.bias)) % (VEC * 4) != 0;
    }

    static size_t workspace(int64_t n, int64_t d, bool cols, bool backward) {
        if (sizeof(A) != 4 || n == 0) return 0;
        int64_t most = 0;
        for (int k = 0; k < 2; ++k) {  // whichever way the pointers turn out to be aligned
            if (cols) {
                const ColPlan p = col_plan(n, d, (int)sizeof(T), k == 0, backward);
                const int64_t need = 2 * p.chunks * n + 2 * n + (backward ? 2 * p.strips * d : 0);
                most = need > most ? need : most;
            } else if (backward) {
                const LinePlan p = line_plan(n, d, VEC, k == 0, true);
                const int64_t need = p.np != 0 ? 2 * p.blocks * d : 0;
                most = need > most ? need : most;
            }
        }
        return (size_t)most * sizeof(A);
    }

    template <int V> static cudaError_t forward_strips(const T* x, T* y, NormArgs<float> a, const ColPlan& p, float* ws,
                                                       cudaStream_t s) {
        float* stats = ws + 2 * a.n;
        if (a.mean == nullptr) a.mean = ws;
        if (a.rstd == nullptr) a.rstd = ws + a.n;
        const dim3 grid((unsigned)p.strips, (unsigned)p.chunks);
        norm_strip_stats_kernel<T, V><<<grid, kColThreads, 0, s>>>(x, a, p.chunk, stats);
        norm_strip_fold_kernel<<<(unsigned)ceil_div64(a.n, 32), 1024, 0, s>>>(stats, a.n, a.d, p.chunk, p.chunks, a.eps, a.mean,
                                                                           a.rstd);
        norm_strip_apply_kernel<T, V, false><<<grid, kColThreads, 0, s>>>(x, nullptr, y, a, p.chunk, a.mean, a.rstd, nullptr,
                                                                          nullptr);
        count_launches(3);
        return cudaGetLastError();
    }

    template <int V> static cudaError_t backward_strips(const T* x, const T* gy, T* gx, float* gw, float* gb,
                                                        const NormArgs<float>& a, const ColPlan& p, float* ws, cudaStream_t s) {
        float *c1 = ws, *c2 = ws + a.n, *sums = ws + 2 * a.n, *part = sums + 2 * p.chunks * a.n;
        const bool weights = gw != nullptr || gb != nullptr;
        const dim3 grid((unsigned)p.strips, (unsigned)p.chunks);
        norm_strip_sums_kernel<T, V><<<grid, kColThreads, 0, s>>>(x, gy, a, p.chunk, sums, weights ? part : nullptr);
        count_launches(1);
        cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return e;
        const Fold samples{sums, p.chunks, a.n, a.n, c1, c2}, features{part, p.strips, a.d, a.d, gw, gb};
        if (gx == nullptr) return weights ? launch_fold(features, Fold{}, s) : cudaSuccess;
        e = launch_fold(samples, weights ? features : Fold{}, s);
        if (e != cudaSuccess) return e;
        norm_strip_apply_kernel<T, V, true><<<grid, kColThreads, 0, s>>>(x, gy, gx, a, p.chunk, a.mean, a.rstd, c1, c2);
        count_launches(1);
        return cudaGetLastError();
    }

    static cudaError_t forward(const void* x, void* y, const NormArgs<A>& a, bool cols, void* ws, cudaStream_t s) {
        if constexpr (sizeof(A) == 4) {
            if (cols) {
                const bool w = wide(x, a.sd, a.d) && wide(y, a.gd, a.d);
                const ColPlan p = col_plan(a.n, a.d, (int)sizeof(T), w, false);
                return w ? forward_strips<VEC>((const T*)x, (T*)y, a, p, (float*)ws, s)
                         : forward_strips<1>((const T*)x, (T*)y, a, p, (float*)ws, s);
            }
            const bool shifted = !wide(x, a.sn, a.n) || !wide(y, a.gn, a.n) || a.d % VEC != 0 || loose(a);
            LinePlan p = line_plan(a.n, a.d, VEC, shifted, false);
            p.plan.loose = loose(a);
            if (p.np != 0) {
                const size_t rows = (size_t)kStages * p.np * 16 * p.plan.g * p.plan.rows;
                auto go = [&](auto k) {
                    constexpr auto kernel = decltype(k)::value;
                    if (const cudaError_t e = allow<kernel, kStages * 4 * 16 * kLineThreads>()) return e;
                    return launch_lines(kernel, p, rows, s, (const T*)x, (T*)y, a, p.plan);
                };
                auto pick = [&](auto mode) {
                    constexpr Windows M = decltype(mode)::value;
                    return p.np == 1   ? go(Kernel<norm_line_kernel<T, 1, M>>())
                           : p.np == 2 ? go(Kernel<norm_line_kernel<T, 2, M>>())
                                       : go(Kernel<norm_line_kernel<T, 4, M>>());
                };
                return form(p, a.d, shifted, pick);
            }
        }
        count_launches(1);
        if constexpr (sizeof(A) == 8) {
            if (cols) {
                norm_cols_kernel<T><<<blocks(ceil_div64(a.n, 32)), dim3(32, 8), 0, s>>>((const T*)x, (T*)y, a);
                return cudaGetLastError();
            }
        }
        norm_rows_kernel<T><<<blocks(a.n), 256, 0, s>>>((const T*)x, (T*)y, a);
        return cudaGetLastError();
    }

    static cudaError_t backward(const void* x, const void* gy, void* gx, A* gw, A* gb, const NormArgs<A>& a, bool cols,
                                void* ws, cudaStream_t s) {
        if constexpr (sizeof(A) == 4) {
            if (cols && a.n > 0) {
                const bool w = wide(x, a.sd, a.d) && wide(gy, a.gd, a.d) && (gx == nullptr || wide(gx, a.od, a.d));
                const ColPlan p = col_plan(a.n, a.d, (int)sizeof(T), w, true);
                return w ? backward_strips<VEC>((const T*)x, (const T*)gy, (T*)gx, gw, gb, a, p, (float*)ws, s)
                         : backward_strips<1>((const T*)x, (const T*)gy, (T*)gx, gw, gb, a, p, (float*)ws, s);
            }
            const bool shifted = !wide(x, a.sn, a.n) || !wide(gy, a.gn, a.n) || (gx != nullptr && !wide(gx, a.on, a.n)) ||
                                 a.d % VEC != 0 || loose(a);
            LinePlan p = line_plan(a.n, a.d, VEC, shifted, true);
            p.plan.loose = loose(a);
            if (a.n > 0 && p.np != 0) {
                float* part = gw != nullptr || gb != nullptr ? (float*)ws : nullptr;
                // the rows on their way; in the end, one group's sums (d floats)
                const size_t rows = (size_t)kStages * 2 * p.np * 16 * p.plan.g * p.plan.rows, sums = (size_t)a.d * 4;
                const size_t shared = part != nullptr && p.plan.rows > 1 && sums > rows ? sums : rows;
                auto go = [&](auto k) {
                    constexpr auto kernel = decltype(k)::value;
                    if (const cudaError_t e = allow<kernel, kStages * 2 * 4 * 16 * 512>()) return e;
                    return launch_lines(kernel, p, shared, s, (const T*)x, (const T*)gy, (T*)gx, a, p.plan, part);
                };
                auto pick = [&](auto mode) {
                    constexpr Windows M = decltype(mode)::value;
                    return p.np == 1   ? go(Kernel<norm_line_grad_kernel<T, 1, M>>())
                           : p.np == 2 ? go(Kernel<norm_line_grad_kernel<T, 2, M>>())
                                       : go(Kernel<norm_line_grad_kernel<T, 4, M>>());
                };
                const cudaError_t e = form(p, a.d, shifted, pick);
                if (e != cudaSuccess || part == nullptr) return e;
                return launch_fold(Fold{part, p.blocks, a.d, a.d, gw, gb}, Fold{}, s);
            }
        }
        if constexpr (sizeof(A) == 8) {
            if (cols) {
                if (gx != nullptr) {
                    norm_cols_grad_kernel<T><<<blocks(ceil_div64(a.n, 32)), dim3(32, 8), 0, s>>>((const T*)x, (const T*)gy,
                                                                                               (T*)gx, a);
                    count_launches(1);
                }
                if (gw != nullptr || gb != nullptr) {
                    norm_weight_cols_kernel<T><<<blocks(a.d), 256, 0, s>>>((const T*)x, (const T*)gy, a, gw, gb);
                    count_launches(1);
                }
                return cudaGetLastError();
            }
        }
        if (gx != nullptr) {
            norm_rows_grad_kernel<T><<<blocks(a.n), 256, 0, s>>>((const T*)x, (const T*)gy, (T*)gx, a);
            count_launches(1);
        }
        if (gw != nullptr || gb != nullptr) {  // also of no rows: zeros
            norm_weight_rows_kernel<T><<<blocks(ceil_div64(a.d, 32)), dim3(32, 8), 0, s>>>((const T*)x, (const T*)gy, a, gw, gb);
            count_launches(1);
        }
        return cudaGetLastError();
    }
};

int check(int dtype, const void* x, int64_t ldx, const void* g, int64_t ldg, int64_t n, int64_t d, int cols) {
    if (dtype != CLB_F32 && dtype != CLB_F64 && dtype != CLB_BF16 && dtype != CLB_F16)
        return set_error(CLB_ERR_DTYPE, "layer_norm: unsupported dtype");
    if (n < 0 || d < 1 || d > (int64_t(1) << 31)) return set_error(CLB_ERR_INVALID, "layer_norm: bad sizes");
    if (n > 0 && (!x || !g)) return set_error(CLB_ERR_INVALID, "layer_norm: null pointer");
    const int64_t outer = cols ? d : n, inner = cols ? n : d;
    if (outer > 1 && (ldx < inner || ldg < inner))
        return set_error(CLB_ERR_INVALID, "layer_norm: row stride below the row length");
    return CLB_OK;
}

template <typename A>
NormArgs<A> args(int64_t n, int64_t d, int cols, int64_t ldx, int64_t ldg, int64_t ldo, const void* w, const void* b,
                 double eps, void* mean, void* rstd) {
    NormArgs<A> a{};
    a.n = n;
    a.d = d;
    a.sn = cols ? 1 : ldx;
    a.sd = cols ? ldx : 1;
    a.gn = cols ? 1 : ldg;
    a.gd = cols ? ldg : 1;
    a.on = cols ? 1 : ldo;
    a.od = cols ? ldo : 1;
    a.weight = (const A*)w;
    a.bias = (const A*)b;
    a.eps = (A)eps;
    a.mean = (A*)mean;
    a.rstd = (A*)rstd;
    return a;
}

int done(cudaError_t e) { return e == cudaSuccess ? CLB_OK : set_error(CLB_ERR_CUDA, cudaGetErrorString(e)); }

}  // namespace
}  // namespace clb

using namespace clb;

extern "C" size_t clb_layer_norm_workspace_bytes(int dtype, int64_t n, int64_t d, int feature_major, int backward) {
    if (n < 0 || d < 1) return 0;
    const bool cols = feature_major != 0, back = backward != 0;
    switch (dtype) {
        case CLB_F32: return Norm<float>::workspace(n, d, cols, back);
        case CLB_F64: return Norm<double>::workspace(n, d, cols, back);
        case CLB_BF16: return Norm<__nv_bfloat16>::workspace(n, d, cols, back);
        case CLB_F16: return Norm<__half>::workspace(n, d, cols, back);
        default: return 0;
    }
}

extern "C" int clb_layer_norm_forward(int dtype, const void* x, int64_t ldx, int64_t n, int64_t d, int feature_major,
                                      const void* weight, const void* bias, double eps, void* y, int64_t ldy, void* mean,
                                      void* rstd, void* workspace, size_t workspace_bytes, clb_stream_t stream) {
    if (const int st = check(dtype, x, ldx, y, ldy, n, d, feature_major)) return st;
    if (!(eps >= 0.0)) return set_error(CLB_ERR_INVALID, "layer_norm: eps must not be negative");
    const size_t need = clb_layer_norm_workspace_bytes(dtype, n, d, feature_major, 0);
    if (need > 0 && (!workspace || workspace_bytes < need)) return set_error(CLB_ERR_WORKSPACE, "layer_norm: workspace too small");
    if (n == 0) return CLB_OK;
    cudaStream_t s = (cudaStream_t)stream;
    const bool cols = feature_major != 0;
    const auto f = args<float>(n, d, cols, ldx, ldy, 0, weight, bias, eps, mean, rstd);
    switch (dtype) {
        case CLB_F32: return done(Norm<float>::forward(x, y, f, cols, workspace, s));
        case CLB_F64:
            return done(Norm<double>::forward(x, y, args<double>(n, d, cols, ldx, ldy, 0, weight, bias, eps, mean, rstd), cols,
                                              workspace, s));
        case CLB_BF16: return done(Norm<__nv_bfloat16>::forward(x, y, f, cols, workspace, s));
        default: return done(Norm<__half>::forward(x, y, f, cols, workspace, s));
    }
}

extern "C" int clb_layer_norm_backward(int dtype, const void* x, int64_t ldx, const void* gy, int64_t ldgy, int64_t n,
                                       int64_t d, int feature_major, const void* weight, const void* mean,
                                       const void* rstd, void* gx, int64_t ldgx, void* gw, void* gb, void* workspace,
                                       size_t workspace_bytes, clb_stream_t stream) {
    if (const int st = check(dtype, x, ldx, gy, ldgy, n, d, feature_major)) return st;
    const int64_t outer = feature_major ? d : n, inner = feature_major ? n : d;
    if (gx != nullptr && outer > 1 && ldgx < inner)
        return set_error(CLB_ERR_INVALID, "layer_norm: row stride below the row length");
    if (n > 0 && (!mean || !rstd)) return set_error(CLB_ERR_INVALID, "layer_norm: null pointer");
    const size_t need = clb_layer_norm_workspace_bytes(dtype, n, d, feature_major, 1);
    if (need > 0 && (!workspace || workspace_bytes < need)) return set_error(CLB_ERR_WORKSPACE, "layer_norm: workspace too small");
    cudaStream_t s = (cudaStream_t)stream;
    const bool cols = feature_major != 0;
    if (n == 0) gx = nullptr;  // the weight's gradients of no rows are zero, and are written below
    const auto f = args<float>(n, d, cols, ldx, ldgy, ldgx, weight, nullptr, 0, (void*)mean, (void*)rstd);
    switch (dtype) {
        case CLB_F32: return done(Norm<float>::backward(x, gy, gx, (float*)gw, (float*)gb, f, cols, workspace, s));
        case CLB_F64:
            return done(Norm<double>::backward(
                x, gy, gx, (double*)gw, (double*)gb,
                args<double>(n, d, cols, ldx, ldgy, ldgx, weight, nullptr, 0, (void*)mean, (void*)rstd), cols, workspace, s));
        case CLB_BF16: return done(Norm<__nv_bfloat16>::backward(x, gy, gx, (float*)gw, (float*)gb, f, cols, workspace, s));
        default: return done(Norm<__half>::backward(x, gy, gx, (float*)gw, (float*)gb, f, cols, workspace, s));
    }
}
