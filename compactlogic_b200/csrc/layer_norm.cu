// Layer norm over the features of [n, d] activations, in either storage layout, forward and backward:
//   mu_n = mean_d x,  r_n = 1 / sqrt(mean_d (x - mu)^2 + eps),  h = (x - mu) r,  y = h w + b
//   t = gy w,  gx = r (t - mean_d t - h mean_d (t h)),  gw = sum_n gy h,  gb = sum_n gy
// Statistics and sums are held in the arithmetic type (fp32; fp64 for fp64 activations).
#include <cuda_runtime.h>

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

// Samples contiguous: a block of 32 x 8 threads per 32 samples, the lanes along the samples.
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

// ... and one block per feature when the samples are.
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

// ---- rows held in registers (fp32 / bf16 / fp16) ----
// G threads own a row (of `parts` blocks of a cluster: a contiguous share of it), E entries each, and walk down the rows
// with the next row's loads in flight; weight, bias and the weight's gradients of a thread's columns stay in its registers
// all the way.  A row is cut into 16-byte windows from the last 16-byte boundary before it, `shift` entries back; thread t of
// a share owns windows t, t + G, ...  The rows of one thread are a multiple of a whole pack's entries apart, so their shift
// is the same and a thread's columns do not move.

template <typename T> __device__ __forceinline__ int shift_of(const T* p) {
    return (int)((reinterpret_cast<uintptr_t>(p) / sizeof(T)) % (16 / sizeof(T)));
}

template <typename T, int E> struct Line {
    static constexpr int VEC = 16 / sizeof(T);
    Pack<T, VEC> p[E / VEC];

    // column of entry e, with c0 = column of the thread's first window (negative before the row)
    static __device__ __forceinline__ int column(int e, int c0, int g) { return c0 + e / VEC * g * VEC + e % VEC; }

    // d = 0: nothing, all zeros.  wide: the row's windows are whole 16-byte words of memory
    __device__ __forceinline__ void load(const T* __restrict__ row, int c0, int g, int d, bool wide) {
        const unsigned whole = wide && d >= VEC ? d - VEC + 1 : 0;
#pragma unroll
        for (int u = 0; u < E / VEC; ++u) {
            const int c = c0 + u * g * VEC;
            if ((unsigned)c < whole) {
                p[u].load(row + c);
            } else {
                p[u] = {};
                if (c < d && c + VEC > 0) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j)
                        if ((unsigned)(c + j) < (unsigned)d) p[u].raw(j, row[c + j]);
                }
            }
        }
    }
    __device__ __forceinline__ void get(float (&f)[E]) const {
#pragma unroll
        for (int u = 0; u < E / VEC; ++u) {
            float v[VEC];
            p[u].get(v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) f[u * VEC + j] = v[j];
        }
    }
    static __device__ __forceinline__ void store(T* __restrict__ row, int c0, int g, int d, bool wide, const float (&f)[E]) {
        const unsigned whole = wide && d >= VEC ? d - VEC + 1 : 0;
#pragma unroll
        for (int u = 0; u < E / VEC; ++u) {
            const int c = c0 + u * g * VEC;
            if (c >= d) break;
            float v[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = f[u * VEC + j];
            Pack<T, VEC> q;
            q.put(v);
            if ((unsigned)c < whole) {
                q.store(row + c);
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if ((unsigned)(c + j) < (unsigned)d) row[c + j] = q.raw(j);
            }
        }
    }
};

constexpr int kMostThreads = 512, kMostParts = 8;

struct RowPlan {
    int g, rows, parts;  // threads a row and block, rows a block, blocks a row
};

// Sum over the G threads of a row within a block (the whole warp for G = 32), through `sh`.
__device__ __forceinline__ float group_sum(float v, float* sh, int g) {
    v = warp_sum(v);
    if (g == 32) return v;
    const int w = g >> 5, warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) sh[warp] = v;
    __syncthreads();
    float t = 0;
    for (int k = warp / w * w, end = k + w; k < end; ++k) t += sh[k];
    return t;
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

template <typename T, int E>
__global__ void __launch_bounds__(kMostThreads) norm_line_kernel(const T* __restrict__ x, T* __restrict__ y, NormArgs<float> a,
                                                                 RowPlan plan) {
    using L = Line<T, E>;
    __shared__ float sums[kMostThreads / 32], squares[kMostThreads / 32];
    __shared__ float2 shares[2][kMostParts];
    const int g = plan.g, t = threadIdx.x % g, rank = (int)(blockIdx.x % (unsigned)plan.parts);
    const int share = g * E, d = (int)a.d;
    if (plan.parts > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    const int64_t step = (int64_t)(gridDim.x / (unsigned)plan.parts) * plan.rows;
    int64_t i = (int64_t)(blockIdx.x / (unsigned)plan.parts) * plan.rows + threadIdx.x / g;
    const int shift = shift_of(x + i * a.sn), c0 = rank * share + t * L::VEC - shift;
    const bool same = shift_of(y + i * a.gn) == shift;
    // entries of the row in block k's share
    auto count = [&](int k) { return min(max(d + shift - k * share, 0), share) - (k == 0 ? shift : 0); };
    float w[E], b[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int c = L::column(e, c0, g);
        const bool in = (unsigned)c < (unsigned)d;
        w[e] = in && a.weight != nullptr ? a.weight[c] : 1.f;
        b[e] = in && a.bias != nullptr ? a.bias[c] : 0.f;
    }
    L next;
    next.load(x + (i < a.n ? i : 0) * a.sn, c0, g, i < a.n ? d : 0, true);
    if (plan.parts > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    // every thread of a block takes the same turns, also where its row lies past the end
    for (int64_t top = i - threadIdx.x / g, turn = 0; top < a.n; top += step, i += step, ++turn) {
        float f[E];
        next.get(f);
        const int64_t below = i + step;
        next.load(x + (below < a.n ? below : 0) * a.sn, c0, g, below < a.n ? d : 0, true);
        float s = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) s += f[e];
        float mu = group_sum(s, sums, g) / (float)max(count(rank), 1);
        float q = 0;
#pragma unroll
        for (int u = 0; u < E / L::VEC; ++u) {
            const int c = c0 + u * g * L::VEC;
            const bool whole = c >= 0 && c + L::VEC <= d;
#pragma unroll
            for (int j = 0; j < L::VEC; ++j) {
                const float v = f[u * L::VEC + j] - mu;
                if (whole || (unsigned)(c + j) < (unsigned)d) q = fmaf(v, v, q);
            }
        }
        q = group_sum(q, squares, g);
        if (plan.parts > 1) {
            float2* slots = shares[turn & 1];
            cluster_share(slots, make_float2(mu, q), rank, plan.parts);
            float m = 0;
            for (int k = 0; k < plan.parts; ++k) m += slots[k].x * ((float)count(k) / (float)d);
            q = 0;
            for (int k = 0; k < plan.parts; ++k) {
                const float c = slots[k].x - m;
                q += slots[k].y + c * c * (float)count(k);
            }
            mu = m;
        }
        const float r = 1.f / sqrtf(q / (float)d + a.eps);
        if (i < a.n) {
#pragma unroll
            for (int e = 0; e < E; ++e) f[e] = fmaf((f[e] - mu) * r, w[e], b[e]);
            L::store(y + i * a.gn, c0, g, d, same, f);
            if (t == 0 && rank == 0) {
                if (a.mean != nullptr) a.mean[i] = mu;
                if (a.rstd != nullptr) a.rstd[i] = r;
            }
        }
    }
}

// part: [2, gridDim.x / parts * rows, d] sums of gy h and gy over a group's rows (null: not wanted).  gx null: not wanted.
template <typename T, int E>
__global__ void __launch_bounds__(kMostThreads) norm_line_grad_kernel(const T* __restrict__ x, const T* __restrict__ gy,
                                                                      T* __restrict__ gx, NormArgs<float> a, RowPlan plan,
                                                                      float* __restrict__ part) {
    using L = Line<T, E>;
    __shared__ float2 sums[2][kMostThreads / 32];
    __shared__ float2 shares[2][kMostParts];
    const int g = plan.g, t = threadIdx.x % g, rank = (int)(blockIdx.x % (unsigned)plan.parts), d = (int)a.d;
    if (plan.parts > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    const int64_t step = (int64_t)(gridDim.x / (unsigned)plan.parts) * plan.rows;
    const int64_t group = (int64_t)(blockIdx.x / (unsigned)plan.parts) * plan.rows + threadIdx.x / g;
    int64_t i = group;
    const int shift = shift_of(x + i * a.sn), c0 = (rank * g * (E / L::VEC) + t) * L::VEC - shift;
    const bool wide = shift_of(gy + i * a.gn) == shift, same = gx != nullptr && shift_of(gx + i * a.on) == shift;
    float w[E], gw[E] = {}, gb[E] = {};
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int c = L::column(e, c0, g);
        w[e] = (unsigned)c < (unsigned)d && a.weight != nullptr ? a.weight[c] : 1.f;
    }
    const float per = 1.f / (float)d;
    L xn, gn;
    float mun = 0, rn = 0;
    auto fetch = [&](int64_t k) {
        const bool in = k < a.n;
        xn.load(x + (in ? k : 0) * a.sn, c0, g, in ? d : 0, true);
        gn.load(gy + (in ? k : 0) * a.gn, c0, g, in ? d : 0, wide);
        mun = in ? a.mean[k] : 0.f;
        rn = in ? a.rstd[k] : 0.f;
    };
    fetch(i);
    if (plan.parts > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    for (int64_t top = i - threadIdx.x / g, turn = 0; top < a.n; top += step, i += step, ++turn) {
        float h[E], f[E];
        xn.get(h);
        gn.get(f);
        const float mu = mun, r = rn;
        fetch(i + step);
        float s1 = 0, s2 = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {  // entries past the row have f = 0
            h[e] = (h[e] - mu) * r;
            gw[e] = fmaf(f[e], h[e], gw[e]);
            gb[e] += f[e];
            f[e] *= w[e];
            s1 += f[e];
            s2 = fmaf(f[e], h[e], s2);
        }
        if (gx == nullptr) continue;  // the same for every thread
        s1 = warp_sum(s1);
        s2 = warp_sum(s2);
        if (g > 32) {
            const int nw = g >> 5, warp = threadIdx.x >> 5;
            float2* at = sums[turn & 1];
            if ((threadIdx.x & 31) == 0) at[warp] = make_float2(s1, s2);
            __syncthreads();
            s1 = s2 = 0;
            for (int k = warp / nw * nw, end = k + nw; k < end; ++k) {
                s1 += at[k].x;
                s2 += at[k].y;
            }
        }
        if (plan.parts > 1) {
            float2* slots = shares[turn & 1];
            cluster_share(slots, make_float2(s1, s2), rank, plan.parts);
            s1 = s2 = 0;
            for (int k = 0; k < plan.parts; ++k) {
                s1 += slots[k].x;
                s2 += slots[k].y;
            }
        }
        s1 *= per;
        s2 *= per;
        if (i < a.n) {
#pragma unroll
            for (int e = 0; e < E; ++e) f[e] = r * (f[e] - fmaf(h[e], s2, s1));
            L::store(gx + i * a.on, c0, g, d, same, f);
        }
    }
    if (part == nullptr) return;
    float* at = part + group * d;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int c = L::column(e, c0, g);
        if ((unsigned)c < (unsigned)d) {
            at[c] = gw[e];
            at[step * d + c] = gb[e];
        }
    }
}

// out[j] = sum over p of part[p * ld + j] for j < d, in a fixed order: 32 columns x 32 shares of the rows a block;
// blockIdx.y picks the first or the second `groups` rows, and gw or gb.
__global__ void __launch_bounds__(1024) norm_fold_kernel(const float* __restrict__ part, int64_t groups, int64_t ld, int64_t d,
                                                         float* gw, float* gb) {
    __shared__ float sh[32][33];
    float* out = blockIdx.y == 0 ? gw : gb;
    if (out == nullptr) return;
    part += blockIdx.y * groups * ld;
    const int64_t j = (int64_t)blockIdx.x * 32 + threadIdx.x;
    float s[4] = {};
    if (j < d) {
        int64_t p = threadIdx.y;
        for (; p + 96 < groups; p += 128) {
#pragma unroll
            for (int u = 0; u < 4; ++u) s[u] += part[(p + 32 * u) * ld + j];
        }
        for (; p < groups; p += 32) s[0] += part[p * ld + j];
    }
    sh[threadIdx.y][threadIdx.x] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    const float t = warp_sum(sh[threadIdx.x][threadIdx.y]);
    const int64_t k = (int64_t)blockIdx.x * 32 + threadIdx.y;
    if (threadIdx.x == 0 && k < d) out[k] = t;
}

// The row plan of a width, the entries a thread holds (0: too wide), and the groups of threads that walk the rows.
struct LinePlan {
    RowPlan plan;
    int e;
    int64_t groups;
};

LinePlan line_plan(int64_t n, int64_t d, int vec, bool shifted, bool backward) {
    LinePlan p{};
    if (shifted) d += vec - 1;  // room for the furthest shift
    for (int e = vec; e <= 16; e *= 2)
        if (d <= 32 * e || e == 16) {
            p.e = e;
            break;
        }
    int64_t g = ceil_div64(d, (int64_t)p.e * 32) * 32;
    p.plan.parts = 1;
    while (p.plan.parts < kMostParts && g > kMostThreads) {
        p.plan.parts *= 2;
        g = ceil_div64(d, (int64_t)p.e * 32 * p.plan.parts) * 32;
    }
    if (g > kMostThreads) return {};
    p.plan.g = (int)g;
    p.plan.rows = g <= 64 ? (int)(128 / g) : 1;
    // what is resident at once: the kernels take up to 128 registers a thread, the forward ones of few entries 64
    const int threads = !backward && p.e <= 8 ? 1024 : 512;
    int64_t blocks = (int64_t)gpu_sms() * (threads / (p.plan.g * p.plan.rows)) / p.plan.parts;
    const int64_t most = ceil_div64(n, p.plan.rows);
    blocks = blocks < 1 ? 1 : blocks;
    // rows of one thread a multiple of a pack's entries apart (see above), where it has more than one
    if (shifted && blocks < most && blocks % vec != 0) blocks = blocks > vec ? blocks - blocks % vec : vec;
    p.groups = (blocks < most ? blocks : most) * p.plan.rows;
    return p;
}

template <typename P> struct Same { using type = P; };  // a parameter that is not deduced

template <typename... P> cudaError_t launch_lines(void (*kernel)(P...), const LinePlan& p, cudaStream_t s,
                                                  typename Same<P>::type... args) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[1];
    cfg.gridDim = dim3((unsigned)(p.groups / p.plan.rows * p.plan.parts));
    cfg.blockDim = dim3((unsigned)(p.plan.g * p.plan.rows));
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
// elementwise, reading the operands again.  A call runs both passes over one slab of samples after the other, as many as
// leave a slab's operands in the L2 cache, so that the second pass does not read memory again.

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

// stats [2, chunks, n]: mean and sum of squared differences of each chunk's features, for the samples from `from` on.
template <typename T, int V>
__global__ void __launch_bounds__(kColThreads) norm_strip_stats_kernel(const T* __restrict__ x, NormArgs<float> a,
                                                                       int64_t from, int64_t to, int64_t chunk,
                                                                       float* __restrict__ stats) {
    constexpr int W = kColThreads / 32;
    __shared__ float sh[W][2][32 * V];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t i = from + ((int64_t)blockIdx.x * 32 + lane) * V, j0 = blockIdx.y * chunk;
    const int left = (int)(to - i < V ? (to > i ? to - i : 0) : V);
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
        const int64_t at = from + (int64_t)blockIdx.x * 32 * V + (c % 32) * V + c / 32;
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
        if (at < to) {
            stats[blockIdx.y * a.n + at] = m;
            stats[(gridDim.y + blockIdx.y) * a.n + at] = q;
        }
    }
}

// mean and rstd from the chunks: 32 samples x 8 shares of the chunks a block
__global__ void __launch_bounds__(256) norm_strip_fold_kernel(const float* __restrict__ stats, int64_t n, int64_t d,
                                                              int64_t from, int64_t to, int64_t chunk, int chunks, float eps,
                                                              float* mean, float* rstd) {
    __shared__ float sh[8][3][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t i = from + (int64_t)blockIdx.x * 32 + lane;
    float m = 0, q = 0, n0 = 0;
    if (i < to)
        for (int k = warp; k < chunks; k += 8) {
            const float nk = (float)(d - k * chunk < chunk ? d - k * chunk : chunk), part = nk / (n0 + nk);
            join(m, q, stats[k * n + i], stats[(chunks + k) * n + i], part, n0 * part);
            n0 += nk;
        }
    sh[warp][0][lane] = m;
    sh[warp][1][lane] = q;
    sh[warp][2][lane] = n0;
    __syncthreads();
    if (warp != 0 || i >= to) return;
    for (int k = 1; k < 8; ++k) {
        const float nk = sh[k][2][lane];
        if (nk == 0) break;
        const float part = nk / (n0 + nk);
        join(m, q, sh[k][0][lane], sh[k][1][lane], part, n0 * part);
        n0 += nk;
    }
    mean[i] = m;
    rstd[i] = 1.f / sqrtf(q / (float)d + eps);
}

// y from x, mean and rstd; or gx from x, gy, and the folded sums c1, c2 (GRAD)
template <typename T, int V, bool GRAD>
__global__ void __launch_bounds__(kColThreads) norm_strip_apply_kernel(const T* __restrict__ x, const T* __restrict__ gy,
                                                                       T* __restrict__ y, NormArgs<float> a, int64_t from,
                                                                       int64_t to, int64_t chunk, const float* mean,
                                                                       const float* rstd, const float* c1, const float* c2) {
    constexpr int W = kColThreads / 32, B = GRAD ? 4 : 8;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t i = from + ((int64_t)blockIdx.x * 32 + lane) * V, j0 = blockIdx.y * chunk;
    const int left = (int)(to - i < V ? (to > i ? to - i : 0) : V);
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
__global__ void __launch_bounds__(kColThreads) norm_strip_sums_kernel(const T* __restrict__ x, const T* __restrict__ gy,
                                                                      NormArgs<float> a, int64_t from, int64_t to,
                                                                      int64_t chunk, float* __restrict__ sums,
                                                                      float* __restrict__ part, int64_t strip0,
                                                                      int64_t strips) {
    constexpr int W = kColThreads / 32, B = kBatch;
    __shared__ float sh[W][2][32 * V];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t i = from + ((int64_t)blockIdx.x * 32 + lane) * V, j0 = blockIdx.y * chunk;
    const int left = (int)(to - i < V ? (to > i ? to - i : 0) : V);
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
            // 2 B sums over the lanes at once: at each step a lane keeps half of them and hands over the rest
#pragma unroll
            for (int o = 16, k = B; k >= 1; o >>= 1, k >>= 1) {
                const bool up = lane & o;
#pragma unroll
                for (int u = 0; u < k; ++u) {
                    const float keep = up ? both[u + k] : both[u], give = up ? both[u] : both[u + k];
                    both[u] = keep + __shfl_xor_sync(0xffffffffu, give, o);
                }
            }
            const float total = both[0] + __shfl_xor_sync(0xffffffffu, both[0], 1);
            const int u = lane >> 1;  // which of the 2 B sums this lane holds
            const int64_t f = j + (u & (B - 1));
            if ((lane & 1) == 0 && f < end) part[((u >= B ? strips : 0) + strip0 + blockIdx.x) * a.d + f] = total;
        }
    }
#pragma unroll
    for (int c = 0; c < V; ++c) {
        sh[warp][0][c * 32 + lane] = s1[c];
        sh[warp][1][c * 32 + lane] = s2[c];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 32 * V; c += kColThreads) {
        const int64_t at = from + (int64_t)blockIdx.x * 32 * V + (c % 32) * V + c / 32;
        float p = 0, q = 0;
        for (int k = 0; k < W; ++k) {
            p += sh[k][0][c];
            q += sh[k][1][c];
        }
        if (at < to) {
            sums[blockIdx.y * a.n + at] = p;
            sums[(gridDim.y + blockIdx.y) * a.n + at] = q;
        }
    }
}

struct ColPlan {
    int v;                 // samples a thread owns
    int64_t slab, strips;  // samples of a slab (whole strips), strips of the call
    int64_t chunk;         // features of a block
    int chunks;
};

ColPlan col_plan(int64_t n, int64_t d, int elem, bool wide, bool backward) {
    ColPlan p{};
    p.v = wide ? 16 / elem : 1;
    const int64_t strip = 32 * p.v, all = ceil_div64(n, strip);
    // Half of the L2 cache for a slab's operands; the whole call where it fits
    const int64_t room = (int64_t)48 << 20, bytes = d * strip * elem * (backward ? 2 : 1);
    int64_t per = room / bytes < 1 ? 1 : room / bytes;
    if (all * bytes <= (int64_t)80 << 20 || bytes > room) per = all;
    p.slab = per * strip;
    p.strips = all;
    const int64_t wanted = ceil_div64((int64_t)gpu_sms() * 3, per < all ? per : all), unit = kColThreads / 32 * kBatch;
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
                const int64_t need = p.e != 0 ? 2 * p.groups * d : 0;
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
        for (int64_t from = 0; from < a.n; from += p.slab) {
            const int64_t to = from + p.slab < a.n ? from + p.slab : a.n;
            const dim3 grid((unsigned)ceil_div64(to - from, 32 * V), (unsigned)p.chunks);
            norm_strip_stats_kernel<T, V><<<grid, kColThreads, 0, s>>>(x, a, from, to, p.chunk, stats);
            norm_strip_fold_kernel<<<(unsigned)ceil_div64(to - from, 32), 256, 0, s>>>(stats, a.n, a.d, from, to, p.chunk,
                                                                                     p.chunks, a.eps, a.mean, a.rstd);
            norm_strip_apply_kernel<T, V, false><<<grid, kColThreads, 0, s>>>(x, nullptr, y, a, from, to, p.chunk, a.mean,
                                                                              a.rstd, nullptr, nullptr);
            count_launches(3);
            const cudaError_t e = cudaGetLastError();
            if (e != cudaSuccess) return e;
        }
        return cudaSuccess;
    }

    template <int V> static cudaError_t backward_strips(const T* x, const T* gy, T* gx, float* gw, float* gb,
                                                        const NormArgs<float>& a, const ColPlan& p, float* ws, cudaStream_t s) {
        float *c1 = ws, *c2 = ws + a.n, *sums = ws + 2 * a.n, *part = sums + 2 * p.chunks * a.n;
        const bool weights = gw != nullptr || gb != nullptr;
        for (int64_t from = 0; from < a.n; from += p.slab) {
            const int64_t to = from + p.slab < a.n ? from + p.slab : a.n;
            const dim3 grid((unsigned)ceil_div64(to - from, 32 * V), (unsigned)p.chunks);
            norm_strip_sums_kernel<T, V><<<grid, kColThreads, 0, s>>>(x, gy, a, from, to, p.chunk, sums,
                                                                      weights ? part : nullptr, from / (32 * V), p.strips);
            count_launches(1);
            if (gx != nullptr) {
                norm_fold_kernel<<<dim3((unsigned)ceil_div64(to - from, 32), 2), dim3(32, 32), 0, s>>>(
                    sums + from, p.chunks, a.n, to - from, c1 + from, c2 + from);
                norm_strip_apply_kernel<T, V, true><<<grid, kColThreads, 0, s>>>(x, gy, gx, a, from, to, p.chunk, a.mean,
                                                                                 a.rstd, c1, c2);
                count_launches(2);
            }
            const cudaError_t e = cudaGetLastError();
            if (e != cudaSuccess) return e;
        }
        if (weights) {
            norm_fold_kernel<<<dim3((unsigned)ceil_div64(a.d, 32), 2), dim3(32, 32), 0, s>>>(part, p.strips, a.d, a.d, gw, gb);
            count_launches(1);
        }
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
            const LinePlan p = line_plan(a.n, a.d, VEC, !wide(x, a.sn, a.n), false);
            if (p.e != 0) {
                auto go = [&](auto kernel) { return launch_lines(kernel, p, s, (const T*)x, (T*)y, a, p.plan); };
                return p.e == 16 ? go(norm_line_kernel<T, 16>) : p.e == 8 ? go(norm_line_kernel<T, 8>) : go(norm_line_kernel<T, VEC>);
            }
        }
        count_launches(1);
        if (cols)
            norm_cols_kernel<T><<<blocks(ceil_div64(a.n, 32)), dim3(32, 8), 0, s>>>((const T*)x, (T*)y, a);
        else
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
            const LinePlan p = line_plan(a.n, a.d, VEC, !wide(x, a.sn, a.n), true);
            if (a.n > 0 && p.e != 0) {
                float* part = gw != nullptr || gb != nullptr ? (float*)ws : nullptr;
                auto go = [&](auto kernel) {
                    return launch_lines(kernel, p, s, (const T*)x, (const T*)gy, (T*)gx, a, p.plan, part);
                };
                const cudaError_t e = p.e == 16  ? go(norm_line_grad_kernel<T, 16>)
                                      : p.e == 8 ? go(norm_line_grad_kernel<T, 8>)
                                                 : go(norm_line_grad_kernel<T, VEC>);
                if (e != cudaSuccess || part == nullptr) return e;
                norm_fold_kernel<<<dim3((unsigned)ceil_div64(a.d, 32), 2), dim3(32, 32), 0, s>>>(part, p.groups, a.d, a.d, gw, gb);
                count_launches(1);
                return cudaGetLastError();
            }
        }
        if (gx != nullptr) {
            if (cols)
                norm_cols_grad_kernel<T><<<blocks(ceil_div64(a.n, 32)), dim3(32, 8), 0, s>>>((const T*)x, (const T*)gy,
                                                                                           (T*)gx, a);
            else
                norm_rows_grad_kernel<T><<<blocks(a.n), 256, 0, s>>>((const T*)x, (const T*)gy, (T*)gx, a);
            count_launches(1);
            const cudaError_t e = cudaGetLastError();
            if (e != cudaSuccess) return e;
        }
        if (gw != nullptr || gb != nullptr) {
            if (cols)
                norm_weight_cols_kernel<T><<<blocks(a.d), 256, 0, s>>>((const T*)x, (const T*)gy, a, gw, gb);
            else
                norm_weight_rows_kernel<T><<<blocks(ceil_div64(a.d, 32)), dim3(32, 8), 0, s>>>((const T*)x, (const T*)gy, a,
                                                                                             gw, gb);
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
            return done(Norm<double>::forward(x, y, args<double>(n, d, cols, ldx, ldy, 0, weight, bias, eps, mean, rstd), cols, workspace, s));
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
