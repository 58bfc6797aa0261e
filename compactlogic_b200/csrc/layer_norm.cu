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
// all the way.  ALIGNED: rows start on 16 bytes and hold whole 16-byte packs, thread t owns packs t, t + G, ...; else single
// elements t, t + G, ..., which stay coalesced whatever the rows' alignment.

template <typename T, int E, bool ALIGNED> struct Line {
    static constexpr int VEC = 16 / sizeof(T);
    Pack<T, VEC> p[E / VEC];

    static __device__ __forceinline__ int column(int e, int t, int g) {
        return ALIGNED ? (e / VEC * g + t) * VEC + e % VEC : e * g + t;
    }
    __device__ __forceinline__ void load(const T* __restrict__ row, int t, int g, int d) {
        if constexpr (ALIGNED) {
#pragma unroll
            for (int u = 0; u < E / VEC; ++u) {
                const int c = (u * g + t) * VEC;
                if (c < d)
                    p[u].load(row + c);
                else
                    p[u] = {};
            }
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int c = e * g + t;
                p[e / VEC].raw(e % VEC, c < d ? row[c] : T(0.f));
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
    static __device__ __forceinline__ void store(T* __restrict__ row, int t, int g, int d, const float (&f)[E]) {
#pragma unroll
        for (int u = 0; u < E / VEC; ++u) {
            if constexpr (ALIGNED) {
                const int c = (u * g + t) * VEC;
                if (c < d) {
                    float v[VEC];
#pragma unroll
                    for (int j = 0; j < VEC; ++j) v[j] = f[u * VEC + j];
                    Pack<T, VEC> q;
                    q.put(v);
                    q.store(row + c);
                }
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const int c = (u * VEC + j) * g + t;
                    if (c < d) row[c] = from_acc<T>(f[u * VEC + j]);
                }
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

template <typename T, int E, bool ALIGNED>
__global__ void __launch_bounds__(kMostThreads) norm_line_kernel(const T* __restrict__ x, T* __restrict__ y, NormArgs<float> a,
                                                                 RowPlan plan) {
    using L = Line<T, E, ALIGNED>;
    __shared__ float sums[kMostThreads / 32], squares[kMostThreads / 32];
    __shared__ float2 shares[2][kMostParts];
    const int g = plan.g, t = threadIdx.x % g, rank = (int)(blockIdx.x % (unsigned)plan.parts);
    const int share = g * E, all = (int)a.d;
    const int off = rank * share, d = min(max(all - off, 0), share);  // this block's columns of a row
    if (plan.parts > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    float w[E], b[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int c = L::column(e, t, g);
        w[e] = c < d && a.weight != nullptr ? a.weight[off + c] : 1.f;
        b[e] = c < d && a.bias != nullptr ? a.bias[off + c] : 0.f;
    }
    const int64_t step = (int64_t)(gridDim.x / (unsigned)plan.parts) * plan.rows;
    int64_t i = (int64_t)(blockIdx.x / (unsigned)plan.parts) * plan.rows + threadIdx.x / g;
    L next;
    next.load(x + (i < a.n ? i : 0) * a.sn + off, t, g, i < a.n ? d : 0);
    if (plan.parts > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    // every thread of a block takes the same turns, also where its row lies past the end
    for (int64_t top = i - threadIdx.x / g, turn = 0; top < a.n; top += step, i += step, ++turn) {
        float f[E];
        next.get(f);
        const int64_t below = i + step;
        next.load(x + (below < a.n ? below : 0) * a.sn + off, t, g, below < a.n ? d : 0);
        float s = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) s += f[e];
        float mu = group_sum(s, sums, g) / (float)max(d, 1);
        float q = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float c = L::column(e, t, g) < d ? f[e] - mu : 0.f;
            q += c * c;
        }
        q = group_sum(q, squares, g);
        if (plan.parts > 1) {
            float2* slots = shares[turn & 1];
            cluster_share(slots, make_float2(mu, q), rank, plan.parts);
            float m = 0;
            for (int k = 0; k < plan.parts; ++k) m += slots[k].x * ((float)min(max(all - k * share, 0), share) / (float)all);
            q = 0;
            for (int k = 0; k < plan.parts; ++k) {
                const float c = slots[k].x - m;
                q += slots[k].y + c * c * (float)min(max(all - k * share, 0), share);
            }
            mu = m;
        }
        const float r = 1.f / sqrtf(q / (float)all + a.eps);
        if (i < a.n) {
#pragma unroll
            for (int e = 0; e < E; ++e) f[e] = fmaf((f[e] - mu) * r, w[e], b[e]);
            L::store(y + i * a.gn + off, t, g, d, f);
            if (t == 0 && rank == 0) {
                if (a.mean != nullptr) a.mean[i] = mu;
                if (a.rstd != nullptr) a.rstd[i] = r;
            }
        }
    }
}

// part: [2, gridDim.x / parts * rows, d] sums of gy h and gy over a group's rows (null: not wanted).  gx null: not wanted.
template <typename T, int E, bool ALIGNED>
__global__ void __launch_bounds__(kMostThreads) norm_line_grad_kernel(const T* __restrict__ x, const T* __restrict__ gy,
                                                                      T* __restrict__ gx, NormArgs<float> a, RowPlan plan,
                                                                      float* __restrict__ part) {
    using L = Line<T, E, ALIGNED>;
    __shared__ float first[2][kMostThreads / 32], second[2][kMostThreads / 32];
    __shared__ float2 shares[2][kMostParts];
    const int g = plan.g, t = threadIdx.x % g, rank = (int)(blockIdx.x % (unsigned)plan.parts);
    const int share = g * E, all = (int)a.d;
    const int off = rank * share, d = min(max(all - off, 0), share);
    if (plan.parts > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    float w[E], gw[E] = {}, gb[E] = {};
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int c = L::column(e, t, g);
        w[e] = c < d && a.weight != nullptr ? a.weight[off + c] : 1.f;
    }
    const float per = 1.f / (float)all;
    const int64_t step = (int64_t)(gridDim.x / (unsigned)plan.parts) * plan.rows;
    const int64_t group = (int64_t)(blockIdx.x / (unsigned)plan.parts) * plan.rows + threadIdx.x / g;
    int64_t i = group;
    L xn, gn;
    float mun = 0, rn = 0;
    auto fetch = [&](int64_t k) {
        const bool in = k < a.n;
        xn.load(x + (in ? k : 0) * a.sn + off, t, g, in ? d : 0);
        gn.load(gy + (in ? k : 0) * a.gn + off, t, g, in ? d : 0);
        mun = in ? a.mean[k] : 0.f;
        rn = in ? a.rstd[k] : 0.f;
    };
    fetch(i);
    if (plan.parts > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    for (int64_t top = i - threadIdx.x / g, turn = 0; top < a.n; top += step, i += step, ++turn) {
        const L xi = xn, gi = gn;
        const float mu = mun, r = rn;
        fetch(i + step);
        float h[E], f[E];
        xi.get(h);
        gi.get(f);
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
            const int nw = g >> 5, warp = threadIdx.x >> 5, b = (int)(turn & 1);
            if ((threadIdx.x & 31) == 0) {
                first[b][warp] = s1;
                second[b][warp] = s2;
            }
            __syncthreads();
            s1 = s2 = 0;
            for (int k = warp / nw * nw, end = k + nw; k < end; ++k) {
                s1 += first[b][k];
                s2 += second[b][k];
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
            L::store(gx + i * a.on + off, t, g, d, f);
        }
    }
    if (part == nullptr) return;
    const int64_t groups = step;
    float* at = part + group * a.d + off;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int c = L::column(e, t, g);
        if (c < d) {
            at[c] = gw[e];
            at[groups * a.d + c] = gb[e];
        }
    }
}

// out[j] = sum over p of part[p, j], in a fixed order: 32 columns x 32 shares of the rows a block; blockIdx.y picks gw or gb.
__global__ void __launch_bounds__(1024) norm_fold_kernel(const float* __restrict__ part, int64_t groups, int64_t d, float* gw,
                                                         float* gb) {
    __shared__ float sh[32][33];
    float* out = blockIdx.y == 0 ? gw : gb;
    if (out == nullptr) return;
    part += blockIdx.y * groups * d;
    const int64_t j = (int64_t)blockIdx.x * 32 + threadIdx.x;
    float s[4] = {};
    if (j < d) {
        int64_t p = threadIdx.y;
        for (; p + 96 < groups; p += 128) {
#pragma unroll
            for (int u = 0; u < 4; ++u) s[u] += part[(p + 32 * u) * d + j];
        }
        for (; p < groups; p += 32) s[0] += part[p * d + j];
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

LinePlan line_plan(int64_t n, int64_t d, int vec, bool backward) {
    LinePlan p{};
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

template <typename T> struct Norm {
    using A = typename Acc<T>::type;
    static constexpr int VEC = 16 / sizeof(T);

    static bool aligned(const void* p, int64_t ld, const NormArgs<A>& a) {
        return reinterpret_cast<uintptr_t>(p) % 16 == 0 && a.d % VEC == 0 && (a.n == 1 || ld % VEC == 0);
    }

    static cudaError_t forward(const void* x, void* y, const NormArgs<A>& a, bool cols, cudaStream_t s) {
        if constexpr (sizeof(A) == 4) {
            const LinePlan p = line_plan(a.n, a.d, VEC, false);
            if (!cols && p.e != 0) {
                auto go = [&](auto wide, auto narrow) {
                    return launch_lines(aligned(x, a.sn, a) && aligned(y, a.gn, a) ? wide : narrow, p, s, (const T*)x, (T*)y, a,
                                        p.plan);
                };
                if (p.e == 16) return go(norm_line_kernel<T, 16, true>, norm_line_kernel<T, 16, false>);
                if (p.e == 8) return go(norm_line_kernel<T, 8, true>, norm_line_kernel<T, 8, false>);
                return go(norm_line_kernel<T, VEC, true>, norm_line_kernel<T, VEC, false>);
            }
        }
        count_launches(1);
        if (cols)
            norm_cols_kernel<T><<<blocks(ceil_div64(a.n, 32)), dim3(32, 8), 0, s>>>((const T*)x, (T*)y, a);
        else
            norm_rows_kernel<T><<<blocks(a.n), 256, 0, s>>>((const T*)x, (T*)y, a);
        return cudaGetLastError();
    }

    static size_t workspace(int64_t n, int64_t d, bool cols, bool backward) {
        if (sizeof(A) != 4 || cols || !backward || n == 0) return 0;
        const LinePlan p = line_plan(n, d, VEC, true);
        return p.e != 0 ? (size_t)(2 * p.groups * d) * sizeof(A) : 0;
    }

    static cudaError_t backward(const void* x, const void* gy, void* gx, A* gw, A* gb, const NormArgs<A>& a, bool cols,
                                void* workspace, cudaStream_t s) {
        if constexpr (sizeof(A) == 4) {
            const LinePlan p = line_plan(a.n, a.d, VEC, true);
            if (!cols && a.n > 0 && p.e != 0) {
                float* part = gw != nullptr || gb != nullptr ? (float*)workspace : nullptr;
                auto go = [&](auto wide, auto narrow) {
                    const bool al = aligned(x, a.sn, a) && aligned(gy, a.gn, a) && (gx == nullptr || aligned(gx, a.on, a));
                    return launch_lines(al ? wide : narrow, p, s, (const T*)x, (const T*)gy, (T*)gx, a, p.plan, part);
                };
                const cudaError_t e =
                    p.e == 16 ? go(norm_line_grad_kernel<T, 16, true>, norm_line_grad_kernel<T, 16, false>)
                    : p.e == 8 ? go(norm_line_grad_kernel<T, 8, true>, norm_line_grad_kernel<T, 8, false>)
                               : go(norm_line_grad_kernel<T, VEC, true>, norm_line_grad_kernel<T, VEC, false>);
                if (e != cudaSuccess || part == nullptr) return e;
                norm_fold_kernel<<<dim3((unsigned)ceil_div64(a.d, 32), 2), dim3(32, 32), 0, s>>>(part, p.groups, a.d, gw, gb);
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
        case CLB_F32: return done(Norm<float>::forward(x, y, f, cols, s));
        case CLB_F64:
            return done(Norm<double>::forward(x, y, args<double>(n, d, cols, ldx, ldy, 0, weight, bias, eps, mean, rstd), cols, s));
        case CLB_BF16: return done(Norm<__nv_bfloat16>::forward(x, y, f, cols, s));
        default: return done(Norm<__half>::forward(x, y, f, cols, s));
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
