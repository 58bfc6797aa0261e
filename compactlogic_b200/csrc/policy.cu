// Losses on class logits z [n, v]: the log-probability of one chosen action a_i per row, and the clipped policy loss built
// on it, forward and backward.
//   lp_i = z[i, a_i] / T - log sum_j exp(z[i, j] / T)
//   ratio = exp(lp - old),  pg = -min(ratio A, clip(ratio, lo, hi) A),  kl = exp(q) - q - 1 with q = ref - lp
//   loss = scale * sum over counted rows of (pg + beta kl),  scale = 1 / (number of counted rows), or 1
//   slope = d loss_i / d lp_i = -A ratio [ratio A <= clip(ratio) A] + beta (1 - exp(q))
//   d loss / d z[i, j] = scale slope / T ([j = a_i] - softmax(z[i] / T)_j)
// A row's softmax is kept as its maximum m and the sum of exp((z - m) / T): z - m is exact where it matters, also for rows
// that hold the type's lowest value or -inf.  A row that is not counted is not read, gives zeros, and has a zero gradient.
// A counted row whose action lies outside [0, v) gives NaN (no memory is read for it).
#include <cuda_runtime.h>

#include "common.cuh"
#include "kernels.h"

namespace clb {

namespace {

// exp((z - m) / T): fp32 through the hardware's base-2 exponential with log2(e) / T folded into one factor.
__device__ __forceinline__ float soft_exp(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ double soft_exp(double x) { return exp(x); }
inline float soft_factor(float inv_t) { return (float)(1.4426950408889634 * (double)inv_t); }
inline double soft_factor(double inv_t) { return inv_t; }

template <typename A> __device__ __forceinline__ A lowest() { return -(A)INFINITY; }

template <typename A> struct RowArgs {
    int64_t n, v, sn, sv;  // element (i, j) of z is z[i * sn + j * sv]
    const int64_t* actions;
    const uint8_t* mask;   // null: every row counts
    A inv_t, factor;
    A* logp;
    A* stats;              // [2, n]: the rows' maxima and sums
    // the policy loss (null `adv`: log-probabilities only)
    const A *adv, *old_lp, *ref;
    A lo, hi, beta;
    A *ratio, *kl, *slope, *row_loss;
};

// One row from its maximum and sum; returns d loss_i / d lp_i before the scale.
template <typename T, typename A = typename Acc<T>::type>
__device__ A finish_row(const T* __restrict__ z, const RowArgs<A>& a, int64_t i, A m, A s) {
    const int64_t act = a.actions[i];
    A lp = (A)NAN;
    if (act >= 0 && act < a.v) lp = (to_acc(z[i * a.sn + act * a.sv]) - m) * a.inv_t - log(s);
    a.logp[i] = lp;
    if (a.stats != nullptr) {
        a.stats[i] = m;
        a.stats[a.n + i] = s;
    }
    if (a.adv == nullptr) return (A)0;
    const A adv = a.adv[i], r = exp(lp - a.old_lp[i]);
    const A held = r < a.lo ? a.lo : r > a.hi ? a.hi : r;  // NaN stays NaN
    const A free_ = r * adv, kept = held * adv;
    A loss = -(free_ <= kept ? free_ : kept), slope = free_ <= kept ? -free_ : (A)0;
    if (free_ != free_) loss = slope = free_;
    a.ratio[i] = r;
    if (a.ref != nullptr) {
        const A q = a.ref[i] - lp, e = expm1(q);
        a.kl[i] = e - q;
        loss += a.beta * (e - q);
        slope -= a.beta * e;
    }
    a.row_loss[i] = loss;
    if (a.slope != nullptr) a.slope[i] = slope;
    return slope;
}

template <typename A> __device__ void skip_row(const RowArgs<A>& a, int64_t i) {
    a.logp[i] = 0;
    if (a.stats != nullptr) {
        a.stats[i] = 0;
        a.stats[a.n + i] = 1;
    }
    if (a.adv == nullptr) return;
    a.ratio[i] = 0;
    if (a.ref != nullptr) a.kl[i] = 0;
    a.row_loss[i] = 0;
    if (a.slope != nullptr) a.slope[i] = 0;
}

// Running maximum and sum.  An empty or all -inf part has m = -inf, s = 0; such a whole row ends with log(0) and NaN, as
// the formula does.
template <typename A> struct Run {
    A m = lowest<A>(), s = 0;
    __device__ __forceinline__ void add(A z, A factor) {
        if (z > m) {
            s *= soft_exp((m - z) * factor);  // m = -inf: 0 * s, and s is still 0 or NaN
            m = z;
        }
        s += soft_exp((z - (m == lowest<A>() ? (A)0 : m)) * factor);
    }
    __device__ __forceinline__ void merge(A m2, A s2, A factor) {
        const A top = m > m2 ? m : m2, safe = top == lowest<A>() ? (A)0 : top;
        s = s * soft_exp((m - safe) * factor) + s2 * soft_exp((m2 - safe) * factor);
        m = top;
    }
};

template <typename A> __device__ __forceinline__ void warp_merge(Run<A>& r, A factor) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const A m2 = __shfl_xor_sync(0xffffffffu, r.m, o), s2 = __shfl_xor_sync(0xffffffffu, r.s, o);
        r.merge(m2, s2, factor);
    }
}

// Logits contiguous: one block per row, which reads its row once.
template <typename T>
__global__ void __launch_bounds__(256) rows_forward_kernel(const T* __restrict__ z, RowArgs<typename Acc<T>::type> a) {
    using A = typename Acc<T>::type;
    __shared__ A sm[8], ss[8];
    for (int64_t i = blockIdx.x; i < a.n; i += gridDim.x) {
        if (a.mask != nullptr && !a.mask[i]) {
            if (threadIdx.x == 0) skip_row(a, i);
            continue;
        }
        Run<A> r;
        for (int64_t j = threadIdx.x; j < a.v; j += blockDim.x) r.add(to_acc(z[i * a.sn + j * a.sv]), a.factor);
        warp_merge(r, a.factor);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) {
            sm[threadIdx.x >> 5] = r.m;
            ss[threadIdx.x >> 5] = r.s;
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < (int)(blockDim.x >> 5); ++w) r.merge(sm[w], ss[w], a.factor);
            finish_row<T>(z, a, i, r.m, r.s);
        }
    }
}

// Samples contiguous: 32 x 8 threads per 32 rows, the lanes along the rows.
template <typename T>
__global__ void __launch_bounds__(256) cols_forward_kernel(const T* __restrict__ z, RowArgs<typename Acc<T>::type> a) {
    using A = typename Acc<T>::type;
    __shared__ A sm[8][33], ss[8][33];
    const int64_t i = (int64_t)blockIdx.x * 32 + threadIdx.x;
    const bool live = i < a.n && (a.mask == nullptr || a.mask[i]);
    Run<A> r;
    if (live)
        for (int64_t j = threadIdx.y; j < a.v; j += blockDim.y) r.add(to_acc(z[i * a.sn + j * a.sv]), a.factor);
    sm[threadIdx.y][threadIdx.x] = r.m;
    ss[threadIdx.y][threadIdx.x] = r.s;
    __syncthreads();
    if (threadIdx.y != 0 || i >= a.n) return;
    if (!live) {
        skip_row(a, i);
        return;
    }
    for (int w = 1; w < (int)blockDim.y; ++w) r.merge(sm[w][threadIdx.x], ss[w][threadIdx.x], a.factor);
    finish_row<T>(z, a, i, r.m, r.s);
}

template <typename A> struct GradArgs {
    int64_t n, v, sn, sv, gn, gv;
    const int64_t* actions;
    const uint8_t* mask;
    A inv_t, factor;
    const A* stats;
    const A* slope;     // null: 1
    const A* scale;     // device scalar; null: 1
    const A* upstream;  // upstream[i * up_stride]; null: 1
    int64_t up_stride;
    int unless_one;     // leave gz alone when the (scalar) upstream gradient is 1
};

template <typename T, bool COLS>
__global__ void __launch_bounds__(256) logit_grad_kernel(const T* __restrict__ z, T* __restrict__ gz,
                                                         GradArgs<typename Acc<T>::type> a) {
    using A = typename Acc<T>::type;
    if (a.unless_one && a.upstream[0] == (A)1) return;
    const A scale = a.scale != nullptr ? a.scale[0] : (A)1;
    // COLS: lanes along the rows, threadIdx.y along the classes; else the whole block along the classes of one row
    for (int64_t b = blockIdx.x; COLS ? b * 32 < a.n : b < a.n; b += gridDim.x) {
        const int64_t i = COLS ? b * 32 + threadIdx.x : b;
        if (i >= a.n) continue;
        const bool live = a.mask == nullptr || a.mask[i];
        A c = 0, m = 0, inv = 0;
        int64_t act = -1;
        if (live) {
            c = (a.slope != nullptr ? a.slope[i] : (A)1) * scale * (a.upstream != nullptr ? a.upstream[i * a.up_stride] : (A)1) *
                a.inv_t;
            m = a.stats[i];
            inv = (A)1 / a.stats[a.n + i];
            act = a.actions[i];
            if (act < 0 || act >= a.v) c = (A)NAN;
        }
        for (int64_t j = COLS ? threadIdx.y : threadIdx.x; j < a.v; j += COLS ? blockDim.y : blockDim.x) {
            A g = 0;
            if (live) {
                g = -c * (soft_exp((to_acc(z[i * a.sn + j * a.sv]) - m) * a.factor) * inv);
                if (j == act) g += c;
            }
            gz[i * a.gn + j * a.gv] = from_acc<T>(g);
        }
    }
}

// Counted rows, and the loss from the rows' losses: one block, a fixed order of summation.
template <typename A>
__global__ void __launch_bounds__(1024) loss_kernel(const A* __restrict__ row_loss, const uint8_t* __restrict__ mask,
                                                    int64_t n, int mean, A* loss, A* scale) {
    __shared__ A sh[32];
    __shared__ long long sc[32];
    A s = 0;
    long long c = 0;
    for (int64_t i = threadIdx.x; i < n; i += blockDim.x) {
        s += row_loss[i];
        c += mask == nullptr || mask[i];
    }
    s = warp_sum(s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
    if ((threadIdx.x & 31) == 0) {
        sh[threadIdx.x >> 5] = s;
        sc[threadIdx.x >> 5] = c;
    }
    __syncthreads();
    if (threadIdx.x >= 32) return;
    s = warp_sum(sh[threadIdx.x]);
    c = sc[threadIdx.x];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
    if (threadIdx.x == 0) {
        const A f = mean ? (A)1 / (A)(c > 0 ? c : 1) : (A)1;
        scale[0] = f;
        if (loss != nullptr) loss[0] = s * f;
    }
}

unsigned blocks(int64_t n) { return (unsigned)(n < (1 << 30) ? n : (1 << 30)); }

template <typename T> struct Logits {
    using A = typename Acc<T>::type;

    static cudaError_t forward(const void* z, const RowArgs<A>& a, bool cols, cudaStream_t s) {
        if (cols)
            cols_forward_kernel<T><<<blocks(ceil_div64(a.n, 32)), dim3(32, 8), 0, s>>>((const T*)z, a);
        else
            rows_forward_kernel<T><<<blocks(a.n), 256, 0, s>>>((const T*)z, a);
        count_launches(1);
        return cudaGetLastError();
    }

    static cudaError_t backward(const void* z, void* gz, const GradArgs<A>& a, bool cols, cudaStream_t s) {
        if (cols)
            logit_grad_kernel<T, true><<<blocks(ceil_div64(a.n, 32)), dim3(32, 8), 0, s>>>((const T*)z, (T*)gz, a);
        else
            logit_grad_kernel<T, false><<<blocks(a.n), 256, 0, s>>>((const T*)z, (T*)gz, a);
        count_launches(1);
        return cudaGetLastError();
    }

    static int logp(const void* z, int64_t ldz, int64_t n, int64_t v, bool cols, const int64_t* actions,
                    const uint8_t* mask, double t, void* logp, void* stats, cudaStream_t s) {
        RowArgs<A> a{};
        fill(a, ldz, n, v, cols, actions, mask, t);
        a.logp = (A*)logp;
        a.stats = (A*)stats;
        return status(forward(z, a, cols, s));
    }

    static void fill(RowArgs<A>& a, int64_t ldz, int64_t n, int64_t v, bool cols, const int64_t* actions,
                     const uint8_t* mask, double t) {
        a.n = n;
        a.v = v;
        a.sn = cols ? 1 : ldz;
        a.sv = cols ? ldz : 1;
        a.actions = actions;
        a.mask = mask;
        a.inv_t = (A)(1.0 / t);
        a.factor = soft_factor(a.inv_t);
    }

    static int status(cudaError_t e) { return e == cudaSuccess ? CLB_OK : set_error(CLB_ERR_CUDA, cudaGetErrorString(e)); }

    static int grad(const void* z, int64_t ldz, int64_t n, int64_t v, bool cols, const int64_t* actions,
                    const uint8_t* mask, double t, const void* stats, const void* slope, const void* scale,
                    const void* upstream, int64_t up_stride, int unless_one, void* gz, int64_t ldgz, cudaStream_t s) {
        GradArgs<A> a{};
        a.n = n;
        a.v = v;
        a.sn = cols ? 1 : ldz;
        a.sv = cols ? ldz : 1;
        a.gn = cols ? 1 : ldgz;
        a.gv = cols ? ldgz : 1;
        a.actions = actions;
        a.mask = mask;
        a.inv_t = (A)(1.0 / t);
        a.factor = soft_factor(a.inv_t);
        a.stats = (const A*)stats;
        a.slope = (const A*)slope;
        a.scale = (const A*)scale;
        a.upstream = (const A*)upstream;
        a.up_stride = up_stride;
        a.unless_one = unless_one;
        return status(backward(z, gz, a, cols, s));
    }

    static int policy(const void* z, int64_t ldz, int64_t n, int64_t v, bool cols, const int64_t* actions,
                      const uint8_t* mask, const void* adv, const void* old_lp, const void* ref, double lo, double hi,
                      double beta, double t, int mean, void* loss, void* scale, void* row_loss, void* logp, void* ratio,
                      void* kl, void* slope, void* stats, void* gz, int64_t ldgz, cudaStream_t s) {
        RowArgs<A> a{};
        fill(a, ldz, n, v, cols, actions, mask, t);
        a.logp = (A*)logp;
        a.stats = (A*)stats;
        a.adv = (const A*)adv;
        a.old_lp = (const A*)old_lp;
        a.ref = (const A*)ref;
        a.lo = (A)lo;
        a.hi = (A)hi;
        a.beta = (A)beta;
        a.ratio = (A*)ratio;
        a.kl = (A*)kl;
        a.slope = (A*)slope;
        a.row_loss = (A*)row_loss;
        if (n > 0)
            if (const int st = status(forward(z, a, cols, s))) return st;
        loss_kernel<A><<<1, 1024, 0, s>>>((const A*)row_loss, mask, n, mean, (A*)loss, (A*)scale);
        count_launches(1);
        if (const int st = status(cudaGetLastError())) return st;
        if (gz == nullptr || n == 0) return CLB_OK;
        return grad(z, ldz, n, v, cols, actions, mask, t, stats, slope, scale, nullptr, 0, 0, gz, ldgz, s);
    }
};

int check(const char* what, int dtype, const void* z, int64_t ldz, int64_t n, int64_t v, int cols, const int64_t* actions,
          double t) {
    if (dtype != CLB_F32 && dtype != CLB_F64 && dtype != CLB_BF16 && dtype != CLB_F16) return set_error(CLB_ERR_DTYPE, what);
    if (n < 0 || v < 1) return set_error(CLB_ERR_INVALID, what);
    if (!(t > 0.0)) return set_error(CLB_ERR_INVALID, "logits: the temperature must be positive");
    if (n > 0 && (!z || !actions)) return set_error(CLB_ERR_INVALID, "logits: null pointer");
    const int64_t outer = cols ? v : n, inner = cols ? n : v;
    if (outer > 1 && ldz < inner) return set_error(CLB_ERR_INVALID, "logits: row stride below the row length");
    return CLB_OK;
}

}  // namespace
}  // namespace clb

using namespace clb;

#define CLB_LOGITS(dtype, call)                                  \
    switch (dtype) {                                             \
        case CLB_F32: return Logits<float>::call;                \
        case CLB_F64: return Logits<double>::call;               \
        case CLB_BF16: return Logits<__nv_bfloat16>::call;       \
        default: return Logits<__half>::call;                    \
    }

extern "C" int clb_action_logp(int dtype, const void* z, int64_t ldz, int64_t n, int64_t v, int class_major,
                               const int64_t* actions, const uint8_t* mask, double temperature, void* logp, void* stats,
                               clb_stream_t stream) {
    if (const int st = check("action_logp: bad dtype or sizes", dtype, z, ldz, n, v, class_major, actions, temperature))
        return st;
    if (n == 0) return CLB_OK;
    if (!logp) return set_error(CLB_ERR_INVALID, "action_logp: null pointer");
    CLB_LOGITS(dtype, logp(z, ldz, n, v, class_major != 0, actions, mask, temperature, logp, stats, (cudaStream_t)stream));
}

extern "C" int clb_logit_grad(int dtype, const void* z, int64_t ldz, int64_t n, int64_t v, int class_major,
                              const int64_t* actions, const uint8_t* mask, double temperature, const void* stats,
                              const void* slope, const void* scale, const void* upstream, int64_t upstream_stride,
                              int unless_one, void* gz, int64_t ldgz, clb_stream_t stream) {
    if (const int st = check("logit_grad: bad dtype or sizes", dtype, z, ldz, n, v, class_major, actions, temperature))
        return st;
    if (n == 0) return CLB_OK;
    if (!stats || !gz || (unless_one && (!upstream || upstream_stride != 0)))
        return set_error(CLB_ERR_INVALID, "logit_grad: null pointer, or unless_one without a scalar upstream gradient");
    if ((class_major ? v : n) > 1 && ldgz < (class_major ? n : v))
        return set_error(CLB_ERR_INVALID, "logit_grad: row stride below the row length");
    CLB_LOGITS(dtype, grad(z, ldz, n, v, class_major != 0, actions, mask, temperature, stats, slope, scale, upstream,
                           upstream_stride, unless_one, gz, ldgz, (cudaStream_t)stream));
}

extern "C" int clb_policy_loss(int dtype, const void* z, int64_t ldz, int64_t n, int64_t v, int class_major,
                               const int64_t* actions, const uint8_t* mask, const void* advantages, const void* old_logp,
                               const void* ref_logp, double clip_low, double clip_high, double kl_coef, double temperature,
                               int mean, void* loss, void* scale, void* row_loss, void* logp, void* ratio, void* kl,
                               void* slope, void* stats, void* gz, int64_t ldgz, clb_stream_t stream) {
    if (const int st = check("policy_loss: bad dtype or sizes", dtype, z, ldz, n, v, class_major, actions, temperature))
        return st;
    if (!(clip_low >= 0.0) || !(clip_high >= 0.0)) return set_error(CLB_ERR_INVALID, "policy_loss: negative clip range");
    if (!scale || (n > 0 && (!advantages || !old_logp || !row_loss || !logp || !ratio || (ref_logp && !kl))))
        return set_error(CLB_ERR_INVALID, "policy_loss: null pointer");
    if (gz != nullptr && (!stats || !slope)) return set_error(CLB_ERR_INVALID, "policy_loss: a gradient needs stats and slope");
    if (gz != nullptr && (class_major ? v : n) > 1 && ldgz < (class_major ? n : v))
        return set_error(CLB_ERR_INVALID, "policy_loss: row stride below the row length");
    CLB_LOGITS(dtype, policy(z, ldz, n, v, class_major != 0, actions, mask, advantages, old_logp, ref_logp, 1.0 - clip_low,
                             1.0 + clip_high, kl_coef, temperature, mean, loss, scale, row_loss, logp, ratio, kl, slope,
                             stats, gz, ldgz, (cudaStream_t)stream));
}
