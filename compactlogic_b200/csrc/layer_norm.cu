// Layer norm over the features of [n, d] activations, in either storage layout, forward and backward:
//   mu_n = mean_d x,  r_n = 1 / sqrt(mean_d (x - mu)^2 + eps),  h = (x - mu) r,  y = h w + b
//   t = gy w,  gx = r (t - mean_d t - h mean_d (t h)),  gw = sum_n gy h,  gb = sum_n gy
// Statistics and sums are held in the arithmetic type (fp32; fp64 for fp64 activations).
#include <cuda_runtime.h>

#include "common.cuh"
#include "kernels.h"

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

// Rows contiguous: one block per row.
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

unsigned blocks(int64_t n) { return (unsigned)(n < (1 << 30) ? n : (1 << 30)); }

template <typename T> struct Norm {
    using A = typename Acc<T>::type;

    static cudaError_t forward(const void* x, void* y, const NormArgs<A>& a, bool cols, cudaStream_t s) {
        if (cols)
            norm_cols_kernel<T><<<blocks(ceil_div64(a.n, 32)), dim3(32, 8), 0, s>>>((const T*)x, (T*)y, a);
        else
            norm_rows_kernel<T><<<blocks(a.n), 256, 0, s>>>((const T*)x, (T*)y, a);
        count_launches(1);
        return cudaGetLastError();
    }

    static cudaError_t backward(const void* x, const void* gy, void* gx, A* gw, A* gb, const NormArgs<A>& a, bool cols,
                                cudaStream_t s) {
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
    (void)dtype, (void)n, (void)d, (void)feature_major, (void)backward;
    return 0;
}

extern "C" int clb_layer_norm_forward(int dtype, const void* x, int64_t ldx, int64_t n, int64_t d, int feature_major,
                                      const void* weight, const void* bias, double eps, void* y, int64_t ldy, void* mean,
                                      void* rstd, void* workspace, size_t workspace_bytes, clb_stream_t stream) {
    if (const int st = check(dtype, x, ldx, y, ldy, n, d, feature_major)) return st;
    if (!(eps >= 0.0)) return set_error(CLB_ERR_INVALID, "layer_norm: eps must not be negative");
    (void)workspace, (void)workspace_bytes;
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
    (void)workspace, (void)workspace_bytes;
    cudaStream_t s = (cudaStream_t)stream;
    const bool cols = feature_major != 0;
    if (n == 0) gx = nullptr;  // the weight's gradients of no rows are zero, and are written below
    const auto f = args<float>(n, d, cols, ldx, ldgy, ldgx, weight, nullptr, 0, (void*)mean, (void*)rstd);
    switch (dtype) {
        case CLB_F32: return done(Norm<float>::backward(x, gy, gx, (float*)gw, (float*)gb, f, cols, s));
        case CLB_F64:
            return done(Norm<double>::backward(
                x, gy, gx, (double*)gw, (double*)gb,
                args<double>(n, d, cols, ldx, ldgy, ldgx, weight, nullptr, 0, (void*)mean, (void*)rstd), cols, s));
        case CLB_BF16: return done(Norm<__nv_bfloat16>::backward(x, gy, gx, (float*)gw, (float*)gb, f, cols, s));
        default: return done(Norm<__half>::backward(x, gy, gx, (float*)gw, (float*)gb, f, cols, s));
    }
}
