// Dropout whose mask is a function of (seed, offset, element) and is never stored: the backward pass draws the same words
// again.  The generator is Philox4x32-10 (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as easy as
// 1, 2, 3", SC 2011), written from the paper.
//
// One counter serves a 2 x 2 block of the logical [n, d] matrix: element (n, d) takes word 2 (n & 1) + (d & 1) of
// Philox(counter = (d >> 1, n >> 1, offset), key = seed).  A thread that walks two neighbouring rows of the contiguous axis
// therefore uses all four words of every call whether features or samples are contiguous, and the mask does not depend on
// the storage layout, on strides, or on how the work is split.
#include <cuda_runtime.h>

#include <cmath>

#include "common.cuh"
#include "kernels.h"

namespace clb {

namespace {

struct Words { uint32_t w[4]; };

__device__ __forceinline__ Words philox(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
        c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)p1;
        c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)p0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {{c0, c1, c2, c3}};
}

struct DropArgs {
    int64_t ldx, ldy, rows, cols;  // rows of the strided axis, entries of the contiguous one
    uint64_t seed, offset;
    const int64_t* rng;            // device {seed, offset}; takes the place of the two above
    uint32_t threshold;            // an element is kept when its word >= threshold
    int none;                      // p == 1: nothing is kept
    double scale;
};

// Each thread owns VEC consecutive entries of two neighbouring rows (2 * VEC elements, VEC / 2 Philox calls).
// BATCH_INNER: the contiguous axis is n (feature-major storage), else d.  WIDE: one vector access per row.
template <typename T, int VEC, bool BATCH_INNER, bool WIDE>
__global__ void __launch_bounds__(256) dropout_kernel(const T* __restrict__ x, T* __restrict__ y, DropArgs a) {
    using A = typename Acc<T>::type;
    uint64_t seed = a.seed, offset = a.offset;
    if (a.rng != nullptr) {
        seed = (uint64_t)a.rng[0];
        offset = (uint64_t)a.rng[1];
    }
    const A scale = (A)a.scale;
    const int64_t pairs = (a.rows + 1) >> 1, steps = (a.cols + VEC - 1) / VEC;
    for (int64_t rp = blockIdx.y; rp < pairs; rp += gridDim.y) {
        for (int64_t st = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; st < steps; st += (int64_t)gridDim.x * blockDim.x) {
            const int64_t c = st * VEC, r = rp * 2;
            A v[2][VEC];
            const bool full = c + VEC <= a.cols;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (r + i >= a.rows) continue;
                const T* p = x + (r + i) * a.ldx + c;
                if (WIDE && full) {
                    load_acc<T, VEC>(p, v[i]);
                } else {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) v[i][j] = c + j < a.cols ? to_acc(p[j]) : (A)0;
                }
            }
#pragma unroll
            for (int j = 0; j < VEC; j += 2) {
                const uint32_t inner = (uint32_t)((c + j) >> 1), outer = (uint32_t)rp;
                const Words w = philox(BATCH_INNER ? outer : inner, BATCH_INNER ? inner : outer, (uint32_t)offset,
                                       (uint32_t)(offset >> 32), (uint32_t)seed, (uint32_t)(seed >> 32));
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const uint32_t word = w.w[BATCH_INNER ? 2 * k + i : 2 * i + k];
                        v[i][j + k] = word >= a.threshold && !a.none ? v[i][j + k] * scale : (A)0;
                    }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (r + i >= a.rows) continue;
                T* p = y + (r + i) * a.ldy + c;
                if (WIDE && full) {
                    store_from_acc<T, VEC>(p, v[i]);
                } else {
#pragma unroll
                    for (int j = 0; j < VEC; ++j)
                        if (c + j < a.cols) p[j] = from_acc<T>(v[i][j]);
                }
            }
        }
    }
}

// Snapshot of a generator state {seed, offset} for one pass, and the step to the next.
__global__ void dropout_advance_kernel(int64_t* state, int64_t* used) {
    used[0] = state[0];
    used[1] = state[1];
    state[1] = (int64_t)((uint64_t)state[1] + 1);
}

template <typename T, int VEC, bool WIDE>
cudaError_t launch(const void* x, void* y, const DropArgs& a, bool batch_inner, cudaStream_t s) {
    const int64_t steps = ceil_div64(a.cols, VEC), pairs = (a.rows + 1) / 2;
    const unsigned threads = steps >= 256 ? 256 : (unsigned)(ceil_div64(steps, 32) * 32);
    const dim3 grid((unsigned)(ceil_div64(steps, threads) < 4096 ? ceil_div64(steps, threads) : 4096),
                    (unsigned)(pairs < 65535 ? pairs : 65535));
    if (batch_inner)
        dropout_kernel<T, VEC, true, WIDE><<<grid, threads, 0, s>>>((const T*)x, (T*)y, a);
    else
        dropout_kernel<T, VEC, false, WIDE><<<grid, threads, 0, s>>>((const T*)x, (T*)y, a);
    return cudaGetLastError();
}

template <typename T>
cudaError_t dispatch(const void* x, void* y, const DropArgs& a, bool batch_inner, cudaStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const uintptr_t at = (uintptr_t)x | (uintptr_t)y;
    const int64_t ld = a.ldx | a.ldy;
    if (at % 16 == 0 && ld % V == 0) return launch<T, V, true>(x, y, a, batch_inner, s);
    return launch<T, 2, false>(x, y, a, batch_inner, s);
}

}  // namespace
}  // namespace clb

using namespace clb;

extern "C" int clb_dropout(int dtype, const void* x, int64_t ldx, int64_t rows, int64_t cols, int batch_inner, double p,
                           int rescale, uint64_t seed, uint64_t offset, const int64_t* rng, void* y, int64_t ldy,
                           clb_stream_t stream) {
    if (dtype != CLB_F32 && dtype != CLB_F64 && dtype != CLB_BF16 && dtype != CLB_F16)
        return set_error(CLB_ERR_DTYPE, "dropout: unsupported dtype");
    const int64_t most = int64_t(1) << 33;  // the block index of either axis is a 32-bit counter word
    if (rows < 0 || cols < 0 || rows > most || cols > most) return set_error(CLB_ERR_INVALID, "dropout: bad sizes");
    if (!(p >= 0.0 && p <= 1.0)) return set_error(CLB_ERR_INVALID, "dropout: p must be in [0, 1]");
    if (rows == 0 || cols == 0) return CLB_OK;
    if (!x || !y) return set_error(CLB_ERR_INVALID, "dropout: null pointer");
    if (rows > 1 && (ldx < cols || ldy < cols)) return set_error(CLB_ERR_INVALID, "dropout: row stride below the row length");
    DropArgs a{};
    a.ldx = rows > 1 ? ldx : 0;
    a.ldy = rows > 1 ? ldy : 0;
    a.rows = rows;
    a.cols = cols;
    a.seed = seed;
    a.offset = offset;
    a.rng = rng;
    const double t = nearbyint(p * 4294967296.0);
    a.none = p == 1.0;
    a.threshold = t >= 4294967296.0 ? 0xFFFFFFFFu : (uint32_t)t;
    a.scale = rescale && p < 1.0 ? 1.0 / (1.0 - p) : 1.0;
    cudaStream_t s = (cudaStream_t)stream;
    cudaError_t e = cudaSuccess;
    switch (dtype) {
        case CLB_F32: e = dispatch<float>(x, y, a, batch_inner != 0, s); break;
        case CLB_F64: e = dispatch<double>(x, y, a, batch_inner != 0, s); break;
        case CLB_BF16: e = dispatch<__nv_bfloat16>(x, y, a, batch_inner != 0, s); break;
        default: e = dispatch<__half>(x, y, a, batch_inner != 0, s); break;
    }
    if (e != cudaSuccess) return set_error(CLB_ERR_CUDA, cudaGetErrorString(e));
    count_launches(1);
    return CLB_OK;
}

extern "C" int clb_dropout_advance(int64_t* state, int64_t* used, clb_stream_t stream) {
    if (!state || !used) return set_error(CLB_ERR_INVALID, "dropout_advance: null pointer");
    dropout_advance_kernel<<<1, 1, 0, (cudaStream_t)stream>>>(state, used);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return set_error(CLB_ERR_CUDA, cudaGetErrorString(e));
    count_launches(1);
    return CLB_OK;
}
