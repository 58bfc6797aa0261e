// Dropout whose mask is a function of (seed, offset, element) and is never stored: the backward pass draws the same words
// again.  The generator is Philox4x32-10 (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as easy as
// 1, 2, 3", SC 2011), written from the paper.
//
// One counter serves a 2 x 2 block of the logical [n, d] matrix: element (n, d) takes word 2 (n & 1) + (d & 1) of
// Philox(counter = (d >> 1, n >> 1, offset), key = seed).  A thread that walks two neighbouring rows of the contiguous axis
// therefore uses all four words of every call whether features or samples are contiguous, and the mask does not depend on
// the storage layout, on strides, or on how the work is split.
//
// What bounds it: 2 bytes in and 2 out an element of 16 bits stand against ten rounds of two 32 x 32 -> 64 multiplies for
// four elements, some 15 instructions an element with the conversion and the choice, so integer issue is as near as memory.
// bf16 64000 x 1024, one pass of 262 MB: 54 us, 4.9 TB/s, 75 % of the card's copy rate; fp32 32000 x 1024, as many bytes for half
// the draws: 47 us, 87 %.  The first kernel, one counter at a
// time and a block per short piece of a row, issued 32 instructions an element and took 97 us.
#include <cuda_runtime.h>

#include <cmath>

#include "common.cuh"
#include "kernels.h"
#include "vec.cuh"

namespace clb {

namespace {

// N counters (c0[i], c1[i], c2, c3) under one key, round by round side by side: the key schedule is shared, and the
// multiplies of one counter hide behind the others'.  On return word w of counter i is c[w][i].
template <int N> __device__ __forceinline__ void philox(uint32_t (&c)[4][N], uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint64_t p0 = (uint64_t)c[0][i] * 0xD2511F53u, p1 = (uint64_t)c[2][i] * 0xCD9E8D57u;
            c[0][i] = (uint32_t)(p1 >> 32) ^ c[1][i] ^ k0;
            c[1][i] = (uint32_t)p1;
            c[2][i] = (uint32_t)(p0 >> 32) ^ c[3][i] ^ k1;
            c[3][i] = (uint32_t)p0;
        }
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
}

struct DropArgs {
    int64_t ldx, ldy, rows, cols;  // rows of the strided axis, entries of the contiguous one
    uint64_t seed, offset;
    const int64_t* rng;            // device {seed, offset}; takes the place of the two above
    uint32_t threshold;            // an element is kept when its word >= threshold
    double scale;
};

// Blocks an SM: the registers of 16-bit elements, twice as many a thread, fit five (bf16 64000 x 1024, both passes: 107 us,
// with six 113), those of fp32 six (32000 x 1024: 93 us, with five 100).
constexpr int kThreads = 128;
template <typename T> constexpr int kBlocks = sizeof(T) == 2 ? 5 : 6;

// The words of NC neighbouring 2 x 2 blocks along the contiguous axis.
template <int NC, bool BATCH_INNER>
__device__ __forceinline__ void draw(uint32_t (&w)[4][NC], uint32_t inner, uint32_t outer, uint64_t seed, uint64_t offset) {
#pragma unroll
    for (int k = 0; k < NC; ++k) {
        w[0][k] = BATCH_INNER ? outer : inner + k;
        w[1][k] = BATCH_INNER ? inner + k : outer;
        w[2][k] = (uint32_t)offset;
        w[3][k] = (uint32_t)(offset >> 32);
    }
    philox<NC>(w, (uint32_t)seed, (uint32_t)(seed >> 32));
}

// The keep decisions of one 2 x VEC block applied to its two packs.
template <typename T, int VEC, bool BATCH_INNER, bool RESCALE>
__device__ __forceinline__ void drop(Pack<T, VEC> (&v)[2], uint32_t inner, uint32_t outer, uint64_t seed, uint64_t offset,
                                     uint32_t threshold, typename Acc<T>::type scale) {
    using A = typename Acc<T>::type;
    constexpr int NC = VEC / 2;
    uint32_t w[4][NC];
    draw<NC, BATCH_INNER>(w, inner, outer, seed, offset);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if constexpr (RESCALE || sizeof(T) != 2) {
            A f[VEC];
            v[i].get(f);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const uint32_t word = w[BATCH_INNER ? 2 * (j & 1) + i : 2 * i + (j & 1)][j >> 1];
                f[j] = word >= threshold ? (RESCALE ? f[j] * scale : f[j]) : (A)0;
            }
            v[i].put(f);
        } else {  // kept values pass bit by bit
#pragma unroll
            for (int k = 0; k < NC; ++k) {
                const uint32_t lo = w[BATCH_INNER ? i : 2 * i][k] >= threshold ? 0x0000FFFFu : 0u;
                const uint32_t hi = w[BATCH_INNER ? 2 + i : 2 * i + 1][k] >= threshold ? 0xFFFF0000u : 0u;
                v[i].w[k] &= lo | hi;
            }
        }
    }
}

// A thread owns VEC consecutive entries of a pair of neighbouring rows at a time and walks down the rows, the next pair's
// loads in flight while it draws the words of the current one.  Rows start on 16 bytes.  BATCH_INNER: the
// contiguous axis is n (feature-major storage), else d.
template <typename T, int VEC, bool BATCH_INNER, bool RESCALE>
__global__ void __launch_bounds__(kThreads, kBlocks<T>) dropout_kernel(const T* __restrict__ x, T* __restrict__ y, DropArgs a) {
    using A = typename Acc<T>::type;
    const int64_t c = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * VEC;
    if (c >= a.cols) return;
    uint64_t seed = a.seed, offset = a.offset;
    if (a.rng != nullptr) {
        seed = (uint64_t)a.rng[0];
        offset = (uint64_t)a.rng[1];
    }
    const A scale = (A)a.scale;
    const int left = a.cols - c < VEC ? (int)(a.cols - c) : VEC;
    const bool full = left == VEC;
    const uint32_t pairs = (uint32_t)((a.rows + 1) >> 1), step = gridDim.y * blockDim.y;
    uint32_t rp = blockIdx.y * blockDim.y + threadIdx.y;
    const uint32_t lone = (a.rows & 1) ? pairs - 1 : 0xFFFFFFFFu;  // the pair that lacks its second row
    const T* p = x + 2 * (int64_t)rp * a.ldx + c;
    T* q = y + 2 * (int64_t)rp * a.ldy + c;
    const int64_t down_x = 2 * (int64_t)step * a.ldx, down_y = 2 * (int64_t)step * a.ldy;
    auto fetch = [&](Pack<T, VEC>(&v)[2], const T* at, bool second) {
        if (full) {
            v[0].load(at);
            if (second) v[1].load(at + a.ldx);
        } else {
            v[0].gather(at, left, 1, T(0.0f));
            if (second) v[1].gather(at + a.ldx, left, 1, T(0.0f));
        }
    };
    Pack<T, VEC> v[2], next[2];
    if (rp < pairs) fetch(v, p, rp != lone);
    while (rp < pairs) {
        const uint32_t below = rp + step;
        p += down_x;
        if (below < pairs && below > rp) fetch(next, p, below != lone);
        drop<T, VEC, BATCH_INNER, RESCALE>(v, (uint32_t)(c >> 1), rp, seed, offset, a.threshold, scale);
        if (full) {
            v[0].store(q);
            if (rp != lone) v[1].store(q + a.ldy);
        } else {
            v[0].scatter(q, left, 1);
            if (rp != lone) v[1].scatter(q + a.ldy, left, 1);
        }
        q += down_y;
        v[0] = next[0];
        v[1] = next[1];
        rp = below;
    }
}

// The same for rows that do not all start on 16 bytes (odd sizes, slices): a row's 16-byte windows then straddle the 2 x VEC
// blocks, by another shift in each row.  The threads put their blocks' keep masks, as wide as the elements, into shared
// memory and each reads the mask of its own windows back from there, shifted, so that global memory sees whole windows.
// Thread t of a block draws the entries from VEC (first - 1 + t) on, and owns window first + t of either row (the last
// thread none); blockDim.x is at most a warp, so no warp waits for another.  gridDim.y * blockDim.y is a multiple of VEC / 2
// wherever a thread has a second pair of rows: the shifts of its rows are then the same all the way down.
template <typename T, bool BATCH_INNER, bool RESCALE>
__global__ void __launch_bounds__(kThreads, kBlocks<T>) dropout_shifted_kernel(const T* __restrict__ x, T* __restrict__ y,
                                                                            DropArgs a) {
    using A = typename Acc<T>::type;
    constexpr int VEC = 16 / sizeof(T), NC = VEC / 2;
    __shared__ uint4 masks[2][2][kThreads];  // by turns, by row of the pair
    const int at = threadIdx.y * blockDim.x + threadIdx.x;
    const int64_t first = (int64_t)blockIdx.x * (blockDim.x - 1), unit = first - 1 + threadIdx.x;
    uint64_t seed = a.seed, offset = a.offset;
    if (a.rng != nullptr) {
        seed = (uint64_t)a.rng[0];
        offset = (uint64_t)a.rng[1];
    }
    const A scale = (A)a.scale;
    const uint32_t pairs = (uint32_t)((a.rows + 1) >> 1), step = gridDim.y * blockDim.y;
    uint32_t rp = blockIdx.y * blockDim.y + threadIdx.y;
    const uint32_t lone = (a.rows & 1) ? pairs - 1 : 0xFFFFFFFFu;  // the pair that lacks its second row
    const T* p[2];
    T* q[2];
    int shift[2], begin[2], end[2];  // the window holds row entries from its element `begin` up to `end`
    bool full[2], same[2];           // ... all of them; y's windows lie as x's
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const T* row = x + (2 * (int64_t)rp + i) * a.ldx;
        T* out = y + (2 * (int64_t)rp + i) * a.ldy;
        shift[i] = (int)((reinterpret_cast<uintptr_t>(row) / sizeof(T)) % VEC);
        same[i] = (int)((reinterpret_cast<uintptr_t>(out) / sizeof(T)) % VEC) == shift[i];
        const int64_t c = VEC * (first + threadIdx.x) - shift[i];
        begin[i] = c < 0 ? (int)-c : 0;
        end[i] = a.cols - c < VEC ? (a.cols > c ? (int)(a.cols - c) : 0) : VEC;
        if (threadIdx.x + 1 == blockDim.x) end[i] = 0;
        full[i] = begin[i] == 0 && end[i] == VEC;
        p[i] = row + c;
        q[i] = out + c;
    }
    const int64_t down_x = 2 * (int64_t)step * a.ldx, down_y = 2 * (int64_t)step * a.ldy;
    auto fetch = [&](Pack<T, VEC>(&v)[2], uint32_t pair) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (i == 1 && pair == lone) continue;
            if (full[i]) {
                v[i].load(p[i]);
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (j >= begin[i] && j < end[i]) v[i].raw(j, p[i][j]);
            }
        }
    };
    Pack<T, VEC> v[2] = {}, next[2] = {};
    if (rp < pairs) fetch(v, rp);
    int turn = 0;
    for (uint32_t base = blockIdx.y * blockDim.y; base < pairs; base += step, turn ^= 1) {
        const bool in = rp < pairs;
        const uint32_t below = rp + step;
        p[0] += down_x;
        p[1] += down_x;
        if (below < pairs) fetch(next, below);
        uint32_t w[4][NC];
        draw<NC, BATCH_INNER>(w, (uint32_t)(unit * NC), rp, seed, offset);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint32_t m[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if constexpr (sizeof(T) == 2) {
                    m[k] = (w[BATCH_INNER ? i : 2 * i][k] >= a.threshold ? 0x0000FFFFu : 0u) |
                           (w[BATCH_INNER ? 2 + i : 2 * i + 1][k] >= a.threshold ? 0xFFFF0000u : 0u);
                } else {
                    const int j = k * 4 / (int)sizeof(T);
                    m[k] = w[BATCH_INNER ? 2 * (j & 1) + i : 2 * i + (j & 1)][j >> 1] >= a.threshold ? ~0u : 0u;
                }
            }
            masks[turn][i][at] = make_uint4(m[0], m[1], m[2], m[3]);
        }
        __syncwarp();  // one a turn: the masks of this turn are next written two turns on
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (in && end[i] > 0 && !(i == 1 && rp == lone)) {
                // the 16 bytes that begin `shift` elements before the thread's next block
                const int back = shift[i] * (int)sizeof(T);
                const uint32_t* from = reinterpret_cast<const uint32_t*>(&masks[turn][i][at + 1]) - (back + 3) / 4;
                uint32_t m[4];
                if (sizeof(T) == 2 && (back & 3)) {
                    uint32_t lo = from[0];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t hi = from[k + 1];
                        m[k] = __funnelshift_r(lo, hi, 16);
                        lo = hi;
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) m[k] = from[k];
                }
                if constexpr (RESCALE) {
                    A f[VEC];
                    v[i].get(f);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) f[j] *= scale;
                    v[i].put(f);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) v[i].w[k] &= m[k];
                if (full[i] && same[i]) {
                    v[i].store(q[i]);
                } else {
#pragma unroll
                    for (int j = 0; j < VEC; ++j)
                        if (j >= begin[i] && j < end[i]) q[i][j] = v[i].raw(j);
                }
            }
            q[i] += down_y;
            v[i] = next[i];
        }
        rp = below;
    }
}

// Snapshot of a generator state {seed, offset} for one pass, and the step to the next.
__global__ void dropout_advance_kernel(int64_t* state, int64_t* used) {
    used[0] = state[0];
    used[1] = state[1];
    state[1] = (int64_t)((uint64_t)state[1] + 1);
}

template <typename T, bool RESCALE>
cudaError_t launch(const T* x, T* y, const DropArgs& a, bool batch_inner, cudaStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const bool wide = ((uintptr_t)x | (uintptr_t)y) % 16 == 0 && (a.ldx | a.ldy) % V == 0;
    // windows of a row, one more where rows are shifted; short rows: several row pairs side by side in a block
    const int64_t steps = wide ? ceil_div64(a.cols, V) : ceil_div64(a.cols + V - 1, V) + 1, pairs = (a.rows + 1) / 2;
    unsigned bx = wide ? 1 : 2;
    while (bx < (wide ? kThreads : 32) && bx < steps) bx *= 2;
    const dim3 block(bx, kThreads / bx);
    const int64_t gx = wide ? ceil_div64(steps, bx) : ceil_div64(steps - 1, bx - 1), gy = ceil_div64(pairs, (int64_t)block.y);
    if (gx > 0x7FFFFFFF) return cudaErrorInvalidValue;
    // As many blocks as are resident at once, each walking down the rows; four times that for shifted rows, whose blocks
    // are rounded to whole shifts and would leave SMs idle (fp16 1001 x 16383, both passes: 75 us with one wave, 51 with
    // four, 57 with eight).
    int64_t most = (int64_t)gpu_sms() * kBlocks<T> * (wide ? 1 : 4) / gx;
    if (!wide) most -= most % (V / 2);
    if (most < V / 2) most = V / 2;
    const dim3 grid((unsigned)gx, (unsigned)(gy < most ? gy : most));
    if (wide && batch_inner)
        dropout_kernel<T, V, true, RESCALE><<<grid, block, 0, s>>>(x, y, a);
    else if (wide)
        dropout_kernel<T, V, false, RESCALE><<<grid, block, 0, s>>>(x, y, a);
    else if (batch_inner)
        dropout_shifted_kernel<T, true, RESCALE><<<grid, block, 0, s>>>(x, y, a);
    else
        dropout_shifted_kernel<T, false, RESCALE><<<grid, block, 0, s>>>(x, y, a);
    return cudaGetLastError();
}

template <typename T>
cudaError_t dispatch(const void* x, void* y, const DropArgs& a, bool batch_inner, cudaStream_t s) {
    return a.scale != 1.0 ? launch<T, true>((const T*)x, (T*)y, a, batch_inner, s)
                          : launch<T, false>((const T*)x, (T*)y, a, batch_inner, s);
}

}  // namespace
}  // namespace clb

using namespace clb;

extern "C" int clb_dropout(int dtype, const void* x, int64_t ldx, int64_t rows, int64_t cols, int batch_inner, double p,
                           int rescale, uint64_t seed, uint64_t offset, const int64_t* rng, void* y, int64_t ldy,
                           clb_stream_t stream) {
    if (dtype != CLB_F32 && dtype != CLB_F64 && dtype != CLB_BF16 && dtype != CLB_F16)
        return set_error(CLB_ERR_DTYPE, "dropout: unsupported dtype");
    const int64_t most = int64_t(1) << 32;  // half of either index is a 32-bit counter word
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
    const bool none = t >= 4294967296.0;  // no word is as large as 2^32: nothing is kept
    a.threshold = none ? 0 : (uint32_t)t;
    a.scale = rescale && p < 1.0 ? 1.0 / (1.0 - p) : 1.0;
    cudaStream_t s = (cudaStream_t)stream;
    cudaError_t e = cudaSuccess;
    if (none) {
        const size_t elem = dtype == CLB_F64 ? 8 : dtype == CLB_F32 ? 4 : 2;
        e = cudaMemset2DAsync(y, (size_t)(rows > 1 ? ldy : cols) * elem, 0, (size_t)cols * elem, (size_t)rows, s);
        return e == cudaSuccess ? CLB_OK : set_error(CLB_ERR_CUDA, cudaGetErrorString(e));
    }
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
