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
//
// The gradient of the loss needs a row's own sum and nothing of the other rows but how many count, so the forward pass makes
// it while the row is on the chip: the logits are read once and the gradient written once.  A backward pass with another
// upstream gradient than 1 makes it anew from the logits (clb_logit_grad), in one rounding.
//
// Forms, by row length and storage: few rows of few classes in one launch (few_kernel); short rows by lanes of a warp
// (rows_group_kernel); long ones by a block or a cluster of up to 8 (rows_block_kernel); samples contiguous (cols_kernel);
// rows beyond a cluster's registers, and fp64 (rows_stream_kernel), read twice.
// Measured on a B200 (6.45 TB/s copy rate): bf16 2048 x 131072 with its gradient 242 us (1.07 GB, 4.4 TB/s, 69 %), fp32 1777 x
// 50001 with a third of the rows masked 147 us (63 %), log-probabilities of bf16 4096 x 32768 with their gradient 135 us (805
// MB over the two calls, 93 %).  What bounds the long rows: two exponentials an entry (16 a clock and SM: 119 of the 242 us)
// among 14 instructions, and the wait of a cluster's blocks for one another between the two halves.  Measured and dropped:
// clusters that walk over the rows with the next row on its way to shared memory (308 us: fewer clusters fit than blocks),
// and one block a row that reads the row again out of the L2 cache (242 to 276 us).
#include <cuda_runtime.h>

#include "common.cuh"
#include "kernels.h"
#include "vec.cuh"

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
    // the gradient of the same pass (null `gz` of the kernels: none): gz[i * gn + j * gv], scaled by `fixed` or scale[0]
    int64_t gn, gv;
    const A* scale;
    A fixed;
};

// The per-row inputs, read before the row's sum is known so that they have arrived by then.
template <typename A> struct RowIn { A at, adv, old_lp, ref; };

template <typename T, typename A = typename Acc<T>::type>
__device__ __forceinline__ RowIn<A> row_in(const T* __restrict__ z, const RowArgs<A>& a, int64_t i) {
    RowIn<A> in{(A)NAN, 0, 0, 0};
    const int64_t act = a.actions[i];
    if (a.adv != nullptr) {
        in.adv = a.adv[i];
        in.old_lp = a.old_lp[i];
        if (a.ref != nullptr) in.ref = a.ref[i];
    }
    if (act >= 0 && act < a.v) in.at = to_acc(z[i * a.sn + act * a.sv]);
    return in;
}

// One row from its maximum and sum; returns d loss_i / d lp_i before the scale.  write: put the results down.
template <typename A> __device__ A finish_row(const RowArgs<A>& a, const RowIn<A>& in, int64_t i, A m, A s, bool write) {
    const A lp = (in.at - m) * a.inv_t - log(s);
    if (write) {
        a.logp[i] = lp;
        if (a.stats != nullptr) {
            a.stats[i] = m;
            a.stats[a.n + i] = s;
        }
    }
    if (a.adv == nullptr) return (A)0;
    const A r = exp(lp - in.old_lp);
    const A held = r < a.lo ? a.lo : r > a.hi ? a.hi : r;  // NaN stays NaN
    const A free_ = r * in.adv, kept = held * in.adv;
    A loss = -(free_ <= kept ? free_ : kept), slope = free_ <= kept ? -free_ : (A)0;
    if (free_ != free_) loss = slope = free_;
    A kl = 0;
    if (a.ref != nullptr) {
        const A q = in.ref - lp, e = expm1(q);
        kl = e - q;
        loss += a.beta * kl;
        slope -= a.beta * e;
    }
    if (write) {
        a.ratio[i] = r;
        if (a.ref != nullptr) a.kl[i] = kl;
        a.row_loss[i] = loss;
        if (a.slope != nullptr) a.slope[i] = slope;
    }
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

// The runs of a warp's lanes, G at a time, as one: the common maximum first, so that each sum is rescaled once.
template <int G = 32, typename A> __device__ __forceinline__ void warp_merge(Run<A>& r, A factor) {
    A top = r.m;
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) {
        const A m2 = __shfl_xor_sync(0xffffffffu, top, o);
        top = top > m2 ? top : m2;
    }
    const A safe = top == lowest<A>() ? (A)0 : top;
    r.s *= soft_exp((r.m - safe) * factor);
    r.m = top;
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) r.s += __shfl_xor_sync(0xffffffffu, r.s, o);
}

// What a row's gradient needs beside its logits: gz_j = c [j = act] + w exp((z_j - m) / T) with w = -c / s.
template <typename A> struct RowGrad { A m, c, w; };

template <typename A> __device__ __forceinline__ RowGrad<A> row_grad(const RowArgs<A>& a, A slope, A m, A s) {
    // in the order of the gradient kernels below, which then give the same bits for an upstream gradient of 1
    const A c = slope * (a.scale != nullptr ? a.scale[0] : a.fixed) * a.inv_t;
    return {m, c, -c / s};
}

template <typename T> struct Two;  // a pair of 16-bit elements as the packed maximum takes it
template <> struct Two<__nv_bfloat16> {
    using type = __nv_bfloat162;
    static __device__ __forceinline__ type of(uint32_t w) { return *reinterpret_cast<const type*>(&w); }
};
template <> struct Two<__half> {
    using type = __half2;
    static __device__ __forceinline__ type of(uint32_t w) { return *reinterpret_cast<const type*>(&w); }
};

// Rows contiguous, held in registers as 16-byte windows: window k of row i has the entries VEC k - shift ..., where `shift`
// is how far the row starts past a 16-byte boundary.  Entries outside the row read as -inf and are not written.  A thread has
// windows a constant distance STRIDE apart, so that they need no arithmetic of their own.  What is known of the windows picks
// the kernels' form: each is in the row as a whole (kFull), or may be in part or not at all (kShifted).  A row held this way
// is short enough for 32-bit indexes.
enum Windows { kFull, kShifted };

template <typename T, int NV, int STRIDE, Windows M> struct RowPart {
    static constexpr int VEC = 16 / sizeof(T), STEP = VEC * STRIDE;
    Pack<T, VEC> x[NV];

    // c: column of the thread's first window
    __device__ __forceinline__ void load(const T* __restrict__ row, int c, int v) {
        const unsigned whole = v >= VEC ? v - VEC + 1 : 0;  // windows that start in [0, whole) lie in the row
        const T* at = row + c;
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            if (M == kFull || (unsigned)(c + u * STEP) < whole) {
                x[u].load(at + u * STEP);
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    x[u].raw(j, (unsigned)(c + u * STEP + j) < (unsigned)v ? at[u * STEP + j] : T(-INFINITY));
            }
        }
    }
    // the largest entry, a NaN left aside (the sum meets it)
    __device__ __forceinline__ float top() const {
        if constexpr (sizeof(T) == 2) {
            typename Two<T>::type m[2] = {Two<T>::of(x[0].w[0]), Two<T>::of(x[0].w[1])};
#pragma unroll
            for (int u = 0; u < NV; ++u)
#pragma unroll
                for (int k = 0; k < 4; ++k) m[k & 1] = __hmax2(m[k & 1], Two<T>::of(x[u].w[k]));
            m[0] = __hmax2(m[0], m[1]);
            return fmaxf(to_acc(m[0].x), to_acc(m[0].y));
        } else {
            float m[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int u = 0; u < NV; ++u)
#pragma unroll
                for (int j = 0; j < VEC; ++j) m[j & 1] = fmaxf(m[j & 1], x[u].raw(j));
            return fmaxf(m[0], m[1]);
        }
    }
    __device__ __forceinline__ void sum(Run<float>& r, float factor) const {
        const float m = fmaxf(top(), -INFINITY);  // NaN where all entries are
        r.m = m;
        const float safe = m == -INFINITY ? 0.f : m;
        // The difference first: one multiply-add with a product -m * factor would leave that product's rounding in every
        // exponent of the row, all the more the larger the logits or the smaller T (bf16 2048 x 131072: 242 us; so 240).
        float f[VEC], s[4] = {};
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            x[u].get(f);
#pragma unroll
            for (int j = 0; j < VEC; ++j) s[j & 3] += soft_exp((f[j] - safe) * factor);
        }
        r.s = (s[0] + s[1]) + (s[2] + s[3]);
    }
    // Between sum and grad: without it the converted logits of 16 bits, twice the registers, are kept from one to the other and
    // spill (bf16 2048 x 131072: 280 us).
    __device__ __forceinline__ void pin() {
#pragma unroll
        for (int u = 0; u < NV; ++u)
#pragma unroll
            for (int k = 0; k < 4; ++k) asm volatile("" : "+r"(x[u].w[k]));
    }
    // the row's gradient without the chosen action's own term; `same`: out's windows lie as the row's
    __device__ __forceinline__ void grad(T* __restrict__ out, int c, bool same, int v, const RowGrad<float>& g,
                                         float factor) const {
        const unsigned whole = same && v >= VEC ? v - VEC + 1 : 0;
        T* at = out + c;
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            if (M != kFull && c + u * STEP >= v) break;
            float f[VEC];
            x[u].get(f);
#pragma unroll
            for (int j = 0; j < VEC; ++j) f[j] = g.w * soft_exp((f[j] - g.m) * factor);
            Pack<T, VEC> y;
            y.put(f);
            put(at + u * STEP, c + u * STEP, whole, v, y);
        }
    }
    static __device__ __forceinline__ void put(T* __restrict__ at, int c, unsigned whole, int v, const Pack<T, VEC>& y) {
        if (M == kFull || (unsigned)c < whole) {
            y.store(at);
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if ((unsigned)(c + j) < (unsigned)v) at[j] = y.raw(j);
        }
    }
    __device__ __forceinline__ static void zero(T* __restrict__ out, int c, bool same, int v) {
        const unsigned whole = same && v >= VEC ? v - VEC + 1 : 0;
        const Pack<T, VEC> y = {};
        for (int u = 0; u < NV; ++u) put(out + c + u * STEP, c + u * STEP, whole, v, y);
    }
};

template <typename T> __device__ __forceinline__ int shift_of(const T* p) {
    return (int)((reinterpret_cast<uintptr_t>(p) / sizeof(T)) % (16 / sizeof(T)));
}

// The chosen action's own entry, written by the thread that wrote its window before.
template <typename T>
__device__ __forceinline__ void put_action(T* out, const T* row, int64_t act, const RowGrad<float>& g, float factor) {
    const float z = to_acc(row[act]);
    out[act] = from_acc<T>(g.c + g.w * soft_exp((z - g.m) * factor));
}

// Short rows: G lanes of a warp per row, the row's windows in their registers.
template <typename T, int NV, int G>
__global__ void __launch_bounds__(128) rows_group_kernel(const T* __restrict__ z, T* __restrict__ gz, RowArgs<float> a) {
    const int lane = threadIdx.x % G, v = (int)a.v;
    const int64_t i = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / G;
    const bool in = i < a.n, live = in && (a.mask == nullptr || a.mask[i]);
    const T* row = z + (in ? i : 0) * a.sn;
    using Part = RowPart<T, NV, G, kShifted>;
    const int shift = shift_of(row), c = Part::VEC * lane - shift;
    Part part;
    Run<float> r;
    RowIn<float> given{};
    if (live) {
        if (lane == 0) given = row_in<T>(z, a, i);
        part.load(row, c, v);
        part.sum(r, a.factor);
    }
    warp_merge<G>(r, a.factor);
    float slope = 0.f;
    if (lane == 0 && in) {
        if (live)
            slope = finish_row(a, given, i, r.m, r.s, true);
        else
            skip_row(a, i);
    }
    if (gz == nullptr) return;
    slope = __shfl_sync(0xffffffffu, slope, 0, G);
    if (!in) return;
    T* out = gz + i * a.gn;
    const bool same = shift_of(out) == shift;
    if (!live) {
        Part::zero(out, c, same, v);
        return;
    }
    const RowGrad<float> g = row_grad(a, slope, r.m, r.s);
    part.pin();
    part.grad(out, c, same, v, g, a.factor);
    const int64_t act = a.actions[i];
    if (act >= 0 && act < v && ((int)act + shift) / Part::VEC % G == lane) put_action(out, row, act, g, a.factor);
}

constexpr int kWindows = 8;

// Longer rows: a cluster of `parts` blocks per row (one block for parts = 1), kWindows windows a thread.  The blocks give each
// other their warps' maxima and sums through distributed shared memory, and every block finishes the row by itself.
template <typename T, Windows M>
__global__ void __launch_bounds__(512, 2) rows_block_kernel(const T* __restrict__ z, T* __restrict__ gz, RowArgs<float> a,
                                                            int parts) {
    using Part = RowPart<T, kWindows, 32, M>;
    constexpr int VEC = Part::VEC;
    __shared__ float2 runs[8 * 16];
    __shared__ RowGrad<float> shared;
    const int64_t i = blockIdx.x / (unsigned)parts;
    const int rank = (int)(blockIdx.x % (unsigned)parts), warps = blockDim.x >> 5, warp = threadIdx.x >> 5,
              lane = threadIdx.x & 31;
    const T* row = z + i * a.sn;
    const int shift = M == kFull ? 0 : shift_of(row), v = (int)a.v;
    const int first = (rank * warps + warp) * 32 * kWindows + lane, c = VEC * first - shift;  // a warp's windows are neighbours
    T* out = gz != nullptr ? gz + i * a.gn : nullptr;
    const bool same = gz != nullptr && (M == kFull || shift_of(out) == shift);
    if (a.mask != nullptr && !a.mask[i]) {  // the same in every block of the cluster
        if (rank == 0 && threadIdx.x == 0) skip_row(a, i);
        if (gz != nullptr) Part::zero(out, c, same, v);
        return;
    }
    if (parts > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // this block has started
    RowIn<float> given{};
    if (threadIdx.x == 0) given = row_in<T>(z, a, i);
    Part part;
    part.load(row, c, v);
    Run<float> r;
    part.sum(r, a.factor);
    warp_merge(r, a.factor);
    if (parts > 1) {
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        if (lane < parts) {
            uint32_t local = (uint32_t)__cvta_generic_to_shared(&runs[rank * warps + warp]), remote;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(lane));
            asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(remote), "f"(r.m), "f"(r.s) : "memory");
        }
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    } else {
        if (lane == 0) runs[warp] = make_float2(r.m, r.s);
        __syncthreads();
    }
    if (warp == 0) {
        Run<float> t;
        for (int k = lane; k < parts * warps; k += 32) t.merge(runs[k].x, runs[k].y, a.factor);
        warp_merge(t, a.factor);
        if (lane == 0) {
            const float slope = finish_row(a, given, i, t.m, t.s, rank == 0);
            if (gz != nullptr) shared = row_grad(a, slope, t.m, t.s);
        }
    }
    if (gz == nullptr) return;
    __syncthreads();
    const RowGrad<float> g = shared;
    part.pin();
    part.grad(out, c, same, v, g, a.factor);
    const int64_t act = a.actions[i];
    if (act >= 0 && act < v) {
        const int k = ((int)act + shift) / VEC;
        if (k / (32 * kWindows) == rank * warps + warp && k % 32 == lane) put_action(out, row, act, g, a.factor);
    }
}

// Any row length, any type: one block per row, which reads its row once for the sum and once more for the gradient.
template <typename T>
__global__ void __launch_bounds__(512) rows_stream_kernel(const T* __restrict__ z, T* __restrict__ gz,
                                                          RowArgs<typename Acc<T>::type> a) {
    using A = typename Acc<T>::type;
    __shared__ A sm[16], ss[16];
    __shared__ RowGrad<A> shared;
    for (int64_t i = blockIdx.x; i < a.n; i += gridDim.x) {
        const T* row = z + i * a.sn;
        T* out = gz != nullptr ? gz + i * a.gn : nullptr;
        if (a.mask != nullptr && !a.mask[i]) {
            if (threadIdx.x == 0) skip_row(a, i);
            if (gz != nullptr)
                for (int64_t j = threadIdx.x; j < a.v; j += blockDim.x) out[j] = T(0.f);
            continue;
        }
        Run<A> r;
        int64_t j = threadIdx.x;
        for (; j + 7 * blockDim.x < a.v; j += 8 * blockDim.x) {
            A f[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) f[u] = to_acc(row[j + u * blockDim.x]);
#pragma unroll
            for (int u = 0; u < 8; ++u) r.add(f[u], a.factor);
        }
        for (; j < a.v; j += blockDim.x) r.add(to_acc(row[j]), a.factor);
        warp_merge(r, a.factor);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) {
            sm[threadIdx.x >> 5] = r.m;
            ss[threadIdx.x >> 5] = r.s;
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < (int)(blockDim.x >> 5); ++w) r.merge(sm[w], ss[w], a.factor);
            const A slope = finish_row(a, row_in<T>(z, a, i), i, r.m, r.s, true);
            if (gz != nullptr) shared = row_grad(a, slope, r.m, r.s);
        }
        if (gz == nullptr) continue;
        __syncthreads();
        const RowGrad<A> g = shared;
        const int64_t act = a.actions[i];
        for (j = threadIdx.x; j < a.v; j += blockDim.x) {
            const A f = to_acc(row[j]);
            const A e = g.w * soft_exp((f - g.m) * a.factor);
            out[j] = from_acc<T>(j == act ? g.c + e : e);
        }
    }
}

constexpr int kMostWarps = 64, kHeld = 16;  // warps of a cluster along the classes, classes a thread holds

// Samples contiguous: 32 rows a block, the lanes along them, blockDim.y warps (and `parts` blocks of a cluster) along the
// classes.  HELD: each thread's classes fit its registers, else the logits are read again for the gradient.
template <typename T, bool HELD>
__global__ void __launch_bounds__(512) cols_kernel(const T* __restrict__ z, T* __restrict__ gz,
                                                   RowArgs<typename Acc<T>::type> a, int parts) {
    using A = typename Acc<T>::type;
    constexpr int R = kHeld;
    __shared__ A sm[kMostWarps][32], ss[kMostWarps][32];
    __shared__ RowGrad<A> shared[32];
    const int64_t i = (int64_t)(blockIdx.x / (unsigned)parts) * 32 + threadIdx.x;
    const int rank = (int)(blockIdx.x % (unsigned)parts), warps = blockDim.y, stride = parts * warps;
    const int64_t first = rank * warps + threadIdx.y;
    const bool in = i < a.n, live = in && (a.mask == nullptr || a.mask[i]);
    const T* row = z + (in ? i : 0);
    if (parts > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    Run<A> r;
    A f[R];
    RowIn<A> given{};
    if (live && threadIdx.y == 0) given = row_in<T>(z, a, i);
    if (live) {
        for (int64_t j = first; j < a.v; j += (int64_t)R * stride) {
#pragma unroll
            for (int u = 0; u < R; ++u) f[u] = j + u * stride < a.v ? to_acc(row[(j + u * stride) * a.sv]) : lowest<A>();
            A top = lowest<A>();
#pragma unroll
            for (int u = 0; u < R; ++u) top = f[u] > top ? f[u] : top;
            if (top > r.m) {
                r.s *= soft_exp((r.m - top) * a.factor);
                r.m = top;
            }
            const A safe = r.m == lowest<A>() ? (A)0 : r.m;
#pragma unroll
            for (int u = 0; u < R; ++u)
                if (j + u * stride < a.v) r.s += soft_exp((f[u] - safe) * a.factor);
            if (HELD) break;
        }
    }
    if (parts > 1) {
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        for (int p = 0; p < parts; ++p) {
            uint32_t at[2] = {(uint32_t)__cvta_generic_to_shared(&sm[first][threadIdx.x]),
                              (uint32_t)__cvta_generic_to_shared(&ss[first][threadIdx.x])};
            const A val[2] = {r.m, r.s};
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                uint32_t remote;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(at[k]), "r"(p));
                if constexpr (sizeof(A) == 4)
                    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote), "f"((float)val[k]) : "memory");
                else
                    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(remote), "d"((double)val[k]) : "memory");
            }
        }
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    } else if (warps > 1) {
        sm[first][threadIdx.x] = r.m;
        ss[first][threadIdx.x] = r.s;
        __syncthreads();
    }
    if (threadIdx.y == 0 && in) {
        if (live) {
            if (stride > 1) {
                r = Run<A>();
                for (int w = 0; w < stride; ++w) r.merge(sm[w][threadIdx.x], ss[w][threadIdx.x], a.factor);
            }
            const A slope = finish_row(a, given, i, r.m, r.s, rank == 0);
            if (gz != nullptr) shared[threadIdx.x] = row_grad(a, slope, r.m, r.s);
        } else if (rank == 0) {
            skip_row(a, i);
        }
    }
    if (gz == nullptr) return;
    __syncthreads();
    if (!in) return;
    T* out = gz + i;
    if (!live) {
        for (int64_t j = first; j < a.v; j += stride) out[j * a.gv] = T(0.f);
        return;
    }
    const RowGrad<A> g = shared[threadIdx.x];
    const int64_t act = a.actions[i];
    for (int64_t j = first; j < a.v; j += (int64_t)R * stride) {
        if (!HELD) {
#pragma unroll
            for (int u = 0; u < R; ++u) f[u] = j + u * stride < a.v ? to_acc(row[(j + u * stride) * a.sv]) : (A)0;
        }
#pragma unroll
        for (int u = 0; u < R; ++u)
            if (j + u * stride < a.v) {
                const A e = g.w * soft_exp((f[u] - g.m) * a.factor);
                out[(j + u * stride) * a.gv] = from_acc<T>(j + u * stride == act ? g.c + e : e);
            }
        if (HELD) break;
    }
}

// Few rows of few classes (decisions out of a group sum): the whole loss in one launch, which is what such a call costs.  One
// cluster, a thread per row with its logits in registers; the blocks add up the counted rows, then the rows' losses, through
// distributed shared memory, in a fixed order.  As many rows as the cluster has threads: 1024 x 10 takes 8.5 us on the device
// (10.9 in three launches), 8192 x 10 would take 18.7 (11.8).
constexpr int kFewClasses = 16, kFewThreads = 256, kFewRows = 8 * kFewThreads;

template <typename A> __device__ A cluster_sum(A v, A* warps, A* slots, int rank, int parts) {
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
    for (int k = 0; k < kFewThreads / 32; ++k) v += warps[k];
    if (parts == 1) return v;
    if (threadIdx.x < parts) {
        uint32_t local = (uint32_t)__cvta_generic_to_shared(slots + rank), remote;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(threadIdx.x));
        if constexpr (sizeof(A) == 4)
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote), "f"((float)v) : "memory");
        else
            asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(remote), "d"((double)v) : "memory");
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    v = 0;
    for (int k = 0; k < parts; ++k) v += slots[k];
    return v;
}

template <typename T>
__global__ void __launch_bounds__(kFewThreads) few_kernel(const T* __restrict__ z, T* __restrict__ gz,
                                                          RowArgs<typename Acc<T>::type> a, int parts, int mean,
                                                          typename Acc<T>::type* loss, typename Acc<T>::type* scale) {
    using A = typename Acc<T>::type;
    __shared__ A warps[2][kFewThreads / 32], slots[2][8];
    const int rank = (int)blockIdx.x;
    const int64_t first = (int64_t)rank * kFewThreads + threadIdx.x, step = (int64_t)parts * kFewThreads;
    if (parts > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    A count = 0;  // exact: at most kFewRows
    for (int64_t i = first; i < a.n; i += step) count += a.mask == nullptr || a.mask[i] ? (A)1 : (A)0;
    if (parts > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // every block has started
    count = cluster_sum(count, warps[0], slots[0], rank, parts);
    a.fixed = mean ? (A)1 / (count > 0 ? count : (A)1) : (A)1;
    a.scale = nullptr;
    A total = 0;
    for (int64_t i = first; i < a.n; i += step) {
        const bool live = a.mask == nullptr || a.mask[i];
        T* out = gz + i * a.gn;
        if (!live) {
            skip_row(a, i);
            if (gz != nullptr)
                for (int64_t j = 0; j < a.v; ++j) out[j * a.gv] = T(0.f);
            continue;
        }
        const RowIn<A> in = row_in<T>(z, a, i);
        const T* row = z + i * a.sn;
        A f[kFewClasses], m = lowest<A>(), s = 0;
#pragma unroll
        for (int j = 0; j < kFewClasses; ++j) f[j] = j < a.v ? to_acc(row[j * a.sv]) : lowest<A>();
#pragma unroll
        for (int j = 0; j < kFewClasses; ++j) m = f[j] > m ? f[j] : m;
        const A safe = m == lowest<A>() ? (A)0 : m;
#pragma unroll
        for (int j = 0; j < kFewClasses; ++j)
            if (j < a.v) s += soft_exp((f[j] - safe) * a.factor);
        const A slope = finish_row(a, in, i, m, s, true);
        total += a.row_loss[i];
        if (gz == nullptr) continue;
        const RowGrad<A> g = row_grad(a, slope, m, s);
        const int64_t act = a.actions[i];
#pragma unroll
        for (int j = 0; j < kFewClasses; ++j)
            if (j < a.v) {
                const A e = g.w * soft_exp((f[j] - g.m) * a.factor);
                out[j * a.gv] = from_acc<T>(j == act ? g.c + e : e);
            }
    }
    total = cluster_sum(total, warps[1], slots[1], rank, parts);
    if (rank == 0 && threadIdx.x == 0) {
        scale[0] = a.fixed;
        if (loss != nullptr) loss[0] = total * a.fixed;
    }
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
        A c = 0, m = 0, w = 0;
        int64_t act = -1;
        if (live) {
            c = (a.slope != nullptr ? a.slope[i] : (A)1) * scale * (a.upstream != nullptr ? a.upstream[i * a.up_stride] : (A)1) *
                a.inv_t;
            m = a.stats[i];
            act = a.actions[i];
            if (act < 0 || act >= a.v) c = (A)NAN;
            w = -c / a.stats[a.n + i];
        }
        for (int64_t j = COLS ? threadIdx.y : threadIdx.x; j < a.v; j += COLS ? blockDim.y : blockDim.x) {
            A g = 0;
            if (live) {
                g = w * soft_exp((to_acc(z[i * a.sn + j * a.sv]) - m) * a.factor);
                if (j == act) g = c + g;
            }
            gz[i * a.gn + j * a.gv] = from_acc<T>(g);
        }
    }
}

// The same for contiguous rows, in 16-byte windows: blockDim.y rows a block, `chunks` blocks along a row.
template <typename T, int NV, int BX, Windows M>
__global__ void __launch_bounds__(256) rows_grad_kernel(const T* __restrict__ z, T* __restrict__ gz, GradArgs<float> a,
                                                        unsigned chunks) {
    if (a.unless_one && a.upstream[0] == 1.f) return;
    const int64_t i = (int64_t)(blockIdx.x / chunks) * (256 / BX) + threadIdx.y;
    if (i >= a.n) return;
    const T* row = z + i * a.sn;
    T* out = gz + i * a.gn;
    using Part = RowPart<T, NV, BX, M>;
    const int shift = M == kFull ? 0 : shift_of(row), v = (int)a.v, chunk = (int)(blockIdx.x % chunks);
    const bool same = M == kFull || shift_of(out) == shift;
    const int c = Part::VEC * (chunk * BX * NV + (int)threadIdx.x) - shift;
    if (a.mask != nullptr && !a.mask[i]) {
        Part::zero(out, c, same, v);
        return;
    }
    Part part;
    part.load(row, c, v);
    const int64_t act = a.actions[i];
    float k = (a.slope != nullptr ? a.slope[i] : 1.f) * (a.scale != nullptr ? a.scale[0] : 1.f) *
              (a.upstream != nullptr ? a.upstream[i * a.up_stride] : 1.f) * a.inv_t;
    if (act < 0 || act >= a.v) k = NAN;
    const RowGrad<float> g = {a.stats[i], k, -k / a.stats[a.n + i]};
    part.grad(out, c, same, v, g, a.factor);
    if (act >= 0 && act < v) {
        const int w = ((int)act + shift) / Part::VEC;
        if (w / (BX * NV) == chunk && w % BX == threadIdx.x) put_action(out, row, act, g, a.factor);
    }
}

// scale = 1 / (number of counted rows): one block.
template <typename A>
__global__ void __launch_bounds__(1024) count_kernel(const uint8_t* __restrict__ mask, int64_t n, A* scale) {
    __shared__ int64_t sc[32];
    int64_t c = 0;
    const int64_t head = (16 - (reinterpret_cast<uintptr_t>(mask) & 15)) & 15;
    const int64_t vecs = n > head ? (n - head) / 16 : 0;
    for (int64_t k = threadIdx.x; k < vecs; k += blockDim.x) {
        const uint4 v = *reinterpret_cast<const uint4*>(mask + head + 16 * k);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int q = 0; q < 4; ++q) c += __popc(__vcmpne4(w[q], 0)) / 8;
    }
    // the up to 15 entries before the first vector and after the last
    const int64_t done = 16 * vecs, rest = n - done;
    if (threadIdx.x < rest) c += mask[threadIdx.x < head ? threadIdx.x : threadIdx.x + done] != 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
    if ((threadIdx.x & 31) == 0) sc[threadIdx.x >> 5] = c;
    __syncthreads();
    if (threadIdx.x >= 32) return;
    c = threadIdx.x < (blockDim.x >> 5) ? sc[threadIdx.x] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
    if (threadIdx.x == 0) scale[0] = (A)1 / (A)(c > 0 ? c : 1);
}

// loss = scale * sum of the rows' losses: one block, a fixed order of summation.  `fixed` (when >= 0) is the scale where no
// count was needed, and is put down for the backward pass.
template <typename A>
__global__ void __launch_bounds__(1024) loss_kernel(const A* __restrict__ row_loss, int64_t n, A fixed, A* loss, A* scale) {
    __shared__ A sh[32];
    A s[4] = {};
    int64_t i = threadIdx.x;
    for (; i + 3 * blockDim.x < n; i += 4 * blockDim.x) {
#pragma unroll
        for (int u = 0; u < 4; ++u) s[u] += row_loss[i + u * blockDim.x];
    }
    for (; i < n; i += blockDim.x) s[0] += row_loss[i];
    A t = warp_sum((s[0] + s[1]) + (s[2] + s[3]));
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = t;
    __syncthreads();
    if (threadIdx.x >= 32) return;
    t = warp_sum(threadIdx.x < (blockDim.x >> 5) ? sh[threadIdx.x] : (A)0);
    if (threadIdx.x == 0) {
        if (fixed >= 0) scale[0] = fixed;
        if (loss != nullptr) loss[0] = t * (fixed >= 0 ? fixed : scale[0]);
    }
}

unsigned blocks(int64_t n) { return (unsigned)(n < (1 << 30) ? n : (1 << 30)); }

template <typename P> struct Same { using type = P; };  // a parameter that is not deduced

// Threads of a block of rows_block_kernel; twice as many for one block a row, and where eight such blocks do not hold it.
constexpr int kBlockMost = 256;

template <typename T> struct Logits {
    using A = typename Acc<T>::type;

    // gz null: no gradient
    static cudaError_t forward(const void* z, void* gz, const RowArgs<A>& a, bool cols, cudaStream_t s) {
        count_launches(1);
        return cols ? forward_cols((const T*)z, (T*)gz, a, s) : forward_rows((const T*)z, (T*)gz, a, s);
    }

    template <typename... P> static cudaError_t launch(void (*kernel)(P...), int64_t grid, dim3 block, int parts, cudaStream_t s,
                                                       typename Same<P>::type... args) {
        if (grid > 0x7FFFFFFF) return cudaErrorInvalidValue;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)grid);
        cfg.blockDim = block;
        cfg.stream = s;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = (unsigned)parts;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = parts > 1 ? 1 : 0;
        return cudaLaunchKernelEx(&cfg, kernel, args...);
    }

    static cudaError_t forward_cols(const T* z, T* gz, const RowArgs<A>& a, cudaStream_t s) {
        // warps along the classes until each thread holds its classes, over up to four blocks of a cluster
        const int64_t need = ceil_div64(a.v, kHeld);
        const int parts = need <= 16 ? 1 : need <= 32 ? 2 : 4;
        const int warps = need < 16 ? (int)need : kMostWarps / 4;
        const int64_t grid = ceil_div64(a.n, 32) * parts;
        return a.v <= (int64_t)kHeld * warps * parts
                   ? launch(cols_kernel<T, true>, grid, dim3(32, warps), parts, s, z, gz, a, parts)
                   : launch(cols_kernel<T, false>, grid, dim3(32, warps), parts, s, z, gz, a, parts);
    }

    static cudaError_t forward_rows(const T* z, T* gz, const RowArgs<A>& a, cudaStream_t s) {
        if constexpr (sizeof(A) == 4) {
            constexpr int VEC = 16 / sizeof(T);
            // the most windows that a row takes, whatever its shift
            const bool aligned = reinterpret_cast<uintptr_t>(z) % 16 == 0 && (a.n == 1 || a.sn % VEC == 0);
            const int64_t w = ceil_div64(a.v + (aligned ? 0 : VEC - 1), VEC);
            auto group = [&](auto kernel, int g) { return launch(kernel, ceil_div64(a.n * g, 128), dim3(128), 1, s, z, gz, a); };
            // a warp holds rows of up to 256 windows, 8 a lane (bf16 30000 x 2000: 63 us, in blocks 67; 16000 x 4096, 512
            // windows, by a warp 74, in blocks 66)
            if (w <= 4) return group(rows_group_kernel<T, 1, 4>, 4);
            if (w <= 16) return group(rows_group_kernel<T, 1, 16>, 16);
            if (w <= 32) return group(rows_group_kernel<T, 1, 32>, 32);
            if (w <= 64) return group(rows_group_kernel<T, 2, 32>, 32);
            if (w <= 128) return group(rows_group_kernel<T, 4, 32>, 32);
            if (w <= 256) return group(rows_group_kernel<T, 8, 32>, 32);
            auto threads = [](int64_t k) { return dim3((unsigned)(ceil_div64(k, 32) * 32)); };
            // every window whole: rows on 16 bytes that fill the threads' windows
            const bool even = aligned && a.v % VEC == 0 &&
                              (gz == nullptr || (reinterpret_cast<uintptr_t>(gz) % 16 == 0 && (a.n == 1 || a.gn % VEC == 0)));
            auto block = [&](int parts) {
                const dim3 t = threads(ceil_div64(w, kWindows * parts));
                return launch(even && (int64_t)t.x * kWindows * parts == w ? rows_block_kernel<T, kFull>
                                                                           : rows_block_kernel<T, kShifted>,
                              a.n * parts, t, parts, s, z, gz, a, parts);
            };
            // 8 windows a thread (with 4, bf16 16000 x 4096 takes 80 us instead of 66, fp32 8000 x 4000 69 instead of 54);
            // up to 512 threads without a cluster (bf16 4096 x 32768: 116 us; two blocks of 256 threads 121), then clusters of
            // smaller blocks, which wait less for their slowest warp (bf16 2048 x 131072: 242 us; blocks of 512 threads 248)
            if (w <= kWindows * 2 * kBlockMost) return block(1);
            for (int most = kBlockMost; most <= 2 * kBlockMost; most *= 2)
                for (int parts = 2; parts <= 8; parts *= 2)
                    if (w <= (int64_t)parts * kWindows * most)
                        return block(parts);
        }
        return launch(rows_stream_kernel<T>, a.n, dim3(512), 1, s, z, gz, a);
    }

    static cudaError_t backward(const void* z, void* gz, const GradArgs<A>& a, bool cols, cudaStream_t s) {
        count_launches(1);
        if (cols) {
            logit_grad_kernel<T, true><<<blocks(ceil_div64(a.n, 32)), dim3(32, 8), 0, s>>>((const T*)z, (T*)gz, a);
            return cudaGetLastError();
        }
        if constexpr (sizeof(A) == 4) {
            if (a.v < (1 << 30)) {
                constexpr int NV = 4, VEC = 16 / sizeof(T);
                auto even = [&](const void* p, int64_t ld) {
                    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (a.n == 1 || ld % VEC == 0);
                };
                const bool on = even(z, a.sn) && even(gz, a.gn);
                const int64_t w = ceil_div64(a.v + (on ? 0 : VEC - 1), VEC);
                auto go = [&](auto full, auto shifted, int bx) {
                    const int64_t chunks = ceil_div64(w, bx * NV);
                    return launch(on && a.v == chunks * bx * NV * VEC ? full : shifted, ceil_div64(a.n, 256 / bx) * chunks,
                                  dim3(bx, 256 / bx), 1, s, (const T*)z, (T*)gz, a, (unsigned)chunks);
                };
                if (w <= 8 * NV) return go(rows_grad_kernel<T, NV, 8, kFull>, rows_grad_kernel<T, NV, 8, kShifted>, 8);
                if (w <= 64 * NV) return go(rows_grad_kernel<T, NV, 64, kFull>, rows_grad_kernel<T, NV, 64, kShifted>, 64);
                return go(rows_grad_kernel<T, NV, 256, kFull>, rows_grad_kernel<T, NV, 256, kShifted>, 256);
            }
        }
        logit_grad_kernel<T, false><<<blocks(a.n), 256, 0, s>>>((const T*)z, (T*)gz, a);
        return cudaGetLastError();
    }

    static int logp(const void* z, int64_t ldz, int64_t n, int64_t v, bool cols, const int64_t* actions,
                    const uint8_t* mask, double t, void* logp, void* stats, cudaStream_t s) {
        RowArgs<A> a{};
        fill(a, ldz, n, v, cols, actions, mask, t);
        a.logp = (A*)logp;
        a.stats = (A*)stats;
        return status(forward(z, nullptr, a, cols, s));
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
        a.gn = cols ? 1 : ldgz;
        a.gv = cols ? ldgz : 1;
        if (n > 0 && n <= kFewRows && v <= kFewClasses) {
            int parts = 1;
            while (parts < 8 && parts * kFewThreads < n) parts *= 2;
            count_launches(1);
            return status(launch(few_kernel<T>, parts, dim3(kFewThreads), parts, s, (const T*)z, (T*)gz, a, parts, mean,
                                 (A*)loss, (A*)scale));
        }
        const bool count = mean && mask != nullptr;  // else the scale is known here
        a.fixed = mean ? (A)1 / (A)(n > 0 ? n : 1) : (A)1;
        if (count) {
            a.scale = (const A*)scale;
            count_kernel<A><<<1, 1024, 0, s>>>(mask, n, (A*)scale);
            count_launches(1);
            if (const int st = status(cudaGetLastError())) return st;
        }
        if (n > 0)
            if (const int st = status(forward(z, gz, a, cols, s))) return st;
        loss_kernel<A><<<1, 1024, 0, s>>>((const A*)row_loss, n, count ? (A)-1 : a.fixed, (A*)loss, (A*)scale);
        count_launches(1);
        return status(cudaGetLastError());
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
