// 16 bytes of activations in registers: loads, stores, and conversion to and from the arithmetic type two elements at a
// time (one conversion instruction packs a pair of 16-bit results).
#pragma once

#include "common.cuh"

namespace clb {

template <typename T> struct Pair;  // two consecutive 16-bit elements in one 32-bit register
template <> struct Pair<__nv_bfloat16> {
    static __device__ __forceinline__ float2 get(uint32_t w) {
        return {__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)};
    }
    static __device__ __forceinline__ uint32_t put(float lo, float hi) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
};
template <> struct Pair<__half> {
    static __device__ __forceinline__ float2 get(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
    static __device__ __forceinline__ uint32_t put(float lo, float hi) {
        const __half2 v = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
};

// N consecutive elements (N * sizeof(T) = 4, 8 or 16 bytes) kept as they lie in memory.
template <typename T, int N> struct Pack {
    using A = typename Acc<T>::type;
    static constexpr int kWords = (int)(N * sizeof(T) / 4);
    uint32_t w[kWords];

    // `p` aligned to the pack's size
    __device__ __forceinline__ void load(const T* __restrict__ p) {
        if constexpr (kWords == 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(p);
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        } else if constexpr (kWords == 2) {
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            w[0] = v.x, w[1] = v.y;
        } else {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        }
    }
    __device__ __forceinline__ void store(T* __restrict__ p) const {
        if constexpr (kWords == 4)
            *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        else if constexpr (kWords == 2)
            *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
        else
            *reinterpret_cast<uint32_t*>(p) = w[0];
    }
    // element by element, the first `n` of them at p[j * stride]; the rest reads as `fill`
    __device__ __forceinline__ void gather(const T* __restrict__ p, int64_t n, int64_t stride, T fill) {
#pragma unroll
        for (int j = 0; j < N; ++j) raw(j, j < n ? p[j * stride] : fill);
    }
    __device__ __forceinline__ void scatter(T* __restrict__ p, int64_t n, int64_t stride) const {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (j < n) p[j * stride] = raw(j);
    }
    // element j as stored (j a constant)
    __device__ __forceinline__ T raw(int j) const {
        if constexpr (sizeof(T) == 2) {
            const unsigned short h = (unsigned short)(w[j >> 1] >> (16 * (j & 1)));
            return *reinterpret_cast<const T*>(&h);
        } else if constexpr (sizeof(T) == 4) {
            return *reinterpret_cast<const T*>(&w[j]);
        } else {
            return __hiloint2double((int)w[2 * j + 1], (int)w[2 * j]);
        }
    }
    __device__ __forceinline__ void raw(int j, T v) {
        if constexpr (sizeof(T) == 2) {
            const uint32_t h = *reinterpret_cast<const unsigned short*>(&v);
            w[j >> 1] = (j & 1) ? (w[j >> 1] & 0xFFFFu) | (h << 16) : (w[j >> 1] & 0xFFFF0000u) | h;
        } else if constexpr (sizeof(T) == 4) {
            w[j] = *reinterpret_cast<const uint32_t*>(&v);
        } else {
            w[2 * j] = (uint32_t)__double2loint(v);
            w[2 * j + 1] = (uint32_t)__double2hiint(v);
        }
    }
    __device__ __forceinline__ void get(A (&v)[N]) const {
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int j = 0; j < N; j += 2) {
                const float2 f = Pair<T>::get(w[j >> 1]);
                v[j] = f.x;
                v[j + 1] = f.y;
            }
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = (A)raw(j);
        }
    }
    __device__ __forceinline__ void put(const A (&v)[N]) {
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int j = 0; j < N; j += 2) w[j >> 1] = Pair<T>::put(v[j], v[j + 1]);
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) raw(j, (T)v[j]);
        }
    }
};

}  // namespace clb
