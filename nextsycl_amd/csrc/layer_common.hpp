// layer_common.hpp: rows of the library's three types read and written in wide pieces, and what the state-space kernels
// share.
#pragma once
#include <cstdint>
#include <hip/hip_runtime.h>

#include "attn_common.hpp"
#include "kv_formats.hpp"
#include "ns_internal.hpp"

// VEC elements of type QT from element i on, as float32 (VEC 1, or pieces of 8 to 16 bytes at any element: global memory is read and
// written in wide pieces whatever their alignment)
typedef uint32_t piece4_t __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t piece2_t __attribute__((ext_vector_type(2), aligned(2)));
typedef float floats4_t __attribute__((ext_vector_type(4), aligned(4)));
template <int QT, int VEC>
__device__ __forceinline__ void load_row(const void* p, int64_t i, float (&v)[VEC]) {
    if constexpr (VEC == 1) v[0] = load_q<QT>(p, i);
    else if constexpr (QT == 0) {
#pragma unroll
        for (int j = 0; j < VEC; j += 4) {
            const floats4_t a = *reinterpret_cast<const floats4_t*>(static_cast<const float*>(p) + i + j);
            v[j] = a.x, v[j + 1] = a.y, v[j + 2] = a.z, v[j + 3] = a.w;
        }
    } else {
        static_assert(VEC == 8);
        const piece4_t w = *reinterpret_cast<const piece4_t*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const uint16_t b = (uint16_t) (j % 2 ? w[j / 2] >> 16 : w[j / 2]);
            v[j] = QT == 1 ? f16_to_f32(b) : bf16_to_f32(b);
        }
    }
}
template <int QT, int VEC>
__device__ __forceinline__ void store_row(void* p, int64_t i, const float (&v)[VEC]) {
    if constexpr (VEC == 1) store_o<QT>(p, i, v[0]);
    else if constexpr (QT == 0) {
#pragma unroll
        for (int j = 0; j < VEC; j += 4) *reinterpret_cast<floats4_t*>(static_cast<float*>(p) + i + j) = floats4_t{v[j], v[j + 1], v[j + 2], v[j + 3]};
    } else {
        uint32_t w[VEC / 2];
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) {
            const uint32_t a = QT == 1 ? f32_to_f16(v[2 * j]) : f32_to_bf16(v[2 * j]), b = QT == 1 ? f32_to_f16(v[2 * j + 1]) : f32_to_bf16(v[2 * j + 1]);
            w[j] = a | b << 16;
        }
        uint16_t* d = static_cast<uint16_t*>(p) + i;
        if constexpr (VEC == 8) *reinterpret_cast<piece4_t*>(d) = piece4_t{w[0], w[1], w[2], w[3]};
        else *reinterpret_cast<piece2_t*>(d) = piece2_t{w[0], w[1]};
    }
}
// the same of the `left` elements that there are (TAIL: there may be fewer than VEC); those that there are not: zeros
template <int QT, int VEC, bool TAIL>
__device__ __forceinline__ void load_piece(const void* p, int64_t i, int left, float (&v)[VEC]) {
    if (!TAIL || left >= VEC) load_row<QT, VEC>(p, i, v);
    else
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = j < left ? load_q<QT>(p, i + j) : 0.0f;
}
template <int QT, int VEC, bool TAIL>
__device__ __forceinline__ void store_piece(void* p, int64_t i, int left, const float (&v)[VEC]) {
    if (!TAIL || left >= VEC) store_row<QT, VEC>(p, i, v);
    else
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            if (j < left) store_o<QT>(p, i + j, v[j]);
}

// v / (1 + e^-v) by the hardware's exponential and reciprocal (one unit in the last place each); where e^-v is infinite, 0
__device__ __forceinline__ float silu(float v) { return v * __builtin_amdgcn_rcpf(1.0f + fast_exp2(v * -1.44269504f)); }
__device__ __forceinline__ float softplus(float v) { return fmaxf(v, 0.0f) + log1pf(expf(-fabsf(v))) + (v != v ? v : 0.0f); }

// A work-group's barrier for what its waves exchange through LDS: memory loads asked for ahead and stores on their
// way out stay in flight across it (a __syncthreads waits for both)
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// the sum over each run of L lanes (4, 8 or 16), in every lane of the run: the run's halves first, then theirs
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
    auto add = [&](auto c) { v += __builtin_bit_cast(float, dpp_u32<decltype(c)::value>(__builtin_bit_cast(uint32_t, v))); };
    if constexpr (L >= 16) add(std::integral_constant<int, 0x140>());
    if constexpr (L >= 8) add(std::integral_constant<int, 0x141>());
    add(std::integral_constant<int, 0x4E>());
    add(std::integral_constant<int, 0xB1>());
    return v;
}

// a state-space layer's sizes, weights and places, as ns_ssm_prompt and ns_ssm_step take them
struct SsmLayer {
    const void *xbc, *dt;
    int64_t xs, dts;
    const float *cw, *cb, *a, *dtb, *d;
    float lo, hi;
    float* conv;
    int64_t cap, p0;
    int H, P, N, G, K, chan;
    const float* h0;
    float* h1;
    void* y;
    int64_t ys;
};

// a head's step size: its row's value with the bias added, through softplus, held to the layer's limits
__device__ __forceinline__ float ssm_dt(const SsmLayer& p, float v) {
    const float s = softplus(v);
    return s < p.lo ? p.lo : s > p.hi ? p.hi : s;
}
// tap k of 4 of a channel: the layer's K taps are the last K of them
__device__ __forceinline__ float ssm_tap(const SsmLayer& p, int ch, int k) { return k >= 4 - p.K ? p.cw[(int64_t) ch * p.K + k - 4 + p.K] : 0.0f; }

// the sizes that the state-space calls take
inline bool ns_ssm_sizes(int64_t H, int64_t P, int64_t N, int64_t G) {
    return H > 0 && P > 0 && N > 0 && G > 0 && H <= 65536 && P <= 65536 && N <= 256 && H % G == 0 && H * P + 2 * G * N <= (int64_t) 1 << 24;
}
// ssm_step.hip: a few successive rows of one sequence from p.p0 on, the last K - 1 of them into the ring (which holds those in front of the
// call and those behind it at once)
void ns_ssm_few(ns_gpu* g, int qt, const SsmLayer& p, int rows);
// ssm_step.hip: what the two state-space calls refuse alike (a ring of fewer than `least` rows among it); 0 or -1
int ns_ssm_check(const char* who, ns_gpu* g, int qt, const SsmLayer& p, int64_t H, int64_t P, int64_t N, int64_t G, int64_t K, int64_t least);
