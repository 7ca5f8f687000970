// kv8_common.hpp: what the kernels over caches of 8-bit values in blocks of tokens share (include/ns_kv8.h).
#pragma once
#include <cmath>
#include <cstdint>
#include <hip/hip_runtime.h>
#include <string>

#include "attn_common.hpp"
#include "kv_formats.hpp"
#include "layer_common.hpp"
#include "ns_internal.hpp"
#include "ns_kv8.h"

constexpr int KV8_TOKENS = 1 << 30;     // of a sequence, at most
constexpr int KV8_HEADS = 4096;         // query heads a key head, at most

// the pools of one cache, and the sequences' tables
struct Kv8Cache {
    uint8_t *kc, *vc;
    float *ksc, *vsc;
    const int32_t* table;
    int64_t tmax, blocks;
    int Hkv, D, block, shift;    // block = 1 << shift tokens
};
// the block of entry e of a sequence's table, or -1. (Some entry is read whatever e is: several of these in a row are under way together, where a
// branch around each would wait for the one in front)
__device__ __forceinline__ int kv8_block(const Kv8Cache& c, const int32_t* table, int64_t seq, int64_t e) {
    const uint32_t b = (uint32_t) table[seq * c.tmax + (e < 0 ? 0 : e < c.tmax ? e : c.tmax - 1)];
    return b < (uint32_t) c.blocks && e >= 0 && e < c.tmax ? (int) b : -1;
}
// where block b's rows of head h begin, in rows
__device__ __forceinline__ int64_t kv8_rows(const Kv8Cache& c, int b, int h) { return ((int64_t) b * c.Hkv + h) * c.block; }

// a sequence's rows in a call: the first, how many, and the tokens in front of them (none: n 0)
struct Kv8Seq {
    int first, n, len;
};
__device__ __forceinline__ Kv8Seq kv8_seq(const int32_t* start, const int32_t* lens, int s, int T, int most) {
    Kv8Seq q;
    q.first = start ? min(max(start[s], 0), T) : min(s, T);
    const int end = start ? min(max(start[s + 1], q.first), T) : min(s + 1, T);
    q.len = lens[s];
    q.n = q.len < 0 || q.len > KV8_TOKENS ? 0 : min(end - q.first, most);
    return q;
}

template <int FORM>
struct Kv8Form {
    static constexpr float MOST = FORM == 0 ? 127.0f : 448.0f;
    // the exponents that a scale is held to, and the exponent of a scale under the exponent of its largest value (2^x m, 1 <= m < 2): the
    // largest code is m TOP, so a larger m takes one more
    static constexpr int LO = FORM == 0 ? -24 : -15, HI = FORM == 0 ? 9 : 7, WIDTH = FORM == 0 ? 6 : 8;
    static constexpr uint32_t TOP = FORM == 0 ? 0x7E0000u : 0x600000u;       // the mantissa of 1.984375, of 1.75
};
// the exponent of the least scale that holds magnitudes up to a (finite, not negative)
template <int FORM>
__device__ __forceinline__ int kv8_exponent(float a) {
    using F = Kv8Form<FORM>;
    const uint32_t u = __builtin_bit_cast(uint32_t, a);
    const int e = (int) (u >> 23) - 127 - F::WIDTH + ((u & 0x7FFFFFu) > F::TOP);
    return min(max(e, F::LO), F::HI);
}

// 4 values in units of their scale -> 4 codes, nearest even, magnitudes held to the largest (NaN: 0)
template <int FORM>
__device__ __forceinline__ uint32_t kv8_codes(float a, float b, float c, float d) {
    constexpr float M = Kv8Form<FORM>::MOST;
    auto hold = [](float x) { return x != x ? 0.0f : fminf(fmaxf(x, -M), M); };
    a = hold(a), b = hold(b), c = hold(c), d = hold(d);
    if constexpr (FORM == 0) {
        auto q = [](float x) { return (uint32_t) (uint8_t) (int8_t) (int) rintf(x); };
        return q(a) | q(b) << 8 | q(c) << 16 | q(d) << 24;
    } else {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
        return (uint32_t) __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    }
}
// code i (0 .. 3) of a word as float32
template <int FORM>
__device__ __forceinline__ float kv8_value(uint32_t w, int i) {
    if constexpr (FORM == 0) return (float) (int8_t) (w >> (8 * i));
    else return i == 0 ? __builtin_amdgcn_cvt_f32_fp8(w, 0) : i == 1 ? __builtin_amdgcn_cvt_f32_fp8(w, 1) : i == 2 ? __builtin_amdgcn_cvt_f32_fp8(w, 2) : __builtin_amdgcn_cvt_f32_fp8(w, 3);
}
// a word's 4 codes in another unit: the old scale over the new one, `ratio`, a power of two of at most 1
template <int FORM>
__device__ __forceinline__ uint32_t kv8_reround(uint32_t w, float ratio) {
    return kv8_codes<FORM>(kv8_value<FORM>(w, 0) * ratio, kv8_value<FORM>(w, 1) * ratio, kv8_value<FORM>(w, 2) * ratio, kv8_value<FORM>(w, 3) * ratio);
}

// two codes of a word (bytes 0 and 1, or 2 and 3) -> two halfs code x scale, exactly (the scales there are): int8 as dq8x2 does, e4m3 in one instruction
template <int FORM>
__device__ __forceinline__ uint32_t kv8_halfs2(uint32_t w, int hi, float scale, _Float16 scale16) {
    if constexpr (FORM == 0) return dq8x2(w ^ 0x80808080u, hi ? 0x04030402u : 0x04010400u, scale16);
    else {
        typedef _Float16 h2v __attribute__((ext_vector_type(2)));
        const h2v r = hi ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, true) : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, false);
        return __builtin_bit_cast(uint32_t, r);
    }
}
// 8 codes in two words, each with a scale of its own -> 8 halfs
template <int FORM>
__device__ __forceinline__ s8v kv8_halfs8(uint32_t w0, uint32_t w1, float s0, float s1) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    const _Float16 h0 = (_Float16) s0, h1 = (_Float16) s1;
    const u4 r = {kv8_halfs2<FORM>(w0, 0, s0, h0), kv8_halfs2<FORM>(w0, 1, s0, h0), kv8_halfs2<FORM>(w1, 0, s1, h1), kv8_halfs2<FORM>(w1, 1, s1, h1)};
    return __builtin_bit_cast(s8v, r);
}
// 8 codes -> 8 halfs without their scale
template <int FORM>
__device__ __forceinline__ s8v kv8_halfs8(uint32_t w0, uint32_t w1) {
    if constexpr (FORM == 0) {
        typedef _Float16 h2v __attribute__((ext_vector_type(2)));
        typedef uint32_t u4 __attribute__((ext_vector_type(4)));
        const uint32_t x0 = w0 ^ 0x80808080u, x1 = w1 ^ 0x80808080u;
        const h2v off = {(_Float16) -1152.0f, (_Float16) -1152.0f};
        auto two = [&](uint32_t x, uint32_t sel) { return __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2v, __builtin_amdgcn_perm(0x64646464u, x, sel)) + off); };
        const u4 r = {two(x0, 0x04010400u), two(x0, 0x04030402u), two(x1, 0x04010400u), two(x1, 0x04030402u)};
        return __builtin_bit_cast(s8v, r);
    } else return kv8_halfs8<FORM>(w0, w1, 1.0f, 1.0f);
}

// ---- host side
// a window as the kernels count it: 0 where it is none, no longer than any sequence
inline int64_t kv8_window(int64_t win) { return win <= 0 ? 0 : win < 2 * (int64_t) KV8_TOKENS ? win : 2 * (int64_t) KV8_TOKENS; }
// what every call over a cache refuses; 0 or -1
int ns_kv8_check(const std::string& who, int form, int64_t Hkv, int64_t D, int64_t block, int64_t blocks, int64_t S, int64_t tmax, const Kv8Cache& c);
inline Kv8Cache kv8_cache(const void* kc, const void* vc, const float* ksc, const float* vsc, const int32_t* table, int64_t tmax, int64_t Hkv, int64_t D, int64_t block,
                          int64_t blocks) {
    const int shift = block == 16 ? 4 : block == 32 ? 5 : block == 64 ? 6 : 7;
    return {(uint8_t*) kc, (uint8_t*) vc, (float*) ksc, (float*) vsc, table, tmax, blocks, (int) Hkv, (int) D, (int) block, shift};
}
// kv8_attend.hip: up to 16 rows' weights (acc1 = acc0 + them) as a token's attention makes them, with the keys as values; 0, -1, or 1: not with so much scratch
int ns_kv8_rows_weights(ns_gpu* g, const std::string& w, int form, int qt, const Kv8Cache& c, const void* q, int64_t qs, int64_t T, int64_t p0, int64_t Hq, int64_t win,
                        float sl2, const float* acc0, float* acc1, float* scratch, int64_t floats);
// kv8_store.hip: tokens from .. from + n - 1 of the table's first sequence as half rows [Hkv][n][D]; 0 or -1
int ns_kv8_widen(ns_gpu* g, int form, const Kv8Cache& c, int64_t from, int64_t n, uint16_t* k, uint16_t* v);
