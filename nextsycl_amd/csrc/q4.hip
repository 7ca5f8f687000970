// q4.hip: 4-bit weights with group scales - their layout (ns_q4_pack) and their product with 1 to 16 rows (ns_q4_product).
//
// y[t][m] = sum over groups of s[m][group] sum over the group's k of (q[m][k] - 8) x[t][k]. Bound: HBM - 0.5625 bytes a
// weight (0.516 with a scale for 128) for 2 operations a row. What stands beside the loads is unpacking: a tile of 16 x 128
// weights is 1 KB that a wave reads as 16 bytes a lane, laid out so that four bytes are a lane's operand of one 16 x 16 x 32
// matrix instruction, and a nibble becomes a half by one and-or (the exponent of 1024 over it) and one exact subtraction -
// 9 instructions for 8 weights, no shuffle, and no sum over lanes: the matrix unit sums. Its operands are exact (whole
// numbers -8 .. 7 as halfs), so a group's scale multiplies its float32 sum afterwards. Rows enter as halfs times a power of
// two a (row, tile) that puts the largest at 2^13 (no overflow, and nothing lost above 2^-37 of the largest): bfloat16 rows
// then fit as they are, float32 rows as two halfs (22 bits, two matrix instructions), half rows need neither.
//
// A work-group of 8 waves takes 16 outputs and shares K among its waves, tile by tile; the waves' sums meet in LDS in a
// fixed order. Its rows lie in LDS as operands, a stretch of K at a time.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "ns_internal.hpp"
#include "ns_layer.h"
#include "layer_common.hpp"

namespace {

constexpr int WAVES = 8, PF = 4, LDS_ROWS = 64 * 1024;

constexpr int64_t q4_tile_bytes(int64_t group) { return 1024 + 16 * (128 / group) * 2; }

struct Q4Params {
    const void* x;
    const uint8_t* w;
    void* y;
    int64_t xs, ys;
    int T, M, K, kt, chunk;      // kt: tiles along K; chunk: tiles of K that LDS holds at a time
    int vec;                     // rows readable in pieces of 8 values
};

// 8 weights of a word as halfs, -8 .. 7 exactly: nibble i under the exponent byte is 1024 + q, one 4 bits up 1024 + 16 q
__device__ __forceinline__ s8v q4_operand(uint32_t w) {
    typedef _Float16 h2v __attribute__((ext_vector_type(2)));
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    const h2v off = {(_Float16) -1032.0f, (_Float16) -1032.0f}, sixteenth = {(_Float16) 0.0625f, (_Float16) 0.0625f}, off16 = {(_Float16) -72.0f, (_Float16) -72.0f};
    auto under = [](uint32_t v, uint32_t mask) { return __builtin_bit_cast(h2v, (v & mask) | 0x64006400u); };
    const uint32_t w8 = w >> 8;
    const u4 r = {__builtin_bit_cast(uint32_t, under(w, 0x000f000fu) + off), __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(under(w, 0x00f000f0u), sixteenth, off16)),
                  __builtin_bit_cast(uint32_t, under(w8, 0x000f000fu) + off), __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(under(w8, 0x00f000f0u), sixteenth, off16))};
    return __builtin_bit_cast(s8v, r);
}

// GR: groups a tile (4, 2, 1)
template <int QT, int GR>
__global__ __launch_bounds__(64 * WAVES) void q4_product_kernel(Q4Params p) {
    constexpr int PLANES = QT == 0 ? 2 : 1, TILE = 1024 + 32 * GR, SW = 2 * GR;     // SW: a lane's scales, in words
    extern __shared__ __align__(16) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, n = lane % 16, g = lane / 16;
    const int col = n < p.T ? n : p.T - 1;             // (columns behind the rows: some row's, never written)
    s8v* xo = reinterpret_cast<s8v*>(lds);             // [plane][tile][16 pieces of 8][row]
    const int plane = p.chunk * 16 * p.T;
    float* xscale = reinterpret_cast<float*>(lds + (size_t) plane * PLANES * 16);   // [tile][row]
    const uint8_t* wt = p.w + (int64_t) blockIdx.x * p.kt * TILE;
    f4v acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int c0 = 0; c0 < p.kt; c0 += p.chunk) {
        const int here = min(p.chunk, p.kt - c0);
        uint4 nib[PF];
        uint32_t sc[PF][SW];
        auto fetch = [&](int i, uint4& q, uint32_t (&s)[SW]) {
            const int at = min(wave + WAVES * i, here - 1);
            const uint8_t* tile = wt + (int64_t) (c0 + at) * TILE;
            q = *reinterpret_cast<const uint4*>(tile + lane * 16);
            const uint32_t* ss = reinterpret_cast<const uint32_t*>(tile + 1024 + g * 8 * GR);
#pragma unroll
            for (int j = 0; j < SW; ++j) s[j] = ss[j];
        };
#pragma unroll
        for (int i = 0; i < PF; ++i) fetch(i, nib[i], sc[i]);
        // the rows' stretch as operands: 16 threads a (row, tile), 8 values each
        if (c0) __syncthreads();
        for (int task = tid / 16; task < here * p.T; task += 64 * WAVES / 16) {
            const int kl = task / p.T, t = task - kl * p.T, u = tid % 16, k = (c0 + kl) * 128 + u * 8;
            float v[8];
            if (p.vec && k + 8 <= p.K) load_row<QT, 8>(p.x, t * p.xs + k, v);
            else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = k + j < p.K ? load_q<QT>(p.x, t * p.xs + k + j) : 0.0f;
            }
            s8v hi, lo;
            float up = 1.0f;
            if constexpr (QT != 1) {
                float big = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) big = fmaxf(big, fabsf(v[j]));
                big = row16_max(big);
                // 2^(13 - exponent of the largest), its exponent field between 12 and 253: it has an inverse
                const int e = min(267 - (int) (__builtin_bit_cast(uint32_t, big) >> 23), 253);
                up = __builtin_bit_cast(float, (uint32_t) e << 23);
                if (u == 0) xscale[kl * p.T + t] = __builtin_bit_cast(float, (uint32_t) (254 - e) << 23);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float f = v[j] * up;
                const _Float16 half = (_Float16) f;
                hi[j] = __builtin_bit_cast(short, half);
                if constexpr (PLANES == 2) lo[j] = to16<false>(fabsf(f) < 65504.0f ? f - (float) half : 0.0f);
            }
            xo[(kl * 16 + u) * p.T + t] = hi;
            if constexpr (PLANES == 2) xo[plane + (kl * 16 + u) * p.T + t] = lo;
        }
        __syncthreads();
        for (int i0 = 0; wave + WAVES * i0 < here; i0 += PF) {
            uint4 nib2[PF];
            uint32_t sc2[PF][SW];
            const bool more = wave + WAVES * (i0 + PF) < here;
            if (more) {
#pragma unroll
                for (int i = 0; i < PF; ++i) fetch(i0 + PF + i, nib2[i], sc2[i]);
            }
#pragma unroll
            for (int i = 0; i < PF; ++i) {
                const int kl = wave + WAVES * (i0 + i);
                if (kl >= here) break;
                f4v tile = {0.0f, 0.0f, 0.0f, 0.0f}, s = tile;
                const uint32_t words[4] = {nib[i].x, nib[i].y, nib[i].z, nib[i].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const s8v a = q4_operand(words[j]);
                    const int at = (kl * 16 + 4 * j + g) * p.T + col;
                    s = mfma16<false>(a, xo[at], s);
                    if constexpr (PLANES == 2) s = mfma16<false>(a, xo[plane + at], s);
                    if ((j + 1) % (4 / GR) == 0) {
                        constexpr int PER = 4 / GR;
                        const int grp = j / PER;
                        const uint32_t s0 = sc[i][grp * 2], s1 = sc[i][grp * 2 + 1];
                        tile[0] = fmaf(f16_to_f32((uint16_t) s0), s[0], tile[0]);
                        tile[1] = fmaf(f16_to_f32((uint16_t) (s0 >> 16)), s[1], tile[1]);
                        tile[2] = fmaf(f16_to_f32((uint16_t) s1), s[2], tile[2]);
                        tile[3] = fmaf(f16_to_f32((uint16_t) (s1 >> 16)), s[3], tile[3]);
                        s = f4v{0.0f, 0.0f, 0.0f, 0.0f};
                    }
                }
                const float down = QT == 1 ? 1.0f : xscale[kl * p.T + col];
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[e] = QT == 1 ? acc[e] + tile[e] : fmaf(down, tile[e], acc[e]);
            }
            if (more) {
#pragma unroll
                for (int i = 0; i < PF; ++i) {
                    nib[i] = nib2[i];
#pragma unroll
                    for (int j = 0; j < SW; ++j) sc[i][j] = sc2[i][j];
                }
            }
        }
    }
    // the waves' sums, in the waves' order
    __syncthreads();
    f4v* part = reinterpret_cast<f4v*>(lds);
    part[wave * 64 + lane] = acc;
    __syncthreads();
    if (tid < 256) {
        const int t = tid / 16, m = tid % 16;
        const float* f = reinterpret_cast<const float*>(part) + ((m / 4) * 16 + t) * 4 + m % 4;
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) sum += f[w * 256];
        const int64_t out = (int64_t) blockIdx.x * 16 + m;
        if (t < p.T && out < p.M) store_o<QT>(p.y, t * p.ys + out, sum);
    }
}

// a thread a (weight row, group): finds its scale, writes its nibbles and the scale where the layout has them
__global__ __launch_bounds__(256) void q4_pack_kernel(int form, const void* src, int64_t ss, int64_t M, int64_t K, int group, int64_t kt, uint8_t* w) {
#pragma clang fp contract(off)
    const int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x, groups = kt * (128 / group), m = i / groups, gr = i - m * groups;
    if (m >= (M + 15) / 16 * 16) return;
    const int64_t k0 = gr * group;
    const float* f = static_cast<const float*>(src) + m * ss;
    const uint8_t* block = static_cast<const uint8_t*>(src) + m * ss + k0 / 32 * 18;
    uint16_t scale = 0;
    float inv = 0.0f;
    if (m < M && form == 0) {
        float most = 0.0f, at = 0.0f;
        for (int64_t k = k0; k < k0 + group && k < K; ++k)
            if (fabsf(f[k]) > most) most = fabsf(f[k]), at = f[k];
        const float d = at / -8.0f;
        inv = d != 0.0f ? 1.0f / d : 0.0f;
        scale = f32_to_f16(d);
    } else if (m < M && k0 < K) scale = (uint16_t) (block[0] | block[1] << 8);
    auto nibble = [&](int64_t k) {
        if (m >= M || k >= K) return 8u;
        if (form == 1) {
            const int j = (int) (k - k0);
            const uint32_t b = block[2 + j % 16];
            return j < 16 ? b & 15 : b >> 4;
        }
        const float v = f[k] * inv + 8.5f;
        return (uint32_t) max(0, min(15, (int) v));
    };
    uint8_t* tile = w + (m / 16 * kt + k0 / 128) * q4_tile_bytes(group);
    const int per = 128 / group, row = (int) (m % 16), first = (int) (k0 % 128);
    reinterpret_cast<uint16_t*>(tile + 1024)[row / 4 * 4 * per + first / group * 4 + row % 4] = scale;
    for (int o = first; o < first + group; o += 8) {
        uint32_t word = 0;
        for (int e = 0; e < 8; ++e) word |= nibble(k0 - first + o + e) << 4 * (e % 2 * 4 + e / 2);
        *reinterpret_cast<uint32_t*>(tile + 16 * (row + 16 * (o / 8 % 4)) + 4 * (o / 32)) = word;
    }
}

bool q4_group(int64_t group) { return group == 32 || group == 64 || group == 128; }

template <int QT, int GR>
void launch_product(ns_gpu* g, Q4Params& p) {
    constexpr int PLANES = QT == 0 ? 2 : 1;
    const int row = p.T * (256 * PLANES + 4);          // bytes of LDS a tile of K
    const int fit = LDS_ROWS / row;
    p.chunk = std::min(p.kt, fit < WAVES ? fit : fit / WAVES * WAVES);
    const size_t lds = std::max<size_t>((size_t) p.chunk * row, WAVES * 64 * sizeof(f4v));
    q4_product_kernel<QT, GR><<<(unsigned) ((p.M + 15) / 16), 64 * WAVES, lds, g->q>>>(p);
}
template <int QT>
void launch_product(ns_gpu* g, Q4Params& p, int64_t group) {
    if (group == 32) launch_product<QT, 4>(g, p);
    else if (group == 64) launch_product<QT, 2>(g, p);
    else launch_product<QT, 1>(g, p);
}

}  // namespace

extern "C" {

int64_t ns_q4_bytes(int64_t M, int64_t K, int64_t group) {
    if (M <= 0 || K <= 0 || !q4_group(group)) return 0;
    return (M + 15) / 16 * ((K + 127) / 128) * q4_tile_bytes(group);
}

int ns_q4_pack(ns_gpu* g, int form, const void* src, int64_t ss, int64_t M, int64_t K, int64_t group, void* w) {
    NS_TRY
    if (M <= 0 || K <= 0) return 0;
    if (form != 0 && form != 1) return ns_fail("ns_q4_pack: form 0 (float32 rows) or 1 (q4_0 blocks)");
    if (!q4_group(group)) return ns_fail("ns_q4_pack: groups of 32, 64 or 128");
    if (form == 1 && (group != 32 || K % 32)) return ns_fail("ns_q4_pack: q4_0 blocks hold groups of 32, a row whole blocks");
    if (M > (int64_t) 1 << 30 || K > (int64_t) 1 << 30) return ns_fail("ns_q4_pack: up to 2^30 rows and values a row");
    if (ss < (form ? K / 32 * 18 : K)) return ns_fail("ns_q4_pack: rows at least as far apart as they are long");
    if ((uintptr_t) w % 16) return ns_fail("ns_q4_pack: weights 16-byte aligned");
    if (!g || !src || !w) return ns_fail("ns_q4_pack: a null buffer");
    const int64_t kt = (K + 127) / 128, threads = (M + 15) / 16 * 16 * kt * (128 / group);
    if ((threads + 255) / 256 > INT32_MAX) return ns_fail("ns_q4_pack: too many weights");
    NS_HIP(hipSetDevice(g->dev));
    q4_pack_kernel<<<(unsigned) ((threads + 255) / 256), 256, 0, g->q>>>(form, src, ss, M, K, (int) group, kt, static_cast<uint8_t*>(w));
    NS_LAUNCHED("q4_pack");
    return 0;
    NS_CATCH
}

int ns_q4_product(ns_gpu* g, int qt, const void* x, int64_t xs, const void* w, int64_t group, void* y, int64_t ys, int64_t T, int64_t M, int64_t K) {
    NS_TRY
    if (T <= 0 || M <= 0) return 0;
    if (qt < 0 || qt > 2) return ns_fail("ns_q4_product: rows of type 0 (float32), 1 (half) or 2 (bfloat16)");
    if (T > 16) return ns_fail("ns_q4_product: 1 to 16 rows");
    if (!q4_group(group)) return ns_fail("ns_q4_product: groups of 32, 64 or 128");
    if (K <= 0 || M > (int64_t) 1 << 30 || K > (int64_t) 1 << 30) return ns_fail("ns_q4_product: 1 to 2^30 outputs and inputs");
    if (xs < K || ys < M) return ns_fail("ns_q4_product: rows at least as far apart as they are long");
    if ((uintptr_t) w % 16) return ns_fail("ns_q4_product: weights 16-byte aligned");
    if (!g || !x || !w || !y) return ns_fail("ns_q4_product: a null buffer");
    NS_HIP(hipSetDevice(g->dev));
    const int64_t e = qt ? 2 : 4;
    Q4Params p{x, static_cast<const uint8_t*>(w), y, xs, ys, (int) T, (int) M, (int) K, (int) ((K + 127) / 128), 0, (uintptr_t) x % 16 == 0 && xs * e % 16 == 0};
    if (qt == 0) launch_product<0>(g, p, group);
    else if (qt == 1) launch_product<1>(g, p, group);
    else launch_product<2>(g, p, group);
    NS_LAUNCHED("q4_product");
    return 0;
    NS_CATCH
}

}  // extern "C"
