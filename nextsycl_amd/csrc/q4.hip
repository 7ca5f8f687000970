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
// A work-group of 8 or 16 waves takes 16 outputs and shares K among its waves, tile by tile; the waves' sums meet in LDS in a
// fixed order. Rows that fit its LDS as operands are laid out there by each work-group, while its first weights are on
// their way; longer ones once, by a kernel in front, in the library's own scratch. A wave asks for a tile while it takes the
// one before. A half row x 18560 outputs of 4096 inputs in groups of 32: 10.4 us, 43 MB, 4.1 TB/s (8.3 us at a copy's rate) - four waves a SIMD ask
// for 1.1 KB each and unpack between (28 vector instructions a matrix instruction). 8 float32 rows x 4096 of 8192 in groups of 128 9.8 us: the rows'
// kernel 2.6, then the weights' 17 MB in 8.3, a work-group a CU, four tiles a wave one behind the other.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "ns_internal.hpp"
#include "ns_layer.h"
#include "attn_host.hpp"
#include "layer_common.hpp"

namespace {

constexpr int LDS_ROWS = 64 * 1024;

constexpr int WIDE_M = 4096;
constexpr int64_t MOST_M = ((int64_t) 1 << 27) - 16;        // (8 waves for 16 of them: what one launch takes)
constexpr int64_t q4_tile_bytes(int64_t group) { return 1024 + 16 * (128 / group) * 2; }

struct Q4Params {
    const void* x;
    const uint8_t* w;
    void* y;
    int64_t xs, ys;
    int T, M, K, kt;             // kt: tiles along K
    uint8_t* ops;                // the rows as operands, where LDS does not hold them
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

// The rows as operands: [plane][tile][16 pieces of 8][row], then a power of two a (tile, row)
template <int QT>
constexpr int PLANES = QT == 0 ? 2 : 1;
__device__ __forceinline__ int64_t q4_plane(const Q4Params& p) { return (int64_t) p.kt * 16 * p.T; }
// 16 threads (u) a (tile kl, row t): 8 values each
template <int QT>
__device__ __forceinline__ void q4_rows(const Q4Params& p, int kl, int t, int u, s8v* xo, float* xscale) {
    const int k = kl * 128 + u * 8;
    float v[8];
    if (k + 8 <= p.K) load_row<QT, 8>(p.x, t * p.xs + k, v);
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
        if constexpr (PLANES<QT> == 2) lo[j] = to16<false>(fabsf(f) < 65504.0f ? f - (float) half : 0.0f);
    }
    const int64_t at = (int64_t) (kl * 16 + u) * p.T + t;
    xo[at] = hi;
    if constexpr (PLANES<QT> == 2) xo[q4_plane(p) + at] = lo;
}
template <int QT>
__global__ __launch_bounds__(256) void q4_rows_kernel(Q4Params p) {
    const int task = blockIdx.x * 16 + threadIdx.x / 16;
    if (task >= p.kt * p.T) return;
    s8v* xo = reinterpret_cast<s8v*>(p.ops);
    q4_rows<QT>(p, task / p.T, task % p.T, threadIdx.x % 16, xo, reinterpret_cast<float*>(xo + q4_plane(p) * PLANES<QT>));
}

// GR: groups a tile (4, 2, 1); MEM: the rows' operands lie in memory, else in LDS; WAVES: 8, or 16
template <int QT, int GR, bool MEM, int WAVES>
__global__ __launch_bounds__(64 * WAVES, MEM && WAVES == 8 ? 2 : 4) void q4_product_kernel(Q4Params p) {
    constexpr int TILE = 1024 + 32 * GR, SW = 2 * GR;             // SW: a lane's scales, in words
    extern __shared__ __align__(16) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64), n = lane % 16, g = lane / 16;
    const int col = n < p.T ? n : p.T - 1;             // (columns behind the rows: some row's, never written)
    const int64_t plane = q4_plane(p);
    s8v* const xo = reinterpret_cast<s8v*>(MEM ? p.ops : lds);
    float* const xscale = reinterpret_cast<float*>(xo + plane * PLANES<QT>);
    const uint8_t* wt = p.w + (int64_t) blockIdx.x * p.kt * TILE;
    f4v acc = {0.0f, 0.0f, 0.0f, 0.0f};
    // a wave's next tiles: their nibbles, scales, and the rows' operands where those come from memory
    // (16 waves: not float32 rows' two planes where a tile has several groups, for which there are no registers)
    constexpr bool XAHEAD = MEM && !(WAVES == 16 && PLANES<QT> == 2 && GR > 1);
    constexpr int XS = XAHEAD ? 4 : 1, XP = XAHEAD ? PLANES<QT> : 1;
    struct Ahead {
        uint4 nib;
        uint32_t sc[SW];
        s8v x[XS][XP];
        float down;
    } ahead[2];
    auto fetch = [&](int i, Ahead& f) {
        const int kl = wave + WAVES * i;
        const uint8_t* tile = wt + (int64_t) kl * TILE;
        f.nib = *reinterpret_cast<const uint4*>(tile + lane * 16);
        const uint32_t* ss = reinterpret_cast<const uint32_t*>(tile + 1024 + g * 8 * GR);
#pragma unroll
        for (int j = 0; j < SW; ++j) f.sc[j] = ss[j];
        if constexpr (XAHEAD) {
            const s8v* x = xo + ((int64_t) kl * 16 + g) * p.T + col;
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int h = 0; h < XP; ++h) f.x[j][h] = x[h * plane + 4 * j * p.T];
            if (QT != 1) f.down = xscale[kl * p.T + col];
        }
    };
    auto compute = [&](int i, const Ahead& f) {
        const int kl = wave + WAVES * i;
        f4v tile = {0.0f, 0.0f, 0.0f, 0.0f}, s = tile;
        const uint32_t words[4] = {f.nib.x, f.nib.y, f.nib.z, f.nib.w};
        const s8v* x = xo + ((int64_t) kl * 16 + g) * p.T + col;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const s8v a = q4_operand(words[j]);
            if constexpr (XAHEAD) {
#pragma unroll
                for (int h = 0; h < XP; ++h) s = mfma16<false>(a, f.x[j][h], s);
            } else {
                s = mfma16<false>(a, x[4 * j * p.T], s);
                if constexpr (PLANES<QT> == 2) s = mfma16<false>(a, x[plane + 4 * j * p.T], s);
            }
            if ((j + 1) % (4 / GR) == 0) {
                const int grp = j / (4 / GR);
                const uint32_t s0 = f.sc[grp * 2], s1 = f.sc[grp * 2 + 1];
                tile[0] = fmaf(f16_to_f32((uint16_t) s0), s[0], tile[0]);
                tile[1] = fmaf(f16_to_f32((uint16_t) (s0 >> 16)), s[1], tile[1]);
                tile[2] = fmaf(f16_to_f32((uint16_t) s1), s[2], tile[2]);
                tile[3] = fmaf(f16_to_f32((uint16_t) (s1 >> 16)), s[3], tile[3]);
                s = f4v{0.0f, 0.0f, 0.0f, 0.0f};
            }
        }
        const float down = QT == 1 ? 1.0f : XAHEAD ? f.down : xscale[kl * p.T + col];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = QT == 1 ? acc[e] + tile[e] : fmaf(down, tile[e], acc[e]);
    };
    if (wave < p.kt) fetch(0, ahead[0]);
    if constexpr (!MEM) {
        for (int task = tid / 16; task < p.kt * p.T; task += 64 * WAVES / 16) q4_rows<QT>(p, task / p.T, task % p.T, tid % 16, xo, xscale);
        lds_barrier();                   // (the weights stay in flight)
    }
    for (int i = 0; wave + WAVES * i < p.kt; i += 2) {
        if (wave + WAVES * (i + 1) < p.kt) fetch(i + 1, ahead[1]);
        compute(i, ahead[0]);
        if (wave + WAVES * (i + 1) >= p.kt) break;
        if (wave + WAVES * (i + 2) < p.kt) fetch(i + 2, ahead[0]);
        compute(i + 1, ahead[1]);
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

template <int QT, int GR, int WAVES>
int launch_product(ns_gpu* g, Q4Params& p) {
    const int64_t rows = (int64_t) p.kt * p.T * (256 * PLANES<QT> + 4), sums = WAVES * 64 * sizeof(f4v);
    const unsigned grid = (unsigned) ((p.M + 15) / 16);
    if (rows <= LDS_ROWS) {
        q4_product_kernel<QT, GR, false, WAVES><<<grid, 64 * WAVES, std::max(rows, sums), g->q>>>(p);
        return 0;
    }
    if ((size_t) (rows + 3) / 4 > ns_own_floats(g)) return ns_fail("ns_q4_product: more scratch than the library has");
    NS_OWN_SCRATCH(g);
    p.ops = reinterpret_cast<uint8_t*>(g->own_scratch);
    q4_rows_kernel<QT><<<(unsigned) ((p.kt * p.T + 15) / 16), 256, 0, g->q>>>(p);
    q4_product_kernel<QT, GR, true, WAVES><<<grid, 64 * WAVES, sums, g->q>>>(p);
    return 0;
}
// 16 waves where each work-group has a CU of its own (up to 256 of them: 4096 outputs), else 8. Of 8192 inputs, a half row in groups of 32: 4096
// outputs 7.2 us with 8 waves, 6.3 with 16; 4112 8.7 and 8.0, 6144 9.4 and 8.7, 8192 9.7 and 9.2, but 18560 of 4096 10.9 and 12.2. 8 float32 rows
// in groups of 128: 4096 10.2 and 9.8, 4112 14.2 and 15.5, 6144 14.8 and 15.6. Whatever the rows' number, so that a row has the same bits alone
// and among others
template <int QT, int GR>
int launch_product(ns_gpu* g, Q4Params& p) {
    return p.M <= WIDE_M ? launch_product<QT, GR, 16>(g, p) : launch_product<QT, GR, 8>(g, p);
}
template <int QT>
int launch_product(ns_gpu* g, Q4Params& p, int64_t group) {
    return group == 32 ? launch_product<QT, 4>(g, p) : group == 64 ? launch_product<QT, 2>(g, p) : launch_product<QT, 1>(g, p);
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
    const int64_t kt = (K + 127) / 128, threads = (M + 15) / 16 * 16 * kt * (128 / group);
    if (!ns_grid_fits((threads + 255) / 256, 256)) return ns_fail("ns_q4_pack: too many weights");
    if (!g || !src || !w) return ns_fail("ns_q4_pack: a null buffer");
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
    if (K <= 0 || M > MOST_M || K > (int64_t) 1 << 22) return ns_fail("ns_q4_product: up to 2^27 - 16 outputs, 1 to 2^22 inputs");
    if (xs < K || ys < M) return ns_fail("ns_q4_product: rows at least as far apart as they are long");
    if ((uintptr_t) w % 16) return ns_fail("ns_q4_product: weights 16-byte aligned");
    if (!g || !x || !w || !y) return ns_fail("ns_q4_product: a null buffer");
    NS_HIP(hipSetDevice(g->dev));
    Q4Params p{x, static_cast<const uint8_t*>(w), y, xs, ys, (int) T, (int) M, (int) K, (int) ((K + 127) / 128)};
    const int rc = qt == 0 ? launch_product<0>(g, p, group) : qt == 1 ? launch_product<1>(g, p, group) : launch_product<2>(g, p, group);
    if (rc) return rc;
    NS_LAUNCHED("q4_product");
    return 0;
    NS_CATCH
}

}  // extern "C"
