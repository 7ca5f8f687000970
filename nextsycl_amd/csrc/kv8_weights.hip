// kv8_weights.hip: what many rows of one sequence give each cached token of their softmax weights, summed over rows and the query heads that
// share its key head (gfx950): column sums of softmax(q K^T), of which no row is kept.
//
// The weights need their row's largest score and sum first, so the product q K^T is made twice. Bound: the matrix unit and, as
// much, the exponentials of both passes. Four kernels: rows into halfs (two of them for float32 rows) with a factor a pair (row, head), keys
// into halfs; a pair's largest score and sum over a split of the tokens (pairs stay in registers, tokens stream past); the splits
// of a pair together; a token's sum over a split of the pairs (tokens stay in registers, pairs stream past); the sums into acc. The streaming
// operand comes from L2 into registers a tile ahead, waves of a work-group take tiles in turn and meet once at the end: no barrier in a loop.
#include <algorithm>
#include <cmath>

#include "attn_host.hpp"
#include "kv8_common.hpp"

namespace {

struct WeightsParams {
    Kv8Cache c;
    const void* q;
    int64_t qs, p0, n, win;     // the rows' first token; tokens in all
    int T, G, h0, nh;           // key heads h0 .. h0 + nh - 1
    int64_t pairs;              // T G, i G + g
    float sl2;
    const uint16_t* k;          // [nh][n][D] half
    uint16_t *qh, *ql;          // [nh][pairs][D] half; the rest of float32 rows
    float4* info;               // [nh][pairs]: factor, largest score, 1 / sum
    float2* part;               // [nh][pairs][ns]: largest score, sum
    int64_t kbs, prs;           // tokens a split; pairs a split
    int ns, rs;
    float* sums;                // [rs][nh][n], or null: into acc at once
    const float* acc0;
    float* acc1;
};

__device__ __forceinline__ int64_t low_of(const WeightsParams& p, int64_t pos) { return p.win > 0 && pos + 1 > p.win ? pos + 1 - p.win : 0; }

// a pair's row brought to exponent 13, as halfs: 16 lanes a pair
template <int D, int QT>
__global__ __launch_bounds__(256) void kv8_rows_kernel(const WeightsParams p) {
    constexpr int E = D / 16;
    const int64_t pair = (int64_t) blockIdx.x * 16 + threadIdx.x / 16;
    const int h = blockIdx.y, li = threadIdx.x % 16;
    const int64_t pc = std::min(pair, p.pairs - 1);
    const int64_t i = pc / p.G, g = pc - i * p.G;
    const int64_t at = i * p.qs + ((int64_t) (p.h0 + h) * p.G + g) * D + li * E;
    float x[E], most = 0.0f;
#pragma unroll
    for (int j = 0; j < E; j += 8) {
        float v[8];
        if constexpr (QT == 0) {
            float a[4], b[4];
            load_row<0, 4>(p.q, at + j, a), load_row<0, 4>(p.q, at + j + 4, b);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = a[k], v[4 + k] = b[k];
        } else load_row<QT, 8>(p.q, at + j, v);
#pragma unroll
        for (int k = 0; k < 8; ++k) x[j + k] = v[k], most = fmaxf(most, fabsf(v[k]));
    }
    most = row16_max(most);
    const int e = std::min(std::max((int) (__builtin_bit_cast(uint32_t, most) >> 23) - 127 - 13, -110), 110);
    const float up = kv8_pow2(-e);
    if (pair >= p.pairs) return;
    const int64_t to = ((int64_t) h * p.pairs + pair) * D + li * E;
#pragma unroll
    for (int j = 0; j < E; j += 8) {
        s8v a, b;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            a[k] = to16<false>(x[j + k] * up);
            if constexpr (QT == 0) b[k] = to16<false>(x[j + k] * up - f16_to_f32((uint16_t) a[k]));
        }
        *reinterpret_cast<s8v*>(p.qh + to + j) = a;
        if constexpr (QT == 0) *reinterpret_cast<s8v*>(p.ql + to + j) = b;
    }
    if (li == 0) p.info[(int64_t) h * p.pairs + pair].x = p.sl2 * kv8_pow2(e);
}

// 16 rows of halfs from row r0 on (past the last: the last again) as an operand: lane (n, g4) row n, features 32 j + 8 g4 ..
template <int D>
__device__ __forceinline__ void operand(s8v (&a)[D / 32], const uint16_t* rows, int64_t r0, int64_t last, int n, int g4) {
    const uint16_t* at = rows + std::min(r0 + n, last) * D + 8 * g4;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) a[j] = *reinterpret_cast<const s8v*>(at + 32 * j);
}

// a pair's largest score and sum of 2^(score - it) over tokens [split kbs, (split + 1) kbs): RT tiles of 16 pairs in registers
template <int D, bool QS, int RT>
__global__ __launch_bounds__(256, 2) void kv8_stats_kernel(const WeightsParams p) {
    constexpr int KB = D / 32;
    __shared__ float red[4][RT * 16][2];
    const int lane = threadIdx.x & 63, n = lane & 15, g4 = lane >> 4, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = blockIdx.x % p.nh, split = blockIdx.x / p.nh % p.ns;
    const int64_t pair0 = (int64_t) (blockIdx.x / p.nh / p.ns) * RT * 16;
    s8v q[RT][KB], ql[QS ? RT : 1][KB];
    float f[RT], m[RT], l[RT];
    int rlo[RT], rhi[RT];                                         // tokens seen, from the split's first on
    const int64_t row0 = pair0 / p.G, row1 = std::min<int64_t>((pair0 + RT * 16 - 1) / p.G, p.T - 1);
    const int64_t j0 = split * p.kbs;
    const int64_t kb = std::max(j0, low_of(p, p.p0 + row0)), ke = std::min(j0 + p.kbs, p.p0 + row1 + 1);
    const uint16_t *qh = p.qh + (int64_t) h * p.pairs * D, *qlo = p.ql + (int64_t) h * p.pairs * D, *k = p.k + (int64_t) h * p.n * D;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int64_t pair = std::min(pair0 + rt * 16 + n, p.pairs - 1), pos = p.p0 + pair / p.G;
        operand<D>(q[rt], qh, pair0 + rt * 16, p.pairs - 1, n, g4);
        if constexpr (QS) operand<D>(ql[rt], qlo, pair0 + rt * 16, p.pairs - 1, n, g4);
        f[rt] = p.info[(int64_t) h * p.pairs + pair].x;
        m[rt] = -INFINITY, l[rt] = 0.0f;
        rlo[rt] = (int) (std::max(low_of(p, pos), j0) - j0), rhi[rt] = (int) (std::min(pos, j0 + p.kbs - 1) - j0);
    }
    // tokens that all of the pairs see
    const int64_t full_lo = low_of(p, p.p0 + row1), full_hi = p.p0 + row0 + 1;
    const int t0 = kb < ke ? (int) ((kb - j0) / 32) : 0, t1 = kb < ke ? (int) ((ke - j0 + 31) / 32) : 0;
    s8v a[2][KB];
    int t = t0 + ((w - t0) & 3);
    if (t < t1)
#pragma unroll
        for (int i = 0; i < 2; ++i) operand<D>(a[i], k, j0 + t * 32 + 16 * i, p.n - 1, n, g4);
    for (; t < t1; t += 4) {
        f4v s[RT][2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                f4v x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < KB; ++j) {
                    x = mfma16<false>(a[i][j], q[rt][j], x);
                    if constexpr (QS) x = mfma16<false>(a[i][j], ql[rt][j], x);
                }
                s[rt][i] = x;
            }
        if (t + 4 < t1)
#pragma unroll
            for (int i = 0; i < 2; ++i) operand<D>(a[i], k, j0 + (t + 4) * 32 + 16 * i, p.n - 1, n, g4);
        const bool edge = j0 + t * 32 < full_lo || j0 + t * 32 + 32 > full_hi;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = s[rt][e / 4][e % 4] * f[rt];
            if (edge)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int key = t * 32 + (e / 4) * 16 + 4 * g4 + e % 4;
                    x[e] = key >= rlo[rt] && key <= rhi[rt] ? x[e] : -INFINITY;
                }
            // (each lane its own tokens' largest: the four lanes of a pair meet at the end)
            float top = m[rt];
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, x[e]);
            const float ref = top == -INFINITY ? 0.0f : top;
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) sum += fast_exp2(x[e] - ref);
            l[rt] = l[rt] * fast_exp2(m[rt] - ref) + sum;
            m[rt] = top;
        }
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const float top = rows_max(m[rt]), ref = top == -INFINITY ? 0.0f : top;
        const float sum = rows_sum(l[rt] * fast_exp2(m[rt] - ref));
        if (g4 == 0) red[w][rt * 16 + n][0] = top, red[w][rt * 16 + n][1] = sum;
    }
    __syncthreads();
    const int64_t pair = pair0 + threadIdx.x;
    if (threadIdx.x < RT * 16 && pair < p.pairs) {
        float top = -INFINITY, sum = 0.0f;
        for (int i = 0; i < 4; ++i) top = fmaxf(top, red[i][threadIdx.x][0]);
        const float ref = top == -INFINITY ? 0.0f : top;
        for (int i = 0; i < 4; ++i) sum += red[i][threadIdx.x][1] * fast_exp2(red[i][threadIdx.x][0] - ref);
        p.part[((int64_t) h * p.pairs + pair) * p.ns + split] = float2{top, sum};
    }
}
// a pair's splits together, in order
__global__ __launch_bounds__(256) void kv8_stats_join_kernel(const WeightsParams p) {
    const int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x;
    if (i >= p.pairs * p.nh) return;
    const float2* at = p.part + i * p.ns;
    float top = -INFINITY, sum = 0.0f;
    for (int s = 0; s < p.ns; ++s) top = fmaxf(top, at[s].x);
    const float ref = top == -INFINITY ? 0.0f : top;
    for (int s = 0; s < p.ns; ++s) sum += at[s].y * fast_exp2(at[s].x - ref);
    p.info[i].y = ref, p.info[i].z = sum == 0.0f ? 0.0f : 1.0f / sum;
}

__device__ __forceinline__ void give(const WeightsParams& p, int h, int64_t t, float sum) {
    const int b = kv8_block(p.c, p.c.table, 0, t >> p.c.shift);
    if (b < 0) return;
    const int64_t at = kv8_rows(p.c, b, p.h0 + h) + (t & (p.c.block - 1));
    p.acc1[at] = (p.acc0 && t < p.p0 ? p.acc0[at] : 0.0f) + sum;
}

// what pairs [rs prs, (rs + 1) prs) give KT tiles of 16 tokens, which stay in registers
template <int D, bool QS, int KT>
__global__ __launch_bounds__(256, 2) void kv8_columns_kernel(const WeightsParams p) {
    constexpr int KB = D / 32;
    __shared__ float red[4][KT * 16];
    const int lane = threadIdx.x & 63, n = lane & 15, g4 = lane >> 4, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = blockIdx.x % p.nh, r = blockIdx.x / p.nh % p.rs;
    const int64_t key0 = (int64_t) (blockIdx.x / p.nh / p.rs) * KT * 16;
    s8v k[KT][KB];
    float sum[KT][4];
    const uint16_t *qh = p.qh + (int64_t) h * p.pairs * D, *qlo = p.ql + (int64_t) h * p.pairs * D, *kr = p.k + (int64_t) h * p.n * D;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
        operand<D>(k[kt], kr, key0 + kt * 16, p.n - 1, n, g4);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[kt][i] = 0.0f;
    }
    // the pairs that see any of these tokens: rows from the first token's own on, to the last that still has the last one in its window
    const int64_t row0 = std::max<int64_t>(0, key0 - p.p0), row1 = p.win > 0 ? std::min<int64_t>(p.T, key0 + KT * 16 - 1 + p.win - p.p0) : p.T;
    const int64_t a0 = std::max(r * p.prs, row0 * p.G / 16 * 16), a1 = std::min(std::min((r + 1) * p.prs, p.pairs), row1 * p.G);
    const float4* info = p.info + (int64_t) h * p.pairs;
    s8v q[KB], ql[QS ? KB : 1];
    float4 f{};
    int64_t pair0 = a0 + 16 * w;
    if (pair0 < a1) {
        operand<D>(q, qh, pair0, p.pairs - 1, n, g4);
        if constexpr (QS) operand<D>(ql, qlo, pair0, p.pairs - 1, n, g4);
        f = info[std::min(pair0 + n, p.pairs - 1)];
    }
    for (; pair0 < a1; pair0 += 64) {
        f4v s[KT];
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
            f4v x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < KB; ++j) {
                x = mfma16<false>(k[kt][j], q[j], x);
                if constexpr (QS) x = mfma16<false>(k[kt][j], ql[j], x);
            }
            s[kt] = x;
        }
        const float4 now = f;
        const int64_t pair = pair0 + n;
        if (pair0 + 64 < a1) {
            operand<D>(q, qh, pair0 + 64, p.pairs - 1, n, g4);
            if constexpr (QS) operand<D>(ql, qlo, pair0 + 64, p.pairs - 1, n, g4);
            f = info[std::min(pair + 64, p.pairs - 1)];
        }
        const int64_t first = p.p0 + pair0 / p.G, last = p.p0 + (std::min(pair0 + 15, p.pairs - 1)) / p.G;
        const bool edge = key0 + KT * 16 > first + 1 || key0 < low_of(p, last) || pair0 + 16 > a1;
        if (edge) {
            const int64_t pos = p.p0 + std::min(pair, p.pairs - 1) / p.G, lo = low_of(p, pos);
            const bool live = pair < a1;
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int64_t key = key0 + kt * 16 + 4 * g4 + i;
                    const float e = fast_exp2(fmaf(s[kt][i], now.x, -now.y)) * now.z;
                    sum[kt][i] += live && key >= lo && key <= pos ? e : 0.0f;
                }
        } else
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[kt][i] = fmaf(fast_exp2(fmaf(s[kt][i], now.x, -now.y)), now.z, sum[kt][i]);
    }
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float v = row16_sum(sum[kt][i]);
            if (n == 0) red[w][kt * 16 + 4 * g4 + i] = v;
        }
    __syncthreads();
    const int64_t t = key0 + threadIdx.x;
    if (threadIdx.x < KT * 16 && t < p.n) {
        const float v = (red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x]);
        if (p.sums) p.sums[((int64_t) r * p.nh + h) * p.n + t] = v;
        else give(p, h, t, v);
    }
}
__global__ __launch_bounds__(256) void kv8_columns_join_kernel(const WeightsParams p) {
    const int64_t t = (int64_t) blockIdx.x * 256 + threadIdx.x;
    const int h = blockIdx.y;
    if (t >= p.n) return;
    float sum = 0.0f;
    for (int r = 0; r < p.rs; ++r) sum += p.sums[((int64_t) r * p.nh + h) * p.n + t];
    give(p, h, t, sum);
}

template <int D, int QT>
int run(ns_gpu* g, const WeightsParams& p) {
    constexpr bool QS = QT == 0;
    constexpr int RT = D == 128 ? 4 : 2, KT = D == 128 ? 4 : 2;
    kv8_rows_kernel<D, QT><<<dim3((unsigned) ((p.pairs + 15) / 16), (unsigned) p.nh), 256, 0, g->q>>>(p);
    NS_LAUNCHED("kv8_rows");
    kv8_stats_kernel<D, QS, RT><<<(unsigned) ((p.pairs + RT * 16 - 1) / (RT * 16) * p.ns * p.nh), 256, 0, g->q>>>(p);
    NS_LAUNCHED("kv8_stats");
    kv8_stats_join_kernel<<<(unsigned) ((p.pairs * p.nh + 255) / 256), 256, 0, g->q>>>(p);
    NS_LAUNCHED("kv8_stats_join");
    kv8_columns_kernel<D, QS, KT><<<(unsigned) ((p.n + KT * 16 - 1) / (KT * 16) * p.rs * p.nh), 256, 0, g->q>>>(p);
    NS_LAUNCHED("kv8_columns");
    if (p.sums) {
        kv8_columns_join_kernel<<<dim3((unsigned) ((p.n + 255) / 256), (unsigned) p.nh), 256, 0, g->q>>>(p);
        NS_LAUNCHED("kv8_columns_join");
    }
    return 0;
}
int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

}  // namespace

extern "C" int ns_kv8_weights(ns_gpu* g, int form, int qt, const void* q, int64_t qs, int64_t T, const int32_t* table, int64_t tmax, int64_t p0, int64_t Hq,
                              int64_t Hkv, int64_t D, int64_t block, int64_t blocks, const void* kc, const float* ksc, int64_t win, float scale, const float* acc0,
                              float* acc1) {
    NS_TRY
    const std::string w("ns_kv8_weights");
    if (T <= 0) return 0;
    WeightsParams p{};
    p.c = kv8_cache(kc, nullptr, ksc, nullptr, table, tmax, Hkv, D, block, blocks);
    if (qt < 0 || qt > 2) return ns_fail(w + ": rows of type 0 (float32), 1 (half) or 2 (bfloat16)");
    if (ns_kv8_check(w, form, Hkv, D, block, blocks, 1, tmax, p.c)) return -1;
    if (Hq <= 0 || Hq % Hkv || Hq > 1 << 20) return ns_fail(w + ": query heads a multiple of the key heads");
    if (p0 < 0 || p0 > KV8_TOKENS || T > KV8_TOKENS) return ns_fail(w + ": positions of 0 to 2^30, up to 2^30 rows");
    if (qs < Hq * D) return ns_fail(w + ": rows at least as far apart as they are long");
    if (!g || !q || !acc1) return ns_fail(w + ": a null buffer");
    NS_HIP(hipSetDevice(g->dev));
    NS_OWN_SCRATCH(g);
    const int64_t own = (int64_t) ns_own_floats(g), G = Hq / Hkv, e = qt == 0 ? 4 : 2;
    // as many key heads at a time as leave their keys half of the scratch, as many rows as the rest holds
    const int64_t one = up((p0 + T) * D / 2 + 16, 64), nh0 = std::min(Hkv, own / 2 / one);
    if (nh0 < 1) return ns_fail(w + ": more tokens than the library's scratch holds");
    constexpr int64_t NS = 64, RS = 16;                           // splits, at most
    // (a pair: its halfs, its four numbers, its splits' two each)
    const int64_t per = nh0 * G * (D / 2 * (qt == 0 ? 2 : 1) + 4 + 2 * NS), sums = RS * nh0 * (p0 + T);
    const int64_t rows = (own - nh0 * one - sums - 1024) / std::max<int64_t>(per, 1);
    if (rows < 1) return ns_fail(w + ": more tokens and heads than the library's scratch holds");
    p.G = (int) G, p.qs = qs, p.win = win > 0 ? win : 0;
    p.sl2 = (scale > 0.0f ? scale : 1.0f / sqrtf((float) D)) * 1.4426950408889634f;
    for (int64_t h = 0; h < Hkv; h += nh0) {
        p.h0 = (int) h, p.nh = (int) std::min(nh0, Hkv - h);
        for (int64_t r = 0; r < T; r += rows) {
            p.T = (int) std::min(rows, T - r), p.p0 = p0 + r, p.n = p.p0 + p.T, p.pairs = p.T * G;
            p.q = (const uint8_t*) q + r * qs * e, p.acc0 = r ? acc1 : acc0, p.acc1 = acc1;
            const int64_t tiles = D == 128 ? 64 : 32, blk = (p.pairs + tiles - 1) / tiles * p.nh, cols = (p.n + tiles - 1) / tiles * p.nh;
            // work-groups enough for two a CU, twice
            const int64_t ns = std::max<int64_t>(1, std::min<int64_t>({(1024 + blk - 1) / blk, NS, (p.n + 255) / 256}));
            p.kbs = up((p.n + ns - 1) / ns, 128), p.ns = (int) ((p.n + p.kbs - 1) / p.kbs);
            const int64_t rs = std::max<int64_t>(1, std::min<int64_t>({(1024 + cols - 1) / cols, RS, (p.pairs + 255) / 256}));
            p.prs = up((p.pairs + rs - 1) / rs, 64), p.rs = (int) ((p.pairs + p.prs - 1) / p.prs);
            if (!ns_grid_fits(blk * p.ns, 256) || !ns_grid_fits(cols * p.rs, 256)) return ns_fail(w + ": more work-groups than a launch takes");
            float* at = g->own_scratch;
            auto take = [&](int64_t floats) { float* was = at; at += up(floats, 64); return was; };
            uint16_t* k = (uint16_t*) take(p.nh * p.n * D / 2);
            p.qh = (uint16_t*) take(p.nh * p.pairs * D / 2);
            p.ql = qt == 0 ? (uint16_t*) take(p.nh * p.pairs * D / 2) : p.qh;
            p.info = (float4*) take(p.nh * p.pairs * 4);
            p.part = (float2*) take(p.nh * p.pairs * p.ns * 2);
            p.sums = p.rs > 1 ? take(p.rs * p.nh * p.n) : nullptr;
            p.k = k;
            if (at - g->own_scratch > own) return ns_fail(w + ": more tokens and heads than the library's scratch holds");
            if (ns_kv8_widen(g, form, p.c, p.h0, p.nh, 0, p.n, k, nullptr)) return -1;
            const int rc = D == 128 ? (qt == 0 ? run<128, 0>(g, p) : qt == 1 ? run<128, 1>(g, p) : run<128, 2>(g, p))
                                    : (qt == 0 ? run<256, 0>(g, p) : qt == 1 ? run<256, 1>(g, p) : run<256, 2>(g, p));
            if (rc) return rc;
        }
    }
    return 0;
    NS_CATCH
}
