// kv8_weights.hip: what many rows of one sequence give each cached token of their softmax weights, summed over rows and the query heads that
// share its key head (gfx950): column sums of softmax(q K^T), of which no row is kept.
//
// The weights need their row's largest score and sum first, so the product q K^T is made twice. Bound: the matrix unit for float32 rows (two halfs, two
// products: 1024 rows behind 3001 tokens, 24 / 4 heads of 256, 167 us, 84 % of a large product's rate in the passes), else the exponentials beside it and the
// passes' starts (64 bfloat16 rows behind 16320, 32 / 8 heads of 128: 44.5 us, two passes of 20). Both passes are one kernel: a wave keeps 64 tokens in registers, codes widened once, and pairs (row,
// head) stream past it through LDS, 16 KiB of operands at a time, for the work-group's four waves at once: 256 neighbouring tokens. First a pair's largest
// score and sum over each 64 tokens, then a token's sum over a split of the pairs. Between them small kernels: rows into halfs, in the order in which the lanes
// of an operand lie, with a factor a pair; a pair's parts together; the splits' sums into acc. Few pairs go the way of a token's attention with weights instead.
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
    int pairs;                  // T G, i G + g
    uint32_t ginv;              // 2^32 / G, rounded up
    float sl2;
    uint8_t* q16;               // [nh][tiles of 16 pairs][D / 32 KiB of halfs, as many of float32 rows' rest]: operands
    int tiles;
    float4* info;               // [nh][pairs]: factor, largest score, 1 / sum
    float2* part;               // [nh][nb][pairs]: largest score, sum over 64 tokens
    int64_t nb;                 // runs of 64 tokens
    int prs, rs;                // pairs a split, splits
    float* sums;                // [rs][nh][n], or null: into acc at once
    const float* acc0;
    float* acc1;
};

// a pair's row (of up to 2^31 / G pairs)
__device__ __forceinline__ int row_of(const WeightsParams& p, int pair) { return p.G == 1 ? pair : (int) __umulhi((uint32_t) pair, p.ginv); }
__device__ __forceinline__ int64_t low_of(const WeightsParams& p, int64_t pos) { return p.win > 0 && pos + 1 > p.win ? pos + 1 - p.win : 0; }

// a pair's row brought to exponent 13, as halfs: 16 lanes a pair. Operand (tile, step 2 j + i), lane 16 g + n: pair n's features 64 j + 16 g + 8 i .. + 7, the
// order in which a lane has a key's 16-byte chunks. (Pairs past the last: the last again)
template <int D, int QT>
__global__ __launch_bounds__(256) void kv8_rows_kernel(const WeightsParams p) {
    constexpr int E = D / 16, KB = D / 32, TILE_BYTES = KB * 1024 * (QT == 0 ? 2 : 1);
    const int pair = (int) blockIdx.x * 16 + threadIdx.x / 16;
    const int h = blockIdx.y, li = threadIdx.x % 16;
    const int pc = std::min(pair, p.pairs - 1), i = row_of(p, pc), g = pc - i * p.G;
    const int64_t at = (int64_t) i * p.qs + ((int64_t) (p.h0 + h) * p.G + g) * D + li * E;
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
    const int e = row_exponent(most);
    const float up = pow2_of(-e);
    uint8_t* to = p.q16 + ((int64_t) h * p.tiles + blockIdx.x) * TILE_BYTES;
#pragma unroll
    for (int j = 0; j < E; j += 8) {
        s8v a, b;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            a[k] = to16<false>(x[j + k] * up);
            if constexpr (QT == 0) b[k] = to16<false>(x[j + k] * up - f16_to_f32((uint16_t) a[k]));
        }
        const int d = li * E + j, place = ((d / 64 * 2 + d / 8 % 2) * 64 + d / 16 % 4 * 16 + (int) (threadIdx.x / 16)) * 16;
        *reinterpret_cast<s8v*>(to + place) = a;
        if constexpr (QT == 0) *reinterpret_cast<s8v*>(to + KB * 1024 + place) = b;
    }
    if (li == 0 && pair < p.pairs) p.info[(int64_t) h * p.pairs + pair].x = row_factor(p.sl2, e);
}

// pairs a key head, and scores in all, up to which the rows go as a token's do, the keys once more in the place of the values: two launches, not four or
// five, and the scores written. (us, instead of: 16 pairs of 8 heads of 128 behind 4000 tokens 15.9 / 20.1, behind 100000 62 / 89; 48 of 4 heads of 256 behind 4000
// 23.7 / 25.6, behind 100000 92.6 / 92.9; 64 of 8 heads of 128 behind 600 17.9 / 22.5, behind 4000 26.4 / 24.7; 96 of 4 of 256 behind 4000 28.1 / 28.1)
constexpr int64_t FEW = 48, FEW_SCORES = 3 << 19;
constexpr int RS = 16;                            // splits of the pairs, at most
constexpr int KT = 4, RUN = 16 * KT;              // tiles of 16 tokens a wave; tokens

__device__ __forceinline__ void give(const WeightsParams& p, int h, int64_t t, float sum) {
    const int b = kv8_block(p.c, p.c.table, 0, t >> p.c.shift);
    if (b < 0) return;
    const int64_t at = kv8_rows(p.c, b, p.h0 + h) + (t & (p.c.block - 1));
    p.acc1[at] = (p.acc0 && t < p.p0 ? p.acc0[at] : 0.0f) + sum;
}

// pass 1 (STATS): each pair's largest score and sum over a wave's 64 tokens; pass 2: what a split of the pairs gives each of them
template <int D, int FORM, bool QS, bool STATS>
__global__ __launch_bounds__(256, 2) void kv8_pass_kernel(const WeightsParams p) {
    // a stage of LDS: TG tiles of operands, and the numbers of 64 pairs; asked for two ahead
    constexpr int KB = D / 32, TILE_BYTES = KB * 1024 * (QS ? 2 : 1), TG = 16384 / TILE_BYTES, STAGE = 16384 + 1024;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[3][STAGE];
    const int lane = threadIdx.x & 63, n = lane & 15, g4 = lane >> 4, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = blockIdx.x % p.nh, r = blockIdx.x / p.nh % p.rs;
    // (the last tokens first: their rows' edges cost more)
    const int64_t run = ((p.nb + 3) / 4 - 1 - (int64_t) (blockIdx.x / p.nh / p.rs)) * 4 + w, key0 = run * RUN, first = (run - w) * RUN;
    // the pairs that see any of the work-group's tokens: rows from the first token's own on, to the last that still has the last one in its window
    const int row0 = (int) std::max<int64_t>(0, first - p.p0), row1 = p.win > 0 ? (int) std::min<int64_t>(p.T, std::max<int64_t>(0, first + 4 * RUN - 1 + p.win - p.p0)) : p.T;
    const int a0 = std::max(r * p.prs, row0 >= p.T ? p.pairs : row0 * p.G / 16 * 16), a1 = std::min(std::min((r + 1) * p.prs, p.pairs), row1 * p.G);
    const float4* info = p.info + (int64_t) h * p.pairs;
    const uint8_t* q16 = p.q16 + (int64_t) h * p.tiles * TILE_BYTES;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t) (uintptr_t) (__attribute__((address_space(3))) uint8_t*) &lds[0][0]);
    const uint32_t off[4] = {(uint32_t) lane * 16, (uint32_t) lane * 16, (uint32_t) lane * 16, (uint32_t) lane * 16};
    // (tiles past the last: the last operands again, masked; numbers past the last: whatever lies behind them, masked too)
    auto ask = [&](int pair0, int buf) __attribute__((always_inline)) {
        const int tile = std::min(pair0 / 16 + w * TG / 4, p.tiles - 1);
        const uint32_t to = lds0 + buf * STAGE;
        lds_fetch_run<false, 4>(q16 + (int64_t) tile * TILE_BYTES + (TG >= 4 ? 0 : w % (4 / TG) * 4096), off, to + w * 4096);
        lds_fetch<false>(reinterpret_cast<const uint8_t*>(info + pair0), off[0], to + 16384);
    };
    if (a0 < a1) ask(a0, 0);
    if (a0 + 16 * TG < a1) ask(a0 + 16 * TG, 1);
    // ---- the tokens
    s8v k[KT][KB];
    int blk[KT];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
        const int64_t t = key0 + kt * 16 + n;
        blk[kt] = kv8_block(p.c, p.c.table, 0, t >> p.c.shift);
        if (t >= p.n) blk[kt] = -1;
    }
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
        const int64_t t = key0 + kt * 16 + n;
        const int b = blk[kt];
        const uint8_t* row = p.c.kc + (kv8_rows(p.c, std::max(b, 0), p.h0 + h) + (t & (p.c.block - 1))) * D + 16 * g4;
        float sc = p.c.ksc[(int64_t) std::max(b, 0) * p.c.Hkv + p.h0 + h];
        if (b < 0) sc = 0.0f;                                     // (no block: nothing may have been stored into the one that was read, its scale be no number)
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
            uint4 x = *reinterpret_cast<const uint4*>(row + 64 * j);
            if (b < 0) x = uint4{0, 0, 0, 0};
            k[kt][2 * j] = kv8_halfs8<FORM>(x.x, x.y, sc, sc), k[kt][2 * j + 1] = kv8_halfs8<FORM>(x.z, x.w, sc, sc);
        }
    }
    float sum[STATS ? 1 : KT][4];
    if constexpr (!STATS)
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[kt][i] = 0.0f;

    int buf = 0, stores = 0;
    for (int group = a0; group < a1; group += 16 * TG, buf = buf == 2 ? 0 : buf + 1) {
        // this stage is there, everyone's; the one two ahead is of a buffer that everyone has read. What may still be under way: the next stage's 5 transfers,
        // and the TG stores behind them where all of the last stage's parts were written
        if (group + 16 * TG >= a1) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        else if (!STATS || stores == 0) asm volatile("s_waitcnt vmcnt(5) lgkmcnt(0)" ::: "memory");
        else if constexpr (TG == 4) asm volatile("s_waitcnt vmcnt(9) lgkmcnt(0)" ::: "memory");
        else if constexpr (TG == 2) asm volatile("s_waitcnt vmcnt(7) lgkmcnt(0)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(6) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (group + 32 * TG < a1) ask(group + 32 * TG, buf == 0 ? 2 : buf - 1);
        const float4* now = reinterpret_cast<const float4*>(&lds[buf][16384]);
        // a tile's scores; what they come to, edge: not every pair sees every token (tokens seen: lo .. hi - 1 from key0 on)
        auto product = [&](int tg, f4v (&s)[KT]) __attribute__((always_inline)) {
            const uint8_t* ql = &lds[buf][tg * TILE_BYTES + lane * 16];
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) s[kt] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < KB * (QS ? 2 : 1); ++j) {
                const s8v q = *reinterpret_cast<const s8v*>(ql + j * 1024);
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) s[kt] = mfma16<false>(k[kt][j % KB], q, s[kt]);
            }
            // (operands are read 4 steps ahead; left alone the compiler reads each pair of them right in front of its products)
            constexpr int N = KB * (QS ? 2 : 1), AHEAD = 4;
            __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
            for (int j = 0; j < N - AHEAD; ++j) __builtin_amdgcn_sched_group_barrier(0x008, KT, 0), __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, KT * AHEAD, 0);
        };
        auto take = [&](int tg, f4v (&s)[KT], auto edge, int lo, int hi) __attribute__((always_inline)) {
            constexpr bool EDGE = decltype(edge)::value;
            const float4 f = now[16 * tg + n];
            if constexpr (STATS) {
                if constexpr (EDGE)
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int key = kt * 16 + 4 * g4 + i;
                            if (key < lo || key >= hi) s[kt][i] = -INFINITY;
                        }
                float big = -INFINITY;
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) big = fmaxf(big, s[kt][i]);
                big = rows_max(big) * f.x;                        // (the factor is positive)
                const float ref = big == -INFINITY ? 0.0f : big;
                float all = 0.0f;
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) all += fast_exp2(fmaf(s[kt][i], f.x, -ref));
                all = rows_sum(all);
                const int pair = group + 16 * tg + n;
                if (g4 == 0 && pair < a1) p.part[((int64_t) h * p.nb + run) * p.pairs + pair] = float2{big, all};
            } else if constexpr (EDGE) {
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = kt * 16 + 4 * g4 + i;
                        const float e = fast_exp2(fmaf(s[kt][i], f.x, -f.y)) * f.z;
                        sum[kt][i] += key >= lo && key < hi ? e : 0.0f;
                    }
            } else
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum[kt][i] = fmaf(fast_exp2(fmaf(s[kt][i], f.x, -f.y)), f.z, sum[kt][i]);
        };
        const int64_t row_first = p.p0 + row_of(p, std::min(group, p.pairs - 1)), row_last = p.p0 + row_of(p, std::min(group + 16 * TG - 1, p.pairs - 1));
        if (group + 16 * TG <= a1 && key0 + RUN <= row_first + 1 && key0 >= low_of(p, row_last)) {
            // every pair sees every token: a tile's products beside the last one's exponentials
            stores = TG;
            f4v s[2][KT];
            product(0, s[0]);
#pragma unroll
            for (int tg = 0; tg < TG; ++tg) {
                if (tg + 1 < TG) product(tg + 1, s[(tg + 1) & 1]);
                take(tg, s[tg & 1], std::false_type(), 0, RUN);
            }
        } else {
            stores = 0;
#pragma unroll
            for (int tg = 0; tg < TG; ++tg) {
                const int pair0 = group + 16 * tg, pair = pair0 + n;
                const int64_t top = p.p0 + row_of(p, std::min(pair0, p.pairs - 1)), last = p.p0 + row_of(p, std::min(pair0 + 15, p.pairs - 1));
                if (pair0 >= a1 || last < key0 || low_of(p, top) >= key0 + RUN) continue;     // (none of them sees this wave's tokens)
                f4v s[KT];
                product(tg, s);
                if (key0 + RUN <= top + 1 && key0 >= low_of(p, last) && pair0 + 16 <= a1) take(tg, s, std::false_type(), 0, RUN);
                else {
                    const int64_t pos = p.p0 + row_of(p, std::min(pair, p.pairs - 1));
                    const int lo = (int) std::min<int64_t>(std::max<int64_t>(low_of(p, pos) - key0, 0), RUN);
                    const int hi = pair < a1 ? (int) std::min<int64_t>(std::max<int64_t>(pos + 1 - key0, 0), RUN) : 0;
                    take(tg, s, std::true_type(), lo, hi);
                }
            }
        }
    }
    if constexpr (!STATS)
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float v = row16_sum(sum[kt][i]);
                const int64_t t = key0 + kt * 16 + 4 * g4 + i;
                if (n == 0 && t < p.n) {
                    if (p.sums) p.sums[((int64_t) r * p.nh + h) * p.n + t] = v;
                    else give(p, h, t, v);
                }
            }
}

// a pair's runs of tokens together: 16 pairs a work-group, 16 threads each a part of the runs
__global__ __launch_bounds__(256) void kv8_stats_join_kernel(const WeightsParams p) {
    __shared__ float2 red[16][17];
    const int h = blockIdx.y, n = threadIdx.x & 15, part = threadIdx.x >> 4;
    const int pair = (int) blockIdx.x * 16 + n, pc = std::min(pair, p.pairs - 1);
    const int64_t pos = p.p0 + row_of(p, pc);
    const float2* at = p.part + (int64_t) h * p.nb * p.pairs + pc;
    float top = -INFINITY, sum = 0.0f;
    const int64_t end = pos / RUN + 1;
#pragma unroll 4
    for (int64_t b = low_of(p, pos) / RUN + part; b < end; b += 16) {
        const float2 v = at[b * p.pairs];
        const float m = fmaxf(top, v.x), ref = m == -INFINITY ? 0.0f : m;
        sum = sum * fast_exp2(top - ref) + v.y * fast_exp2(v.x - ref);
        top = m;
    }
    red[part][n] = float2{top, sum};
    __syncthreads();
    if (part || pair >= p.pairs) return;
    top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, red[i][n].x);
    const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int i = 0; i < 16; ++i) sum += red[i][n].y * fast_exp2(red[i][n].x - ref);
    float4* to = p.info + (int64_t) h * p.pairs + pair;
    to->y = ref, to->z = sum == 0.0f ? 0.0f : 1.0f / sum;
}
__global__ __launch_bounds__(256) void kv8_columns_join_kernel(const WeightsParams p) {
    const int64_t t = (int64_t) blockIdx.x * 256 + threadIdx.x;
    const int h = blockIdx.y;
    if (t >= p.n) return;
    float v[RS], sum = 0.0f;
#pragma unroll
    for (int r = 0; r < RS; ++r) v[r] = r < p.rs ? p.sums[((int64_t) r * p.nh + h) * p.n + t] : 0.0f;
#pragma unroll
    for (int r = 0; r < RS; ++r) sum += v[r];
    give(p, h, t, sum);
}

template <int D, int FORM, int QT>
int run(ns_gpu* g, const WeightsParams& p) {
    constexpr bool QS = QT == 0;
    const unsigned grid = (unsigned) ((p.nb + 3) / 4 * p.rs * p.nh);
    kv8_rows_kernel<D, QT><<<dim3((unsigned) ((p.pairs + 15) / 16), (unsigned) p.nh), 256, 0, g->q>>>(p);
    NS_LAUNCHED("kv8_rows");
    kv8_pass_kernel<D, FORM, QS, true><<<grid, 256, 0, g->q>>>(p);
    NS_LAUNCHED("kv8_pass");
    kv8_stats_join_kernel<<<dim3((unsigned) ((p.pairs + 15) / 16), (unsigned) p.nh), 256, 0, g->q>>>(p);
    NS_LAUNCHED("kv8_stats_join");
    kv8_pass_kernel<D, FORM, QS, false><<<grid, 256, 0, g->q>>>(p);
    NS_LAUNCHED("kv8_pass");
    if (p.sums) {
        kv8_columns_join_kernel<<<dim3((unsigned) ((p.n + 255) / 256), (unsigned) p.nh), 256, 0, g->q>>>(p);
        NS_LAUNCHED("kv8_columns_join");
    }
    return 0;
}
template <int D, int FORM>
int run(ns_gpu* g, int qt, const WeightsParams& p) { return qt == 0 ? run<D, FORM, 0>(g, p) : qt == 1 ? run<D, FORM, 1>(g, p) : run<D, FORM, 2>(g, p); }
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
    if (Hq <= 0 || Hq % Hkv || Hq / Hkv > KV8_HEADS) return ns_fail(w + ": query heads a multiple of the key heads, up to 4096 times");
    if (p0 < 0 || p0 > KV8_TOKENS || T > KV8_TOKENS) return ns_fail(w + ": positions of 0 to 2^30, up to 2^30 rows");
    if (qs < Hq * D) return ns_fail(w + ": rows at least as far apart as they are long");
    if (!g || !q || !acc1) return ns_fail(w + ": a null buffer");
    NS_HIP(hipSetDevice(g->dev));
    NS_OWN_SCRATCH(g);
    const int64_t own = (int64_t) ns_own_floats(g), G = Hq / Hkv, e = qt == 0 ? 4 : 2;
    p.sl2 = (scale > 0.0f ? scale : 1.0f / sqrtf((float) D)) * 1.4426950408889634f;
    if (T <= 16 && (T * G <= FEW || T * Hq * (p0 + T) <= FEW_SCORES)) {
        const int rc = ns_kv8_rows_weights(g, w, form, qt, p.c, q, qs, T, p0, Hq, kv8_window(win), p.sl2, acc0, acc1, g->own_scratch, own);
        if (rc <= 0) return rc;
    }
    // as many rows as the scratch holds - a pair its halfs, its four numbers, its two for each 64 tokens -, else fewer key heads at a time
    const int64_t runs = (p0 + T + RUN - 1) / RUN, per = G * (D / 2 * (qt == 0 ? 2 : 1) + 4 + 2 * runs), sums = RS * (p0 + T) + 16 * D + 1024;
    const int64_t nh0 = std::min(Hkv, own / (per + sums));
    if (nh0 < 1) return ns_fail(w + ": more tokens and heads than the library's scratch holds");
    const int64_t rows = std::min({T, (own / nh0 - sums) / per, std::max<int64_t>(1, ((int64_t) 1 << 31) / (G * G) - 64)});
    p.G = (int) G, p.ginv = (uint32_t) ((((int64_t) 1 << 32) + G - 1) / G), p.qs = qs, p.win = kv8_window(win);
    for (int64_t h = 0; h < Hkv; h += nh0) {
        p.h0 = (int) h, p.nh = (int) std::min(nh0, Hkv - h);
        for (int64_t r = 0; r < T; r += rows) {
            p.T = (int) std::min(rows, T - r), p.p0 = p0 + r, p.n = p.p0 + p.T, p.pairs = (int) (p.T * G);
            p.q = (const uint8_t*) q + r * qs * e, p.acc0 = r ? acc1 : acc0, p.acc1 = acc1;
            // splits: as fine as a stage of LDS until the chip's places, two a CU, are taken once; of 64 pairs and more until they are taken twice. (Once, the 1024
            // rows above 186 us, the 64 rows 49.0 where it is 47.1; three times the same. Always 64: 64 float32 rows behind 40, 24 / 4 heads of 256, 32.5 us where it
            // is 28.1; always a stage: behind 4000 46 where it is 36.6)
            p.nb = (p.n + RUN - 1) / RUN;
            const int64_t stage = 16384 / (D * (qt == 0 ? 4 : 2)), blocks = (p.nb + 3) / 4 * p.nh;
            auto splits = [&](int64_t places, int64_t least) { return std::min((places + blocks - 1) / blocks, (p.pairs + least - 1) / least); };
            const int64_t fine = splits(512, stage), coarse = splits(1024, 64), rs = std::min<int64_t>(RS, std::max(fine, coarse));
            p.prs = (int) up((p.pairs + rs - 1) / rs, fine > coarse ? stage : 64), p.rs = (p.pairs + p.prs - 1) / p.prs;
            if (!ns_grid_fits(blocks * p.rs, 256) || !ns_grid_fits((p.pairs + 15) / 16, 256)) return ns_fail(w + ": more work-groups than a launch takes");
            float* at = g->own_scratch;
            auto take = [&](int64_t floats) { float* was = at; at += up(floats, 64); return was; };
            p.tiles = (p.pairs + 15) / 16;
            p.q16 = (uint8_t*) take((int64_t) p.nh * p.tiles * 16 * D / 2 * (qt == 0 ? 2 : 1));
            p.info = (float4*) take((int64_t) p.nh * p.pairs * 4 + 256);     // (64 pairs are read at a time)
            p.part = (float2*) take(p.nh * p.pairs * p.nb * 2);
            p.sums = p.rs > 1 ? take((int64_t) p.rs * p.nh * p.n) : nullptr;
            if (at - g->own_scratch > own) return ns_fail(w + ": more tokens and heads than the library's scratch holds");
            const int rc = D == 128 ? (form == 0 ? run<128, 0>(g, qt, p) : run<128, 1>(g, qt, p)) : (form == 0 ? run<256, 0>(g, qt, p) : run<256, 1>(g, qt, p));
            if (rc) return rc;
        }
    }
    return 0;
    NS_CATCH
}
