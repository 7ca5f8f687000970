// kv8_attend.hip: attention of a token, or the few rows of a verify pass, of each of several sequences over a cache of 8-bit values in
// blocks of tokens (gfx950).
//
// Bound: HBM - every visible key and value byte read once for all rows and query heads of its key head; 4 D flops a (row, head,
// token), far under the matrix unit's ridge. (64 sequences of 126 to 8000 tokens x 32 / 8 heads of 128, 258 MB: 55.6 us, 6.0 TB/s between a start of 7 us and the
// merge's 5; a half row behind 131071 tokens with weights, 64 / 4 heads: 49.3; 7 float32 rows of 3 sequences behind 2398 to 43003, 24 / 4 heads of 256: 40.1, the
// widening's and the two halfs' instructions beside 131 MB; a row behind 4095, 32 / 8 heads: 11.2, two launches)
//
// Work split: the lengths are known on the device only, and differ. Short contexts are a work-group's each; a few longer ones take a work-group a chunk of 128
// tokens; else the tokens of all sequences and key heads lie end to end in chunks, and each work-group takes an equal run of them (with a grid over the longest
// sequence's splits 64 sequences of 125 to 8000 tokens kept a quarter of the waves' places busy). A run that ends inside a (sequence, key head) leaves a partial there,
// one that begins inside it another: two places a work-group hold them, and a second kernel puts a unit's pieces together. Wave w takes a chunk's tile w of 32 tokens
// through one buffer of keys and one of values of its own in LDS, asked for again as soon as their values lie in registers: no barrier in the loop. The waves'
// (O, m, l) meet in LDS in wave order. A wave holds its next 128 table entries and scales in two registers a lane and picks them by lane reads.
//
// A tile in the transposed orientation, as in attn_decode.hip: S^T[token][pair] = K Q^T with K's codes as halfs and the block's scale on
// the score; online softmax in base 2, float32; O^T[d][pair] += V^T P^T with V as halfs code x scale - exactly - read by the
// transposing 8-bit LDS read (16 lanes, 8 rows x 16 bytes: lane i gets byte i of every row). Rows are brought to exponent 13, which rejoins the scores'
// factor: half and bfloat16 rows are halfs then, exactly down to 2^-27 of their largest, and float32 rows two of them. The softmax weights are two halfs, 22
// bits, whatever the rows: 16-bit outputs are the sum rounded once. (One half a weight beside 16-bit rows: 64 sequences 56.1 us, two 57.0; the other calls of one row the
// same to 0.2)
#include <algorithm>
#include <cmath>

#include "attn_host.hpp"
#include "kv8_common.hpp"
#include "ns_attn.h"

namespace {

constexpr int WAVES = 4, TILE = 32, CHUNK = WAVES * TILE;
// log2 of what a row's largest weight is in the second product, if nothing larger came since: weights lie up to 2^15, a half's range ends above that, and
// its steps begin to widen for those under 2^-14: 2^-21 to 2^-29 of the largest
constexpr float LIFT = 7.0f;

struct AttendParams {
    Kv8Cache c;
    const void* q;
    int64_t qs;
    const int32_t *start, *lens;
    int64_t p0;                 // lens null: the one sequence's tokens in front of the call, its T rows
    int T, most, S, Hq, G;
    uint32_t ginv;              // 2^32 / G, rounded up
    int64_t longest, win;
    int nw, nz;                 // work-groups the chunks are dealt to; chunks of pairs
    int per, ns;                // a work-group's chunks, `per` of one unit, and how many of these a unit may be in; 0: runs
    float sl2;                  // scale x log2(e)
    void* out;
    float* part;                // [nw][most G][D]: O of a piece; runs: [nw][2]..: of one that begins inside a unit; of one that ends in it
    float2* ml;                 // [nw]..[most G]: its m, l
    int2* units;                // runs: [S][Hkv]: the first and the last work-group with tokens of a unit
    int pg;                     // groups of pairs that a sum of weights is shared by
    bool alone;                 // a work-group has all of a unit's scores and sums them up itself
    float* scores;              // [S][Hkv][most G][pad]: scores in log2 units, or null
    float2* stats;              // [S][Hkv][most G]: the largest score and 1 / sum of a pair whose unit is in one piece, or null
    int64_t pad;
    const float* acc0;
    float* acc1;
};

__device__ __forceinline__ Kv8Seq seq_of(const AttendParams& p, int s) {
    if (p.lens) return kv8_seq(p.start, p.lens, s, p.T, p.most);
    return {0, p.T, (int) p.p0};
}
// a sequence's tokens that its rows may see: [lo, hi)
__device__ __forceinline__ void span_of(const AttendParams& p, const Kv8Seq& q, int64_t& lo, int64_t& hi) {
    hi = std::min<int64_t>((int64_t) q.len + q.n, p.longest);
    lo = p.win > 0 ? std::max<int64_t>(0, (int64_t) q.len + 1 - p.win) : 0;
}

// (a 64-bit division takes some hundred instructions, a 32-bit one a few tens)
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) { return (a | b) >> 31 ? a / b : (int64_t) ((uint32_t) a / (uint32_t) b); }
__device__ __forceinline__ int64_t lane_of(int64_t v, int lane) {
    return (int64_t) (uint32_t) __builtin_amdgcn_readlane((int) (uint32_t) v, lane) | (int64_t) __builtin_amdgcn_readlane((int) (v >> 32), lane) << 32;
}
// the row of a pair (16 G of them, G up to 4096: pair x G under 2^32)
__device__ __forceinline__ int row_of(const AttendParams& p, int pair) { return p.G == 1 ? pair : (int) __umulhi((uint32_t) pair, p.ginv); }

// what 4 tokens in a row (a block holds them) have been given
struct Given {
    static constexpr int U = 8;
    int64_t t0, at, scores;
    bool live, seen;
    f4v sum, was;
    __device__ __forceinline__ Given(const AttendParams& p, const Kv8Seq& q, int s, int hk, int64_t t, bool first = true) {
        t0 = t;
        const int64_t end = (int64_t) q.len + q.n;
        const int b = kv8_block(p.c, p.c.table, s, t0 >> p.c.shift);
        live = t0 < end && b >= 0;
        at = kv8_rows(p.c, std::max(b, 0), hk) + (t0 & (p.c.block - 1));
        scores = ((int64_t) s * p.c.Hkv + hk) * p.most * p.G * p.pad + t0;
        int64_t lo, hi;
        span_of(p, q, lo, hi);
        seen = live && lo < hi && t0 < hi;
        sum = was = f4v{0.0f, 0.0f, 0.0f, 0.0f};
        if (p.acc0 && live && first) {
            if (t0 + 4 <= q.len) was = __builtin_bit_cast(f4v, *reinterpret_cast<const floats4_t*>(p.acc0 + at));
            else
#pragma unroll
                for (int i = 0; i < 4; ++i) was[i] = t0 + i < q.len ? p.acc0[at + i] : 0.0f;
        }
    }
    // the scores of pairs `pair` and on, up to `end`. (Only what a pair has seen was written, in whole tiles: tokens of these that one of its rows sees lie in one, the
    // others are 0 there. A tile that none of them lies in may hold anything)
    __device__ __forceinline__ void ask(const AttendParams& p, const Kv8Seq& q, int pair, int end, f4v (&x)[U]) const {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            x[i] = f4v{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            if (pair + i >= end) continue;
            const int64_t pos = (int64_t) q.len + row_of(p, pair + i);
            if (seen && t0 <= pos && (p.win <= 0 || t0 + 3 + p.win > pos)) x[i] = *reinterpret_cast<const f4v*>(p.scores + scores + (pair + i) * p.pad);
        }
    }
    // stat[i]: a pair's largest score and 1 / sum
    __device__ __forceinline__ void add(const f4v (&x)[U], const float2* stat, int i, int last) {
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const float2 f = stat[std::min(i + j, last)];
#pragma unroll
            for (int k = 0; k < 4; ++k) sum[k] = fmaf(fast_exp2(x[j][k] - f.x), f.y, sum[k]);
        }
    }
    __device__ __forceinline__ void give(const AttendParams& p, const Kv8Seq& q) const {
        const int64_t end = (int64_t) q.len + q.n;
        if (!live) return;
        if (t0 + 4 <= end) *reinterpret_cast<floats4_t*>(p.acc1 + at) = __builtin_bit_cast(floats4_t, was + sum);
        else
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (t0 + i < end) p.acc1[at + i] = was[i] + sum[i];
    }
};

// What a unit - a sequence's key head - costs besides its chunks, in chunks: its rows' way in, its sums' way out (2.2 us, where a chunk's bytes take
// 3 of a full chip's). Runs are dealt by chunks and that where there are more chunks than work-groups. (64 sequences of 125 to 8000 tokens x 8 heads:
// 72 us without it, 61.4 with 1, 57.2 with 2, 57.8 with 3; up to 4 float32 rows of each x 4 heads of 256, 62 to 4000 tokens, 84 / 63.8 / 59.2 / 57.2; of 3 sequences of up
// to 43003 48.2 / 46.5 / 44.8 / 44.0)
constexpr int EXTRA = 2;
// a sequence's chunks a key head: chunk `first` and on (a sequence with rows has one at least)
__device__ __forceinline__ int chunks_of(const AttendParams& p, const Kv8Seq& q, int& first) {
    int64_t lo, hi;
    span_of(p, q, lo, hi);
    first = (int) (lo / CHUNK);
    return q.n <= 0 ? 0 : std::max(1, (int) ((hi + CHUNK - 1) / CHUNK) - first);
}

// QT: the rows' type; RT row tiles of 16 pairs a wave; ACC: the scores are kept
template <int D, int RT, int FORM, int QT, bool ACC>
__global__ __launch_bounds__(WAVES * 64, 2) void kv8_attend_kernel(const AttendParams p) {
    constexpr bool QS = QT == 0;                                  // rows in two parts
    constexpr int CH = D / 16, KJ = D / 64, DT = D / 16;          // 16-byte chunks a row; chunks a lane reads of a key; tiles of 16 features
    constexpr int TB = TILE * D, NI = TB / 1024;                  // bytes a tile and stream; transfers
    constexpr int OROW = D + 4, MERGE = RT * 16 * OROW * 4;
    constexpr int WREG = ((2 * TB > MERGE ? 2 * TB : MERGE) + 1023) / 1024 * 1024;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[WAVES * WREG];
    __shared__ __attribute__((aligned(16))) float ml[RT * 16][2][WAVES];
    __shared__ float2 stat[ACC ? RT * 16 : 1];

    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g4 = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    // consecutive work-groups go round the 8 XCDs; a run's chunks of pairs follow each other on one of them (the grid is then a multiple of 8)
    int wg = blockIdx.x, z = 0;
    if (p.nz > 1) {
        const int xj = blockIdx.x / 8;
        wg = (xj / p.nz) * 8 + (int) (blockIdx.x % 8), z = xj % p.nz;
        if (wg >= p.nw) return;
    }
    const int Hkv = p.c.Hkv;
    // (all of the arguments at once: the compiler would ask for each group of them where it is used, one wait behind the other)
    asm volatile("" ::"s"(p.c.kc), "s"(p.c.vc), "s"(p.c.ksc), "s"(p.c.vsc), "s"(p.c.table), "s"(p.c.tmax), "s"(p.c.blocks), "s"(p.c.shift), "s"(p.q), "s"(p.qs), "s"(p.start), "s"(p.lens),
                 "s"(p.T), "s"(p.longest), "s"(p.win), "s"(p.sl2), "s"(p.ginv), "s"(p.nw));
    // ---- this work-group's run of chunks: `left` of them, from the `rest`th of sequence s on (its heads one behind the other)
    int s = 0, first, nch, extra = 0;
    int64_t rest = 0, run = 0, left = 0;
    int raw0 = 0, raw1 = 0;                                       // a piece's first entries where they are known in front of its length
    Kv8Seq q;
    if (p.per) {
        const int unit = wg / p.ns, e0 = (wg - unit * p.ns) * (p.per * CHUNK >> p.c.shift) + lane;
        s = unit / Hkv;
        raw0 = p.c.table[s * p.c.tmax + std::min<int64_t>(e0, p.c.tmax - 1)], raw1 = p.c.table[s * p.c.tmax + std::min<int64_t>(e0 + 64, p.c.tmax - 1)];
        q = seq_of(p, s);
        nch = chunks_of(p, q, first);
        if ((wg - unit * p.ns) * p.per >= nch) return;
    } else {
        // (chunks of a key head, and sequences that have some in bits 40 and up: both sums at once)
        constexpr int64_t ONE = (int64_t) 1 << 40;
        auto chunks = [](int64_t x) { return x & (ONE - 1); };
        auto deal = [&](int64_t all) {
            extra = chunks(all) * Hkv <= p.nw ? 0 : EXTRA;
            const int64_t total = (chunks(all) + (all >> 40) * extra) * Hkv;
            run = quotient(total + p.nw - 1, p.nw);
            rest = wg * run;
            left = std::max<int64_t>(0, std::min(run, total - rest));
        };
        if (p.S == 1) {
            q = seq_of(p, 0);
            nch = chunks_of(p, q, first);
            deal(nch ? nch + ONE : 0);
            if (left <= 0) return;
        } else {
            // (each wave for itself: a lane some of the sequences in a row)
            const int per = (p.S + 63) / 64, s0 = std::min(lane * per, p.S), s1 = std::min(s0 + per, p.S);
            int64_t mine = 0;
            int its;                                              // (a sequence's first chunk)
            auto some = [&](int i) { const int c = chunks_of(p, seq_of(p, i), its); return c ? c + ONE : 0; };
            for (int i = s0; i < s1; ++i) mine += some(i);
            int64_t x = mine;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int64_t y = __shfl_up(x, d);
                if (lane >= d) x += y;
            }
            deal(lane_of(x, 63));
            if (left <= 0) return;
            auto cost = [&](int64_t x) { return (chunks(x) + (x >> 40) * extra) * Hkv; };
            int64_t before = x - mine, at = 0;
            int found = 0;
            const bool here = cost(before) <= rest && rest < cost(x);
            if (here)
                for (int i = s0; i < s1; ++i) {
                    const int64_t y = some(i);
                    if (rest < cost(before + y)) {
                        found = i, at = rest - cost(before);
                        break;
                    }
                    before += y;
                }
            const int lane0 = __builtin_ctzll(__builtin_amdgcn_ballot_w64(here));
            s = __builtin_amdgcn_readlane(found, lane0);
            rest = lane_of(at, lane0);
            q = seq_of(p, s);
            nch = chunks_of(p, q, first);
        }
    }
    uint8_t* stage = lds + w * WREG;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t) (uintptr_t) (__attribute__((address_space(3))) uint8_t*) stage);
    // ---- transfers: chunk position cp of token kk holds the row's chunk cp ^ kk % CH (keys: 16 tokens' same chunk meet no bank
    // conflict), cp ^ (4 (kk / 16) + kk % 4) (values: the 8 rows of a group's transposing read). A transfer is 1024 / D rows; 16 tokens lie in one block
    uint32_t koff[NI], voff[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int r = lane / CH, kk = i * (1024 / D) + r, cp = lane % CH;
        koff[i] = (uint32_t) (r * D + (cp ^ (kk % CH)) * 16);
        voff[i] = (uint32_t) (r * D + (cp ^ (4 * (kk / 16) + kk % 4)) * 16);
    }

    for (;;) {
        // ---- a piece of the run: chunks c0 .. c1 - 1 of one unit
        int64_t lo, hi;
        span_of(p, q, lo, hi);
        const int cost = nch + extra;
        int hk, from, to;
        if (p.per) hk = wg / p.ns - s * Hkv, from = (wg - wg / p.ns * p.ns) * p.per, to = std::min(cost, from + p.per);
        else hk = (int) quotient(rest, cost), from = (int) (rest - (int64_t) hk * cost), to = (int) std::min<int64_t>(cost, from + left);
        const int c0 = std::max(from - extra, 0), c1 = to - extra;
        const int pairs = q.n * p.G, pair0 = z * RT * 16;
        if (pair0 < pairs && c1 > c0) {
            // from here on tokens are counted from the piece's first
            const int64_t j0 = (int64_t) (first + c0) * CHUNK;
            const int jb = (int) (std::max(j0, lo) - j0), je = (int) (std::min(j0 + (int64_t) (c1 - c0) * CHUNK, hi) - j0), pos0 = (int) std::max<int64_t>(q.len - j0, -(1 << 30));
            int blk[2];                                           // entries from the span's first on: lane, 64 + lane; none: -1
            float sk[2], sv[2];
            auto entries = [&](int at) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int e = i * 64 + lane;
                    blk[i] = kv8_block(p.c, p.c.table, s, ((j0 + at) >> p.c.shift) + e);
                    if (at + (e << p.c.shift) >= je) blk[i] = -1;
                }
            };
            auto scales = [&]() __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int64_t at = (int64_t) std::max(blk[i], 0) * Hkv + hk;
                    sk[i] = p.c.ksc[at], sv[i] = p.c.vsc[at];
                    if (blk[i] < 0) sk[i] = 0.0f, sv[i] = 0.0f;
                }
            };
            auto pick = [&](auto (&v)[2], int e) __attribute__((always_inline)) {
                const int x = __builtin_amdgcn_readlane(__builtin_bit_cast(int, v[0]), e & 63), y = __builtin_amdgcn_readlane(__builtin_bit_cast(int, v[1]), e & 63);
                return e < 64 ? x : y;
            };
            auto picked = [&](float (&v)[2], int e) __attribute__((always_inline)) { return __builtin_bit_cast(float, pick(v, e)); };
            auto place_of = [&](int at) __attribute__((always_inline)) {
                const int b = std::max(pick(blk, at >> p.c.shift), 0);
                return (kv8_rows(p.c, b, hk) + (at & (p.c.block - 1))) * D;
            };
            // (at: from the span's first token on)
            auto fetch_keys = [&](int at) __attribute__((always_inline)) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (p.nz == 1) lds_fetch_run<true, NI / 2>(p.c.kc + place_of(at + h * 16), koff + h * (NI / 2), lds0 + h * (TB / 2));
                    else lds_fetch_run<false, NI / 2>(p.c.kc + place_of(at + h * 16), koff + h * (NI / 2), lds0 + h * (TB / 2));
                }
            };
            auto fetch_values = [&](int at) __attribute__((always_inline)) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (p.nz == 1) lds_fetch_run<true, NI / 2>(p.c.vc + place_of(at + h * 16), voff + h * (NI / 2), lds0 + TB + h * (TB / 2));
                    else lds_fetch_run<false, NI / 2>(p.c.vc + place_of(at + h * 16), voff + h * (NI / 2), lds0 + TB + h * (TB / 2));
                }
            };
            const int span = 128 << p.c.shift;                    // tokens of the entries held
            const int t0 = jb / TILE;
            if (p.per && p.win <= 0) {
                const int e0 = (int) (j0 >> p.c.shift) + lane;
                blk[0] = e0 < p.c.tmax && (uint32_t) raw0 < (uint32_t) p.c.blocks && (lane << p.c.shift) < je ? raw0 : -1;
                blk[1] = e0 + 64 < p.c.tmax && (uint32_t) raw1 < (uint32_t) p.c.blocks && ((64 + lane) << p.c.shift) < je ? raw1 : -1;
            } else entries(0);

            // ---- this lane's rows: first and last token seen, operands
            s8v qh[RT][2 * KJ], ql[QS ? RT : 1][2 * KJ];
            float qm[RT];                                         // what a score takes besides the block's scale
            int rlo[RT], rhi[RT];                                 // tokens seen: rlo .. rhi
            float x[RT][2 * KJ][8], most[RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const int pair = pair0 + rt * 16 + n;
                const bool live = pair < pairs;
                const int i = live ? row_of(p, pair) : 0, g = live ? pair - i * p.G : 0;
                rhi[rt] = live ? std::min(pos0 + i, je - 1) : -1;
                rlo[rt] = p.win > 0 ? (int) std::max<int64_t>(jb, pos0 + i + 1 - p.win) : jb;
                const int64_t at = (int64_t) (q.first + i) * p.qs + (int64_t) (hk * p.G + g) * D;
                most[rt] = 0.0f;
#pragma unroll
                for (int j = 0; j < 2 * KJ; ++j) {
                    const int64_t d = at + 64 * (j / 2) + 16 * g4 + 8 * (j % 2);
                    if constexpr (QT == 0) {
                        float a[4], b[4];
                        load_row<0, 4>(p.q, d, a), load_row<0, 4>(p.q, d + 4, b);
#pragma unroll
                        for (int k = 0; k < 4; ++k) x[rt][j][k] = a[k], x[rt][j][4 + k] = b[k];
                    } else load_row<QT, 8>(p.q, d, x[rt][j]);
#pragma unroll
                    for (int k = 0; k < 8; ++k) most[rt] = fmaxf(most[rt], fabsf(x[rt][j][k]));
                }
            }
            // (the rows are there, as the entries are; the scales and the first tile are under way while they become operands)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) asm volatile("" : "+v"(most[rt]));
            scales();
            if (const int t = t0 + ((w - t0) & (WAVES - 1)); t * TILE < std::min(je, span)) fetch_keys(t * TILE), fetch_values(t * TILE);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const float top = rows_max(most[rt]);
                const int e = row_exponent(top);
                const float up = pow2_of(-e);
                qm[rt] = row_factor(p.sl2, e);
#pragma unroll
                for (int j = 0; j < 2 * KJ; ++j)
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const float v = x[rt][j][k] * up;
                        qh[rt][j][k] = to16<false>(v);
                        if constexpr (QS) ql[rt][j][k] = to16<false>(v - f16_to_f32((uint16_t) qh[rt][j][k]));
                    }
            }

            // m: what a row's weights are taken against, LIFT under the largest score it was moved to - moved where a weight would be past a half's range;
            // l: this lane's part of their sum
            float m[RT], l[RT];
            f4v o[RT][DT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                m[rt] = -INFINITY, l[rt] = 0.0f;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) o[rt][dt] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
            }
            // tiles that need no mask: every token seen by every row there is
            const int full_hi = std::min(pos0 + row_of(p, pair0) + 1, je);
            const int full_lo = p.win > 0 ? (int) std::max<int64_t>(jb, pos0 + q.n - p.win) : jb;

            for (int sp = 0; sp < je; sp += span) {
                const int t1 = (std::min(je, sp + span) + TILE - 1) / TILE;
                int t = std::max(t0, sp / TILE);
                t += (w - t) & (WAVES - 1);
                if (sp > 0) {
                    entries(sp), scales();
                    if (t < t1) fetch_keys(t * TILE - sp), fetch_values(t * TILE - sp);
                }
                // (the scales are there before the loop: in it the compiler would wait for them, and what is under way behind them, every turn)
                asm volatile("" : "+v"(sk[0]), "+v"(sk[1]), "+v"(sv[0]), "+v"(sv[1]));
                for (; t < t1; t += WAVES) {
                    const bool more = t + WAVES < t1;
                    const int key0 = t * TILE, at0 = key0 - sp, next = at0 + CHUNK;
                    // (the keys are there, the values behind them still under way)
                    if constexpr (NI == 4) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
                    else asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
                    uint4 raw[2][KJ];
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int j = 0; j < KJ; ++j) {
                            const int kk = h * 16 + n, c = 4 * j + g4;
                            raw[h][j] = *reinterpret_cast<const uint4*>(stage + kk * D + ((c ^ (kk % CH)) << 4));
                        }
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                    if (more) fetch_keys(next);
                    const int ent0 = at0 >> p.c.shift, ent1 = (at0 + 16) >> p.c.shift;
                    const bool bad0 = pick(blk, ent0) < 0, bad1 = pick(blk, ent1) < 0;
                    const bool edge = key0 + TILE > full_hi || key0 < full_lo || bad0 || bad1;

                    f4v sc[RT][2];
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) sc[rt][0] = sc[rt][1] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int j = 0; j < KJ; ++j)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const s8v a = kv8_halfs8<FORM>(raw[h][j].x, raw[h][j].y), b = kv8_halfs8<FORM>(raw[h][j].z, raw[h][j].w);
#pragma unroll
                            for (int rt = 0; rt < RT; ++rt) {
                                sc[rt][h] = mfma16<false>(a, qh[rt][2 * j], sc[rt][h]);
                                sc[rt][h] = mfma16<false>(b, qh[rt][2 * j + 1], sc[rt][h]);
                                if constexpr (QS) {
                                    sc[rt][h] = mfma16<false>(a, ql[rt][2 * j], sc[rt][h]);
                                    sc[rt][h] = mfma16<false>(b, ql[rt][2 * j + 1], sc[rt][h]);
                                }
                            }
                        }
                    const float k0 = picked(sk, ent0), k1 = picked(sk, ent1);
                    s8v ph[RT], pl[RT];
                    float kept[ACC ? RT : 1][8];
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        float x[8];
                        const float f0 = qm[rt] * k0, f1 = qm[rt] * k1;
#pragma unroll
                        for (int i = 0; i < 4; ++i) x[i] = sc[rt][0][i] * f0, x[4 + i] = sc[rt][1][i] * f1;
                        if (edge) {
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const int key = key0 + (i / 4) * 16 + 4 * g4 + i % 4;
                                if (i < 4 ? bad0 : bad1) x[i] = 0.0f;      // (no block: a key of zeros)
                                x[i] = key >= rlo[rt] && key <= rhi[rt] ? x[i] : -INFINITY;
                            }
                        }
                        if constexpr (ACC)
#pragma unroll
                            for (int i = 0; i < 8; ++i) kept[rt][i] = x[i];
                        const float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
                        if (__builtin_amdgcn_ballot_w64(top > m[rt] + 15.0f)) {
                            const float m1 = fmaxf(m[rt], rows_max(top) - LIFT), c = m1 == -INFINITY ? 1.0f : fast_exp2(m[rt] - m1);
                            m[rt] = m1;
                            l[rt] *= c;
#pragma unroll
                            for (int dt = 0; dt < DT; ++dt) o[rt][dt] *= c;
                        }
                        const float ref = m[rt] == -INFINITY ? 0.0f : m[rt];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float e = fast_exp2(x[i] - ref);
                            l[rt] += e;
                            ph[rt][i] = to16<false>(e);
                            pl[rt][i] = to16<false>(e - f16_to_f32((uint16_t) ph[rt][i]));
                        }
                    }
                    const float v0 = picked(sv, ent0), v1 = picked(sv, ent1);
                    if (!more) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                    else if constexpr (NI == 4) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
                    else asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
                    typedef int v2i __attribute__((ext_vector_type(2)));
                    v2i val[DT];
                    {
                        // lane n of group g4 addresses token row n / 2 of the group's 8, half n % 2 of the chunk
                        const int r = n >> 1, kk = (r >> 2) * 16 + 4 * g4 + (r & 3), x = 4 * (kk / 16) + kk % 4;
                        uint8_t* at = stage + TB + kk * D + (n & 1) * 8;
#pragma unroll
                        for (int dt = 0; dt < DT; ++dt) val[dt] = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) v2i*) (at + ((dt ^ x) << 4)));
                    }
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                    if constexpr (ACC) {
                        // (in front of the values' transfers: the wait for the keys ahead of them then counts these too, and no more; leaving them under way as well is no
                        // faster)
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt)
                            if (const int pair = pair0 + rt * 16 + n; pair < pairs) {
                                float* at = p.scores + (((int64_t) s * Hkv + hk) * p.most * p.G + pair) * p.pad + j0 + key0 + 4 * g4;
                                *reinterpret_cast<f4v*>(at) = f4v{kept[rt][0], kept[rt][1], kept[rt][2], kept[rt][3]};
                                *reinterpret_cast<f4v*>(at + 16) = f4v{kept[rt][4], kept[rt][5], kept[rt][6], kept[rt][7]};
                            }
                    }
                    if (more) fetch_values(next);
                    if (edge) {
                        // (bytes of tokens that there are not may hold anything)
                        uint32_t live0 = 0, live1 = 0;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int a = key0 + 4 * g4 + i, b = a + 16;
                            live0 |= !bad0 && a >= jb && a < je ? 0xFFu << (8 * i) : 0u;
                            live1 |= !bad1 && b >= jb && b < je ? 0xFFu << (8 * i) : 0u;
                        }
#pragma unroll
                        for (int dt = 0; dt < DT; ++dt) val[dt][0] &= (int) live0, val[dt][1] &= (int) live1;
                    }
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) {
                        const s8v a = kv8_halfs8<FORM>((uint32_t) val[dt][0], (uint32_t) val[dt][1], v0, v1);
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt) {
                            o[rt][dt] = mfma16<false>(a, ph[rt], o[rt][dt]);
                            o[rt][dt] = mfma16<false>(a, pl[rt], o[rt][dt]);
                        }
                    }
                }
            }

            // ---- the waves' sums, each parked in the wave's own region
            float* own = reinterpret_cast<float*>(stage);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const float sum = rows_sum(l[rt]);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f4v*>(own + (rt * 16 + n) * OROW + dt * 16 + 4 * g4) = o[rt][dt];
                if (g4 == 0) ml[rt * 16 + n][0][w] = m[rt], ml[rt * 16 + n][1][w] = sum;
            }
            __syncthreads();
            const bool whole = c0 == 0 && c1 == nch;
            const int64_t unit = (int64_t) s * Hkv + hk;
            const int64_t piece = (p.per ? wg : (int64_t) wg * 2 + (c0 == 0)) * p.most * p.G;
            for (int i = tid; i < RT * 16 * (D / 4); i += WAVES * 64) {
                const int row = i / (D / 4), d = i % (D / 4) * 4, pair = pair0 + row;
                if (pair >= pairs) break;
                float top = -INFINITY;
#pragma unroll
                for (int k = 0; k < WAVES; ++k) top = fmaxf(top, ml[row][0][k]);
                const float ref = top == -INFINITY ? 0.0f : top;
                f4v sum = {0.0f, 0.0f, 0.0f, 0.0f};
                float all = 0.0f;
#pragma unroll
                for (int k = 0; k < WAVES; ++k) {
                    const float c = fast_exp2(ml[row][0][k] - ref);
                    all += ml[row][1][k] * c;
                    sum += *reinterpret_cast<const f4v*>(reinterpret_cast<const float*>(lds + k * WREG) + row * OROW + d) * c;
                }
                if (whole) {
                    const float inv = all == 0.0f ? 0.0f : 1.0f / all;
                    const int i2 = row_of(p, pair), g = pair - i2 * p.G;
                    const float v[4] = {sum[0] * inv, sum[1] * inv, sum[2] * inv, sum[3] * inv};
                    const int64_t at = ((int64_t) (q.first + i2) * p.Hq + hk * p.G + g) * D + d;
#pragma unroll
                    for (int k = 0; k < 4; ++k) store_o<QT>(p.out, at + k, v[k]);
                    if (ACC && d == 0) {
                        if (p.alone) stat[row] = float2{ref, inv};
                        else p.stats[unit * p.most * p.G + pair] = float2{ref, inv};
                    }
                } else {
                    *reinterpret_cast<f4v*>(p.part + (piece + pair) * D + d) = sum;
                    if (d == 0) p.ml[piece + pair] = float2{top, all};
                }
            }
            if constexpr (ACC)
                if (p.alone) {
                    __syncthreads();                              // (the scores are written, the numbers there)
                    for (int64_t t = tid * 4; t < (int64_t) q.len + q.n; t += WAVES * 64 * 4) {
                        Given x(p, q, s, hk, t);
                        for (int at = 0; at < pairs; at += Given::U) {
                            f4v v[Given::U];
                            x.ask(p, q, at, pairs, v);
                            x.add(v, stat, at, pairs - 1);
                        }
                        x.give(p, q);
                    }
                }
            if (z == 0 && c0 == 0 && tid == 0 && p.units) p.units[unit] = int2{wg, whole ? wg : wg + (int) quotient(cost - to + run - 1, run)};
        }
        left -= to - from;
        if (left <= 0) break;                                     // (a piece alone: at once)
        rest += to - from;
        if (rest >= (int64_t) cost * Hkv) {
            rest = 0;
            do q = seq_of(p, ++s), nch = chunks_of(p, q, first);
            while (nch == 0 && s < p.S - 1);
            if (nch == 0) return;
        }
        __syncthreads();                                          // (the regions are read: the next piece's transfers may begin)
    }
}

// What comes behind the tokens, in one launch: `rows` work-groups put the pieces of a (sequence, key head, pair) together, others (with acc) sum up what 1024 tokens
// of a key head, or fewer of many pairs, have been given, from the scores and the pieces' m and l. (131072 tokens x 4 key heads of 16 rows, 192 pieces each: a launch each took 6.4 and
// 8.0 us one behind the other, 50.2 us the call instead of 53.4)
constexpr int TH = 256;

// where a unit's pieces lie, and how many there are: of runs the first one lies in its work-group's second place, the others in their first
struct Pieces {
    int64_t first;
    int last;
    bool runs;
    __device__ __forceinline__ int64_t at(int k) const { return runs ? 2 * (first + k) + (k == 0) : first + k; }
    __device__ __forceinline__ int count(const AttendParams& p, const Kv8Seq& q) const {
        int its;
        return runs ? last - (int) first + 1 : (chunks_of(p, q, its) + p.per - 1) / p.per;
    }
};
__device__ __forceinline__ Pieces pieces_of(const AttendParams& p, int64_t unit) {
    if (p.per) return {unit * p.ns, 0, false};
    const int2 ws = p.units[unit];
    return {ws.x, ws.y, true};
}

// out = sum over a unit's pieces of O 2^(m - M) / sum of l 2^(m - M): D / 4 threads x SG pieces at a time in a fixed shape, each of them against the largest m
// of its own
template <int D, int QT>
__device__ __forceinline__ void merge(const AttendParams& p, int64_t place, uint8_t* lds) {
    constexpr int L = D / 4, SG = TH / L, U = 8;
    float* sums = reinterpret_cast<float*>(lds);                  // [SG][D]
    float2* ml = reinterpret_cast<float2*>(lds + SG * D * 4);     // [SG]
    const int tid = threadIdx.x;
    const int64_t unit = place / (p.most * p.G);
    const int pair = (int) (place - unit * p.most * p.G), s = (int) (unit / p.c.Hkv), hk = (int) (unit - (int64_t) s * p.c.Hkv);
    const Pieces ps = pieces_of(p, unit);
    const Kv8Seq q = seq_of(p, s);
    const int64_t row = (int64_t) p.most * p.G;
    const int count = ps.count(p, q), sg = tid / L, d = tid % L * 4;
    if (pair >= q.n * p.G || count == 1) return;
    float m = -INFINITY, l = 0.0f;
    f4v sum = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k0 = sg; k0 < count; k0 += SG * U) {
        f4v o[U];
        float2 x[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int k = std::min(k0 + i * SG, count - 1);
            const int64_t at = ps.at(k) * row + pair;
            o[i] = *reinterpret_cast<const f4v*>(p.part + at * D + d), x[i] = p.ml[at];
            if (k0 + i * SG >= count) x[i].x = -INFINITY;
        }
        float top = m;
#pragma unroll
        for (int i = 0; i < U; ++i) top = fmaxf(top, x[i].x);
        const float ref = top == -INFINITY ? 0.0f : top, c0 = fast_exp2(m - ref);
        sum *= c0, l *= c0, m = top;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const float c = fast_exp2(x[i].x - ref);
            if (k0 + i * SG < count) sum += o[i] * c, l += x[i].y * c;
        }
    }
    *reinterpret_cast<f4v*>(sums + sg * D + d) = sum;
    if (d == 0) ml[sg] = float2{m, l};
    __syncthreads();
    if (tid >= L) return;
    float top = -INFINITY, all = 0.0f;
#pragma unroll 8
    for (int k = 0; k < SG; ++k) top = fmaxf(top, ml[k].x);
    const float ref = top == -INFINITY ? 0.0f : top;
    sum = f4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int k = 0; k < SG; ++k) {
        const float c = fast_exp2(ml[k].x - ref);
        sum += *reinterpret_cast<const f4v*>(sums + k * D + d) * c, all += ml[k].y * c;
    }
    const float inv = all == 0.0f ? 0.0f : 1.0f / all;
    const int i = row_of(p, pair), g = pair - i * p.G;
    const int64_t at = ((int64_t) (q.first + i) * p.Hq + hk * p.G + g) * D + d;
#pragma unroll
    for (int k = 0; k < 4; ++k) store_o<QT>(p.out, at + k, sum[k] * inv);
}

// acc1 = acc0 + the weights of the pairs: a thread 4 tokens and one of `pg` groups of the pairs, 8 at a time; 256 pairs' largest scores and sums at a time in
// LDS; the groups' sums meet there in their order
constexpr int PAIRS = 256;
__device__ __forceinline__ void give(const AttendParams& p, int64_t place, uint8_t* lds) {
    constexpr int U = Given::U;
    float2* stat = reinterpret_cast<float2*>(lds);                // [PAIRS]: m, 1 / l
    float2* part = stat + PAIRS;                                  // [TH]
    f4v* sums = reinterpret_cast<f4v*>(part);                     // [TH], behind the last of `part`
    const int tid = threadIdx.x, tokens = TH / p.pg, pg = tid / tokens, slot = tid - pg * tokens;
    const int64_t runs = (p.longest + 4 * tokens - 1) / (4 * tokens), unit = place / runs;
    const int s = (int) (unit / p.c.Hkv), hk = (int) (unit - (int64_t) s * p.c.Hkv);
    const int64_t t0 = ((place - unit * runs) * tokens + slot) * 4;
    const Kv8Seq q = seq_of(p, s);
    if (q.n <= 0 || t0 - 4 * slot >= (int64_t) q.len + q.n) return;
    const Pieces ps = pieces_of(p, unit);
    const int count = ps.count(p, q);
    Given given(p, q, s, hk, t0, pg == 0);
    const int64_t row = (int64_t) p.most * p.G;
    const int pairs = q.n * p.G, step = p.pg * U;
    for (int p0 = 0; p0 < pairs; p0 += PAIRS) {
        const int n = std::min(PAIRS, pairs - p0);
        f4v x[U];
        given.ask(p, q, p0 + pg * U, p0 + n, x);
        // the pairs' m and l over their pieces: up to 16 threads a pair
        const int bits = n > 1 ? 32 - __builtin_clz(n - 1) : 0, mine = tid & ((1 << bits) - 1), sub = tid >> bits, subs = std::min(TH >> bits, 16);
        if (count == 1) {
            if (tid < n) stat[tid] = p.stats[unit * row + p0 + tid];
        } else {
            float m = -INFINITY, l = 0.0f;
            if (mine < n && sub < subs)
                for (int k0 = sub; k0 < count; k0 += subs * U) {
                    float2 v[U];
                    float top = m;
#pragma unroll
                    for (int i = 0; i < U; ++i) {
                        const int k = std::min(k0 + i * subs, count - 1);
                        v[i] = p.ml[ps.at(k) * row + p0 + mine];
                        if (k0 + i * subs >= count) v[i] = float2{-INFINITY, 0.0f};
                    }
#pragma unroll
                    for (int i = 0; i < U; ++i) top = fmaxf(top, v[i].x);
                    const float ref = top == -INFINITY ? 0.0f : top;
                    l *= fast_exp2(m - ref), m = top;
#pragma unroll
                    for (int i = 0; i < U; ++i) l += v[i].y * fast_exp2(v[i].x - ref);
                }
            part[tid] = float2{m, l};
            __syncthreads();
            if (tid < n) {
                for (int k = 1; k < subs; ++k) m = fmaxf(m, part[(k << bits) + tid].x);
                const float ref = m == -INFINITY ? 0.0f : m;
                l = 0.0f;
                for (int k = 0; k < subs; ++k) l += part[(k << bits) + tid].y * fast_exp2(part[(k << bits) + tid].x - ref);
                stat[tid] = float2{ref, l == 0.0f ? 0.0f : 1.0f / l};
            }
        }
        __syncthreads();
        for (int at = pg * U; at < n; at += step) {
            f4v next[U];
            if (at + step < n) given.ask(p, q, p0 + at + step, p0 + n, next);
            given.add(x, stat, at, n - 1);
#pragma unroll
            for (int i = 0; i < U; ++i) x[i] = next[i];
        }
        __syncthreads();                                          // (the numbers are read)
    }
    // (tokens from `longest` on, if a sequence has any: nothing was given to them. Its last work-group's)
    if (place - unit * runs == runs - 1)
        for (int64_t t = (runs * tokens + tid) * 4; t < (int64_t) q.len + q.n; t += TH * 4) Given(p, q, s, hk, t).give(p, q);
    if (p.pg > 1) {
        sums[tid] = given.sum;
        __syncthreads();
        if (pg) return;
        for (int i = 1; i < p.pg; ++i) given.sum += sums[i * tokens + slot];
    }
    given.give(p, q);
}

template <int D, int QT, bool ACC>
__global__ __launch_bounds__(TH) void kv8_join_kernel(const AttendParams p, int64_t rows) {
    constexpr int SG = TH / (D / 4), MERGE = SG * D * 4 + SG * 8, GIVE = ACC ? PAIRS * 8 + TH * 16 : 0;
    __shared__ __attribute__((aligned(16))) uint8_t lds[MERGE > GIVE ? MERGE : GIVE];
    if (!ACC || (int64_t) blockIdx.x < rows) merge<D, QT>(p, blockIdx.x, lds);
    else give(p, (int64_t) blockIdx.x - rows, lds);
}

template <int D, int RT, int QT>
void launch_attend(ns_gpu* g, int form, const AttendParams& p, dim3 grid) {
    if (p.acc1) form == 0 ? kv8_attend_kernel<D, RT, 0, QT, true><<<grid, WAVES * 64, 0, g->q>>>(p) : kv8_attend_kernel<D, RT, 1, QT, true><<<grid, WAVES * 64, 0, g->q>>>(p);
    else form == 0 ? kv8_attend_kernel<D, RT, 0, QT, false><<<grid, WAVES * 64, 0, g->q>>>(p) : kv8_attend_kernel<D, RT, 1, QT, false><<<grid, WAVES * 64, 0, g->q>>>(p);
}
template <int QT>
void launch_attend(ns_gpu* g, int form, const AttendParams& p, int64_t D, int RT, dim3 grid) {
    if (D == 128) RT == 1 ? launch_attend<128, 1, QT>(g, form, p, grid) : launch_attend<128, 2, QT>(g, form, p, grid);
    else launch_attend<256, 1, QT>(g, form, p, grid);
}
template <int D, int QT>
void launch_join(ns_gpu* g, const AttendParams& p, int64_t rows, int64_t grid) {
    if (p.acc1) kv8_join_kernel<D, QT, true><<<(unsigned) grid, TH, 0, g->q>>>(p, rows);
    else kv8_join_kernel<D, QT, false><<<(unsigned) grid, TH, 0, g->q>>>(p, rows);
}

// 16-pair tiles a wave: two where more than 16 pairs share a key head of 128 (heads of 256 have no registers for a second: 16 pairs a work-group,
// the next ones read the tokens from L2)
int tiles_of(int64_t pairs, int64_t D) { return pairs > 16 && D == 128 ? 2 : 1; }
int64_t pair_chunks(int64_t pairs, int64_t D) { const int64_t rows = 16 * tiles_of(pairs, D); return (pairs + rows - 1) / rows; }
// chunks up to which work-groups take a unit each, by the number of units: nothing is put together behind them then, and no run is looked for. 2 of 4 units, 4 of
// 8, 10 of 64, 12 of 128, 16 of 512 and more. (us, a unit each against runs: 8 units of 400 tokens 10.3 / 11.4, of 800 14.5 / 11.6; 4 units of 24 rows of 256
// features, 200 tokens 11.9 / 14.4, 400 15.6 / 13.9; 128 units of 800 tokens 14.9 / 18.3, of 1600 22.6 / 21.0; 512 units of 1600 38.5 / 43.0)
int64_t whole_chunks(int64_t units) {
    int64_t log2 = 0;
    while (units >> (log2 + 1)) ++log2;
    return std::max<int64_t>(1, std::min<int64_t>(2 * log2 - 2, 16));
}
// How the tokens are dealt out. A work-group a piece of at most `per` chunks of a unit: all of its chunks where contexts are short (above), one where 512
// work-groups, two a CU, are enough for that - its table entries are asked for beside its length then, not behind it (us, beside runs: 3 sequences of 800
// tokens x 8 heads 11.5 / 13.0, 4 rows of each x 4 heads of 256 15.1 / 17.1, a token behind 4095 12.0 / 12.0; the wrong side, 3 sequences of 25 to 1600 - every
// one's places are counted at the longest - 18.3 / 16.8). Else
// runs, on as many work-groups. (64 sequences of 125 to 8000 tokens x 8 heads of 128: 448 work-groups 59.0 us, 512 57.2, 640 64.5, 768 59.4; all of 8000: 180 / 171 /
// 195 / 181; 4 rows of each of 64 x 24 / 4 heads of 256, two chunks of pairs, 4000 tokens: 192 pairs of work-groups 172, 256 136)
struct Deal {
    int64_t nw, per, ns;
};
Deal deal_of(int64_t S, int64_t pairs, int64_t Hkv, int64_t D, int64_t longest) {
    const int64_t chunks = (longest + CHUNK - 1) / CHUNK, units = S * Hkv, places = std::max<int64_t>(1, 512 / pair_chunks(pairs, D));
    if (chunks <= whole_chunks(units)) return {units, chunks, 1};
    if (units * chunks <= places) return {units * chunks, 1, chunks};
    return {std::min(places, units * (chunks + EXTRA)), 0, 0};
}

struct Scratch {
    int64_t part, ml, units, scores, stats, pad;
    int64_t all() const { return part + ml + units + scores + stats; }
};
Scratch scratch_of(int64_t S, int64_t most, int64_t Hq, int64_t Hkv, int64_t D, int64_t longest, bool acc, const Deal& deal) {
    const int64_t rows = S * most * Hq, pairs = most * (Hq / Hkv), pieces = deal.per ? (deal.ns > 1 ? deal.nw : 0) : 2 * deal.nw;
    Scratch x{};
    x.pad = (longest + 31) / 32 * 32;
    x.part = pieces * pairs * D, x.ml = (pieces * pairs * 2 + 3) / 4 * 4;
    x.units = deal.per ? 0 : (S * Hkv * 2 + 3) / 4 * 4;
    x.scores = acc ? rows * x.pad : 0;
    x.stats = acc ? rows * 2 : 0;
    return x;
}
bool sizes_fit(int64_t S, int64_t most, int64_t Hq, int64_t Hkv, int64_t D, int64_t longest) {
    return S > 0 && S <= 65535 && most > 0 && most <= DECODE_ROWS && Hkv > 0 && Hkv <= 32767 && Hq > 0 && Hq % Hkv == 0 && Hq / Hkv <= KV8_HEADS && S * most * Hq <= INT32_MAX && (D == 128 || D == 256) && longest > 0 &&
           longest <= 2 * (int64_t) KV8_TOKENS;
}

Scratch scratch_of(int64_t S, int64_t most, int64_t Hq, int64_t Hkv, int64_t D, int64_t longest, bool acc) {
    return scratch_of(S, most, Hq, Hkv, D, longest, acc, deal_of(S, most * (Hq / Hkv), Hkv, D, longest));
}

// a checked call, its scratch at hand: scratch_of's floats
int attend(ns_gpu* g, const std::string& w, int form, int qt, AttendParams p, int64_t Hkv, int64_t D, const Deal& deal, float* scratch) {
    const int64_t pairs = (int64_t) p.most * p.G, nz = pair_chunks(pairs, D), rows = (int64_t) p.S * p.most * p.Hq;
    const Scratch x = scratch_of(p.S, p.most, p.Hq, Hkv, D, p.longest, p.acc1 != nullptr, deal);
    p.nw = (int) deal.nw, p.per = (int) deal.per, p.ns = (int) deal.ns, p.nz = (int) nz, p.pad = x.pad;
    p.ginv = (uint32_t) ((((int64_t) 1 << 32) + p.G - 1) / p.G);
    const int64_t grid = nz > 1 ? (deal.nw + 7) / 8 * 8 * nz : deal.nw;
    const bool pieces = x.part > 0;
    p.part = scratch;
    p.ml = (float2*) (scratch + x.part);
    p.units = deal.per ? nullptr : (int2*) (scratch + x.part + x.ml);
    p.scores = p.acc1 ? scratch + x.part + x.ml + x.units : nullptr;
    p.stats = p.acc1 ? (float2*) (scratch + x.part + x.ml + x.units + x.scores) : nullptr;
    // (a unit's work-group, where it has all its pairs, sums up their weights too: 8 heads behind 100 tokens 9.2 us, in a launch of their own 11.6; 64 sequences behind
    // 800 28.1 / 30.7)
    p.alone = p.acc1 && deal.per && deal.ns == 1 && nz == 1;
    // (up to 16 pairs a thread's, while that leaves the chip empty: 256 pairs of 4 key heads behind 500 tokens 21.0 us, all by one thread 60.1; behind 30000 104, 128)
    for (p.pg = 1; p.pg < 16 && p.pg * 16 < pairs && (p.longest * p.pg + 4 * TH - 1) / (4 * TH) * Hkv * p.S < 512;) p.pg *= 2;
    const int64_t merges = pieces ? rows : 0, tokens = 4 * TH / p.pg, gives = p.acc1 && !p.alone ? (p.longest + tokens - 1) / tokens * Hkv * p.S : 0;
    if (!ns_grid_fits(grid, 256) || !ns_grid_fits(merges + gives, TH)) return ns_fail(w + ": more work-groups than a launch takes");
    const int RT = tiles_of(pairs, D);
    if (qt == 0) launch_attend<0>(g, form, p, D, RT, dim3((unsigned) grid));
    else if (qt == 1) launch_attend<1>(g, form, p, D, RT, dim3((unsigned) grid));
    else launch_attend<2>(g, form, p, D, RT, dim3((unsigned) grid));
    NS_LAUNCHED("kv8_attend");
    if (merges + gives > 0) {
        if (D == 128) qt == 0 ? launch_join<128, 0>(g, p, merges, merges + gives) : qt == 1 ? launch_join<128, 1>(g, p, merges, merges + gives) : launch_join<128, 2>(g, p, merges, merges + gives);
        else qt == 0 ? launch_join<256, 0>(g, p, merges, merges + gives) : qt == 1 ? launch_join<256, 1>(g, p, merges, merges + gives) : launch_join<256, 2>(g, p, merges, merges + gives);
        NS_LAUNCHED("kv8_join");
    }
    return 0;
}

}  // namespace

int ns_kv8_rows_weights(ns_gpu* g, const std::string& w, int form, int qt, const Kv8Cache& c, const void* q, int64_t qs, int64_t T, int64_t p0, int64_t Hq, int64_t win,
                        float sl2, const float* acc0, float* acc1, float* scratch, int64_t floats) {
    AttendParams p{};
    p.c = c, p.c.vc = c.kc, p.c.vsc = c.ksc;
    p.q = q, p.qs = qs, p.p0 = p0, p.T = p.most = (int) T, p.S = 1, p.Hq = (int) Hq, p.G = (int) (Hq / c.Hkv), p.longest = p0 + T, p.win = win, p.sl2 = sl2;
    p.acc0 = acc0, p.acc1 = acc1;
    const Deal deal = deal_of(1, T * p.G, c.Hkv, c.D, p.longest);
    const int64_t rows = (T * Hq * c.D + 3) / 4 * 4, need = scratch_of(1, T, Hq, c.Hkv, c.D, p.longest, true, deal).all();
    if (T > DECODE_ROWS || need + rows > floats) return 1;
    p.out = scratch + need;
    return attend(g, w, form, qt, p, c.Hkv, c.D, deal, scratch);
}

extern "C" {

int64_t ns_kv8_attend_scratch(int64_t S, int64_t most, int64_t Hq, int64_t Hkv, int64_t D, int64_t longest, int acc) {
    return sizes_fit(S, most, Hq, Hkv, D, longest) ? scratch_of(S, most, Hq, Hkv, D, longest, acc != 0).all() : 0;
}

int ns_kv8_attend(ns_gpu* g, int form, int qt, const void* q, int64_t qs, int64_t T, const int32_t* start, const int32_t* lens, int64_t S, int64_t most,
                  int64_t longest, const int32_t* table, int64_t tmax, int64_t Hq, int64_t Hkv, int64_t D, int64_t block, int64_t blocks, const void* kc,
                  const void* vc, const float* ksc, const float* vsc, int64_t win, float scale, void* out, const float* acc0, float* acc1, float* scratch) {
    NS_TRY
    const std::string w("ns_kv8_attend");
    if (T <= 0 || S <= 0 || most <= 0) return 0;
    AttendParams p{};
    p.c = kv8_cache(kc, vc, ksc, vsc, table, tmax, Hkv, D, block, blocks);
    if (qt < 0 || qt > 2) return ns_fail(w + ": rows of type 0 (float32), 1 (half) or 2 (bfloat16)");
    if (ns_kv8_check(w, form, Hkv, D, block, blocks, S, tmax, p.c)) return -1;
    if (Hq <= 0 || Hq % Hkv || Hq / Hkv > KV8_HEADS) return ns_fail(w + ": query heads a multiple of the key heads, up to 4096 times");
    if (most > DECODE_ROWS) return ns_fail(w + ": 1 to 16 rows a sequence");
    if (S * most * Hq > INT32_MAX) return ns_fail(w + ": up to 2^31 - 1 rows x heads");
    if (T > KV8_TOKENS) return ns_fail(w + ": up to 2^30 rows");
    if (longest <= 0 || longest > 2 * (int64_t) KV8_TOKENS) return ns_fail(w + ": contexts of 1 to 2^31 tokens");
    if (qs < Hq * D) return ns_fail(w + ": rows at least as far apart as they are long");
    p.S = (int) S, p.most = (int) most, p.Hq = (int) Hq, p.G = (int) (Hq / Hkv), p.longest = longest, p.T = (int) T;
    const int64_t need = scratch_of(S, p.most, Hq, Hkv, D, longest, acc1 != nullptr).all();
    if (!g || !q || !lens || !vc || !vsc || !out || (need && !scratch)) return ns_fail(w + ": a null buffer");
    if (need && (uintptr_t) scratch % 16) return ns_fail(w + ": scratch 16-byte aligned");
    p.q = q, p.qs = qs, p.start = start, p.lens = lens, p.win = kv8_window(win), p.out = out, p.acc0 = acc0, p.acc1 = acc1;
    p.sl2 = (scale > 0.0f ? scale : 1.0f / sqrtf((float) D)) * 1.4426950408889634f;
    NS_HIP(hipSetDevice(g->dev));
    return attend(g, w, form, qt, p, Hkv, D, deal_of(S, most * p.G, Hkv, D, longest), scratch);
    NS_CATCH
}

int ns_kv8_prompt(ns_gpu* g, int form, int qt, const void* q, int64_t qs, int64_t T, const int32_t* table, int64_t tmax, int64_t p0, int64_t Hq, int64_t Hkv,
                  int64_t D, int64_t block, int64_t blocks, const void* kc, const void* vc, const float* ksc, const float* vsc, int64_t win, float scale,
                  void* out) {
    NS_TRY
    const std::string w("ns_kv8_prompt");
    if (T <= 0) return 0;
    Kv8Cache c = kv8_cache(kc, vc, ksc, vsc, table, tmax, Hkv, D, block, blocks);
    if (qt < 0 || qt > 2) return ns_fail(w + ": rows of type 0 (float32), 1 (half) or 2 (bfloat16)");
    if (ns_kv8_check(w, form, Hkv, D, block, blocks, 1, tmax, c)) return -1;
    if (Hq <= 0 || Hq % Hkv || Hq / Hkv > KV8_HEADS) return ns_fail(w + ": query heads a multiple of the key heads, up to 4096 times");
    if (p0 < 0 || p0 > KV8_TOKENS || T > KV8_TOKENS) return ns_fail(w + ": positions of 0 to 2^30, up to 2^30 rows");
    if (qs < Hq * D) return ns_fail(w + ": rows at least as far apart as they are long");
    if (!g || !q || !vc || !vsc || !out) return ns_fail(w + ": a null buffer");
    const int64_t e = qt == 0 ? 4 : 2;
    if ((uintptr_t) q % 16 || qs * e % 16 || (uintptr_t) out % 16) return ns_fail(w + ": query and output rows 16-byte aligned");
    NS_HIP(hipSetDevice(g->dev));
    NS_OWN_SCRATCH(g);
    const size_t own = ns_own_floats(g);
    win = kv8_window(win);
    // the tokens that the rows see, from a block's first on, widened at the scratch's end; the pass plans with what is in front of them. (From the 17th row
    // on: 32 x 32 / 8 heads behind 4000 28.4 us, as tokens, 16 rows a trip, 37.8; 64 x 16 / 2 of 256 behind 20000 53.5, 118. The wrong side, which the rule does not
    // count: few heads a key head, or very many tokens, 17 x 8 / 8 behind 20000 42.5, 34.6, 32 x 32 / 8 behind 100000 188, 156)
    const int64_t from = win > 0 ? std::max<int64_t>(0, p0 + 1 - win) >> c.shift << c.shift : 0, n = p0 + T - from;
    const size_t wide = (size_t) (Hkv * n * D);                   // floats, both streams of halfs
    if (T > DECODE_ROWS && wide <= own / 4 * 3 && n * D * 2 < (int64_t) 1 << 32) {
        uint16_t* k = reinterpret_cast<uint16_t*>(g->own_scratch + (own - wide) / 64 * 64);
        if (ns_kv8_widen(g, form, c, from, n, k, k + Hkv * n * D)) return -1;
        return ns_attn_prompt_any(g, "ns_kv8_prompt", qt, 0, 0, q, qs, k, k + Hkv * n * D, T, Hq, Hkv, D, n, p0 - from, win, 1, -1, scale, out,
                                  (own - wide) / 64 * 64, true);
    }
    AttendParams p{};
    p.c = c, p.qs = qs, p.S = 1, p.Hq = (int) Hq, p.G = (int) (Hq / Hkv), p.win = win;
    p.sl2 = (scale > 0.0f ? scale : 1.0f / sqrtf((float) D)) * 1.4426950408889634f;
    for (int64_t t = 0; t < T; t += DECODE_ROWS) {
        const int64_t rows = std::min(DECODE_ROWS, T - t);
        p.q = (const uint8_t*) q + t * qs * e, p.out = (uint8_t*) out + t * Hq * D * e, p.T = p.most = (int) rows, p.p0 = p0 + t, p.longest = p0 + t + rows;
        // (runs on as many work-groups as have places for their pieces, where the scratch does not hold them all)
        Deal deal = deal_of(1, rows * p.G, Hkv, D, p.longest);
        if (scratch_of(1, rows, Hq, Hkv, D, p.longest, false, deal).all() > (int64_t) own) {
            const Scratch one = scratch_of(1, rows, Hq, Hkv, D, p.longest, false, {1, 0, 0});
            deal = {std::min(deal.nw, ((int64_t) own - one.units) / (one.part + one.ml + 4)), 0, 0};
            if (deal.nw < 1) return ns_fail(w + ": more rows and heads than the library's scratch holds");
        }
        if (attend(g, w, form, qt, p, Hkv, D, deal, g->own_scratch)) return -1;
    }
    return 0;
    NS_CATCH
}

}  // extern "C"
