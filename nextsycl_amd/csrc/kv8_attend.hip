// kv8_attend.hip: attention of a token, or the few rows of a verify pass, of each of several sequences over a cache of 8-bit values in
// blocks of tokens (gfx950).
//
// Bound: HBM - every visible key and value byte read once for all rows and query heads of its key head; 4 D flops a (row, head,
// token), far under the matrix unit's ridge.
//
// Work split: a work-group of 4 waves takes tokens [s kbs, (s + 1) kbs) of one sequence and key head (and 16 or 32 of its row, head
// pairs, i G + g); wave w the 32-token tiles t % 4 == w, each through two buffers of its own in LDS (the next tile's transfers under
// way while this one is worked on): no barrier in the loop. The waves' (O, m, l) meet in LDS in wave order; of several splits a second
// kernel makes one. A wave holds its split's table entries and scales in two registers a lane and picks them by lane reads.
//
// A tile in the transposed orientation, as in attn_decode.hip: S^T[token][pair] = K Q^T with K's codes as halfs and the block's scale on
// the score; online softmax in base 2, float32; O^T[d][pair] += V^T P^T with V as halfs code x scale - exactly - read by the
// transposing 8-bit LDS read (16 lanes, 8 rows x 16 bytes: lane i gets byte i of every row). Float32 rows enter the first product
// as two halfs, softmax weights the second one as two: 22 bits of each. Rows are brought to exponent 13 first, so that the second half of no value
// that matters is below a half's range, and their exponent rejoins the scores' factor.
#include <algorithm>
#include <cmath>

#include "attn_host.hpp"
#include "kv8_common.hpp"
#include "ns_attn.h"

namespace {

constexpr int WAVES = 4, TILE = 32;
constexpr int MOST_SPLIT = 2048;                  // tokens a split, at most: 128 table entries of 16 tokens, two a lane

struct AttendParams {
    Kv8Cache c;
    const void* q;
    int64_t qs;
    const int32_t *start, *lens;
    int64_t p0;                 // lens null: the one sequence's tokens in front of the call, its T rows
    int T, most, S, Hq, G;
    int64_t longest, win, kbs;
    int ns, nz;                 // splits of the longest sequence; chunks of pairs
    float sl2;                  // scale x log2(e)
    void* out;
    float* part;                // [S][Hkv][most G][ns] x (D + 4): O, m, l, -, -
    float* scores;              // [S][Hkv][most G][pad]: scores in log2 units, or null
    float* stats;               // [S][Hkv][most G][2]: a pair's largest score and its sum, or null
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

// QT: the rows' type; RT row tiles of 16 pairs a wave
template <int D, int RT, int FORM, int QT>
__global__ __launch_bounds__(WAVES * 64, D == 128 ? 2 : 1) void kv8_attend_kernel(const AttendParams p) {
    constexpr bool QS = QT == 0;                                  // rows in two parts
    constexpr int CH = D / 16, KJ = D / 64, DT = D / 16;          // 16-byte chunks a row; chunks a lane reads of a key; tiles of 16 features
    constexpr int TB = TILE * D, NI = TB / 1024;                  // bytes a tile and stream; transfers
    constexpr int STAGE = 4 * TB;                                 // two buffers of keys and values
    constexpr int OROW = D + 4, MERGE = RT * 16 * OROW * 4;
    constexpr int WREG = ((STAGE > MERGE ? STAGE : MERGE) + 1023) / 1024 * 1024;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[WAVES * WREG];
    __shared__ __attribute__((aligned(16))) float ml[RT * 16][2][WAVES];

    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g4 = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    // consecutive work-groups go round the 8 XCDs; the chunks of one (split, key head, sequence) follow each other on one of them
    const int xj = blockIdx.x / 8, u = (xj / p.nz) * 8 + (int) (blockIdx.x % 8), z = xj % p.nz;
    const int Hkv = p.c.Hkv;
    if (u >= p.ns * Hkv * p.S) return;
    const int split = u % p.ns, hk = u / p.ns % Hkv, s = u / (p.ns * Hkv);
    const Kv8Seq q = seq_of(p, s);
    const int pairs = q.n * p.G, pair0 = z * RT * 16;
    if (q.n <= 0 || pair0 >= pairs) return;
    int64_t lo, hi;
    span_of(p, q, lo, hi);
    const int64_t j0 = split * p.kbs, jb = std::max(j0, lo), je = std::min(j0 + p.kbs, hi);
    if (jb >= je && p.ns > 1) return;                             // (the merge passes this split over, by the same rule)

    // ---- the split's blocks and scales: entry e0 + lane, e0 + 64 + lane
    const int64_t e0 = j0 >> p.c.shift;
    int blk[2];
    float sk[2], sv[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int64_t e = e0 + i * 64 + lane;
        blk[i] = (e << p.c.shift) < je ? kv8_block(p.c, p.c.table, s, e) : -1;
    }
    // ---- this lane's rows: position, first and last token seen, operands
    s8v qh[RT][2 * KJ], ql[QS ? RT : 1][2 * KJ];
    float qm[RT];                                                 // what a score takes besides the block's scale
    int64_t rlo[RT], rhi[RT];                                     // tokens seen: rlo .. rhi
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int pair = pair0 + rt * 16 + n;
        const bool live = pair < pairs;
        const int i = live ? pair / p.G : 0, g = live ? pair - i * p.G : 0;
        const int64_t pos = (int64_t) q.len + i;
        rlo[rt] = live ? (p.win > 0 ? std::max<int64_t>(0, pos + 1 - p.win) : 0) : 1;
        rhi[rt] = live ? std::min(pos, hi - 1) : 0;
        const int64_t at = (int64_t) (q.first + i) * p.qs + (int64_t) (hk * p.G + g) * D;
        float x[2 * KJ][8], most = 0.0f;
#pragma unroll
        for (int j = 0; j < 2 * KJ; ++j) {
            const int64_t d = at + 64 * (j / 2) + 16 * g4 + 8 * (j % 2);
            if constexpr (QT == 0) {
                float a[4], b[4];
                load_row<0, 4>(p.q, d, a), load_row<0, 4>(p.q, d + 4, b);
#pragma unroll
                for (int k = 0; k < 4; ++k) x[j][k] = a[k], x[j][4 + k] = b[k];
            } else load_row<QT, 8>(p.q, d, x[j]);
#pragma unroll
            for (int k = 0; k < 8; ++k) most = fmaxf(most, fabsf(x[j][k]));
        }
        most = rows_max(most);
        const int e = std::min(std::max((int) (__builtin_bit_cast(uint32_t, most) >> 23) - 127 - 13, -110), 110);
        const float up = kv8_pow2(-e);
        qm[rt] = p.sl2 * kv8_pow2(e);
#pragma unroll
        for (int j = 0; j < 2 * KJ; ++j)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float v = x[j][k] * up;
                qh[rt][j][k] = to16<false>(v);
                if constexpr (QS) ql[rt][j][k] = to16<false>(v - f16_to_f32((uint16_t) qh[rt][j][k]));
            }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int64_t at = (int64_t) std::max(blk[i], 0) * Hkv + hk;
        sk[i] = p.c.ksc[at], sv[i] = p.c.vsc[at];
        if (blk[i] < 0) sk[i] = 0.0f, sv[i] = 0.0f;
    }
    auto pick = [&](auto (&v)[2], int e) __attribute__((always_inline)) {
        const int x = __builtin_amdgcn_readlane(__builtin_bit_cast(int, v[0]), e & 63), y = __builtin_amdgcn_readlane(__builtin_bit_cast(int, v[1]), e & 63);
        return e < 64 ? x : y;
    };
    auto picked = [&](float (&v)[2], int e) __attribute__((always_inline)) { return __builtin_bit_cast(float, pick(v, e)); };

    // ---- transfers: chunk position cp of token kk holds the row's chunk cp ^ kk % CH (keys: 16 tokens' same chunk meet no bank
    // conflict), cp ^ (4 (kk / 16) + kk % 4) (values: the 8 rows of a group's transposing read). A transfer is 1024 / D rows; 16 tokens lie in one block
    uint8_t* stage = lds + w * WREG;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t) (uintptr_t) (__attribute__((address_space(3))) uint8_t*) stage);
    uint32_t koff[NI], voff[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int r = lane / CH, kk = i * (1024 / D) + r, cp = lane % CH;
        koff[i] = (uint32_t) (r * D + (cp ^ (kk % CH)) * 16);
        voff[i] = (uint32_t) (r * D + (cp ^ (4 * (kk / 16) + kk % 4)) * 16);
    }
    const int nt = (int) ((je - j0 + TILE - 1) / TILE), t0 = (int) ((jb - j0) / TILE);
    auto fetch = [&](int t, int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = t * TILE + h * 16, b = std::max(pick(blk, at >> p.c.shift), 0);
            const int64_t off = (kv8_rows(p.c, b, hk) + (at & (p.c.block - 1))) * D;
            lds_fetch_run<true, NI / 2>(p.c.kc + off, koff + h * (NI / 2), lds0 + buf * 2 * TB + h * (TB / 2));
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = t * TILE + h * 16, b = std::max(pick(blk, at >> p.c.shift), 0);
            const int64_t off = (kv8_rows(p.c, b, hk) + (at & (p.c.block - 1))) * D;
            lds_fetch_run<true, NI / 2>(p.c.vc + off, voff + h * (NI / 2), lds0 + buf * 2 * TB + TB + h * (TB / 2));
        }
    };

    float m[RT], l[RT];
    f4v o[RT][DT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -INFINITY, l[rt] = 0.0f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[rt][dt] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
    }
    // tiles that need no mask: every token seen by every row there is
    const int64_t full_hi = std::min<int64_t>((int64_t) q.len + pair0 / p.G + 1, hi);
    const int64_t full_lo = p.win > 0 ? std::max<int64_t>(0, (int64_t) q.len + q.n - p.win) : 0;

    int t = t0 + ((w - t0) & (WAVES - 1)), buf = 0;
    if (t < nt) fetch(t, 0);
    if (t + WAVES < nt) fetch(t + WAVES, 1);
    // (the scales are there before the loop: in it the compiler would wait for them, and the tiles behind them, every turn)
    asm volatile("" : "+v"(sk[0]), "+v"(sk[1]), "+v"(sv[0]), "+v"(sv[1]));
    for (; t < nt; t += WAVES, buf ^= 1) {
        if (t + WAVES < nt) {
            if constexpr (NI == 4) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
            else asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
        } else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const uint8_t* kl = stage + buf * 2 * TB;
        uint8_t* vl = stage + buf * 2 * TB + TB;
        const int64_t key0 = j0 + t * TILE;
        const int ent0 = (t * TILE) >> p.c.shift, ent1 = (t * TILE + 16) >> p.c.shift;
        const bool bad0 = pick(blk, ent0) < 0, bad1 = pick(blk, ent1) < 0;
        const bool edge = key0 + TILE > full_hi || key0 < full_lo || bad0 || bad1;

        f4v sc[RT][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int j = 0; j < KJ; ++j) {
                const int kk = h * 16 + n, c = 4 * j + g4;
                const uint4 r = *reinterpret_cast<const uint4*>(kl + kk * D + ((c ^ (kk % CH)) << 4));
                const s8v a = kv8_halfs8<FORM>(r.x, r.y), b = kv8_halfs8<FORM>(r.z, r.w);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    f4v x = j == 0 ? f4v{0.0f, 0.0f, 0.0f, 0.0f} : sc[rt][h];
                    x = mfma16<false>(a, qh[rt][2 * j], x);
                    x = mfma16<false>(b, qh[rt][2 * j + 1], x);
                    if constexpr (QS) {
                        x = mfma16<false>(a, ql[rt][2 * j], x);
                        x = mfma16<false>(b, ql[rt][2 * j + 1], x);
                    }
                    sc[rt][h] = x;
                }
            }
        }
        const float k0 = picked(sk, ent0), k1 = picked(sk, ent1);
        s8v ph[RT], pl[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float x[8];
            const float f0 = qm[rt] * k0, f1 = qm[rt] * k1;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = sc[rt][0][i] * f0, x[4 + i] = sc[rt][1][i] * f1;
            if (edge) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int64_t key = key0 + (i / 4) * 16 + 4 * g4 + i % 4;
                    if (i < 4 ? bad0 : bad1) x[i] = 0.0f;         // (no block: a key of zeros)
                    x[i] = key >= rlo[rt] && key <= rhi[rt] ? x[i] : -INFINITY;
                }
            }
            if (p.scores) {
                const int pair = pair0 + rt * 16 + n;
                if (pair < pairs) {
                    float* at = p.scores + (((int64_t) s * Hkv + hk) * p.most * p.G + pair) * p.pad + key0 + 4 * g4;
                    *reinterpret_cast<f4v*>(at) = f4v{x[0], x[1], x[2], x[3]};
                    *reinterpret_cast<f4v*>(at + 16) = f4v{x[4], x[5], x[6], x[7]};
                }
            }
            float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
            top = rows_max(top);
            if (__builtin_amdgcn_ballot_w64(top > m[rt])) {       // some row's largest score moves
                const float m1 = fmaxf(m[rt], top), c = m1 == -INFINITY ? 1.0f : fast_exp2(m[rt] - m1);
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
        // which of the 8 tokens of a lane's operand there are (bytes of others may hold anything)
        uint32_t live0 = ~0u, live1 = ~0u;
        if (edge) {
            live0 = live1 = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t a = key0 + 4 * g4 + i, b = a + 16;
                live0 |= !bad0 && a >= lo && a < hi ? 0xFFu << (8 * i) : 0u;
                live1 |= !bad1 && b >= lo && b < hi ? 0xFFu << (8 * i) : 0u;
            }
        }
        {
            // lane n of group g4 addresses token row n / 2 of the group's 8, half n % 2 of the chunk
            const int r = n >> 1, kk = (r >> 2) * 16 + 4 * g4 + (r & 3), x = 4 * (kk / 16) + kk % 4;
            uint8_t* at = vl + kk * D + (n & 1) * 8;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                typedef int v2i __attribute__((ext_vector_type(2)));
                const v2i raw = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) v2i*) (at + ((dt ^ x) << 4)));
                const s8v a = kv8_halfs8<FORM>((uint32_t) raw[0] & live0, (uint32_t) raw[1] & live1, v0, v1);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    o[rt][dt] = mfma16<false>(a, ph[rt], o[rt][dt]);
                    o[rt][dt] = mfma16<false>(a, pl[rt], o[rt][dt]);
                }
            }
        }
        // this buffer's reads have returned: the tile after the next may have it
        if (t + 2 * WAVES < nt) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            fetch(t + 2 * WAVES, buf);
        }
    }

    // ---- the waves' sums, each parked in the wave's own region
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    float* own = reinterpret_cast<float*>(stage);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const float sum = rows_sum(l[rt]);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f4v*>(own + (rt * 16 + n) * OROW + dt * 16 + 4 * g4) = o[rt][dt];
        if (g4 == 0) ml[rt * 16 + n][0][w] = m[rt], ml[rt * 16 + n][1][w] = sum;
    }
    __syncthreads();
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
        const int64_t place = ((int64_t) s * Hkv + hk) * p.most * p.G + pair;
        if (p.ns == 1) {
            const float inv = all == 0.0f ? 0.0f : 1.0f / all;
            const int i2 = pair / p.G, g = pair - i2 * p.G;
            const float v[4] = {sum[0] * inv, sum[1] * inv, sum[2] * inv, sum[3] * inv};
            const int64_t at = ((int64_t) (q.first + i2) * p.Hq + hk * p.G + g) * D + d;
#pragma unroll
            for (int k = 0; k < 4; ++k) store_o<QT>(p.out, at + k, v[k]);
            if (p.stats && d == 0) p.stats[2 * place] = ref, p.stats[2 * place + 1] = inv;
        } else {
            float* to = p.part + (place * p.ns + split) * (D + 4);
            *reinterpret_cast<f4v*>(to + d) = sum;
            if (d == 0) to[D] = top, to[D + 1] = all;
        }
    }
}

// out = sum over the splits of O 2^(m - M) / sum of l 2^(m - M): a work-group a (sequence, key head, pair), its lanes a split each for the
// weights, then D / 4 threads x 256 / (D / 4) splits at a time in a fixed shape
template <int D, int QT>
__global__ __launch_bounds__(256) void kv8_merge_kernel(const AttendParams p) {
    constexpr int L = D / 4, SG = 256 / L;
    __shared__ __attribute__((aligned(16))) float sums[SG][D];
    __shared__ float wsum[SG];
    const int tid = threadIdx.x, lane = tid & 63;
    const int64_t place = blockIdx.x;
    const int pair = (int) (place % (p.most * p.G)), hk = (int) (place / (p.most * p.G) % p.c.Hkv), s = (int) (place / ((int64_t) p.most * p.G * p.c.Hkv));
    const Kv8Seq q = seq_of(p, s);
    if (pair >= q.n * p.G) return;
    int64_t lo, hi;
    span_of(p, q, lo, hi);
    const int first = (int) (lo / p.kbs), end = (int) ((hi + p.kbs - 1) / p.kbs);
    const float* part = p.part + place * p.ns * (D + 4);
    float top = -INFINITY;
    for (int k = first + lane; k < end; k += 64) top = fmaxf(top, part[(int64_t) k * (D + 4) + D]);
    top = wave_max(top);
    const float ref = top == -INFINITY ? 0.0f : top;
    const int sg = tid / L, d = tid % L * 4;
    f4v sum = {0.0f, 0.0f, 0.0f, 0.0f};
    float all = 0.0f;
    for (int k = first + sg; k < end; k += SG) {
        const float* at = part + (int64_t) k * (D + 4);
        const float c = fast_exp2(at[D] - ref);
        all += at[D + 1] * c;
        sum += *reinterpret_cast<const f4v*>(at + d) * c;
    }
    *reinterpret_cast<f4v*>(&sums[sg][d]) = sum;
    if (d == 0) wsum[sg] = all;
    __syncthreads();
    if (tid >= L) return;
    sum = f4v{0.0f, 0.0f, 0.0f, 0.0f}, all = 0.0f;
#pragma unroll
    for (int k = 0; k < SG; ++k) sum += *reinterpret_cast<const f4v*>(&sums[k][d]), all += wsum[k];
    const float inv = all == 0.0f ? 0.0f : 1.0f / all;
    const int i = pair / p.G, g = pair - i * p.G;
    const int64_t at = ((int64_t) (q.first + i) * p.Hq + hk * p.G + g) * D + d;
#pragma unroll
    for (int k = 0; k < 4; ++k) store_o<QT>(p.out, at + k, sum[k] * inv);
    if (p.stats && tid == 0) p.stats[2 * place] = ref, p.stats[2 * place + 1] = inv;
}

// acc1 = acc0 + the weights of the pairs: a thread a token
__global__ __launch_bounds__(256) void kv8_given_kernel(const AttendParams p) {
    const int hk = blockIdx.y, s = blockIdx.z;
    const Kv8Seq q = seq_of(p, s);
    const int64_t t = (int64_t) blockIdx.x * 256 + threadIdx.x;
    int64_t lo, hi;
    span_of(p, q, lo, hi);
    if (q.n <= 0 || t >= (int64_t) q.len + q.n) return;
    const int b = kv8_block(p.c, p.c.table, s, t >> p.c.shift);
    if (b < 0) return;
    const int64_t at = kv8_rows(p.c, b, hk) + (t & (p.c.block - 1));
    float sum = 0.0f;
    if (t < hi) {
        const int64_t place = ((int64_t) s * p.c.Hkv + hk) * p.most * p.G;
        for (int pair = 0; pair < q.n * p.G; ++pair) {
            // (only what the pair has seen was written)
            const int64_t pos = (int64_t) q.len + pair / p.G;
            if (t > pos || (p.win > 0 && t + p.win <= pos)) continue;
            sum += fast_exp2(p.scores[(place + pair) * p.pad + t] - p.stats[2 * (place + pair)]) * p.stats[2 * (place + pair) + 1];
        }
    }
    p.acc1[at] = (p.acc0 && t < q.len ? p.acc0[at] : 0.0f) + sum;
}

template <int D, int QT>
void launch_attend(ns_gpu* g, int form, const AttendParams& p, int RT, unsigned grid) {
    if (form == 0) RT == 1 ? kv8_attend_kernel<D, 1, 0, QT><<<grid, WAVES * 64, 0, g->q>>>(p) : kv8_attend_kernel<D, 2, 0, QT><<<grid, WAVES * 64, 0, g->q>>>(p);
    else RT == 1 ? kv8_attend_kernel<D, 1, 1, QT><<<grid, WAVES * 64, 0, g->q>>>(p) : kv8_attend_kernel<D, 2, 1, QT><<<grid, WAVES * 64, 0, g->q>>>(p);
}
template <int D, int QT>
void launch_merge(ns_gpu* g, const AttendParams& p, int64_t rows) { kv8_merge_kernel<D, QT><<<(unsigned) rows, 256, 0, g->q>>>(p); }

// tokens a split and how many splits of `longest` there are. Work-groups enough for two a CU, splits of 128 to 2048 tokens
struct Splits {
    int64_t kbs, ns;
};
Splits splits_of(int64_t S, int64_t nz, int64_t Hkv, int64_t longest) {
    const int64_t want = std::max<int64_t>(1, 512 / std::max<int64_t>(1, S * Hkv * nz));
    const int64_t kbs = std::min<int64_t>(MOST_SPLIT, std::max<int64_t>(128, ((longest + want - 1) / want + 127) / 128 * 128));
    return {kbs, (longest + kbs - 1) / kbs};
}
int64_t chunks_of(int64_t pairs) { return pairs <= 16 ? 1 : (pairs + 31) / 32; }

struct Scratch {
    int64_t part, scores, stats, pad;
    int64_t all() const { return part + scores + stats; }
};
Scratch scratch_of(int64_t S, int64_t most, int64_t Hq, int64_t Hkv, int64_t D, int64_t longest, bool acc) {
    const Splits sp = splits_of(S, chunks_of(most * (Hq / Hkv)), Hkv, longest);
    const int64_t rows = S * most * Hq;
    Scratch x{};
    x.pad = (longest + 31) / 32 * 32;
    x.part = sp.ns > 1 ? rows * sp.ns * (D + 4) : 0;
    x.scores = acc ? rows * x.pad : 0;
    x.stats = acc ? rows * 2 : 0;
    return x;
}
bool sizes_fit(int64_t S, int64_t most, int64_t Hq, int64_t Hkv, int64_t D, int64_t longest) {
    return S > 0 && S <= 65535 && most > 0 && most <= DECODE_ROWS && Hkv > 0 && Hkv <= 32767 && Hq > 0 && Hq <= 1 << 20 && Hq % Hkv == 0 && (D == 128 || D == 256) && longest > 0 &&
           longest <= 2 * (int64_t) KV8_TOKENS;
}

// a checked call, its scratch at hand
int attend(ns_gpu* g, const std::string& w, int form, int qt, AttendParams p, int64_t Hkv, int64_t D, float* scratch) {
    const int64_t nz = chunks_of((int64_t) p.most * p.G);
    const Splits sp = splits_of(p.S, nz, Hkv, p.longest);
    const Scratch x = scratch_of(p.S, p.most, p.Hq, Hkv, D, p.longest, p.acc1 != nullptr);
    const int64_t units = sp.ns * Hkv * p.S, rows = (int64_t) p.S * p.most * p.Hq;
    if ((units + 7) / 8 * 8 * nz > (int64_t) 1 << 30 || !ns_grid_fits((units + 7) / 8 * 8 * nz, 256) || !ns_grid_fits(rows, 256))
        return ns_fail(w + ": more work-groups than a launch takes");
    p.kbs = sp.kbs, p.ns = (int) sp.ns, p.nz = (int) nz, p.pad = x.pad;
    p.part = scratch;
    p.scores = p.acc1 ? scratch + x.part : nullptr;
    p.stats = p.acc1 ? scratch + x.part + x.scores : nullptr;
    const unsigned grid = (unsigned) ((units + 7) / 8 * 8 * nz);
    const int RT = p.most * p.G <= 16 ? 1 : 2;
    if (D == 128) qt == 0 ? launch_attend<128, 0>(g, form, p, RT, grid) : qt == 1 ? launch_attend<128, 1>(g, form, p, RT, grid) : launch_attend<128, 2>(g, form, p, RT, grid);
    else qt == 0 ? launch_attend<256, 0>(g, form, p, RT, grid) : qt == 1 ? launch_attend<256, 1>(g, form, p, RT, grid) : launch_attend<256, 2>(g, form, p, RT, grid);
    NS_LAUNCHED("kv8_attend");
    if (p.ns > 1) {
        if (D == 128) qt == 0 ? launch_merge<128, 0>(g, p, rows) : qt == 1 ? launch_merge<128, 1>(g, p, rows) : launch_merge<128, 2>(g, p, rows);
        else qt == 0 ? launch_merge<256, 0>(g, p, rows) : qt == 1 ? launch_merge<256, 1>(g, p, rows) : launch_merge<256, 2>(g, p, rows);
        NS_LAUNCHED("kv8_merge");
    }
    if (p.acc1) {
        kv8_given_kernel<<<dim3((unsigned) ((p.longest + 255) / 256), (unsigned) Hkv, (unsigned) p.S), 256, 0, g->q>>>(p);
        NS_LAUNCHED("kv8_given");
    }
    return 0;
}

}  // namespace

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
    if (Hq <= 0 || Hq % Hkv || Hq > 1 << 20) return ns_fail(w + ": query heads a multiple of the key heads");
    if (most > DECODE_ROWS) return ns_fail(w + ": 1 to 16 rows a sequence");
    if (T > KV8_TOKENS) return ns_fail(w + ": up to 2^30 rows");
    if (longest <= 0 || longest > 2 * (int64_t) KV8_TOKENS) return ns_fail(w + ": contexts of 1 to 2^31 tokens");
    if (qs < Hq * D) return ns_fail(w + ": rows at least as far apart as they are long");
    p.S = (int) S, p.most = (int) most, p.Hq = (int) Hq, p.G = (int) (Hq / Hkv), p.longest = longest, p.T = (int) T;
    const int64_t need = scratch_of(S, p.most, Hq, Hkv, D, longest, acc1 != nullptr).all();
    if (!g || !q || !lens || !vc || !vsc || !out || (need && !scratch)) return ns_fail(w + ": a null buffer");
    if (need && (uintptr_t) scratch % 16) return ns_fail(w + ": scratch 16-byte aligned");
    p.q = q, p.qs = qs, p.start = start, p.lens = lens, p.win = win, p.out = out, p.acc0 = acc0, p.acc1 = acc1;
    p.sl2 = (scale > 0.0f ? scale : 1.0f / sqrtf((float) D)) * 1.4426950408889634f;
    NS_HIP(hipSetDevice(g->dev));
    return attend(g, w, form, qt, p, Hkv, D, scratch);
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
    if (Hq <= 0 || Hq % Hkv || Hq > 1 << 20) return ns_fail(w + ": query heads a multiple of the key heads");
    if (p0 < 0 || p0 > KV8_TOKENS || T > KV8_TOKENS) return ns_fail(w + ": positions of 0 to 2^30, up to 2^30 rows");
    if (qs < Hq * D) return ns_fail(w + ": rows at least as far apart as they are long");
    if (!g || !q || !vc || !vsc || !out) return ns_fail(w + ": a null buffer");
    const int64_t e = qt == 0 ? 4 : 2;
    if ((uintptr_t) q % 16 || qs * e % 16 || (uintptr_t) out % 16) return ns_fail(w + ": query and output rows 16-byte aligned");
    NS_HIP(hipSetDevice(g->dev));
    NS_OWN_SCRATCH(g);
    const size_t own = ns_own_floats(g);
    // the tokens that the rows see, from a block's first on, widened at the scratch's end; the pass plans with what is in front of them
    const int64_t from = win > 0 ? std::max<int64_t>(0, p0 + 1 - win) >> c.shift << c.shift : 0, n = p0 + T - from;
    const size_t wide = (size_t) (Hkv * n * D);                   // floats, both streams of halfs
    if (T > DECODE_ROWS && wide <= own / 4 * 3 && n * D * 2 < (int64_t) 1 << 32) {
        uint16_t* k = reinterpret_cast<uint16_t*>(g->own_scratch + (own - wide) / 64 * 64);
        if (ns_kv8_widen(g, form, c, 0, (int) Hkv, from, n, k, k + Hkv * n * D)) return -1;
        return ns_attn_prompt_any(g, "ns_kv8_prompt", qt, 0, 0, q, qs, k, k + Hkv * n * D, T, Hq, Hkv, D, n, p0 - from, win > 0 ? win : 0, 1, -1, scale, out,
                                  (own - wide) / 64 * 64);
    }
    AttendParams p{};
    p.c = c, p.qs = qs, p.S = 1, p.Hq = (int) Hq, p.G = (int) (Hq / Hkv), p.win = win;
    p.sl2 = (scale > 0.0f ? scale : 1.0f / sqrtf((float) D)) * 1.4426950408889634f;
    for (int64_t t = 0; t < T; t += DECODE_ROWS) {
        const int64_t rows = std::min(DECODE_ROWS, T - t);
        p.q = (const uint8_t*) q + t * qs * e, p.out = (uint8_t*) out + t * Hq * D * e, p.T = p.most = (int) rows, p.p0 = p0 + t, p.longest = p0 + t + rows;
        if ((size_t) scratch_of(1, rows, Hq, Hkv, D, p.longest, false).all() > own) return ns_fail(w + ": more rows, heads and tokens than the library's scratch holds");
        if (attend(g, w, form, qt, p, Hkv, D, g->own_scratch)) return -1;
    }
    return 0;
    NS_CATCH
}

}  // extern "C"
