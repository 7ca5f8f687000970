// kv8_evict.hip: a cache of 8-bit values in blocks of tokens shortened to the tokens of the largest accumulated softmax weights (gfx950).
//
// Which tokens, a (sequence, key head) a work-group: the weights' bits, as whole numbers, are searched from the top 11 bits down for the value at the
// last kept place (three histograms in LDS; zeros, of which there can be many, are not counted but left over). Up to 32768 weights are in registers, a
// wave's tokens in a row, so a kept token's place is the waves' counts in front of it, its wave's own in front and its lane's place in a ballot: tokens keep their
// order, and of equal weights the earliest stay. Move: a work-group a block to be written, key head and
// stream - its rows gathered, re-rounded to the largest of their scales. In place the blocks go through the library's scratch, since a block is read by
// those in front of it; blocks whose tokens stay where they are are left out. Bound: the kept rows' bytes, read and written; the search by one CU's instructions.
// (32768 tokens of 8 heads of 128 to 8192: 26.6 us, the search 17 - 42 vector instructions a weight -, the move 9.6, 3.5 TB/s. 12 sequences of 59 to 3001 tokens x
// 4 heads of 256 to 517: 14.7, 8.2 + 6.6. With thread-strided tokens and counts in LDS the search took 20; with a list of the first bin's weights for the
// second and third sweep 26)
#include <algorithm>

#include "attn_host.hpp"
#include "kv8_common.hpp"

namespace {

constexpr int SEL = 1024;                         // threads of the search
constexpr uint32_t NONE = ~0u;                    // (no weight's bits, no row)

struct EvictParams {
    Kv8Cache c;
    const int32_t *lens, *to;
    int32_t* lens1;
    int64_t s0, longest, keep, first, last;
    float* acc;
    int64_t cap;                // places of a list: min(keep, longest)
    int nh;                     // = Hkv
    int32_t* idx;               // [group's S][Hkv][cap]: kept tokens, in order
    int2* info;                 // [group's S]: tokens to move, the new length
    uint8_t* stage;             // in place: [group's S][blocks of cap][Hkv][2][block x D], then scales [..][2], then acc [..][block]
    float *stage_scale, *stage_acc;
    int nb;                     // blocks of cap tokens
};

// the sum over this lane and those in front of it: each row of 16, then the rows' last lanes over the rows behind them
__device__ __forceinline__ int lanes_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);        // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);       // row_bcast 15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);       // row_bcast 31 into rows 2 and 3
    return v;
}
// a work-group's exclusive prefix sum of v, and the total (a call's last read of `sums` comes before the next one's barrier)
__device__ __forceinline__ int scan1024(int v, int* sums, int& total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, x = lanes_scan(v);
    if (lane == 63) sums[w] = x;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < SEL / 64; ++i) {
        const int y = sums[i];
        if (i < w) before += y;
        total += y;
    }
    return before + x - v;
}

// this lane's place among the lanes of m
__device__ __forceinline__ int lane_place(uint64_t m) { return __builtin_amdgcn_mbcnt_hi((uint32_t) (m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t) m, 0)); }

// (what follows from v is made again where it is used: the compiler would keep all of it in registers from its first use on)
__device__ __forceinline__ int again(int v) {
    asm volatile("" : "+v"(v));
    return v;
}
__device__ __forceinline__ uint32_t again_s(uint32_t v) {
    v = __builtin_amdgcn_readfirstlane(v);
    asm volatile("" : "+s"(v));
    return v;
}

// R weights a thread, a wave's in a row (token 64 R w + 64 i + lane); longer contexts in pieces of 1024 R, read again for each step. (One CU has the whole of a
// key head's search: what counts is the instructions a weight)
template <int R>
__global__ __launch_bounds__(SEL) void kv8_select_kernel(const EvictParams p) {
    constexpr int PIECE = SEL * R;
    __shared__ int hist[2048];
    __shared__ int entries[PIECE / 16];                           // where a piece's blocks begin in acc, in 16 tokens (none: -1; behind the last: 0)
    __shared__ int sums[4][SEL / 64];                             // (of scans in turn)
    __shared__ int found[3];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), hk = blockIdx.x, gs = blockIdx.y;
    const int64_t s = p.s0 + gs;
    const int n = p.lens[s];
    const bool over = n < 0 || n > p.longest, whole = n <= p.keep;
    const int rows = over || (whole && !p.to) ? 0 : whole ? n : (int) p.keep;
    if (hk == 0 && tid == 0) p.info[gs] = int2{rows, over || whole ? n : (int) p.keep};
    if (rows == 0) return;
    int32_t* idx = p.idx + ((int64_t) gs * p.nh + hk) * p.cap;
    const int cap = (int) p.cap;
    if (whole) {
        for (int t = tid; t < n; t += SEL) idx[t] = t;
        return;
    }
    // the weights of the tokens between those that stay anyhow, as whole numbers in the same order
    const int lo = (int) p.first, hi = n - (int) p.last, pieces = (n + PIECE - 1) / PIECE;
    const int mine = w * 64 * R, mask = p.c.block - 1;
    uint32_t key[R];
    auto load = [&](int piece) __attribute__((always_inline)) {
        const int t0 = piece * PIECE, m = std::min(n - t0, PIECE), count = (m + p.c.block - 1) >> p.c.shift;
        for (int i = tid; i < PIECE >> p.c.shift; i += SEL) {
            const int b = i < count ? kv8_block(p.c, p.c.table, s, (t0 >> p.c.shift) + i) : -1;
            entries[i] = b >= 0 ? (int) (kv8_rows(p.c, b, hk) >> 4) : i < count ? -1 : 0;
        }
        __syncthreads();
        const int g0 = t0 + mine, lane0 = again(lane), in = lane0 & mask;
        float a[R];
        int none = 0;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int e = entries[(lane0 >> p.c.shift) + ((mine + i * 64) >> p.c.shift)];   // (64 tokens from a multiple of 64 on)
            none |= e;
            a[i] = p.acc[(uint64_t) (((uint32_t) std::max(e, 0) << 4) + (uint32_t) ((i * 64 & mask) + in))];
        }
        // (not a number, and below 0: 0)
#pragma unroll
        for (int i = 0; i < R; ++i) key[i] = __builtin_bit_cast(uint32_t, a[i]) > 0x7F800000u ? 0 : __builtin_bit_cast(uint32_t, a[i]);
        if (__builtin_amdgcn_ballot_w64(none < 0)) {
            const int lane1 = again(lane);
#pragma unroll
            for (int i = 0; i < R; ++i)
                if (entries[(lane1 >> p.c.shift) + ((mine + i * 64) >> p.c.shift)] < 0) key[i] = 0;
        }
        if (g0 < lo || g0 + 64 * R > hi)
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const int t = g0 + i * 64 + lane0;
                if ((uint32_t) (t - lo) >= (uint32_t) (hi - lo)) key[i] = t < n ? NONE : 0;
                __builtin_amdgcn_sched_barrier(0);                // (one after the other: else 64 masks at once)
            }
    };
    for (int i = tid; i < 2048; i += SEL) hist[i] = 0;
    load(0);
    // the value at place `need` from the top: 11, 10, 10 bits. `at`: what is known of it
    int need = (int) (p.keep - p.first - p.last);
    uint32_t at = need > 0 ? 0 : NONE;                            // (NONE: none of them)
    for (int pass = 0; pass < 3 && at != NONE; ++pass) {
        const int shift = pass == 0 ? 20 : pass == 1 ? 10 : 0, bins = pass == 0 ? 2048 : 1024;
        for (int piece = 0; piece < pieces; ++piece) {
            if (pieces > 1) {
                __syncthreads();                                  // (the entries are read)
                load(piece);
            }
            // (weights from `from` on, `width` of them: in the first pass all but 0)
            const uint32_t from = pass == 0 ? 1 : at, width = pass == 0 ? 0x7FFFFFFFu : 1u << (shift + 10);
#pragma unroll
            for (int i = 0; i < R; ++i)
                if (key[i] - from < width) atomicAdd(&hist[key[i] >> shift & (bins - 1)], 1);
        }
        __syncthreads();
        // bins from the largest down, bins / 1024 a thread; they are cleared for the next pass
        const int per = bins / SEL, top = bins - 1 - tid * per;
        const int h0 = hist[top], h1 = per > 1 ? hist[top - 1] : 0;
        hist[top] = 0;
        if (per > 1) hist[top - 1] = 0;
        int all;
        const int before = scan1024(h0 + h1, sums[pass & 1], all);
        if (pass == 0 && all < need) {                            // (all that are above 0, and the first zeros)
            need -= all;
            break;
        }
        if (before < need && before + h0 + h1 >= need) {
            const bool second = before + h0 < need;
            found[0] = top - second, found[1] = need - before - (second ? h0 : 0), found[2] = second ? h1 : h0;
        }
        __syncthreads();
        at |= (uint32_t) found[0] << shift, need = found[1];
        if (need == found[2] && at > 0) {                         // (the whole bin: all that are no less than its least value)
            --at, need = 0;
            break;
        }
    }
    // `need` of the tokens equal to `at`, the earliest, and all above it
    int same0 = 0, kept0 = 0;                                     // in the pieces in front
    for (int piece = 0; piece < pieces; ++piece) {
        if (pieces > 1) {
            __syncthreads();
            load(piece);
        }
        // how many of a mask the waves in front of this one have; all of them
        auto before = [&](auto mask, int* sums, int& all) __attribute__((always_inline)) {
            int c = 0;
#pragma unroll
            for (int i = 0; i < R; ++i) c += __builtin_popcountll(mask(i));
            if (lane == 0) sums[w] = c;
            __syncthreads();
            int x = 0;
            all = 0;
#pragma unroll
            for (int i = 0; i < SEL / 64; ++i) {
                const int y = sums[i];
                if (i < w) x += y;
                all += y;
            }
            return __builtin_amdgcn_readfirstlane(x);
        };
        if (need > 0) {
            // the equal ones that stay become larger than `at`, the others smaller
            uint32_t equal = at;
            auto mask = [&](int i) { return __builtin_amdgcn_ballot_w64(key[i] == equal); };
            int same, first = same0 + before(mask, sums[2], same);
            equal = again_s(equal);
#pragma unroll
            for (int i = 0; i < R; ++i)
                if (const uint64_t m = mask(i); m) {
                    if (key[i] == equal) key[i] = first + lane_place(m) < need ? at + 1 : 0;
                    first += __builtin_popcountll(m);
                }
            same0 += same;
        }
        // (the first and the last tokens are NONE, above all; those behind the last one 0)
        uint32_t least = at == NONE ? NONE : at + 1;
        auto mask = [&](int i) { return __builtin_amdgcn_ballot_w64(key[i] >= least); };
        int kept, place = kept0 + before(mask, sums[3], kept);
        least = again_s(least);
        const int t0 = piece * PIECE + mine + lane;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const uint64_t m = mask(i);
            if (key[i] >= least)
                if (const int to = place + lane_place(m); to < cap) *reinterpret_cast<int32_t*>(reinterpret_cast<uint8_t*>(idx) + (uint32_t) to * 4u) = t0 + i * 64;
            place += __builtin_popcountll(m);
            __builtin_amdgcn_sched_barrier(0);
        }
        kept0 += kept;
        if (pieces > 1) __syncthreads();
    }
}

// one block to be written: key head and stream blockIdx.y, group's sequence blockIdx.z; a thread 16 bytes of NR rows
template <int FORM, int NR>
__global__ __launch_bounds__(256) void kv8_move_kernel(const EvictParams p) {
    __shared__ uint32_t src[128];                                 // a row's place in the pool (NONE: none)
    __shared__ float scale[128];
    __shared__ int differ[2];
    const int tid = threadIdx.x, j = blockIdx.x, hk = blockIdx.y >> 1, val = blockIdx.y & 1, gs = blockIdx.z, B = p.c.block;
    const int64_t s = p.s0 + gs;
    const int2 info = p.info[gs];
    const int dst = kv8_block(p.c, p.to ? p.to : p.c.table, s, j);
    const int t = tid < B && j * B + tid < p.cap ? p.idx[((int64_t) gs * p.nh + hk) * p.cap + j * B + tid] : 0;
    if (j == 0 && blockIdx.y == 0 && tid == 0) p.lens1[s] = info.y;
    const int rows = std::min(info.x - j * B, B);
    if (rows <= 0 || dst < 0) return;
    const uint32_t to0 = (uint32_t) kv8_rows(p.c, dst, hk);
    uint32_t mine = NONE;
    if (tid < 128) {
        if (tid < rows)
            if (const int b = kv8_block(p.c, p.c.table, s, t >> p.c.shift); b >= 0) mine = (uint32_t) kv8_rows(p.c, b, hk) + (t & (B - 1));
        src[tid] = mine;
        const uint64_t other = __builtin_amdgcn_ballot_w64(tid < rows && t != j * B + tid);
        if (tid % 64 == 0) differ[tid / 64] = other != 0;
    }
    __syncthreads();
    if (!p.to && !(differ[0] | differ[1])) return;                // (all of them stay where they are)
    // rows and scales are asked for together. (A block's scale and its rows are as far into their arrays)
    const uint8_t* pool = val ? p.c.vc : p.c.kc;
    const int tpr = p.c.D / 16, row0 = tid / tpr, col = tid % tpr * 16, step = 256 / tpr;
    uint4 x[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        const int r = row0 + i * step;
        x[i] = uint4{0, 0, 0, 0};
        if (r < rows && src[r] != NONE) x[i] = *reinterpret_cast<const uint4*>(pool + (int64_t) src[r] * p.c.D + col);
    }
    if (tid < 128) scale[tid] = mine == NONE ? 0.0f : (val ? p.c.vsc : p.c.ksc)[mine >> p.c.shift];
    const float a = !val && tid < rows && mine != NONE ? p.acc[mine] : 0.0f;
    __syncthreads();
    const float most = wave_max(fmaxf(pow2_of(Kv8Form<FORM>::LO), fmaxf(scale[tid % 64], scale[64 + tid % 64])));
    const int64_t place = ((int64_t) gs * p.nb + j) * p.nh + hk;
    uint8_t* out = p.to ? (val ? p.c.vc : p.c.kc) + (int64_t) to0 * p.c.D : p.stage + (place * 2 + val) * B * p.c.D;
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        const int r = row0 + i * step;
        if (r >= rows) break;
        uint4 w = x[i];
        if (scale[r] != most) {
            const float ratio = scale[r] / most;
            w = uint4{kv8_reround<FORM>(w.x, ratio), kv8_reround<FORM>(w.y, ratio), kv8_reround<FORM>(w.z, ratio), kv8_reround<FORM>(w.w, ratio)};
        }
        *reinterpret_cast<uint4*>(out + r * p.c.D + col) = w;
    }
    if (tid == 0) {
        if (p.to) (val ? p.c.vsc : p.c.ksc)[(int64_t) dst * p.c.Hkv + hk] = most;
        else p.stage_scale[place * 2 + val] = most;
    }
    if (!val && tid < rows) {
        if (p.to) p.acc[to0 + tid] = a;
        else p.stage_acc[place * B + tid] = a;
    }
}

template <int FORM>
void launch_move(ns_gpu* g, const EvictParams& p, dim3 grid) {
    const int values = p.c.block * p.c.D;
    if (values <= 4096) kv8_move_kernel<FORM, 1><<<grid, 256, 0, g->q>>>(p);
    else if (values == 8192) kv8_move_kernel<FORM, 2><<<grid, 256, 0, g->q>>>(p);
    else if (values == 16384) kv8_move_kernel<FORM, 4><<<grid, 256, 0, g->q>>>(p);
    else kv8_move_kernel<FORM, 8><<<grid, 256, 0, g->q>>>(p);
}

// in place: what the scratch holds into the sequence's first blocks
__global__ __launch_bounds__(256) void kv8_settle_kernel(const EvictParams p) {
    __shared__ int differ;
    const int tid = threadIdx.x, j = blockIdx.x, hk = blockIdx.y >> 1, val = blockIdx.y & 1, gs = blockIdx.z, B = p.c.block;
    const int rows = std::min(p.info[gs].x - j * B, B);
    if (rows <= 0) return;
    const int b = kv8_block(p.c, p.c.table, p.s0 + gs, j);
    if (b < 0) return;
    if (tid == 0) differ = 0;
    __syncthreads();
    if (tid < rows && p.idx[((int64_t) gs * p.nh + hk) * p.cap + j * B + tid] != j * B + tid) differ = 1;
    __syncthreads();
    if (!differ) return;
    const int64_t place = ((int64_t) gs * p.nb + j) * p.nh + hk;
    const uint8_t* from = p.stage + (place * 2 + val) * B * p.c.D;
    uint8_t* out = (val ? p.c.vc : p.c.kc) + kv8_rows(p.c, b, hk) * p.c.D;
    for (int i = tid * 16; i < rows * p.c.D; i += 256 * 16) *reinterpret_cast<uint4*>(out + i) = *reinterpret_cast<const uint4*>(from + i);
    if (tid == 0) (val ? p.c.vsc : p.c.ksc)[(int64_t) b * p.c.Hkv + hk] = p.stage_scale[place * 2 + val];
    if (!val && tid < rows) p.acc[kv8_rows(p.c, b, hk) + tid] = p.stage_acc[place * B + tid];
}

}  // namespace

extern "C" int ns_kv8_evict(ns_gpu* g, int form, const int32_t* lens, int32_t* lens1, int64_t S, int64_t longest, int64_t keep, int64_t first, int64_t last,
                            const int32_t* table, const int32_t* to, int64_t tmax, int64_t Hkv, int64_t D, int64_t block, int64_t blocks, void* kc, void* vc,
                            float* ksc, float* vsc, float* acc) {
    NS_TRY
    const std::string w("ns_kv8_evict");
    if (S <= 0) return 0;
    EvictParams p{};
    p.c = kv8_cache(kc, vc, ksc, vsc, table, tmax, Hkv, D, block, blocks);
    if (ns_kv8_check(w, form, Hkv, D, block, blocks, S, tmax, p.c)) return -1;
    if (keep <= 0 || first < 0 || last < 0 || first > keep || last > keep - first) return ns_fail(w + ": 1 token or more kept, the first and last ones among them");
    if (longest <= 0 || longest > KV8_TOKENS) return ns_fail(w + ": contexts of 1 to 2^30 tokens");
    if (blocks * Hkv > (int64_t) (UINT32_MAX / block)) return ns_fail(w + ": a pool of fewer than 2^32 rows");
    if (!g || !lens || !lens1 || !vc || !vsc || !acc) return ns_fail(w + ": a null buffer");
    if (to == table) return ns_fail(w + ": fresh blocks, or null for the sequences' own");
    p.lens = lens, p.lens1 = lens1, p.to = to, p.longest = longest, p.first = first, p.last = last, p.acc = acc, p.nh = (int) Hkv;
    p.cap = std::min(keep, longest), p.keep = std::min(keep, longest);
    p.nb = (int) ((p.cap + block - 1) / block);
    if (!ns_grid_fits(p.nb, 256)) return ns_fail(w + ": more blocks than a launch takes");
    NS_HIP(hipSetDevice(g->dev));
    NS_OWN_SCRATCH(g);
    auto up = [](int64_t v) { return (v + 63) / 64 * 64; };
    const int64_t own = (int64_t) ns_own_floats(g) - 8 * 64;
    // floats a sequence: its lists, its two numbers, and in place its blocks
    const int64_t lists = Hkv * p.cap + 2, places = Hkv * p.nb, staged = to ? 0 : places * (block * D / 2 + 2 + block);
    const int64_t most = std::min<int64_t>(S, own / (lists + staged));
    if (most < 1) return ns_fail(w + ": a sequence of more tokens and heads than the library's scratch holds");
    for (int64_t s = 0; s < S; s += most) {
        const int64_t n = std::min(most, S - s);
        p.s0 = s;
        float* at = g->own_scratch;
        auto take = [&](int64_t floats) { float* was = at; at += up(floats); return was; };
        p.idx = (int32_t*) take(n * Hkv * p.cap);
        p.info = (int2*) take(2 * n);
        if (!to) {
            p.stage = (uint8_t*) take(n * places * block * D / 2);
            p.stage_scale = take(n * places * 2);
            p.stage_acc = take(n * places * block);
        }
        // (weights a thread: 8 heads of 1000 tokens 10.5 us with 2, 12.1 with 8; of 8000 13.8 with 8)
        if (longest <= 2 * SEL) kv8_select_kernel<2><<<dim3((unsigned) Hkv, (unsigned) n), SEL, 0, g->q>>>(p);
        else if (longest <= 8 * SEL) kv8_select_kernel<8><<<dim3((unsigned) Hkv, (unsigned) n), SEL, 0, g->q>>>(p);
        else kv8_select_kernel<32><<<dim3((unsigned) Hkv, (unsigned) n), SEL, 0, g->q>>>(p);
        NS_LAUNCHED("kv8_select");
        const dim3 grid((unsigned) p.nb, (unsigned) (2 * Hkv), (unsigned) n);
        form == 0 ? launch_move<0>(g, p, grid) : launch_move<1>(g, p, grid);
        NS_LAUNCHED("kv8_move");
        if (!to) {
            kv8_settle_kernel<<<grid, 256, 0, g->q>>>(p);
            NS_LAUNCHED("kv8_settle");
        }
    }
    return 0;
    NS_CATCH
}
