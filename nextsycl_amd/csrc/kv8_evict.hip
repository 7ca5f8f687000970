// kv8_evict.hip: a cache of 8-bit values in blocks of tokens shortened to the tokens of the largest accumulated softmax weights (gfx950).
//
// Three steps a (sequence, key head). Which tokens: the weights' bits, as whole numbers, are searched from the top 11 bits down for the
// value at the last kept place (three histograms in LDS); the kept tokens' places follow from one scan over runs of tokens, so they keep their
// order and of equal weights the earliest stay. Move: a work-group a block to be written, key head and stream - its rows gathered, re-rounded to the largest
// of their scales. In place the blocks go through the library's scratch, since a block is read by those in front of it; blocks whose tokens stay
// where they are are left out. Bound: the kept rows' bytes, read and written; the search by one work-group's latencies.
#include <algorithm>

#include "attn_host.hpp"
#include "kv8_common.hpp"

namespace {

constexpr int SEL = 1024, CACHE = 32768;          // threads of the search; tokens whose weights it keeps in LDS

struct EvictParams {
    Kv8Cache c;
    const int32_t *lens, *to;
    int32_t* lens1;
    int64_t s0, longest, keep, first, last;
    float* acc;
    int64_t cap;                // places of a list: min(keep, longest)
    int nh;                     // = Hkv
    int32_t* idx;               // [group's S][Hkv][cap]
    int2* info;                 // [group's S]: tokens to move, the new length
    uint8_t* stage;             // in place: [group's S][blocks of cap][Hkv][2][block x D], then scales [..][2], then acc [..][block]
    float *stage_scale, *stage_acc;
    int nb;                     // blocks of cap tokens
};

// a work-group's exclusive prefix sum of v, and the total
__device__ __forceinline__ int scan1024(int v, int* sums, int& total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(x, d);
        if (lane >= d) x += y;
    }
    __syncthreads();
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

template <bool CACHED>
__global__ __launch_bounds__(SEL) void kv8_select_kernel(const EvictParams p) {
    __shared__ uint32_t keys[CACHED ? CACHE : 1];
    __shared__ int hist[2048];
    __shared__ int sums[SEL / 64];
    __shared__ int found[2];
    const int tid = threadIdx.x, hk = blockIdx.x, gs = blockIdx.y;
    const int64_t s = p.s0 + gs;
    const int n = p.lens[s];
    const bool over = n < 0 || n > p.longest, whole = n <= p.keep;
    const int rows = over || (whole && !p.to) ? 0 : whole ? n : (int) p.keep;
    if (hk == 0 && tid == 0) p.info[gs] = int2{rows, over || whole ? n : (int) p.keep};
    if (rows == 0 || (CACHED && n > CACHE) || (!CACHED && n <= CACHE)) return;
    int32_t* idx = p.idx + ((int64_t) gs * p.nh + hk) * p.cap;
    if (whole) {
        for (int t = tid; t < n; t += SEL) idx[t] = t;
        return;
    }
    // the weights of the tokens between those that stay anyhow, as whole numbers in the same order
    const int lo = (int) p.first, hi = n - (int) p.last;
    auto weight = [&](int t) -> uint32_t {
        const int b = kv8_block(p.c, p.c.table, s, t >> p.c.shift);
        if (b < 0) return 0;
        const float a = p.acc[kv8_rows(p.c, b, hk) + (t & (p.c.block - 1))];
        return a > 0.0f ? __builtin_bit_cast(uint32_t, a) : 0;
    };
    if constexpr (CACHED) {
        for (int t = lo + tid; t < hi; t += SEL) keys[t] = weight(t);
        __syncthreads();
    }
    auto key = [&](int t) -> uint32_t {
        if constexpr (CACHED) return keys[t];
        else return weight(t);
    };
    // the value at place `need` from the top: 11, 10, 10 bits. `at`: what is known of it
    int need = (int) (p.keep - p.first - p.last);
    uint32_t at = 0;
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 20 : pass == 1 ? 10 : 0, bins = pass == 0 ? 2048 : 1024;
        const uint32_t known = pass == 0 ? 0 : ~0u << (shift + 10);
        for (int i = tid; i < bins; i += SEL) hist[i] = 0;
        __syncthreads();
        for (int t = lo + tid; t < hi; t += SEL) {
            const uint32_t k = key(t);
            if ((k & known) == at) atomicAdd(&hist[k >> shift & (bins - 1)], 1);
        }
        __syncthreads();
        // bins from the largest down, bins / 1024 a thread
        const int per = bins / SEL, top = bins - 1 - tid * per;
        int mine = 0;
        for (int i = 0; i < per; ++i) mine += hist[top - i];
        int all;
        const int before = scan1024(mine, sums, all);
        if (before < need && before + mine >= need) {
            int b = before;
            for (int i = 0; i < per; ++i) {
                if (b + hist[top - i] >= need) {
                    found[0] = top - i, found[1] = need - b;
                    break;
                }
                b += hist[top - i];
            }
        }
        __syncthreads();
        if (need > 0) at |= (uint32_t) found[0] << shift, need = found[1];
        else at = ~0u;                                            // (none of them)
        __syncthreads();
        if (at == ~0u) break;
    }
    // `need` of the tokens equal to `at`, the earliest, and all above it. A thread a run of tokens, of odd length: LDS banks
    const int run = ((n + SEL - 1) / SEL) | 1, t0 = (int) std::min<int64_t>((int64_t) tid * run, n), t1 = std::min<int64_t>((int64_t) t0 + run, n);
    int same = 0, more = 0;
    for (int t = t0; t < t1; ++t) {
        const bool sure = t < lo || t >= hi;
        const uint32_t k = sure ? 0 : key(t);
        more += sure || k > at;
        same += !sure && k == at;
    }
    int all;
    const int same0 = scan1024(same, sums, all), kept = std::min(std::max(need - same0, 0), same);
    int place = scan1024(more + kept, sums, all), left = kept;
    for (int t = t0; t < t1; ++t) {
        const bool sure = t < lo || t >= hi;
        const uint32_t k = sure ? 0 : key(t);
        bool keep = sure || k > at;
        if (!sure && k == at && left > 0) keep = true, --left;
        if (keep) {
            if (place < p.cap) idx[place] = t;
            ++place;
        }
    }
}

// one block to be written: key head and stream blockIdx.y, group's sequence blockIdx.z
template <int FORM>
__global__ __launch_bounds__(256) void kv8_move_kernel(const EvictParams p) {
    __shared__ int64_t src[128];                                  // a row's place in the pool, in rows (-1: none)
    __shared__ float scale[128];
    __shared__ int differ;
    const int tid = threadIdx.x, j = blockIdx.x, hk = blockIdx.y >> 1, val = blockIdx.y & 1, gs = blockIdx.z, B = p.c.block;
    const int64_t s = p.s0 + gs;
    const int2 info = p.info[gs];
    if (j == 0 && blockIdx.y == 0 && tid == 0) p.lens1[s] = info.y;
    const int rows = std::min(info.x - j * B, B);
    if (rows <= 0) return;
    int dst = -1;
    if (p.to) {
        dst = kv8_block(p.c, p.to, s, j);
        if (dst < 0) return;
    }
    if (tid == 0) differ = 0;
    __syncthreads();
    if (tid < rows) {
        const int t = p.idx[((int64_t) gs * p.nh + hk) * p.cap + j * B + tid];
        const int b = kv8_block(p.c, p.c.table, s, t >> p.c.shift);
        src[tid] = b < 0 ? -1 : kv8_rows(p.c, b, hk) + (t & (B - 1));
        scale[tid] = b < 0 ? 0.0f : (val ? p.c.vsc : p.c.ksc)[(int64_t) b * p.c.Hkv + hk];
        if (t != j * B + tid) differ = 1;
    }
    __syncthreads();
    if (!p.to && !differ) return;                                 // (all of them stay where they are)
    float most = kv8_pow2(Kv8Form<FORM>::LO);
    for (int r = tid & 63; r < rows; r += 64) most = fmaxf(most, scale[r]);
    most = wave_max(most);
    const int64_t place = ((int64_t) gs * p.nb + j) * p.nh + hk;
    const uint8_t* pool = val ? p.c.vc : p.c.kc;
    uint8_t* out = p.to ? (val ? p.c.vc : p.c.kc) + kv8_rows(p.c, dst, hk) * p.c.D : p.stage + (place * 2 + val) * B * p.c.D;
    const int tpr = p.c.D / 16, row0 = tid / tpr, col = tid % tpr * 16;
    for (int r = row0; r < rows; r += 256 / tpr) {
        uint4 w = {0, 0, 0, 0};
        if (src[r] >= 0) {
            w = *reinterpret_cast<const uint4*>(pool + src[r] * p.c.D + col);
            if (scale[r] != most) {
                const float ratio = scale[r] / most;
                w = uint4{kv8_reround<FORM>(w.x, ratio), kv8_reround<FORM>(w.y, ratio), kv8_reround<FORM>(w.z, ratio), kv8_reround<FORM>(w.w, ratio)};
            }
        }
        *reinterpret_cast<uint4*>(out + r * p.c.D + col) = w;
    }
    if (tid == 0) {
        if (p.to) (val ? p.c.vsc : p.c.ksc)[(int64_t) dst * p.c.Hkv + hk] = most;
        else p.stage_scale[place * 2 + val] = most;
    }
    if (!val && tid < rows) {
        const float a = src[tid] < 0 ? 0.0f : p.acc[src[tid]];
        if (p.to) p.acc[kv8_rows(p.c, dst, hk) + tid] = a;
        else p.stage_acc[place * B + tid] = a;
    }
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
    if (longest <= 0 || longest > 2 * (int64_t) KV8_TOKENS - 1) return ns_fail(w + ": contexts of 1 to 2^31 - 1 tokens");
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
        kv8_select_kernel<true><<<dim3((unsigned) Hkv, (unsigned) n), SEL, 0, g->q>>>(p);
        NS_LAUNCHED("kv8_select");
        if (longest > CACHE) {
            kv8_select_kernel<false><<<dim3((unsigned) Hkv, (unsigned) n), SEL, 0, g->q>>>(p);
            NS_LAUNCHED("kv8_select");
        }
        const dim3 grid((unsigned) p.nb, (unsigned) (2 * Hkv), (unsigned) n);
        if (form == 0) kv8_move_kernel<0><<<grid, 256, 0, g->q>>>(p);
        else kv8_move_kernel<1><<<grid, 256, 0, g->q>>>(p);
        NS_LAUNCHED("kv8_move");
        if (!to) {
            kv8_settle_kernel<<<grid, 256, 0, g->q>>>(p);
            NS_LAUNCHED("kv8_settle");
        }
    }
    return 0;
    NS_CATCH
}
