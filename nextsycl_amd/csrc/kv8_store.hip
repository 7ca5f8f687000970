// kv8_store.hip: key and value rows into a cache of 8-bit values in blocks of tokens, and blocks widened to half rows (gfx950).
//
// A block's scale is a power of two: 2^x m / M against the largest magnitude 2^x m needs only its exponent and a comparison of m, a value
// over it is exact, its code the one rounding. In a block that holds rows the scale only grows; the codes that were there, whole numbers
// (or e4m3) of the old unit, are re-rounded to the new one, 2^k of it: half a step of the new unit at most, and over any number of
// growths 1/2 + 1/4 + .. of the final one.
//
// Bound: HBM, rows read once and codes written (8192 float32 rows of 8 heads of 128: 15.6 us, 5.4 TB/s; a row of each of 64 sequences: 4.4, the lengths',
// entries', scale's and rows' reads behind one another). A work-group takes one block of one key head and stream, all of its new rows
// in registers - a thread 8 float32 or 16 half values -: their largest magnitude, then their codes. (8192 bfloat16 rows in blocks of 16 11.7 us, 4.3 TB/s; with 8
// values a thread 13.7)
#include <type_traits>

#include "attn_host.hpp"
#include "kv8_common.hpp"

namespace {

struct StoreParams {
    Kv8Cache c;
    const void *k, *v;
    int64_t ks, vs;
    const int32_t *start, *lens;
    int T, most;
};

// TH threads of E values, NP passes over a block's rows: block x D = E TH NP values
template <int QT, int FORM, int D, int TH, int NP>
__global__ __launch_bounds__(TH) void kv8_store_kernel(const StoreParams p) {
    constexpr int E = QT == 0 ? 8 : 16, TPR = D / E, RPP = TH / TPR, B = RPP * NP;      // values a thread, threads a row, rows a pass, rows a block
    using codes_t = std::conditional_t<E == 8, uint2, uint4>;
    __shared__ float red[TH / 64];
    const int tid = threadIdx.x, s = blockIdx.z;
    const int h = blockIdx.y >> 1, val = blockIdx.y & 1;
    const Kv8Seq q = kv8_seq(p.start, p.lens, s, p.T, p.most);
    const int64_t e = q.len / B + (int) blockIdx.x;
    const int64_t t0 = e * B, end = (int64_t) q.len + q.n;        // the block's tokens from t0 on; the call's end at `end`
    if (q.n <= 0 || t0 >= end) return;
    const int b = kv8_block(p.c, p.c.table, s, e);
    if (b < 0) return;
    const bool fresh = t0 >= q.len;
    uint8_t* pool = (val ? p.c.vc : p.c.kc) + kv8_rows(p.c, b, h) * D;
    float* scale = (val ? p.c.vsc : p.c.ksc) + (int64_t) b * p.c.Hkv + h;
    const void* src = val ? p.v : p.k;
    const int64_t stride = val ? p.vs : p.ks;
    const int row = tid / TPR, col = tid % TPR * E;
    const float s0 = fresh ? 0.0f : *scale;

    float x[NP][E], most = 0.0f;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int64_t t = t0 + i * RPP + row;
        if (t < q.len || t >= end) continue;
        const int64_t at = (q.first + (t - q.len)) * stride + (int64_t) h * D + col;
        if constexpr (QT == 0) {
            float lo[4], hi[4];
            load_row<0, 4>(src, at, lo), load_row<0, 4>(src, at + 4, hi);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[i][j] = lo[j], x[i][4 + j] = hi[j];
        } else {
            float lo[8], hi[8];
            load_row<QT, 8>(src, at, lo), load_row<QT, 8>(src, at + 8, hi);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[i][j] = lo[j], x[i][8 + j] = hi[j];
        }
#pragma unroll
        for (int j = 0; j < E; ++j) most = fmaxf(most, fabsf(x[i][j]));      // (fmaxf: NaN counts as nothing)
    }
    most = wave_max(most);
    if (tid % 64 == 0) red[tid / 64] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < TH / 64; ++w) most = fmaxf(most, red[w]);
    const float s1 = fmaxf(s0, pow2_of(kv8_exponent<FORM>(most))), inv = 1.0f / s1, ratio = s0 * inv;
    if (!fresh && s1 > s0) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int64_t t = t0 + i * RPP + row;
            if (t >= q.len && t < end) continue;
            codes_t* at = reinterpret_cast<codes_t*>(pool + (i * RPP + row) * D + col);
            codes_t w = *at;
            w.x = kv8_reround<FORM>(w.x, ratio), w.y = kv8_reround<FORM>(w.y, ratio);
            if constexpr (E == 16) w.z = kv8_reround<FORM>(w.z, ratio), w.w = kv8_reround<FORM>(w.w, ratio);
            *at = w;
        }
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int64_t t = t0 + i * RPP + row;
        if (t < q.len || t >= end) continue;
        auto four = [&](int j) { return kv8_codes<FORM>(x[i][j] * inv, x[i][j + 1] * inv, x[i][j + 2] * inv, x[i][j + 3] * inv); };
        codes_t w;
        w.x = four(0), w.y = four(4);
        if constexpr (E == 16) w.z = four(8), w.w = four(12);
        *reinterpret_cast<codes_t*>(pool + (i * RPP + row) * D + col) = w;
    }
    if (tid == 0 && (fresh || s1 > s0)) *scale = s1;
}

template <int QT, int FORM, int D>
void launch_store(ns_gpu* g, const StoreParams& p, dim3 grid) {
    // (16 rows' threads of 8 values; of 16 values 32 rows' where there are as many)
    constexpr int TH = 2 * D, S = QT == 0 ? 1 : 2;
    if (p.c.block == 16) kv8_store_kernel<QT, FORM, D, TH / S, 1><<<grid, TH / S, 0, g->q>>>(p);
    else if (p.c.block == 32) kv8_store_kernel<QT, FORM, D, TH, 2 / S><<<grid, TH, 0, g->q>>>(p);
    else if (p.c.block == 64) kv8_store_kernel<QT, FORM, D, TH, 4 / S><<<grid, TH, 0, g->q>>>(p);
    else kv8_store_kernel<QT, FORM, D, TH, 8 / S><<<grid, TH, 0, g->q>>>(p);
}
template <int QT>
void launch_store(ns_gpu* g, int form, const StoreParams& p, dim3 grid) {
    if (p.c.D == 128) form == 0 ? launch_store<QT, 0, 128>(g, p, grid) : launch_store<QT, 1, 128>(g, p, grid);
    else form == 0 ? launch_store<QT, 0, 256>(g, p, grid) : launch_store<QT, 1, 256>(g, p, grid);
}

// tokens from .. from + n of one sequence as half rows, k and v [Hkv][n][D]: a thread 8 values of each of 8 rows, asked for together. (20126 tokens of 2
// heads of 256: 11.2 us, 5.5 TB/s)
template <int FORM, int D>
__global__ __launch_bounds__(256) void kv8_widen_kernel(const Kv8Cache c, int64_t from, int64_t n, uint16_t* __restrict__ k, uint16_t* __restrict__ v) {
    constexpr int TPR = D / 8, RPP = 256 / TPR, U = 8;
    const int h = blockIdx.y, col = threadIdx.x % TPR * 8;
    const int64_t j0 = (int64_t) blockIdx.x * RPP * U + threadIdx.x / TPR;
    const uint8_t* pool = blockIdx.z ? c.vc : c.kc;
    const float* scale = blockIdx.z ? c.vsc : c.ksc;
    uint16_t* out = (blockIdx.z ? v : k) + (int64_t) h * n * D + col;
    int b[U];
    uint2 w[U];
    float s[U];
#pragma unroll
    for (int i = 0; i < U; ++i) b[i] = kv8_block(c, c.table, 0, (from + std::min(j0 + i * RPP, n - 1)) >> c.shift);
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int64_t t = from + std::min(j0 + i * RPP, n - 1);
        const int bc = std::max(b[i], 0);
        w[i] = *reinterpret_cast<const uint2*>(pool + (kv8_rows(c, bc, h) + (t & (c.block - 1))) * D + col);
        s[i] = scale[(int64_t) bc * c.Hkv + h];
    }
    // (no block: codes and scale 0 - the block read in its place may never have been stored into, its scale be anything, NaN and infinity too)
#pragma unroll
    for (int i = 0; i < U; ++i) {
        if (b[i] < 0) w[i] = uint2{0, 0}, s[i] = 0.0f;
        if (j0 + i * RPP < n) *reinterpret_cast<s8v*>(out + (j0 + i * RPP) * D) = kv8_halfs8<FORM>(w[i].x, w[i].y, s[i], s[i]);
    }
}

}  // namespace

int ns_kv8_widen(ns_gpu* g, int form, const Kv8Cache& c, int64_t from, int64_t n, uint16_t* k, uint16_t* v) {
    const int64_t rows = 8 * 256 / (c.D / 8);
    const dim3 grid((unsigned) ((n + rows - 1) / rows), (unsigned) c.Hkv, 2);
    if (c.D == 128) form == 0 ? kv8_widen_kernel<0, 128><<<grid, 256, 0, g->q>>>(c, from, n, k, v) : kv8_widen_kernel<1, 128><<<grid, 256, 0, g->q>>>(c, from, n, k, v);
    else form == 0 ? kv8_widen_kernel<0, 256><<<grid, 256, 0, g->q>>>(c, from, n, k, v) : kv8_widen_kernel<1, 256><<<grid, 256, 0, g->q>>>(c, from, n, k, v);
    NS_LAUNCHED("kv8_widen");
    return 0;
}

int ns_kv8_check(const std::string& who, int form, int64_t Hkv, int64_t D, int64_t block, int64_t blocks, int64_t S, int64_t tmax, const Kv8Cache& c) {
    if (form < 0 || form > 1) return ns_fail(who + ": a cache form 0 (int8) or 1 (e4m3)");
    if (D != 128 && D != 256) return ns_fail(who + ": heads of 128 or 256");
    if (block != 16 && block != 32 && block != 64 && block != 128) return ns_fail(who + ": blocks of 16, 32, 64 or 128 tokens");
    if (Hkv <= 0 || Hkv > 32767) return ns_fail(who + ": 1 to 32767 key heads");
    if (blocks <= 0 || blocks > INT32_MAX || tmax <= 0 || tmax > INT32_MAX) return ns_fail(who + ": a pool and tables of 1 to 2^31 - 1 blocks");
    if (S <= 0 || S > 65535) return ns_fail(who + ": 1 to 65535 sequences");
    if (!c.kc || !c.ksc || !c.table) return ns_fail(who + ": a null buffer");
    if (((uintptr_t) c.kc | (uintptr_t) c.vc) % 16) return ns_fail(who + ": pools 16-byte aligned");
    return 0;
}

extern "C" int ns_kv8_store(ns_gpu* g, int form, int qt, const void* k, int64_t ks, const void* v, int64_t vs, int64_t T, const int32_t* start, const int32_t* lens,
                            int64_t S, int64_t most, const int32_t* table, int64_t tmax, int64_t Hkv, int64_t D, int64_t block, int64_t blocks, void* kc,
                            void* vc, float* ksc, float* vsc) {
    NS_TRY
    const std::string w("ns_kv8_store");
    if (T <= 0 || S <= 0 || most <= 0) return 0;
    StoreParams p{kv8_cache(kc, vc, ksc, vsc, table, tmax, Hkv, D, block, blocks), k, v, ks, vs, start, lens, 0, 0};
    if (qt < 0 || qt > 2) return ns_fail(w + ": rows of type 0 (float32), 1 (half) or 2 (bfloat16)");
    if (ns_kv8_check(w, form, Hkv, D, block, blocks, S, tmax, p.c)) return -1;
    if (T > KV8_TOKENS || most > KV8_TOKENS) return ns_fail(w + ": up to 2^30 rows");
    if (ks < Hkv * D || vs < Hkv * D) return ns_fail(w + ": rows at least as far apart as they are long");
    if (!g || !k || !v || !lens || !vc || !vsc) return ns_fail(w + ": a null buffer");
    most = std::min(most, T);
    p.T = (int) T, p.most = (int) most;
    const dim3 grid((unsigned) ((most + block - 2) / block + 1), (unsigned) (2 * Hkv), (unsigned) S);
    if (!ns_grid_fits(grid.x, 16 * D / 8)) return ns_fail(w + ": more rows than a launch takes");
    NS_HIP(hipSetDevice(g->dev));
    if (qt == 0) launch_store<0>(g, form, p, grid);
    else if (qt == 1) launch_store<1>(g, form, p, grid);
    else launch_store<2>(g, form, p, grid);
    NS_LAUNCHED("kv8_store");
    return 0;
    NS_CATCH
}
