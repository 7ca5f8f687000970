// ssm_prompt.hip: a prompt's rows through a state-space layer's convolution and scan (ns_ssm_prompt).
//
// The recurrence h_t = exp(dt_t a) h_{t-1} + dt_t x_t (outer) B_t, y_t = h_t C_t + d x_t, in chunks of 64 rows: with cum_l the sum of
// dt a over a chunk's rows up to l, and h the state in front of the chunk,
//   y_l = exp(cum_l) C_l h + sum over s <= l of [(C_l . B_s) exp(cum_l - cum_s) dt_s + (s = l) d] x_s
//   h'  = exp(cum_63) h + sum over s of exp(cum_63 - cum_s) dt_s x_s (outer) B_s
// three matrix products a chunk and head, and one (C . B) a chunk and group. They run on the matrix unit: an operand is two
// halfs (22 bits), scaled by a power of two that puts the largest value of its column, row or block at 2^13, and three
// instructions a product drop nothing above 2^-22; sums, states and scales are float32. (bfloat16 rows: the products that
// reach y alone take their operands' first halfs, 2^-11 beside the rows' own rounding of 2^-8; Y3 below.)
//
// ssm_prep_kernel, 8 waves a (chunk, group): convolves B and C (a thread half a channel's rows), leaves them in LDS as [feature]
// [row] - an operand's rows are a thread's own, C's come back through transposing reads - and multiplies them; the work-groups
// behind sum the exponents (ssm_header).
// ssm_scan_kernel, a work-group a (head, up to 64 of its features, segment of the prompt): walks its chunks with the state in
// the accumulators of 4 waves, a quarter of its features each (wave w 32 w .. 32 w + 31 of 128). In a chunk wave w convolves 16 columns of x into the
// operands that all read (LDS), splits its part of the state into another, then takes 16 rows of y and its part of h'. Matrix
// results come as (column, 4 consecutive rows) a lane, operands go in as (row or column, 8 values of the summed index) a
// lane; the summed index may come in any order that both sides share, so in runs of 4 of two neighbouring tiles a result
// is an operand as it stands: neither the state nor C . B is ever moved between lanes. A wave's barriers wait for LDS alone:
// what it has asked memory for stays on its way.
// Where heads alone do not fill the chip the prompt is cut in segments: the same kernel first leaves the states of their
// pieces from a start of zero (STATE: half of the work), and each segment's scan starts from those before it, decayed.
//
// Bound: no unit's rate, but steps that wait for one another. 8192 bfloat16 rows of 128 heads of 64 x 128 (308 MB in and out: 60 us at a copy's
// rate; 121 GFLOP of half products as executed, the segments' states and C . B among them: 113 us at a large product's) take 298 - 306 us: 40 in
// the first kernel (51 MB read, 94 written), 87 for the segments' states, 178 for the scan - 8 to 12 vector instructions a matrix instruction, of
// x's convolution, the splits, the decays and the state's scaling and sums, in three waves a SIMD that spend 24 % of their life issuing one, 29 %
// ready for it and the rest at barriers and loads (matrix unit 19 - 23 % busy). 2051 float32 rows of 64 heads (80 MB: 16 us; 22 GFLOP: 21) 71 - 76
// us (10 + 22 + 45), 85 half rows of 128 heads of 80 24: two launches and two chunks of 5 us each. Work-groups a CU, 8192 bfloat16 rows: three of
// the scan 300 us, two - with x and the operands asked for a chunk ahead, for which they have the registers - 320; of the segments' states two or
// three alike. Float32 and half rows have both halfs of each operand in LDS, and so two.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "ns_internal.hpp"
#include "ns_layer.h"
#include "layer_common.hpp"

namespace {

constexpr int L = 64;                     // rows a chunk
constexpr int64_t PASS_ROWS = 8192;       // rows a pass works on: what bounds the scratch
constexpr int MOST_SEGS = 32;
// up to these row by row, as steps: bfloat16 rows of 128 heads of 64 x 128 4 7.6 us and 17.3 as a chunk, 16 16.7 and 17.3, 20 19.9 and 17.4; of 24
// heads of them 16 16.1 and 16.4, 20 19.3 and 16.5; of 80 heads of 64 x 64 16 12.8 and 15.1, 20 15.3 and 15.1; of 64 heads of 32 x 256 16
// 20.2 and 24.7, 24 28.2 and 25.1; only of few and small heads are more (7 of 64 x 16: 24 14.4 and 16.9)
constexpr int64_t FEW_ROWS = 16;
// a chunk and head's header, exponents base 2. Rows' exponents from their run of 16's start, step sizes, weights in the chunk's state, decays from the
// chunk's start; exponents between a run's end and a later one's start [later][run], the whole chunk's exponent and decay, what the weights
// are to be multiplied with (the states' kernel reads up to here); rows' own exponents, to their run's end, from their quarter of the run's
// start. All are sums of rows' exponents, which have one sign, and an exponent between two rows is the sum of those that lie between the two:
// none is larger than what it enters. (As differences of 64-bit sums that floats held from a run's start, rows behind a step of 50 lost 9 of
// their decays' bits. 2051 float32 rows 72.8 us so, 74.6 now, 8192 bfloat16 rows 293 and 298)
constexpr int HDR_L = 0, HDR_DT = 64, HDR_W = 128, HDR_E = 192, HDR_BD = 256, HDR_END = 272, HDR_STATE = 288, HDR_A = 288, HDR_R = 352, HDR_Q = 416, HDR = 480;
// a row's exponent is held to these: 2 to it is 0 or infinite in 32 bits, a chunk's sums are finite
constexpr double MOST_EXPONENT = 4096.0;

// bytes of a chunk and group's operands: C (hi, lo), B (hi, lo) of KK = padded N / 32 steps, C . B as float32
constexpr int64_t op_c(int kk) { return (int64_t) 4 * kk * 1024; }
constexpr int64_t op_bytes(int kk) { return 4 * op_c(kk) + 16 * 1024; }

struct ScanParams {
    SsmLayer l;
    int64_t t0, all;            // the pass's first row, the call's rows
    int64_t slot0;              // the ring's slot of the call's first row
    int T, chunks, segs, per;   // rows and chunks of the pass; segments, chunks a segment
    int sub, piece;             // pieces a segment whose states are found apart, chunks a piece
    int blocks, vec_y, vec_h;   // blocks of 64 features a head; y in pieces of 4 values, the state too
    uint8_t* ops;               // [chunk][group] operands
    float* scales;              // [chunk][group]: what B's and C's operands are to be multiplied with
    float* hdr;                 // [chunk][head]
    float* hist;                // [3][chan]: the raw rows in front of the call's first
    float* segst;               // [1 + piece][head, block]: the pass's first state, then what each piece of the segments but the
                                // last leaves - the first from that state, the others from zero
    float* segtot;              // [piece][head]: their exponents
};

// a power of two that takes `big` to 2^13 .. 2^14, and its inverse
__device__ __forceinline__ void to_half_range(float big, float& up, float& down) {
    const int e = min(267 - (int) (__builtin_bit_cast(uint32_t, big) >> 23 & 255), 253);
    up = __builtin_bit_cast(float, (uint32_t) e << 23);
    down = __builtin_bit_cast(float, (uint32_t) (254 - e) << 23);
}
// 8 floats as two operands: halfs and the halfs of what they leave. (The first halfs are opaque from where they are made: the
// compiler would round a float a second time for the difference, and may round it otherwise there - fused with the product it
// comes from -, which leaves two operands that do not belong together.)
__device__ __forceinline__ s8v half8(const float (&v)[8]) {
    h8v a;
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = (_Float16) v[j];
    return __builtin_bit_cast(s8v, a);
}
__device__ __forceinline__ void split8(const float (&v)[8], s8v& hi, s8v& lo) {
    hi = half8(v);
    asm volatile("" : "+v"(hi));
    const h8v a = __builtin_bit_cast(h8v, hi);
    float r[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = fmaf((float) a[j], -1.0f, v[j]);
    lo = half8(r);
}

// the largest of 4 lanes 16 apart, without the canonicalising copies of fmaxf
__device__ __forceinline__ float rows_most(float v) {
    float a, b;
    pair16(v, a, b);
    pair32(__builtin_elementwise_maximum(a, b), a, b);
    return __builtin_elementwise_maximum(a, b);
}

// the ring's value `at` rows (negative) from the call's first: zeros in front of the sequence, and of taps that there are not
__device__ __forceinline__ float ring_row(const ScanParams& s, int at, int ch) {
    const SsmLayer& p = s.l;
    if (at < 1 - p.K || p.p0 + at < 0) return 0.0f;
    const int64_t slot = s.slot0 + at;                         // (the ring has K - 1 slots at least)
    return p.conv[(slot < 0 ? slot + p.cap : slot) * p.chan + ch];
}

// a row's value out of its bits
template <int QT>
__device__ __forceinline__ float raw_value(uint32_t b) {
    return QT == 0 ? __builtin_bit_cast(float, b) : QT == 1 ? f16_to_f32((uint16_t) b) : bf16_to_f32((uint16_t) b);
}

// a head's step sizes and exponents in a chunk, a lane a row
template <int QT>
__device__ __forceinline__ void ssm_header(const ScanParams& s, int chunk, int head, int lane) {
    const SsmLayer& p = s.l;
    const int t = chunk * L + lane;
    const float dt = t < s.T ? ssm_dt(p, load_q<QT>(p.dt, (s.t0 + t) * p.dts + head) + (p.dtb ? p.dtb[head] : 0.0f)) : 0.0f;
    const double own = (double) dt * (double) p.a[head] * 1.4426950408889634074;
    const float add = (float) (own < -MOST_EXPONENT ? -MOST_EXPONENT : own > MOST_EXPONENT ? MOST_EXPONENT : own);       // (a NaN stays one)
    // its sums with the rows in front of it in its quarter of its run of 16, in its run, and of the rows behind it in its run (0x110 + n: the value of
    // n lanes in front within 16, 0x100 + n: behind; 0 where there is none)
    auto of = [](auto at, float v) { return __builtin_bit_cast(float, dpp_u32<decltype(at)::value>(__builtin_bit_cast(uint32_t, v))); };
    using std::integral_constant;
    const float add1 = of(integral_constant<int, 0x111>(), add);
    float quarter = add + (lane % 4 > 0 ? add1 : 0.0f), run = add + add1, behind = of(integral_constant<int, 0x101>(), add);
    const float quarter2 = of(integral_constant<int, 0x112>(), quarter);
    quarter += lane % 4 > 1 ? quarter2 : 0.0f;
    run += of(integral_constant<int, 0x112>(), run);
    run += of(integral_constant<int, 0x114>(), run);
    run += of(integral_constant<int, 0x118>(), run);
    behind += of(integral_constant<int, 0x101>(), behind);
    behind += of(integral_constant<int, 0x102>(), behind);
    behind += of(integral_constant<int, 0x104>(), behind);
    behind += of(integral_constant<int, 0x108>(), behind);
    // the runs' own
    float whole[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) whole[k] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, run), 16 * k + 15));
    auto runs = [&](int first, int last) {       // of runs first .. last
        float v = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) v += k >= first && k <= last ? whole[k] : 0.0f;
        return v;
    };
    const float end = runs(0, 3), between = runs(lane % 4 + 1, lane % 16 / 4 - 1);
    float* to = s.hdr + ((int64_t) chunk * p.H + head) * HDR;
    to[HDR_DT + lane] = dt;
    to[HDR_E + lane] = exp2f(run + runs(0, lane / 16 - 1));
    to[HDR_A + lane] = add;
    to[HDR_L + lane] = run;
    to[HDR_R + lane] = behind;
    to[HDR_Q + lane] = quarter;
    // (the weights times a power of two that puts the largest between 1/2 and 1: they enter operands)
    const float weight = exp2f(behind + runs(lane / 16 + 1, 3)) * dt, most = wave_max(fabsf(weight));
    const int e = min(max((int) (__builtin_bit_cast(uint32_t, most) >> 23 & 255), 1), 252);
    to[HDR_W + lane] = weight * __builtin_bit_cast(float, (uint32_t) (253 - e) << 23);
    if (lane < 16) to[HDR_BD + lane] = between;         // (run lane % 4, the later lane / 4)
    if (lane < 3) to[HDR_END + lane] = lane == 0 ? end : lane == 1 ? exp2f(end) : __builtin_bit_cast(float, (uint32_t) (e + 1) << 23);
}

// KT: tiles of 16 features that each of 4 waves of the scan holds: 1 up to 64 features, 2 up to 128, 4 up to 256 (bfloat16 rows of 80 heads of
// 64 x 64: 4096 112 us with 1, 144 with 2, 588 33.8 and 40.0)
template <int QT, int KT>
__global__ __launch_bounds__(512, KT == 4 ? 1 : 2) void ssm_prep_kernel(ScanParams s) {
    constexpr int KW = KT == 4 ? 2 : 1, NP = 128 * KW, KK = 2 * KT, ROW = L + 4;     // (34 words: a column of LDS banks on for each feature)
    __shared__ __align__(16) short plane[2][2][NP * ROW];      // [B, C][hi, lo][feature][row]
    __shared__ float part[2][8];
    const SsmLayer& p = s.l;
    const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64), n16 = lane % 16, g = lane / 16;
    if ((int) blockIdx.x >= s.chunks * p.G) {
        // work-groups behind those: headers, a wave a (chunk, head)
        const int64_t i = (int64_t) (blockIdx.x - s.chunks * p.G) * 8 + wave, heads = (int64_t) s.chunks * p.H;
        if (i < heads) ssm_header<QT>(s, (int) (i / p.H), (int) (i % p.H), lane);
        else if (s.t0 == 0) {
            // and x's rows in front of the call, for the scan: the ring is written while that runs
            const int64_t at = (i - heads) * 64 + lane, inner = (int64_t) p.H * p.P;
            if (at < 3 * inner) s.hist[at / inner * p.chan + at % inner] = ring_row(s, (int) (at / inner) - 3, (int) (at % inner));
        }
        return;
    }
    const int chunk = blockIdx.x / p.G, group = blockIdx.x % p.G;
    const int here = min(L, s.T - chunk * L);
    const int64_t first = s.t0 + (int64_t) chunk * L;
    uint8_t* ops = s.ops + (int64_t) blockIdx.x * op_bytes(KK);
    float downs[2] = {1.0f, 1.0f};
#pragma unroll
    for (int j = 0; j < KW; ++j) {
        // a thread half a channel: its 32 rows
        const int half = tid / 256, r0 = 32 * half;
        const int isc = KW == 1 ? tid / 128 % 2 : j, n = KW == 1 ? tid % 128 : tid % 256, ch = p.H * p.P + (isc * p.G + group) * p.N + n;
        float v[L / 2], big = 0.0f;
        if (n < p.N) {
            float a0, a1, a2;
            const float w0 = ssm_tap(p, ch, 0), w1 = ssm_tap(p, ch, 1), w2 = ssm_tap(p, ch, 2), w3 = ssm_tap(p, ch, 3), b = p.cb ? p.cb[ch] : 0.0f;
            auto row = [&](int t) { return load_q<QT>(p.xbc, (first + min(t, here - 1)) * p.xs + ch); };
            if (half || first >= 3) a0 = row(r0 - 3), a1 = row(r0 - 2), a2 = row(r0 - 1);
            else a0 = ring_row(s, -3, ch), a1 = ring_row(s, -2, ch), a2 = ring_row(s, -1, ch);      // (first is 0)
#pragma unroll
            for (int t = 0; t < L / 2; ++t) v[t] = row(r0 + t);
            auto convolve = [&](auto all) {
                // (FEW taps: of those that there are not 0, as 0 times what is not finite is not)
                constexpr bool FEW = !decltype(all)::value;
                if (FEW) a0 = 0.0f, a1 = p.K > 2 ? a1 : 0.0f, a2 = p.K > 1 ? a2 : 0.0f;
#pragma unroll
                for (int t = 0; t < L / 2; ++t) {
                    const float a3 = v[t];
                    const float c = silu(fmaf(w3, a3, fmaf(w2, a2, fmaf(w1, a1, fmaf(w0, a0, b)))));
                    if (FEW) a1 = p.K > 2 ? a2 : 0.0f, a2 = p.K > 1 ? a3 : 0.0f;
                    else a0 = a1, a1 = a2, a2 = a3;
                    v[t] = r0 + t < here ? c : 0.0f;
                    // (what is not finite has no part in the scale: it would leave the other rows' values none)
                    big = fabsf(v[t]) < __builtin_inff() ? fmaxf(big, fabsf(v[t])) : big;
                }
            };
            if (p.K == 4) convolve(std::true_type());
            else convolve(std::false_type());
        } else {
#pragma unroll
            for (int t = 0; t < L / 2; ++t) v[t] = 0.0f;
        }
        big = wave_max(big);
        if (lane == 0) part[j][wave] = big;
        __syncthreads();
        auto most = [&](int from, int n) {
            float m = 0.0f;
            for (int i = 0; i < n; ++i) m = fmaxf(m, fmaxf(part[j][from + i], part[j][from + 4 + i]));
            return m;
        };
        float up;
        if constexpr (KW == 1) {
            float ups[2];
            to_half_range(most(0, 2), ups[0], downs[0]);
            to_half_range(most(2, 2), ups[1], downs[1]);
            up = isc ? ups[1] : ups[0];
        } else to_half_range(most(0, 4), up, downs[j]);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            // rows 32 half + 4 q .. + 3 and 16 behind them: an operand's 8
            float e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = v[16 * (i / 4) + 4 * q + i % 4] * up;
            s8v hi, lo;
            split8(e, hi, lo);
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
                const int at = n * ROW + r0 + 4 * i + 4 * q;
                *reinterpret_cast<s4v*>(plane[isc][0] + at) = s4v{hi[i], hi[i + 1], hi[i + 2], hi[i + 3]};
                *reinterpret_cast<s4v*>(plane[isc][1] + at) = s4v{lo[i], lo[i + 1], lo[i + 2], lo[i + 3]};
            }
            if (!isc && (KT > 1 || n < 64)) {
                s8v* to = reinterpret_cast<s8v*>(ops + 2 * op_c(KK)) + ((n / 16) * 2 + half) * 64 + n % 16 + 16 * q;
                to[0] = hi;
                to[op_c(KK) / 16] = lo;
            }
        }
    }
    if (tid < 2) s.scales[(int64_t) blockIdx.x * 2 + tid] = tid ? downs[1] : downs[0];
    __syncthreads();
    // 16 rows of a plane as operands: (row, features 32 kk + 4 g .. + 3 and 16 behind them)
    auto operand = [&](short* from, int tile, int kk) {
        short* at = from + (32 * kk + 4 * g + n16 / 4) * ROW + 16 * tile + 4 * (n16 % 4);
        const s4v a = lds_read_tr16(at), b = lds_read_tr16(at + 16 * ROW);
        return s8v{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    };
    const int w = wave % 4, h = wave / 4;
    // (of bfloat16 rows the scan takes C's first halfs alone)
    if (QT != 2 || h == 0) {
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) reinterpret_cast<s8v*>(ops + h * op_c(KK))[(w * KK + kk) * 64 + lane] = operand(plane[1][h], w, kk);
    }
    // C . B of 16 rows of C against the rows of B that they see: column a row of C, 4 consecutive rows of B a lane
    const float down = downs[0] * downs[1];
    for (int st = h; st <= w; st += 2) {
        f4v acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            const s8v bh = operand(plane[0][0], st, kk), bl = operand(plane[0][1], st, kk), chh = operand(plane[1][0], w, kk), cl = operand(plane[1][1], w, kk);
            acc = mfma16<false>(bh, chh, acc);
            acc = mfma16<false>(bl, chh, acc);
            acc = mfma16<false>(bh, cl, acc);
        }
        reinterpret_cast<f4v*>(ops + 4 * op_c(KK))[((w * 2 + st / 2) * 64 + lane) * 2 + st % 2] = acc * down;
    }
}

// work-groups a CU: what LDS has room for, and the registers that leaves a wave
template <int QT, int KT, bool STATE>
constexpr int SCAN_WGS = KT == 4 ? 1 : STATE || QT == 2 ? 3 : 2;
template <int QT, int KT, int CT, bool STATE>
__global__ __launch_bounds__(256, (SCAN_WGS<QT, KT, STATE>)) void ssm_scan_kernel(ScanParams s) {
    constexpr int KK = 2 * KT;
    constexpr bool AHEAD = STATE || SCAN_WGS<QT, KT, STATE> <= 2;     // x and the operands asked for early, where there are registers for them
    // y's products from both halfs of their operands - the state, C, x, C . B with its decays -, but for bfloat16 rows: what first halfs lose, 2^-11
    // each, is an eighth of y's own rounding (8192 rows' error against 64 bits is 1.680e-3 of y, 1.658e-3 with both), and one plane of the state and of x
    // leaves LDS and registers for three work-groups a CU (298 us; 365 with both halfs, two work-groups)
    constexpr bool Y3 = QT != 2;
    // x weighted for the state (hi, lo) and as it is (hi, for Y3 lo): [32 rows][16 columns][lane]; the state: [32 features][..]
    constexpr int WH = 0, WL = 1, XH = 2, XL = 3, PLANES = STATE ? 2 : Y3 ? 4 : 3, HP = STATE ? 0 : Y3 ? 2 : 1;
    __shared__ __align__(16) s8v xop[PLANES][2][CT][64];
    __shared__ __align__(16) s8v hop[HP + !HP][STATE ? 1 : KK][CT][64];
    __shared__ __align__(16) float xs[16 * CT], hs[16 * CT];                // what their results are to be multiplied with, a column
    __shared__ __align__(16) float hmax[16 * CT][4];                   // the largest of each wave's part of the state, a column
    constexpr int HDRS = STATE ? HDR_STATE : HDR;
    __shared__ __align__(16) float hdrs[2][HDRS];
    __shared__ int bad[16 * CT];
    __shared__ __align__(16) int spoilt[4];                       // a column's first row that is not finite; whether 16 columns have one
    const SsmLayer& p = s.l;
    const int tid = threadIdx.x, lane = tid % 64, w = __builtin_amdgcn_readfirstlane(tid / 64), n = lane % 16, g = lane / 16;
    // heads of a group read the same operands: consecutive work-groups of one XCD (every eighth of the launch)
    int id = blockIdx.x;
    const int total = gridDim.x;
    if (total % 8 == 0) id = id % 8 * (total / 8) + id / 8;
    const int per = p.H / p.G, hb = per * s.blocks;
    const int in_group = id % hb, seg = id / hb % s.segs, group = id / (hb * s.segs);       // (STATE: seg counts pieces)
    const int head = group * per + in_group / s.blocks, block = in_group % s.blocks, c0 = block * 16 * CT;
    const int col = c0 + 16 * w + n;                              // the column of x this lane convolves
    const bool has = (CT == 4 || w < CT) && col < p.P;            // (fewer column tiles than waves: the last have none)
    const int xch = head * p.P + (has ? col : 0);
    // (the taps times log2 e: x comes out times it too, which its operand's scale takes back, and the exponential takes it as it is; a tap that
    // there is not is 0 times what is not finite for rows whose column that has already ended)
    constexpr float LOG2E = 1.44269504f, LN2 = 0.693147181f;
    const float w0 = ssm_tap(p, xch, 0) * LOG2E, w1 = ssm_tap(p, xch, 1) * LOG2E, w2 = ssm_tap(p, xch, 2) * LOG2E, w3 = ssm_tap(p, xch, 3) * LOG2E;
    const float bias = p.cb ? p.cb[xch] * LOG2E : 0.0f;
    const float skip = p.d ? p.d[head] : 0.0f;
    const int from = STATE ? seg / s.sub * s.per + seg % s.sub * s.piece : seg * s.per;
    const int to = min(s.chunks, STATE ? min(from + s.piece, (seg / s.sub + 1) * s.per) : from + s.per);
    const int64_t owner = (int64_t) head * s.blocks + block, owners = (int64_t) p.H * s.blocks;

    // features 16 (w KT + i) + 4 g .. + 3 of column 16 ct + n
    f4v st[KT][CT];
    auto feature = [&](int i) { return 16 * (w * KT + i) + 4 * g; };
    auto kept = [&](int slot) { return reinterpret_cast<f4v*>(s.segst) + ((slot * owners + owner) * 4 + w) * (KT * CT * 64) + lane; };
    // (a cut pass's first state is read from where the state kernel has put it: the last segment may write h1 = h0 meanwhile)
    if (STATE ? seg == 0 : s.segs == 1) {
        const float* h0 = s.t0 ? p.h1 : p.h0;
#pragma unroll
        for (int i = 0; i < KT; ++i)
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                f4v v = {0.0f, 0.0f, 0.0f, 0.0f};
                const int f = feature(i), c = c0 + 16 * ct + n;
                if (h0 && c < p.P && f < p.N) {
                    const float* src = h0 + ((int64_t) head * p.P + c) * p.N + f;
                    if (s.vec_h) v = *reinterpret_cast<const f4v*>(src);
                    else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (f + e < p.N) v[e] = src[e];
                    }
                }
                st[i][ct] = v;
                if (STATE) kept(0)[(i * CT + ct) * 64] = v;
            }
    } else {
        const f4v* src = kept(seg > 0 && !STATE);
#pragma unroll
        for (int i = 0; i < KT; ++i)
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) st[i][ct] = STATE ? f4v{0.0f, 0.0f, 0.0f, 0.0f} : src[(i * CT + ct) * 64];
        for (int r = 1; !STATE && r < seg * s.sub; ++r) {
            const float keep = exp2f(s.segtot[(int64_t) r * p.H + head]);
            const f4v* add = kept(1 + r);
#pragma unroll
            for (int i = 0; i < KT; ++i)
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) st[i][ct] = st[i][ct] * keep + add[(i * CT + ct) * 64];
        }
    }
    if (CT < 4 && tid < 4) spoilt[tid] = 0;
    float exponent = 0.0f;
    // a chunk's header, through registers into LDS; x: 16 rows of this lane's column - 16 j + 4 g .. + 3 - and 3 in front of each 4
    float head0, head1;
    auto fetch_header = [&](int c) {
        const float* hd = s.hdr + ((int64_t) min(c, s.chunks - 1) * p.H + head) * HDR;
        head0 = hd[tid];
        head1 = hd[256 + tid % (HDRS - 256)];
    };
    auto put_header = [&](int c) {
        hdrs[c % 2][tid] = head0;
        if (tid < HDRS - 256) hdrs[c % 2][256 + tid] = head1;
    };
    // (as they are loaded: widened to 32 bits they would be awaited at once)
    typedef std::conditional_t<QT == 0, uint32_t, uint16_t> raw_t;
    raw_t raw[28];
    const int64_t row_bytes = p.xs * (QT ? 2 : 4);
    const uint32_t lane_off = (uint32_t) (4 * g * row_bytes + (int64_t) xch * (QT ? 2 : 4));
    auto fetch_x = [&](int c, int g) {
        if (AHEAD && CT < 4 && w >= CT) return;           // (without AHEAD the branch costs more registers than the loads)
        const int here = min(L, s.T - c * L);
        const int64_t first = s.t0 + (int64_t) c * L;
        // as a buffer of its own, from the first row of the chunk that there is in front of its first: a lane's offset in a vector
        // register, a row's in a scalar one
        const int front = first > 0 ? 3 : 0;
        const auto rows = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(static_cast<const char*>(p.xbc) + (first - front) * row_bytes), (short) 0, -1, 0x00020000);
        auto at = [&](uint32_t lane_off, uint32_t off) {
            if constexpr (QT == 0) return (raw_t) __builtin_amdgcn_raw_buffer_load_b32(rows, lane_off, off, 0);
            else return (raw_t) __builtin_amdgcn_raw_buffer_load_b16(rows, lane_off, off, 0);
        };
        if (front && here == L) {
            uint32_t step = (uint32_t) row_bytes;
            asm volatile("" : "+s"(step));           // (or the compiler carries 28 offsets from chunk to chunk)
#pragma unroll
            for (int j = 0; j < 28; ++j) raw[j] = at(lane_off, (16 * (j / 7) + j % 7) * step);
        } else {
            // the call's first chunk, or one that is not whole: rows held to those that there are (those in front of the call come from the ring)
#pragma unroll
            for (int j = 0; j < 28; ++j) {
                const int r = min(max(16 * (j / 7) + 4 * g + j % 7 - 3 + front, 0), here - 1 + front);
                raw[j] = at((uint32_t) r * (uint32_t) row_bytes + (uint32_t) xch * (QT ? 2 : 4), 0);
            }
        }
    };
    // each column's largest in this wave's part of the state: what the next chunk's operands of it are scaled by
    auto column_max = [&] {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            float big = 0.0f;
#pragma unroll
            for (int i = 0; i < KT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) big = __builtin_elementwise_maximum(big, fabsf(st[i][ct][e]));
            big = rows_most(big);
            if (g == 0) hmax[16 * ct + n][w] = big;
        }
    };
    if constexpr (!STATE) column_max();
    fetch_header(from);
    put_header(from);
    if constexpr (AHEAD) fetch_x(from, g);
    __syncthreads();

    for (int c = from; c < to; ++c) {
        const float* hdr = hdrs[c % 2];
        const uint8_t* ops = s.ops + ((int64_t) c * p.G + group) * op_bytes(KK);
        const float scale_b = s.scales[((int64_t) c * p.G + group) * 2], sc = s.scales[((int64_t) c * p.G + group) * 2 + 1];
        // (opaque copies: addresses and comparisons made of them are a few instructions where they are needed, and not a
        // hundred registers kept over the loop)
        int ln = n, lg = g;
        asm volatile("" : "+v"(ln), "+v"(lg));
        fetch_header(c + 1);
        // this chunk's operands, on their way while x and the state become theirs
        s8v bop[KT][2][2], cop[STATE ? 1 : KK][2];
        f4v cbv[2][2];
        auto fetch_b = [&] {
            const s8v* b = reinterpret_cast<const s8v*>(ops + 2 * op_c(KK)) + lane;
#pragma unroll
            for (int i = 0; i < KT; ++i)
#pragma unroll
                for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                    for (int h = 0; h < 2; ++h) bop[i][ks][h] = b[((w * KT + i) * 2 + ks) * 64 + h * (op_c(KK) / 16)];
        };
        auto fetch_c = [&] {
            const s8v* cp = reinterpret_cast<const s8v*>(ops) + w * KK * 64 + lane;
#pragma unroll
            for (int kk = 0; kk < KK; ++kk)
#pragma unroll
                for (int h = 0; h < (Y3 ? 2 : 1); ++h) cop[kk][h] = cp[kk * 64 + h * (op_c(KK) / 16)];
            const f4v* cbp = reinterpret_cast<const f4v*>(ops + 4 * op_c(KK)) + w * 2 * 64 * 2;
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (ks <= w / 2) cbv[ks][h] = cbp[(ks * 64 + lane) * 2 + h];
        };
        if constexpr (AHEAD) {
            fetch_b();
            if constexpr (!STATE) fetch_c();
        } else fetch_x(c, lg);
        // x's operands
        if (CT == 4 || w < CT) {
            const int here = min(L, s.T - c * L);
            const bool whole = here == L;
            float x[2][8], big = 0.0f;
            f4v wt[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                // rows 16 j + 4 g .. + 3
                wt[j] = *reinterpret_cast<const f4v*>(hdr + HDR_W + 16 * j + 4 * lg);
                float u[7];
#pragma unroll
                for (int i = 0; i < 7; ++i) u[i] = raw_value<QT>(raw[7 * j + i]);
                if (j == 0 && c == 0 && s.t0 == 0) {
                    // (in front of the call: float32 from the ring, whatever the rows' type; awaited here, or every chunk would
                    // wait for all that it has asked for where the two ways meet)
                    float old[3];
#pragma unroll
                    for (int i = 0; i < 3; ++i) old[i] = s.hist[(int64_t) i * p.chan + xch];
                    asm volatile("" : "+v"(old[0]), "+v"(old[1]), "+v"(old[2]));
#pragma unroll
                    for (int i = 0; i < 3; ++i) u[i] = lg == 0 ? old[i] : u[i];
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float v = fmaf(w3, u[i + 3], fmaf(w2, u[i + 2], fmaf(w1, u[i + 1], fmaf(w0, u[i], bias))));
                    x[j / 2][4 * (j % 2) + i] = v * __builtin_amdgcn_rcpf(1.0f + fast_exp2(-v));
                }
            }
            if (!whole) {
                asm volatile("");        // (a branch, not 32 instructions of every chunk)
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i / 8][i % 8] = 16 * (i / 4) + 4 * lg + i % 4 < here ? x[i / 8][i % 8] : 0.0f;
            }
            // (a NaN among them stays one)
#pragma unroll
            for (int i = 0; i < 16; ++i) big = __builtin_elementwise_maximum(big, fabsf(x[i / 8][i % 8]));
            auto operands = [&](float big, auto held) {
                float up, down;
                to_half_range(rows_most(big), up, down);
                if (g == 0) xs[16 * w + n] = down * LN2;
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
                    float v[8], r[8];
                    s8v hi, lo;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        v[i] = x[ks][i] * up;
                        r[i] = v[i] * wt[2 * ks + i / 4][i % 4];
                    }
                    split8(r, hi, lo);
                    xop[WH][ks][w][lane] = hi;
                    xop[WL][ks][w][lane] = lo;
                    if constexpr (!STATE) {
                        if constexpr (decltype(held)::value) {
#pragma unroll
                            for (int i = 0; i < 8; ++i) v[i] = fabsf(v[i]) < __builtin_inff() ? v[i] : 0.0f;
                        }
                        if constexpr (Y3) {
                            split8(v, hi, lo);
                            xop[XL][ks][w][lane] = lo;
                        } else hi = half8(v);
                        xop[XH][ks][w][lane] = hi;
                    }
                }
            };
            const bool fine = STATE || !__ballot(!(big < __builtin_inff()));
            if (!STATE && lane == 0) spoilt[w] = !fine;
            if (fine) operands(big, std::false_type());
            else {
                // a row that is not finite must not reach the rows in front of it (0 times it is not 0): among x's operands it is
                // 0, and from it on the column is NaN
                int where = L;
                big = 0.0f;
#pragma unroll
                for (int i = 15; i >= 0; --i) {
                    const float y = fabsf(x[i / 8][i % 8]);
                    if (y < __builtin_inff()) big = fmaxf(big, y);
                    else where = 16 * (i / 4) + 4 * lg + i % 4;
                }
                where = min(where, __shfl_xor(where, 16));
                where = min(where, __shfl_xor(where, 32));
                operands(big, std::true_type());
                if (g == 0) bad[16 * w + n] = where;
            }
        }
        if constexpr (!AHEAD && !STATE) fetch_c();
        // this wave's part of the state
        if constexpr (!STATE) {
            f4v parts[CT];
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) parts[ct] = *reinterpret_cast<const f4v*>(hmax[16 * ct + n]);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                const int at = 16 * ct + n;
                const float most = __builtin_elementwise_maximum(__builtin_elementwise_maximum(parts[ct][0], parts[ct][1]), __builtin_elementwise_maximum(parts[ct][2], parts[ct][3]));
                float up, down;
                to_half_range(most, up, down);
                if (w == 0 && g == 0) hs[at] = down;
                if constexpr (KT == 1) {
                    // (half an operand: its neighbour's tile is the other)
                    const float v[8] = {st[0][ct][0] * up, st[0][ct][1] * up, st[0][ct][2] * up, st[0][ct][3] * up, 0.0f, 0.0f, 0.0f, 0.0f};
                    s8v hi, lo;
                    if constexpr (Y3) {
                        split8(v, hi, lo);
                        reinterpret_cast<s4v*>(&hop[1][w / 2][ct][lane])[w % 2] = s4v{lo[0], lo[1], lo[2], lo[3]};
                    } else hi = half8(v);
                    reinterpret_cast<s4v*>(&hop[0][w / 2][ct][lane])[w % 2] = s4v{hi[0], hi[1], hi[2], hi[3]};
                }
#pragma unroll
                for (int j = 0; j < KT / 2; ++j) {
                    float v[8];
                    s8v hi, lo;
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = st[2 * j + i / 4][ct][i % 4] * up;
                    if constexpr (Y3) {
                        split8(v, hi, lo);
                        hop[1][w * (KT / 2) + j][ct][lane] = lo;
                    } else hi = half8(v);
                    hop[0][w * (KT / 2) + j][ct][lane] = hi;
                }
            }
        }
        lds_barrier();
        if constexpr (AHEAD)
            if (c + 1 < to) fetch_x(c + 1, lg);
        if constexpr (!STATE) {
            const int row = 16 * w + ln;
            // of rows of one run: those of s's quarter of it behind s, up to this row; then whole quarters; then this row's up to it
            f4v in_run;
            {
                const f4v own = *reinterpret_cast<const f4v*>(hdr + HDR_A + 16 * w + 4 * lg);
                const float* quarters = hdr + HDR_Q + 16 * w;
                const float q1 = quarters[min(4 * lg + 7, 15)], q2 = quarters[min(4 * lg + 11, 15)], q = quarters[ln];
                const int apart = ln / 4 - lg;
                float past = (apart > 0 ? q : 0.0f) + ((apart > 1 ? q1 : 0.0f) + (apart > 2 ? q2 : 0.0f));
#pragma unroll
                for (int i = 3; i >= 0; --i) {
                    in_run[i] = past;
                    past += 4 * lg + i <= ln ? own[i] : 0.0f;
                }
            }
            // 16 rows of y: this lane row 16 w + n, columns 16 ct + 4 g .. + 3
            f4v y[CT], yi[CT];
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) y[ct] = yi[ct] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) {
                    yi[ct] = mfma16<false>(hop[0][kk][ct][lane], cop[kk][0], yi[ct]);
                    if constexpr (Y3) {
                        yi[ct] = mfma16<false>(hop[HP - 1][kk][ct][lane], cop[kk][0], yi[ct]);
                        yi[ct] = mfma16<false>(hop[0][kk][ct][lane], cop[kk][1], yi[ct]);
                    }
                }
            }
            // the chunk's own rows: C . B decayed, d on the diagonal
            const float cl = hdr[HDR_L + row];
            float m[2][8], big = 0.0f;
            const f4v bd = *reinterpret_cast<const f4v*>(hdr + HDR_BD + 4 * w);
#pragma unroll
            for (int st = 0; st < 4; ++st) {
                float* to_m = m[st / 2] + 4 * (st % 2);
                if (st > w) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) to_m[i] = 0.0f;
                    continue;
                }
                const f4v dts = *reinterpret_cast<const f4v*>(hdr + HDR_DT + 16 * st + 4 * lg);
                // from s to its run's end, to this row's run's start, to this row
                const f4v apart = *reinterpret_cast<const f4v*>(hdr + HDR_R + 16 * st + 4 * lg) + (cl + bd[st]), between = st < w ? apart : in_run;
                const f4v cb = cbv[st / 2][st % 2];
#pragma unroll
                for (int i = 0; i < 4; ++i) to_m[i] = cb[i] * dts[i] * fast_exp2(between[i]);
                if (st == w) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        to_m[i] = 4 * lg + i == ln ? to_m[i] + skip : to_m[i];
                        to_m[i] = 4 * lg + i > ln ? 0.0f : to_m[i];
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) big = __builtin_elementwise_maximum(big, fabsf(to_m[i]));
            }
            float up, down;
            to_half_range(rows_most(big), up, down);
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                if (ks > w / 2) break;
                s8v hi, lo;
#pragma unroll
                for (int i = 0; i < 8; ++i) m[ks][i] *= up;
                if constexpr (Y3) split8(m[ks], hi, lo);
                else hi = half8(m[ks]);
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) {
                    y[ct] = mfma16<false>(xop[XH][ks][ct][lane], hi, y[ct]);
                    if constexpr (Y3) {
                        y[ct] = mfma16<false>(xop[PLANES - 1][ks][ct][lane], hi, y[ct]);
                        y[ct] = mfma16<false>(xop[XH][ks][ct][lane], lo, y[ct]);
                    }
                }
            }
            if constexpr (!AHEAD) fetch_b();
            const int t = c * L + row;
            const float el = hdr[HDR_E + row] * sc;
            const int4 sp = *reinterpret_cast<const int4*>(spoilt);
            const bool finite = !__builtin_amdgcn_readfirstlane(sp.x | sp.y | sp.z | sp.w);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                const f4v f = *reinterpret_cast<const f4v*>(&xs[16 * ct + 4 * lg]), fi = *reinterpret_cast<const f4v*>(&hs[16 * ct + 4 * lg]);
#pragma unroll
                for (int e = 0; e < 4; ++e) y[ct][e] = fmaf(y[ct][e], f[e] * down, yi[ct][e] * (fi[e] * el));
                if (!AHEAD) asm volatile("" : "+v"(y[ct]));          // (few registers: one column tile after another)
            }
            if (!finite) {
#pragma unroll
                for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (spoilt[ct] && row >= bad[16 * ct + 4 * lg + e]) y[ct][e] = __builtin_nanf("");
            }
            if (t < s.T) {
                const int64_t at = (s.t0 + t) * p.ys + (int64_t) head * p.P + c0 + 4 * lg;
                if (s.vec_y) {
#pragma unroll
                    for (int ct = 0; ct < CT; ++ct) {
                        const float v[4] = {y[ct][0], y[ct][1], y[ct][2], y[ct][3]};
                        if (c0 + 16 * ct + 4 * lg < p.P) store_row<QT, 4>(p.y, at + 16 * ct, v);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4 * CT; ++i)
                        if (c0 + 16 * (i / 4) + 4 * lg + i % 4 < p.P) store_o<QT>(p.y, at + 16 * (i / 4) + i % 4, y[i / 4][i % 4]);
                }
            }
        }
        // the state behind the chunk
        {
            const float keep = hdr[HDR_END + 1], sb = scale_b * hdr[HDR_END + 2];
            exponent += hdr[HDR_END];
            s8v ahead[2][2][2];
            // (in registers of its own, that a product's first step starts from: the compiler would clear each sum apart)
            f4v zero = {0.0f, 0.0f, 0.0f, 0.0f};
            if constexpr (!STATE) asm volatile("" : "+v"(zero));
            float fs[CT];
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) fs[ct] = xs[16 * ct + n];
            auto operands = [&](int ct) {
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) ahead[ct % 2][ks][0] = xop[WH][ks][ct][lane], ahead[ct % 2][ks][1] = xop[WL][ks][ct][lane];
            };
            // (a column tile ahead, but in the states' kernel: its three work-groups a CU hide the reads)
            if constexpr (!STATE) operands(0);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                if constexpr (STATE) operands(ct);
                else if (ct < CT - 1) operands(ct + 1);
                f4v a[KT];
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
                    const s8v hi = ahead[ct % 2][ks][0], lo = ahead[ct % 2][ks][1];
#pragma unroll
                    for (int i = 0; i < KT; ++i) a[i] = mfma16<false>(bop[i][ks][0], hi, ks ? a[i] : zero);
#pragma unroll
                    for (int i = 0; i < KT; ++i) a[i] = mfma16<false>(bop[i][ks][1], hi, a[i]);
#pragma unroll
                    for (int i = 0; i < KT; ++i) a[i] = mfma16<false>(bop[i][ks][0], lo, a[i]);
                }
                const float f = sb * fs[ct];
#pragma unroll
                for (int i = 0; i < KT; ++i) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) st[i][ct][e] = fmaf(st[i][ct][e], keep, a[i][e] * f);
                    // (here: the compiler would ask for all columns' operands at once)
                    asm volatile("" : "+v"(st[i][ct]));
                }
            }
        }
        put_header(c + 1);
        if constexpr (!STATE) column_max();
        lds_barrier();
    }

    if constexpr (STATE) {
        f4v* dst = kept(1 + seg);
#pragma unroll
        for (int i = 0; i < KT; ++i)
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) dst[(i * CT + ct) * 64] = st[i][ct];
        if (tid == 0 && block == 0) s.segtot[(int64_t) seg * p.H + head] = exponent;
    } else {
        if (seg == s.segs - 1) {
#pragma unroll
            for (int i = 0; i < KT; ++i)
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) {
                    const int f = feature(i), cc = c0 + 16 * ct + n;
                    if (cc >= p.P || f >= p.N) continue;
                    float* dst = p.h1 + ((int64_t) head * p.P + cc) * p.N + f;
                    if (s.vec_h) *reinterpret_cast<f4v*>(dst) = st[i][ct];
                    else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (f + e < p.N) dst[e] = st[i][ct][e];
                    }
                }
        }
        // the call's last raw rows into the ring: this block's x, and the group's B and C
        if (seg == 0 && s.t0 + s.T == s.all) {
            for (int64_t t = max((int64_t) 0, s.all - (p.K - 1)); t < s.all; ++t) {
                float* dst = p.conv + (p.p0 + t) % p.cap * p.chan;
                if (tid < 16 * CT && c0 + tid < p.P) dst[head * p.P + c0 + tid] = load_q<QT>(p.xbc, t * p.xs + head * p.P + c0 + tid);
                if (in_group == 0)
                    for (int i = tid; i < 2 * p.N; i += 256) {
                        const int ch = p.H * p.P + (i / p.N * p.G + group) * p.N + i % p.N;
                        dst[ch] = load_q<QT>(p.xbc, t * p.xs + ch);
                    }
            }
        }
    }
}

// how a pass of T rows is cut, and where its scratch lies
struct Plan {
    int kk, chunks, segs, per, sub, piece, blocks;
    int64_t ops, scales, hdr, hist, segst, segtot, floats;
};
Plan plan_of(int64_t T, int64_t H, int64_t P, int64_t N, int64_t G, int wgs) {
    Plan q{};
    q.kk = N <= 64 ? 2 : N <= 128 ? 4 : 8;
    q.chunks = (int) ((T + L - 1) / L);
    q.blocks = (int) ((P + 63) / 64);
    const int64_t owners = H * q.blocks;
    // as many segments as fill the chip's places for the scan's work-groups, of 2 chunks at least. (bfloat16 rows of 32 heads of 64 x 128:
    // 512 44.6 us in segments of 4 chunks, 32.5 in those of 2, and 256 rows, left whole, 29.8 - in two segments 30.4; 8192 rows of
    // 8 heads of 64 x 64 91.2 us with up to 8 segments, 49.9 with up to 32, 52.3 with 64: a segment's start walks the states in
    // front of it)
    const int64_t segs = std::max<int64_t>(1, std::min<int64_t>({MOST_SEGS, 256 * wgs / owners, q.chunks < 6 ? 1 : q.chunks / 2}));
    q.per = (int) ((q.chunks + segs - 1) / segs);
    q.segs = (q.chunks + q.per - 1) / q.per;
    // their states in as many pieces as fill those of the state kernel's, of 4 chunks at least (2: 2051 float32 rows of 64 heads of
    // 64 x 128 76.1 us for 73.6)
    q.sub = q.segs == 1 ? 1 : (int) std::max<int64_t>(1, std::min<int64_t>(q.per / 4, (768 + owners * (q.segs - 1) - 1) / (owners * (q.segs - 1))));
    q.piece = (q.per + q.sub - 1) / q.sub;
    int64_t at = 0;
    auto take = [&](int64_t floats) {
        const int64_t here = at;
        at += (floats + 3) / 4 * 4;
        return here;
    };
    q.ops = take(q.chunks * G * op_bytes(q.kk) / 4);
    q.scales = take(q.chunks * G * 2);
    q.hdr = take(q.chunks * H * HDR);
    q.hist = take(3 * (H * P + 2 * G * N));
    const int64_t pieces = (q.segs - 1) * (int64_t) q.sub;
    q.segst = take(pieces ? (1 + pieces) * owners * 64 * q.kk * 32 : 0);
    q.segtot = take(pieces * H);
    q.floats = at;
    return q;
}

// column tiles of 16 a work-group: what a head's fewest work-groups of up to 4 share out evenly (bfloat16 rows: 796 of 128 heads of
// 80 x 128 58.7 us with 3 tiles a work-group, 65.3 with 4; 4096 of 64 heads of 32 x 128 66.7 with 2, 89.8 with 4, of 32 x 256 146.8 and 193.8)
template <int QT, int KT, bool STATE>
void launch_scan(ns_gpu* g, const ScanParams& s, unsigned blocks) {
    const int tiles = ((s.l.P + 15) / 16 + s.blocks - 1) / s.blocks;
    if (tiles <= 2) ssm_scan_kernel<QT, KT, 2, STATE><<<blocks, 256, 0, g->q>>>(s);
    else if (tiles == 3) ssm_scan_kernel<QT, KT, 3, STATE><<<blocks, 256, 0, g->q>>>(s);
    else ssm_scan_kernel<QT, KT, 4, STATE><<<blocks, 256, 0, g->q>>>(s);
}

template <int QT, int KT>
void launch_pass(ns_gpu* g, ScanParams& s, const Plan& q) {
    const int64_t waves = (int64_t) q.chunks * s.l.H + (s.t0 ? 0 : (3 * (int64_t) s.l.H * s.l.P + 63) / 64);
    ssm_prep_kernel<QT, KT><<<(unsigned) (q.chunks * s.l.G + (waves + 7) / 8), 512, 0, g->q>>>(s);
    const unsigned owners = (unsigned) (s.l.H * q.blocks);
    if (q.segs > 1) {
        ScanParams f = s;
        f.segs = (q.segs - 1) * q.sub;      // (the last segment's state is the scan's own)
        launch_scan<QT, KT, true>(g, f, owners * f.segs);
    }
    launch_scan<QT, KT, false>(g, s, owners * q.segs);
}

template <int QT>
void run_prompt(ns_gpu* g, const SsmLayer& p, int64_t T, float* scratch) {
    for (int64_t t0 = 0; t0 < T; t0 += PASS_ROWS) {
        const int64_t n = std::min(PASS_ROWS, T - t0);
        const Plan q = plan_of(n, p.H, p.P, p.N, p.G, p.N <= 128 ? SCAN_WGS<QT, 2, false> : SCAN_WGS<QT, 4, false>);
        ScanParams s{p, t0, T, p.p0 % p.cap, (int) n, q.chunks, q.segs, q.per, q.sub, q.piece, q.blocks};
        s.vec_y = p.P % 4 == 0;
        s.vec_h = p.N % 4 == 0 && (uintptr_t) p.h0 % 16 == 0 && (uintptr_t) p.h1 % 16 == 0;
        s.ops = reinterpret_cast<uint8_t*>(scratch + q.ops);
        s.scales = scratch + q.scales, s.hdr = scratch + q.hdr, s.hist = scratch + q.hist, s.segst = scratch + q.segst, s.segtot = scratch + q.segtot;
        if (q.kk == 2) launch_pass<QT, 1>(g, s, q);
        else if (q.kk == 4) launch_pass<QT, 2>(g, s, q);
        else launch_pass<QT, 4>(g, s, q);
    }
}

}  // namespace

extern "C" {

int64_t ns_ssm_prompt_scratch(int64_t T, int64_t H, int64_t P, int64_t N, int64_t G, int64_t K) {
    if (T <= 0 || !ns_ssm_sizes(H, P, N, G) || K < 1 || K > 4) return 0;
    // (whatever the rows' type; and a last pass of fewer rows may be cut in more segments than a full one)
    int64_t most = 0;
    for (int wgs = 1; wgs <= 3; ++wgs) {
        most = std::max(most, plan_of(std::min(T, PASS_ROWS), H, P, N, G, wgs).floats);
        if (T > PASS_ROWS && T % PASS_ROWS) most = std::max(most, plan_of(T % PASS_ROWS, H, P, N, G, wgs).floats);
    }
    return most;
}

int ns_ssm_prompt(ns_gpu* g, int qt, const void* xbc, int64_t xs, const void* dt, int64_t dts, const float* cw, const float* cb, const float* a,
                  const float* dtb, const float* d, float dt_lo, float dt_hi, float* conv, int64_t cap, int64_t p0, int64_t T, int64_t H,
                  int64_t P, int64_t N, int64_t G, int64_t K, const float* h0, float* h1, void* y, int64_t ys, float* scratch) {
    NS_TRY
    if (T <= 0) return 0;
    SsmLayer p{xbc, dt, xs, dts, cw, cb, a, dtb, d, dt_lo, dt_hi, conv, cap, p0, (int) H, (int) P, (int) N, (int) G, (int) K, 0, h0, h1, y, ys};
    if (ns_ssm_check("ns_ssm_prompt", g, qt, p, H, P, N, G, K, K - 1)) return -1;
    if (!scratch) return ns_fail("ns_ssm_prompt: a null buffer");
    if (xs > (int64_t) 1 << 23) return ns_fail("ns_ssm_prompt: rows up to 2^23 values apart");
    if ((uintptr_t) scratch % 16) return ns_fail("ns_ssm_prompt: scratch 16-byte aligned");
    p.chan = (int) (H * P + 2 * G * N);
    if (K == 1) p.conv = nullptr, p.cap = 1;
    NS_HIP(hipSetDevice(g->dev));
    if (T <= FEW_ROWS && p.cap >= K - 1 + (K > 1 ? T : 0) && p.cap <= INT32_MAX) ns_ssm_few(g, qt, p, (int) T);
    else if (qt == 0) run_prompt<0>(g, p, T, scratch);
    else if (qt == 1) run_prompt<1>(g, p, T, scratch);
    else run_prompt<2>(g, p, T, scratch);
    NS_LAUNCHED("ssm_prompt");
    return 0;
    NS_CATCH
}

}  // extern "C"
