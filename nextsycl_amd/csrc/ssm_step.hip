// ssm_step.hip: a token, or a few successive ones, of each of several sequences through a state-space layer's convolution
// and recurrence (ns_ssm_step).
//
// A row's head: h = exp(dt a) h + dt x (outer) B, y = h C + d x over a state of P x N floats that nothing else of the call
// touches. Bound: HBM - the state is read and written once (8 H P N bytes a sequence, 8.4 MB at 128 heads of 64 x 128) for
// 5 operations a float. So a lane holds 4 consecutive features of a few of the head's P rows and asks for them right behind
// what the convolution reads, which (a few hundred channels, each group's B and C by every head of the group: 4 multiply-adds and
// a few KB that the cache holds) runs while they are on their way; y is a sum over a row's lanes. Rows of one slot
// are walked with the state in registers, their convolutions four rows at a time.
// 128 heads of 64 x 128: 64 tokens (548 MB) 107 - 109 us, 5.1 TB/s - a copy's rate; one token 5.4 us, a launch and the two latencies of
// its loads and sums (1.6 us of bytes); 12 half rows of 3 slots, 128 heads of 80 x 128, 14.7 us (33 MB: 6.3): a row of each 9.3, each further
// row 1.9. Four work-groups a CU (those
// rows with three, 8 state rows a lane: 17.0, for 15.8), four rows at a time (two: 16.5).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "ns_internal.hpp"
#include "ns_layer.h"
#include "layer_common.hpp"

namespace {

constexpr int64_t MOST_ROWS = 4096;

// The sums over each run of LR lanes of U values, value lane / (LR / U) in a lane: at each step two values' halves of the run
// change places, so that U values take U - 1 additions (and as many exchanges) until one a lane is left, not U each. (The lanes of a value are
// added in lanes_sum's order, whatever U: a state row's sum has the same bits from every instance)
template <int LR, int U>
__device__ __forceinline__ float lanes_sums(const float (&v)[U], int lane) {
    if constexpr (U == 1) return lanes_sum<LR>(v[0]);
    else {
        float w[U / 2];
#pragma unroll
        for (int u = 0; u < U / 2; ++u) {
            const float a = v[u], b = v[u + U / 2];
            if constexpr (LR >= 32) {
                const uint32_t x = __builtin_bit_cast(uint32_t, a), y = __builtin_bit_cast(uint32_t, b);
                const auto r = LR == 64 ? __builtin_amdgcn_permlane32_swap(x, y, false, false) : __builtin_amdgcn_permlane16_swap(x, y, false, false);
                w[u] = __builtin_bit_cast(float, (uint32_t) r[0]) + __builtin_bit_cast(float, (uint32_t) r[1]);
            } else {
                const bool upper = lane & LR / 2;
                const float mine = upper ? b : a, other = upper ? a : b;
                static_assert(LR == 16 || LR == 8);
                w[u] = mine + __builtin_bit_cast(float, dpp_u32<LR == 16 ? 0x140 : 0x141>(__builtin_bit_cast(uint32_t, other)));
            }
        }
        return lanes_sums<LR / 2, U / 2>(w, lane);
    }
}

struct StepParams {
    SsmLayer l;
    const int32_t *pos, *slots;
    int64_t nslots;
    int R, pblocks;
    int one;              // all R rows are one sequence's, as a short prompt's are: of those only the last K - 1 go into the ring
};

// LR lanes a state row, U rows a lane; VEC: a lane's 4 floats as one piece
template <int QT, int LR, int U, bool VEC>
__global__ __launch_bounds__(256, VEC ? 4 : 3) void ssm_step_kernel(StepParams s) {
    constexpr int RW = 256 / LR, PB = RW * U, UP = U > 4 ? 8 : U, AHEAD = 4, NMAX = 4 * LR, CH = (2 * NMAX + PB + 255) / 256;
    __shared__ __align__(16) float row_in[AHEAD][2 * NMAX + PB];      // B, C, the block's x of a row
    __shared__ float step[AHEAD][2];                                  // its step size and decay
    __shared__ uint64_t mine[MOST_ROWS / 64];
    __shared__ uint16_t list[MOST_ROWS];
    const SsmLayer& p = s.l;
    const int tid = threadIdx.x, lane = tid % 64, head = blockIdx.x / s.pblocks, pb = blockIdx.x % s.pblocks, r0 = blockIdx.y;
    const int group = head / (p.H / p.G), n0 = tid % LR * 4, prow = pb * PB + tid / LR;
    const int64_t slot = s.slots ? s.slots[r0] : r0;
    const int64_t first = s.pos ? (int64_t) s.pos[r0] : p.p0;
    if (slot < 0 || slot >= s.nslots || first < 0) return;
    // the slot's rows in their order, as many as its ring has room for: this work-group is the first's, or has nothing to do
    const int cap = (int) p.cap;
    int count = s.one ? s.R : 1;
    if (s.slots) {
        for (int w = tid / 64; w * 64 < s.R; w += 4) {
            const int at = w * 64 + lane;
            const uint64_t m = __ballot(at < s.R && s.slots[at < s.R ? at : 0] == (int32_t) slot);
            if (lane == 0) mine[w] = m;
        }
        __syncthreads();
        for (int w = 0; w <= r0 / 64; ++w) {
            const uint64_t m = w == r0 / 64 ? mine[w] & (((uint64_t) 1 << r0 % 64) - 1) : mine[w];
            if (m) return;
        }
        const int most = p.K > 1 ? cap - p.K + 1 : s.R;
        count = 0;
        for (int w = r0 / 64; w * 64 < s.R; ++w) {
            const uint64_t m = mine[w];
            const int rank = count + __builtin_popcountll(m & (((uint64_t) 1 << lane) - 1));
            if (tid < 64 && (m >> lane & 1) && rank < most) list[rank] = (uint16_t) (w * 64 + lane);
            count += __builtin_popcountll(m);
        }
        count = min(count, most);
        if (count > 1) __syncthreads();
    }
    auto row_of = [&](int i) { return s.slots && count > 1 ? (int64_t) list[i] : (int64_t) (r0 + i); };
    const int kept_from = s.one ? count - (p.K - 1) : 0;
    // this thread's channels: B, C, then the block's part of x; their taps and the raw values in front of the first row
    int ch[CH];
    float w4[CH][4], bias[CH], past[CH][3];
    int to[CH];
    bool keep[CH];
    // the ring's slot of the first row (one division, of 32 bits where they do), those behind it one further each
    const int slot0 = (uint64_t) first >> 32 ? (int) (first % p.cap) : (int) ((uint32_t) first % (uint32_t) cap);
    float* ring = p.conv + slot * p.cap * p.chan;
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        const int c = tid + 256 * j;
        ch[j] = -1, to[j] = c < 2 * NMAX + PB ? c : -1, keep[j] = false;
        if (c < NMAX) {
            if (c < p.N) ch[j] = p.H * p.P + group * p.N + c;
            keep[j] = true;
        } else if (c < 2 * NMAX) {
            if (c - NMAX < p.N) ch[j] = p.H * p.P + (p.G + group) * p.N + c - NMAX;
            keep[j] = true;
        } else if (c < 2 * NMAX + PB) {
            const int pr = pb * PB + c - 2 * NMAX;
            if (pr < p.P) ch[j] = head * p.P + pr;
        }
        // a group's B and C are kept by its first head's first block, x by its own
        keep[j] = ch[j] >= 0 && p.K > 1 && (!keep[j] || (head % (p.H / p.G) == 0 && pb == 0));
#pragma unroll
        for (int k = 0; k < 4; ++k) w4[j][k] = ch[j] >= 0 ? ssm_tap(p, ch[j], k) : 0.0f;
        bias[j] = ch[j] >= 0 && p.cb ? p.cb[ch[j]] : 0.0f;
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            const int at = slot0 - 3 + k;
            past[j][k] = ch[j] >= 0 && k >= 4 - p.K && first - 3 + k >= 0 ? ring[(int64_t) (at < 0 ? at + cap : at) * p.chan + ch[j]] : 0.0f;
        }
    }
    const float rate = p.a[head], skip = p.d ? p.d[head] : 0.0f, dtb = p.dtb ? p.dtb[head] : 0.0f;
    // (a lane a row, of the wave that has no channels of x)
    float raw[AHEAD][CH], size = 0.0f;
    auto fetch = [&](int i0) {
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            if (i0 + a >= count) break;
            const int64_t r = row_of(i0 + a);
#pragma unroll
            for (int j = 0; j < CH; ++j) raw[a][j] = ch[j] >= 0 ? load_q<QT>(p.xbc, r * p.xs + ch[j]) : 0.0f;
        }
        if (tid >= 192 && lane < AHEAD && i0 + lane < count) size = load_q<QT>(p.dt, row_of(i0 + lane) * p.dts + head);
    };
    fetch(0);
    // the state, asked for last: the convolution waits for what it reads alone (a load a piece whatever the lane, so that their number is known:
    // what a lane has no place for is a neighbour's, and set to 0 before its first use)
    float h[U][4];
    const int64_t hrow = (slot * p.H + head) * p.P;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int pr = prow + u * RW;
        if constexpr (VEC) {
            const floats4_t v = *reinterpret_cast<const floats4_t*>((p.h0 ? p.h0 : p.h1) + (hrow + min(pr, p.P - 1)) * p.N + (n0 < p.N ? n0 : 0));
            h[u][0] = v.x, h[u][1] = v.y, h[u][2] = v.z, h[u][3] = v.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) h[u][i] = p.h0 && pr < p.P && n0 + i < p.N ? p.h0[(hrow + pr) * p.N + n0 + i] : 0.0f;
        }
    }
    int here = slot0;
    for (int i0 = 0; i0 < count; i0 += AHEAD) {
        // four rows at a time: their convolutions and step sizes, in LDS, then the state through them
        const int rows = min(AHEAD, count - i0);
        if (i0) lds_barrier();           // the rows before have been read
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            if (a >= rows) break;
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                if (to[j] < 0) continue;
                const float v = raw[a][j];
                row_in[a][to[j]] = ch[j] >= 0 ? silu(fmaf(w4[j][3], v, fmaf(w4[j][2], past[j][2], fmaf(w4[j][1], past[j][1], fmaf(w4[j][0], past[j][0], bias[j]))))) : 0.0f;
                // (of taps that there are not: 0 times what is not finite is not 0)
                past[j][0] = p.K > 3 ? past[j][1] : 0.0f, past[j][1] = p.K > 2 ? past[j][2] : 0.0f, past[j][2] = p.K > 1 ? v : 0.0f;
                if (keep[j] && i0 + a >= kept_from) ring[(int64_t) here * p.chan + ch[j]] = v;
            }
            here = here + 1 == cap ? 0 : here + 1;
        }
        if (tid >= 192 && lane < rows) {
            const float dt = ssm_dt(p, size + dtb);
            step[lane][0] = dt, step[lane][1] = expf(dt * rate);
        }
        lds_barrier();
        if (i0 + AHEAD < count) fetch(i0 + AHEAD);
        if (VEC && i0 == 0 && (!p.h0 || n0 >= p.N)) {
#pragma unroll
            for (int u = 0; u < U; ++u) h[u][0] = h[u][1] = h[u][2] = h[u][3] = 0.0f;
        }
        for (int a = 0; a < rows; ++a) {
            const float dt = step[a][0], decay = step[a][1];
            const float4 b = *reinterpret_cast<const float4*>(row_in[a] + n0), c = *reinterpret_cast<const float4*>(row_in[a] + NMAX + n0);
            const float bx = dt * b.x, by = dt * b.y, bz = dt * b.z, bw = dt * b.w;
            float sum[UP] = {};
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float x = row_in[a][2 * NMAX + tid / LR + u * RW];
                h[u][0] = fmaf(h[u][0], decay, x * bx), h[u][1] = fmaf(h[u][1], decay, x * by);
                h[u][2] = fmaf(h[u][2], decay, x * bz), h[u][3] = fmaf(h[u][3], decay, x * bw);
                sum[u] = fmaf(h[u][3], c.w, fmaf(h[u][2], c.z, fmaf(h[u][1], c.y, h[u][0] * c.x)));
            }
            // (a lane then holds the sum of one of its U state rows; the first of those that hold the same one writes it)
            const int mine_u = tid % LR / (LR / UP), mine_p = prow + mine_u * RW;
            const float out = fmaf(skip, row_in[a][2 * NMAX + tid / LR + min(mine_u, U - 1) * RW], lanes_sums<LR, UP>(sum, lane));
            if (tid % (LR / UP) == 0 && mine_u < U && mine_p < p.P) store_o<QT>(p.y, row_of(i0 + a) * p.ys + head * p.P + mine_p, out);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int pr = prow + u * RW;
        if (pr >= p.P) continue;
        float* dst = p.h1 + (hrow + pr) * p.N + n0;
        if constexpr (VEC) {
            if (n0 < p.N) *reinterpret_cast<floats4_t*>(dst) = floats4_t{h[u][0], h[u][1], h[u][2], h[u][3]};
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n0 + i < p.N) dst[i] = h[u][i];
        }
    }
}

template <int QT, int LR, int U>
void launch_step(ns_gpu* g, StepParams& s, bool vec) {
    s.pblocks = (s.l.P + 256 / LR * U - 1) / (256 / LR * U);
    const dim3 grid((unsigned) (s.l.H * s.pblocks), (unsigned) (s.one ? 1 : s.R));
    if (vec) ssm_step_kernel<QT, LR, U, true><<<grid, 256, 0, g->q>>>(s);
    else ssm_step_kernel<QT, LR, U, false><<<grid, 256, 0, g->q>>>(s);
}
template <int QT>
void launch_step(ns_gpu* g, StepParams& s, bool vec) {
    const int N = s.l.N;
    if (N <= 16) launch_step<QT, 4, 1>(g, s, vec);
    else if (N <= 32) launch_step<QT, 8, 2>(g, s, vec);
    else if (N <= 64) launch_step<QT, 16, 4>(g, s, vec);
    else if (N <= 128) {
        // as many state rows a lane as share a head's out evenly, 8 at most, and 4 while there is no work-group of more for each CU (12 half rows
        // of 3 slots, heads of 80, 14.7 us with 5 of them, 16.2 with 8 and 4; 20 tokens, heads of 32, 18.4 with 4, 20.1 with 8; a token, heads of
        // 64, 5.5 with 4, 6.0 with 8; 64 of them 107 with 8, 115 with 4)
        const int per = 64 * ((s.l.P + 63) / 64), need = (s.l.P + per / 8 - 1) / (per / 8);
        if (need <= 4 || (int64_t) s.l.H * (per / 64) * (s.one ? 1 : s.R) <= 128) launch_step<QT, 32, 4>(g, s, vec);
        else if (need == 5) launch_step<QT, 32, 5>(g, s, vec);
        else if (need == 6) launch_step<QT, 32, 6>(g, s, vec);
        else launch_step<QT, 32, 8>(g, s, vec);
    }
    else launch_step<QT, 64, 4>(g, s, vec);
}

void launch_step(ns_gpu* g, int qt, StepParams& s) {
    const bool vec = s.l.N % 4 == 0;
    if (qt == 0) launch_step<0>(g, s, vec);
    else if (qt == 1) launch_step<1>(g, s, vec);
    else launch_step<2>(g, s, vec);
}

}  // namespace

void ns_ssm_few(ns_gpu* g, int qt, const SsmLayer& p, int rows) {
    StepParams s{};
    s.l = p, s.nslots = 1, s.R = rows, s.one = 1;
    launch_step(g, qt, s);
}

// what the two state-space calls refuse alike
int ns_ssm_check(const char* who, ns_gpu* g, int qt, const SsmLayer& p, int64_t H, int64_t P, int64_t N, int64_t G, int64_t K,
                 int64_t least) {
    const std::string s(who);
    if (qt < 0 || qt > 2) return ns_fail(s + ": rows of type 0 (float32), 1 (half) or 2 (bfloat16)");
    if (!ns_ssm_sizes(H, P, N, G))
        return ns_fail(s + ": heads a multiple of the groups, a state of 1 to 256 features, up to 2^24 channels");
    if (K < 1 || K > 4) return ns_fail(s + ": 1 to 4 taps");
    if (p.xs < H * P + 2 * G * N || p.dts < H || p.ys < H * P) return ns_fail(s + ": rows at least as far apart as they are long");
    if (!(p.lo <= p.hi)) return ns_fail(s + ": step sizes between dt_lo and dt_hi");
    if (p.p0 < 0 || p.p0 > INT64_MAX / 2) return ns_fail(s + ": positions from 0 to 2^62");
    if (K > 1 && p.cap < least) return ns_fail(s + ": a ring of at least " + std::to_string(least) + " rows");
    if (!g || !p.xbc || !p.dt || !p.cw || !p.a || !p.h1 || !p.y || (K > 1 && !p.conv)) return ns_fail(s + ": a null buffer");
    return 0;
}

extern "C" int ns_ssm_step(ns_gpu* g, int qt, const void* xbc, int64_t xs, const void* dt, int64_t dts, const float* cw, const float* cb,
                           const float* a, const float* dtb, const float* d, float dt_lo, float dt_hi, float* conv, int64_t cap, int64_t p0,
                           const int32_t* pos, const int32_t* slots, int64_t nslots, int64_t R, int64_t H, int64_t P, int64_t N, int64_t G,
                           int64_t K, const float* h0, float* h1, void* y, int64_t ys) {
    NS_TRY
    if (R <= 0) return 0;
    StepParams s{};
    s.l = SsmLayer{xbc, dt, xs, dts, cw, cb, a, dtb, d, dt_lo, dt_hi, conv, cap, p0, (int) H, (int) P, (int) N, (int) G, (int) K, 0, h0, h1, y, ys};
    if (R > MOST_ROWS) return ns_fail("ns_ssm_step: up to 4096 rows");
    if (nslots <= 0 || (!slots && R > nslots) || nslots > INT32_MAX) return ns_fail("ns_ssm_step: more rows than slots");
    if (ns_ssm_check("ns_ssm_step", g, qt, s.l, H, P, N, G, K, K)) return -1;
    if (cap > INT32_MAX) return ns_fail("ns_ssm_step: a ring of up to 2^31 - 1 rows");
    if (K == 1) s.l.conv = nullptr, s.l.cap = 1;      // (nothing is kept)
    s.l.chan = (int) (H * P + 2 * G * N);
    s.pos = pos, s.slots = slots, s.nslots = nslots, s.R = (int) R;
    NS_HIP(hipSetDevice(g->dev));
    launch_step(g, qt, s);
    NS_LAUNCHED("ssm_step");
    return 0;
    NS_CATCH
}
