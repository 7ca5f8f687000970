// norm_rows.hip: the norms around a block of a layer - the gated group norm behind the scan (ns_norm_gated), and a block's
// output into the residual stream with the norm in front of the next block (ns_norm_residual).
//
// Bound: HBM for prompts (each row read once and written once: 6 bytes a value of bfloat16 rows for the gated norm), a
// launch and one memory latency for a token. A unit - a group of a row, or a row - is held in registers by 1 to 16
// waves, so nothing is read twice; sums of squares and everything between load and store are float32, rounded once at
// the end. A unit of more than 4096 pieces of 16 bytes is read twice.
// 8192 bfloat16 rows of 8192 in 8 groups 73 us (403 MB, 5.5 TB/s; a large copy 5.1), 4001 bfloat16 rows of 5120 into a float32 stream
// with both norms and a gate 52 us (246 MB, 4.7 TB/s: two sums over a row's waves, each in front of the next step); a token's
// row 3.0 - 3.3 us of kernel, 4.2 a call.
#include <algorithm>
#include <type_traits>

#include "ns_internal.hpp"
#include "ns_layer.h"
#include "layer_common.hpp"

namespace {

// the sum over a unit's threads, in all of them (WIDE: a unit is its whole block; else a wave)
template <bool WIDE>
__device__ __forceinline__ float unit_sum(float v, float* part) {
    v = wave_sum(v);
    if constexpr (WIDE) {
        __syncthreads();                 // (what an earlier sum of the unit left has been read)
        if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = v;
        __syncthreads();
        v = 0.0f;
        for (int i = 0; i < (int) blockDim.x / 64; ++i) v += part[i];
    }
    return v;
}
// VEC weights from element i on, or ones
template <int VEC, bool TAIL>
__device__ __forceinline__ void load_weights(const float* w, int64_t i, int left, float (&v)[VEC]) {
    if (w) load_piece<0, VEC, TAIL>(w, i, left, v);
    else
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = 1.0f;
}
__device__ __forceinline__ float inverse_root(float sum, int n, float eps) { return 1.0f / sqrtf(sum / (float) n + eps); }

struct GatedParams {
    const void *y, *z;
    const float* w;
    void* out;
    int64_t ys, zs, os, units;
    int W, groups, order;
    float eps;
};

// IT pieces of VEC values a thread (TAIL: the unit's last is not whole); IT 0: any number, read twice
template <int QT, int VEC, bool TAIL, bool WIDE, int IT>
__global__ __launch_bounds__(WIDE ? 1024 : 256) void norm_gated_kernel(GatedParams p) {
    __shared__ float part[16];
    const int tpu = WIDE ? blockDim.x : 64, tid = WIDE ? threadIdx.x : threadIdx.x % 64;
    const int64_t unit = WIDE ? blockIdx.x : (int64_t) blockIdx.x * (blockDim.x / 64) + threadIdx.x / 64;
    if (unit >= p.units) return;         // (whole waves; a unit of more than one is its whole block)
    const int64_t t = unit / p.groups, c0 = unit % p.groups * p.W;
    auto values = [&](int at, float (&v)[VEC], float (&s)[VEC]) {
        load_piece<QT, VEC, TAIL>(p.y, t * p.ys + c0 + at, p.W - at, v);
        load_piece<QT, VEC, TAIL>(p.z, t * p.zs + c0 + at, p.W - at, s);
    };
    auto result = [&](int at, float (&v)[VEC], const float (&s)[VEC], float inv) {
        float w[VEC];
        load_weights<VEC, TAIL>(p.w, c0 + at, p.W - at, w);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] *= p.order ? inv * w[j] * s[j] : inv * w[j];
        store_piece<QT, VEC, TAIL>(p.out, t * p.os + c0 + at, p.W - at, v);
    };
    float sum = 0.0f;
    auto square = [&](float (&v)[VEC], float (&s)[VEC]) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            s[j] = silu(s[j]);
            if (!p.order) v[j] *= s[j];
            sum = fmaf(v[j], v[j], sum);
        }
    };
    if constexpr (IT > 0) {
        float v[IT][VEC], s[IT][VEC];
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int at = (i * tpu + tid) * VEC;
            if (at < p.W) values(at, v[i], s[i]);
        }
#pragma unroll
        for (int i = 0; i < IT; ++i)
            if ((i * tpu + tid) * VEC < p.W) square(v[i], s[i]);
        const float inv = inverse_root(unit_sum<WIDE>(sum, part), p.W, p.eps);
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int at = (i * tpu + tid) * VEC;
            if (at < p.W) result(at, v[i], s[i], inv);
        }
    } else {
        float v[VEC], s[VEC];
        for (int at = tid * VEC; at < p.W; at += tpu * VEC) {
            values(at, v, s);
            square(v, s);
        }
        const float inv = inverse_root(unit_sum<WIDE>(sum, part), p.W, p.eps);
        for (int at = tid * VEC; at < p.W; at += tpu * VEC) {
            values(at, v, s);
            square(v, s);
            result(at, v, s, inv);
        }
    }
}

struct ResidualParams {
    const void *x, *h;
    const float *post, *gate, *pre;
    void *h1, *out;
    int64_t xs, hs, h1s, os, T;
    int D;
    float eps, scale;
};

template <int QT, int RT, int VEC, bool TAIL, bool WIDE, int IT>
__global__ __launch_bounds__(WIDE ? 1024 : 256) void norm_residual_kernel(ResidualParams p) {
    __shared__ float part[16];
    const int tpu = WIDE ? blockDim.x : 64, tid = WIDE ? threadIdx.x : threadIdx.x % 64;
    const int64_t t = WIDE ? blockIdx.x : (int64_t) blockIdx.x * (blockDim.x / 64) + threadIdx.x / 64;
    if (t >= p.T) return;
    auto load_x = [&](int at, float (&v)[VEC]) {
        if (p.x) load_piece<QT, VEC, TAIL>(p.x, t * p.xs + at, p.D - at, v);
        else
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = 0.0f;
    };
    // s = h + scale gate post (x inv)
    auto stream = [&](int at, float (&v)[VEC], const float (&h)[VEC], float inv) {
        if (!p.x) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = h[j];
            return;
        }
        float w[VEC];
        if (p.post) {
            load_weights<VEC, TAIL>(p.post, at, p.D - at, w);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = v[j] * inv * w[j];
        }
        if (p.gate) {
            load_weights<VEC, TAIL>(p.gate, at, p.D - at, w);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] *= w[j];
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = fmaf(p.scale, v[j], h[j]);
    };
    auto result = [&](int at, float (&v)[VEC], float inv) {
        float w[VEC];
        load_weights<VEC, TAIL>(p.pre, at, p.D - at, w);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = v[j] * inv * w[j];
        store_piece<QT, VEC, TAIL>(p.out, t * p.os + at, p.D - at, v);
    };
    auto squares = [&](const float (&v)[VEC]) {
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum = fmaf(v[j], v[j], sum);
        return sum;
    };
    if constexpr (IT > 0) {
        float v[IT][VEC], h[IT][VEC];
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int at = (i * tpu + tid) * VEC;
            if (at < p.D) {
                load_x(at, v[i]);
                load_piece<RT, VEC, TAIL>(p.h, t * p.hs + at, p.D - at, h[i]);
            }
        }
        float inv = 1.0f;
        if (p.post) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < IT; ++i)
                if ((i * tpu + tid) * VEC < p.D) sum += squares(v[i]);
            inv = inverse_root(unit_sum<WIDE>(sum, part), p.D, p.eps);
        }
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int at = (i * tpu + tid) * VEC;
            if (at >= p.D) continue;
            stream(at, v[i], h[i], inv);
            sum += squares(v[i]);
            if (p.h1) store_piece<RT, VEC, TAIL>(p.h1, t * p.h1s + at, p.D - at, v[i]);
        }
        if (!p.out) return;
        inv = inverse_root(unit_sum<WIDE>(sum, part), p.D, p.eps);
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int at = (i * tpu + tid) * VEC;
            if (at < p.D) result(at, v[i], inv);
        }
    } else {
        // too long for registers: x and h are read again for each step, the stream written last (h1 may be h)
        float v[VEC], h[VEC], inv = 1.0f, sum = 0.0f;
        if (p.post) {
            for (int at = tid * VEC; at < p.D; at += tpu * VEC) {
                load_x(at, v);
                sum += squares(v);
            }
            inv = inverse_root(unit_sum<WIDE>(sum, part), p.D, p.eps);
            sum = 0.0f;
        }
        for (int at = tid * VEC; at < p.D; at += tpu * VEC) {
            load_x(at, v);
            load_piece<RT, VEC, TAIL>(p.h, t * p.hs + at, p.D - at, h);
            stream(at, v, h, inv);
            sum += squares(v);
        }
        const float inv2 = inverse_root(unit_sum<WIDE>(sum, part), p.D, p.eps);
        for (int at = tid * VEC; at < p.D; at += tpu * VEC) {
            load_x(at, v);
            load_piece<RT, VEC, TAIL>(p.h, t * p.hs + at, p.D - at, h);
            stream(at, v, h, inv);
            if (p.h1) store_piece<RT, VEC, TAIL>(p.h1, t * p.h1s + at, p.D - at, v);
            if (p.out) result(at, v, inv2);
        }
    }
}

// How `units` units of n pieces run: f(WIDE, IT, threads a block, blocks). A wave a unit of up to 64 pieces, in blocks of 4 waves; longer
// ones a block of as many waves as leave a thread one piece, and more only where 16 waves do not do: with two pieces a thread there are
// fewer waves to ask for memory (65536 groups of 128 pieces 77.5 us as a wave's two each, 72.7 as two waves; 4001 rows of 640 pieces
// 54.9 and 52.2)
template <typename F>
void by_size(int64_t n, int64_t units, F f) {
    using std::false_type, std::true_type, std::integral_constant;
    if (n <= 64) return f(false_type(), integral_constant<int, 1>(), 256, (units + 3) / 4);
    if (n <= 1024) return f(true_type(), integral_constant<int, 1>(), (int) ((n + 63) / 64 * 64), units);
    if (n <= 2048) return f(true_type(), integral_constant<int, 2>(), (int) ((n + 127) / 128 * 64), units);
    if (n <= 4096) return f(true_type(), integral_constant<int, 4>(), 1024, units);
    return f(true_type(), integral_constant<int, 0>(), 1024, units);
}

// Pieces of 16 bytes of the rows' type, wherever rows start; where the last is not whole and a wave's lanes have room for all of a unit one by
// one, single values (17048 groups of 35 half values 5.2 us, 9.9 in pieces; 4608 groups of 541 13.1 us in pieces, 28.6 one by one)
template <int VEC>
bool one_by_one(int64_t n) { return n % VEC && n <= 64; }
template <int QT, int VEC, bool TAIL>
void launch_gated(ns_gpu* g, const GatedParams& p) {
    by_size((p.W + VEC - 1) / VEC, p.units, [&](auto wide, auto it, int threads, int64_t blocks) {
        if constexpr (VEC > 1 || (!decltype(wide)::value && decltype(it)::value == 1))
            norm_gated_kernel<QT, VEC, TAIL, decltype(wide)::value, decltype(it)::value><<<(unsigned) blocks, threads, 0, g->q>>>(p);
    });
}
template <int QT>
void launch_gated(ns_gpu* g, const GatedParams& p) {
    constexpr int VEC = QT ? 8 : 4;
    return one_by_one<VEC>(p.W) ? launch_gated<QT, 1, false>(g, p) : p.W % VEC ? launch_gated<QT, VEC, true>(g, p) : launch_gated<QT, VEC, false>(g, p);
}
template <int QT, int RT, int VEC, bool TAIL>
void launch_residual(ns_gpu* g, const ResidualParams& p) {
    by_size((p.D + VEC - 1) / VEC, p.T, [&](auto wide, auto it, int threads, int64_t blocks) {
        if constexpr (VEC > 1 || (!decltype(wide)::value && decltype(it)::value == 1))
            norm_residual_kernel<QT, RT, VEC, TAIL, decltype(wide)::value, decltype(it)::value><<<(unsigned) blocks, threads, 0, g->q>>>(p);
    });
}
template <int QT, int RT>
void launch_residual(ns_gpu* g, const ResidualParams& p) {
    constexpr int VEC = QT ? 8 : 4;
    return one_by_one<VEC>(p.D) ? launch_residual<QT, RT, 1, false>(g, p) : p.D % VEC ? launch_residual<QT, RT, VEC, true>(g, p) : launch_residual<QT, RT, VEC, false>(g, p);
}

// whether `units` units of n values run in one launch
bool one_launch(int qt, int64_t n, int64_t units) {
    const int64_t vec = qt ? 8 : 4;
    bool fits = units <= (int64_t) 1 << 40;
    if (fits) by_size((qt ? one_by_one<8>(n) : one_by_one<4>(n)) ? n : (n + vec - 1) / vec, units, [&](auto, auto, int threads, int64_t blocks) { fits = ns_grid_fits(blocks, threads); });
    return fits;
}

}  // namespace

extern "C" {

int ns_norm_gated(ns_gpu* g, int qt, const void* y, int64_t ys, const void* z, int64_t zs, const float* w, void* out, int64_t os, int64_t T,
                  int64_t D, int64_t groups, float eps, int order) {
    NS_TRY
    if (T <= 0 || D <= 0) return 0;
    if (qt < 0 || qt > 2) return ns_fail("ns_norm_gated: rows of type 0 (float32), 1 (half) or 2 (bfloat16)");
    if (groups <= 0 || D % groups || D > (int64_t) 1 << 24) return ns_fail("ns_norm_gated: up to 2^24 values in equal groups");
    if (order != 0 && order != 1) return ns_fail("ns_norm_gated: order 0 (gate, then norm) or 1 (norm, then gate)");
    if (ys < D || zs < D || os < D) return ns_fail("ns_norm_gated: rows at least as far apart as they are long");
    if (T > ((int64_t) 1 << 40) / groups || !one_launch(qt, D / groups, T * groups)) return ns_fail("ns_norm_gated: too many rows");
    if (!g || !y || !z || !out) return ns_fail("ns_norm_gated: a null buffer");
    NS_HIP(hipSetDevice(g->dev));
    const GatedParams p{y, z, w, out, ys, zs, os, T * groups, (int) (D / groups), (int) groups, order, eps};
    if (qt == 0) launch_gated<0>(g, p);
    else if (qt == 1) launch_gated<1>(g, p);
    else launch_gated<2>(g, p);
    NS_LAUNCHED("norm_gated");
    return 0;
    NS_CATCH
}

int ns_norm_residual(ns_gpu* g, int qt, int rt, const void* x, int64_t xs, const void* h, int64_t hs, void* h1, int64_t h1s, void* out, int64_t os,
                     int64_t T, int64_t D, float eps, float scale, const float* post, const float* gate, const float* pre) {
    NS_TRY
    if (T <= 0 || D <= 0) return 0;
    if (qt < 0 || qt > 2) return ns_fail("ns_norm_residual: rows of type 0 (float32), 1 (half) or 2 (bfloat16)");
    if (rt != 0 && rt != qt) return ns_fail("ns_norm_residual: a stream of float32 or of the rows' type");
    if (D > (int64_t) 1 << 24) return ns_fail("ns_norm_residual: up to 2^24 values");
    if ((x && xs < D) || hs < D || (h1 && h1s < D) || (out && os < D)) return ns_fail("ns_norm_residual: rows at least as far apart as they are long");
    if (!one_launch(qt, D, T)) return ns_fail("ns_norm_residual: too many rows");
    if (!g || !h || (!h1 && !out)) return ns_fail("ns_norm_residual: a null buffer");
    if (!x && (post || gate)) return ns_fail("ns_norm_residual: a norm or gate of no block");
    NS_HIP(hipSetDevice(g->dev));
    const ResidualParams p{x, h, post, gate, pre, h1, out, xs, hs, h1s, os, T, (int) D, eps, scale};
    if (qt == 0) launch_residual<0, 0>(g, p);
    else if (qt == 1) rt == 0 ? launch_residual<1, 0>(g, p) : launch_residual<1, 1>(g, p);
    else rt == 0 ? launch_residual<2, 0>(g, p) : launch_residual<2, 2>(g, p);
    NS_LAUNCHED("norm_residual");
    return 0;
    NS_CATCH
}

}  // extern "C"
