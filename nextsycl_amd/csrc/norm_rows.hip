// norm_rows.hip: the norms around a block of a layer - the gated group norm behind the scan (ns_norm_gated), and a block's
// output into the residual stream with the norm in front of the next block (ns_norm_residual).
//
// Bound: HBM for prompts (each row read once and written once: 6 bytes a value of bfloat16 rows for the gated norm), a
// launch and one memory latency for a token. A unit - a group of a row, or a row - is held in registers by 64, 256 or 1024
// threads, so nothing is read twice; sums of squares and everything between load and store are float32, rounded once at
// the end. A unit too long for 1024 threads' registers is read twice (ranges past 16384 to 32768 values).
#include <algorithm>
#include <type_traits>

#include "ns_internal.hpp"
#include "ns_layer.h"
#include "layer_common.hpp"

namespace {

// the sum over a unit's TPU threads, in all of them (units of more than a wave: one a block)
template <int TPU>
__device__ __forceinline__ float unit_sum(float v, float* part) {
    v = wave_sum(v);
    if constexpr (TPU > 64) {
        __syncthreads();                 // (what an earlier sum of the unit left has been read)
        if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int i = 0; i < TPU / 64; ++i) v += part[i];
    }
    return v;
}

struct GatedParams {
    const void *y, *z;
    const float* w;
    void* out;
    int64_t ys, zs, os, units;
    int W, groups, order;
    float eps;
};

// IT pieces of VEC values a thread; IT 0: any number, read twice
template <int QT, int VEC, int TPU, int IT>
__global__ __launch_bounds__(TPU > 256 ? TPU : 256) void norm_gated_kernel(GatedParams p) {
    constexpr int UNITS = TPU > 256 ? 1 : 256 / TPU;
    __shared__ float part[16];
    const int64_t unit = (int64_t) blockIdx.x * UNITS + threadIdx.x / TPU;
    if (unit >= p.units) return;         // (whole waves; a unit of more than one is its whole block)
    const int tid = threadIdx.x % TPU;
    const int64_t t = unit / p.groups, c0 = unit % p.groups * p.W;
    auto values = [&](int at, float (&v)[VEC], float (&s)[VEC]) {
        load_row<QT, VEC>(p.y, t * p.ys + c0 + at, v);
        load_row<QT, VEC>(p.z, t * p.zs + c0 + at, s);
    };
    auto result = [&](int at, float (&v)[VEC], const float (&s)[VEC], float inv) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            v[j] *= inv;
            if (p.w) v[j] *= p.w[c0 + at + j];
            if (p.order) v[j] *= s[j];
        }
        store_row<QT, VEC>(p.out, t * p.os + c0 + at, v);
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
            const int at = (i * TPU + tid) * VEC;
            if (at < p.W) values(at, v[i], s[i]);
        }
#pragma unroll
        for (int i = 0; i < IT; ++i)
            if ((i * TPU + tid) * VEC < p.W) square(v[i], s[i]);
        const float inv = 1.0f / sqrtf(unit_sum<TPU>(sum, part) / (float) p.W + p.eps);
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int at = (i * TPU + tid) * VEC;
            if (at < p.W) result(at, v[i], s[i], inv);
        }
    } else {
        float v[VEC], s[VEC];
        for (int at = tid * VEC; at < p.W; at += TPU * VEC) {
            values(at, v, s);
            square(v, s);
        }
        const float inv = 1.0f / sqrtf(unit_sum<TPU>(sum, part) / (float) p.W + p.eps);
        for (int at = tid * VEC; at < p.W; at += TPU * VEC) {
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

template <int QT, int RT, int VEC, int TPU, int IT>
__global__ __launch_bounds__(TPU > 256 ? TPU : 256) void norm_residual_kernel(ResidualParams p) {
    constexpr int UNITS = TPU > 256 ? 1 : 256 / TPU;
    __shared__ float part[16];
    const int64_t t = (int64_t) blockIdx.x * UNITS + threadIdx.x / TPU;
    if (t >= p.T) return;
    const int tid = threadIdx.x % TPU;
    const float mean = 1.0f / (float) p.D;
    auto load_x = [&](int at, float (&v)[VEC]) {
        if (p.x) load_row<QT, VEC>(p.x, t * p.xs + at, v);
        else
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = 0.0f;
    };
    // s = h + scale gate post (x inv)
    auto stream = [&](int at, float (&v)[VEC], const float (&h)[VEC], float inv) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            float a = v[j];
            if (p.post) a = a * inv * p.post[at + j];
            if (p.gate) a *= p.gate[at + j];
            v[j] = p.x ? fmaf(p.scale, a, h[j]) : h[j];
        }
    };
    auto result = [&](int at, float (&v)[VEC], float inv) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = v[j] * inv * (p.pre ? p.pre[at + j] : 1.0f);
        store_row<QT, VEC>(p.out, t * p.os + at, v);
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
            const int at = (i * TPU + tid) * VEC;
            if (at < p.D) {
                load_x(at, v[i]);
                load_row<RT, VEC>(p.h, t * p.hs + at, h[i]);
            }
        }
        float inv = 1.0f;
        if (p.post) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < IT; ++i)
                if ((i * TPU + tid) * VEC < p.D) sum += squares(v[i]);
            inv = 1.0f / sqrtf(unit_sum<TPU>(sum, part) * mean + p.eps);
        }
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int at = (i * TPU + tid) * VEC;
            if (at >= p.D) continue;
            stream(at, v[i], h[i], inv);
            sum += squares(v[i]);
            if (p.h1) store_row<RT, VEC>(p.h1, t * p.h1s + at, v[i]);
        }
        if (!p.out) return;
        inv = 1.0f / sqrtf(unit_sum<TPU>(sum, part) * mean + p.eps);
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int at = (i * TPU + tid) * VEC;
            if (at < p.D) result(at, v[i], inv);
        }
    } else {
        // too long for registers: x and h are read again for each step, the stream written last (h1 may be h)
        float v[VEC], h[VEC], inv = 1.0f, sum = 0.0f;
        if (p.post) {
            for (int at = tid * VEC; at < p.D; at += TPU * VEC) {
                load_x(at, v);
                sum += squares(v);
            }
            inv = 1.0f / sqrtf(unit_sum<TPU>(sum, part) * mean + p.eps);
            sum = 0.0f;
        }
        for (int at = tid * VEC; at < p.D; at += TPU * VEC) {
            load_x(at, v);
            load_row<RT, VEC>(p.h, t * p.hs + at, h);
            stream(at, v, h, inv);
            sum += squares(v);
        }
        const float inv2 = 1.0f / sqrtf(unit_sum<TPU>(sum, part) * mean + p.eps);
        for (int at = tid * VEC; at < p.D; at += TPU * VEC) {
            load_x(at, v);
            load_row<RT, VEC>(p.h, t * p.hs + at, h);
            stream(at, v, h, inv);
            if (p.h1) store_row<RT, VEC>(p.h1, t * p.h1s + at, v);
            if (p.out) result(at, v, inv2);
        }
    }
}

// threads a unit and pieces a thread for a unit of n pieces: a wave while its lanes hold the unit in 4 pieces, then 4, then 16 waves
template <typename F>
void by_size(int64_t n, F f) {
    using std::integral_constant;
    auto it = [&](auto tpu) {
        constexpr int TPU = decltype(tpu)::value;
        if (n <= TPU) f(tpu, integral_constant<int, 1>());
        else if (n <= 2 * TPU) f(tpu, integral_constant<int, 2>());
        else f(tpu, integral_constant<int, 4>());
    };
    if (n <= 256) it(integral_constant<int, 64>());
    else if (n <= 1024) it(integral_constant<int, 256>());
    else if (n <= 4096) it(integral_constant<int, 1024>());
    else f(integral_constant<int, 1024>(), integral_constant<int, 0>());
}

template <int QT, int VEC>
int launch_gated(ns_gpu* g, const GatedParams& p) {
    int rc = 0;
    by_size((p.W + VEC - 1) / VEC, [&](auto tpu, auto it) {
        constexpr int TPU = decltype(tpu)::value, UNITS = TPU > 256 ? 1 : 256 / TPU;
        if ((p.units + UNITS - 1) / UNITS > INT32_MAX) rc = ns_fail("ns_norm_gated: too many rows");
        else norm_gated_kernel<QT, VEC, TPU, decltype(it)::value><<<(unsigned) ((p.units + UNITS - 1) / UNITS), TPU > 256 ? TPU : 256, 0, g->q>>>(p);
    });
    return rc;
}
template <int QT, int RT, int VEC>
int launch_residual(ns_gpu* g, const ResidualParams& p) {
    int rc = 0;
    by_size((p.D + VEC - 1) / VEC, [&](auto tpu, auto it) {
        constexpr int TPU = decltype(tpu)::value, UNITS = TPU > 256 ? 1 : 256 / TPU;
        if ((p.T + UNITS - 1) / UNITS > INT32_MAX) rc = ns_fail("ns_norm_residual: too many rows");
        else norm_residual_kernel<QT, RT, VEC, TPU, decltype(it)::value><<<(unsigned) ((p.T + UNITS - 1) / UNITS), TPU > 256 ? TPU : 256, 0, g->q>>>(p);
    });
    return rc;
}

// whether rows of type t at p, s elements apart, can be read in pieces of vec values
bool wide(const void* p, int64_t s, int t, int vec) {
    const int64_t e = t ? 2 : 4, piece = std::min<int64_t>(16, vec * e);
    return (uintptr_t) p % piece == 0 && s * e % piece == 0;
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
    if (!g || !y || !z || !out) return ns_fail("ns_norm_gated: a null buffer");
    if (T > ((int64_t) 1 << 40) / groups) return ns_fail("ns_norm_gated: too many rows");
    NS_HIP(hipSetDevice(g->dev));
    const GatedParams p{y, z, w, out, ys, zs, os, T * groups, (int) (D / groups), (int) groups, order, eps};
    const int vec = qt ? 8 : 4;
    const bool v = D / groups % vec == 0 && wide(y, ys, qt, vec) && wide(z, zs, qt, vec) && wide(out, os, qt, vec);
    const int rc = qt == 0 ? (v ? launch_gated<0, 4>(g, p) : launch_gated<0, 1>(g, p))
                 : qt == 1 ? (v ? launch_gated<1, 8>(g, p) : launch_gated<1, 1>(g, p))
                           : (v ? launch_gated<2, 8>(g, p) : launch_gated<2, 1>(g, p));
    if (rc) return rc;
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
    if (!g || !h || (!h1 && !out)) return ns_fail("ns_norm_residual: a null buffer");
    if (!x && (post || gate)) return ns_fail("ns_norm_residual: a norm or gate of no block");
    NS_HIP(hipSetDevice(g->dev));
    const ResidualParams p{x, h, post, gate, pre, h1, out, xs, hs, h1s, os, T, (int) D, eps, scale};
    const int vec = qt ? 8 : 4;
    const bool v = D % vec == 0 && (!x || wide(x, xs, qt, vec)) && wide(h, hs, rt, vec) && (!h1 || wide(h1, h1s, rt, vec)) && (!out || wide(out, os, qt, vec));
    const int rc = qt == 0   ? (v ? launch_residual<0, 0, 4>(g, p) : launch_residual<0, 0, 1>(g, p))
                   : rt == 0 ? (qt == 1 ? (v ? launch_residual<1, 0, 8>(g, p) : launch_residual<1, 0, 1>(g, p))
                                        : (v ? launch_residual<2, 0, 8>(g, p) : launch_residual<2, 0, 1>(g, p)))
                   : qt == 1 ? (v ? launch_residual<1, 1, 8>(g, p) : launch_residual<1, 1, 1>(g, p))
                             : (v ? launch_residual<2, 2, 8>(g, p) : launch_residual<2, 2, 1>(g, p));
    if (rc) return rc;
    NS_LAUNCHED("norm_residual");
    return 0;
    NS_CATCH
}

}  // extern "C"
