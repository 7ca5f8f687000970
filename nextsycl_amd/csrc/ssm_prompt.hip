// ssm_prompt.hip: a prompt's rows through a state-space layer's convolution and scan (ns_ssm_prompt).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "ns_internal.hpp"
#include "ns_layer.h"
#include "layer_common.hpp"

namespace {

constexpr int64_t PASS_ROWS = 8192;   // rows a pass works on: what bounds the scratch

// the convolved rows and step sizes of rows t0 .. t0 + T - 1, as float32: u [T][chan], dt [T][H]
template <int QT>
__global__ __launch_bounds__(256) void ssm_conv_kernel(SsmLayer p, int64_t t0, int T, float* __restrict__ u, float* __restrict__ dt) {
    const int c = blockIdx.x * 256 + threadIdx.x, t = blockIdx.y;
    if (c < p.chan) {
        float acc = p.cb ? p.cb[c] : 0.0f;
        for (int k = 4 - p.K; k < 4; ++k) {
            const int64_t at = t0 + t - 3 + k;
            const float v = at >= 0 ? load_q<QT>(p.xbc, at * p.xs + c) : p.p0 + at >= 0 ? p.conv[(p.p0 + at) % p.cap * p.chan + c] : 0.0f;
            acc = fmaf(ssm_tap(p, c, k), v, acc);
        }
        u[(int64_t) t * p.chan + c] = silu(acc);
    }
    if (c < p.H) dt[(int64_t) t * p.H + c] = ssm_dt<QT>(p, t0 + t, c);
}

// a wave a state row at a time: one lane a few of its features
template <int QT>
__global__ __launch_bounds__(64) void ssm_scan_kernel(SsmLayer p, int64_t t0, int T, const float* __restrict__ u, const float* __restrict__ dt) {
    const int head = blockIdx.x / p.P, pr = blockIdx.x % p.P, lane = threadIdx.x, group = head / (p.H / p.G);
    const float* src = t0 ? p.h1 : p.h0;
    const int64_t hrow = ((int64_t) head * p.P + pr) * p.N;
    float h[4];
    for (int i = 0; i < 4; ++i) h[i] = src && lane + 64 * i < p.N ? src[hrow + lane + 64 * i] : 0.0f;
    const float rate = p.a[head], skip = p.d ? p.d[head] : 0.0f;
    for (int t = 0; t < T; ++t) {
        const float* row = u + (int64_t) t * p.chan;
        const float x = row[head * p.P + pr], s = dt[(int64_t) t * p.H + head], decay = expf(s * rate);
        const float *b = row + p.H * p.P + group * p.N, *c = b + p.G * p.N;
        float sum = 0.0f;
        for (int i = 0; i < 4; ++i) {
            const int n = lane + 64 * i;
            if (n >= p.N) continue;
            h[i] = fmaf(h[i], decay, s * x * b[n]);
            sum = fmaf(h[i], c[n], sum);
        }
        sum = lanes_sum<64>(sum);
        if (lane == 0) store_o<QT>(p.y, (t0 + t) * p.ys + head * p.P + pr, fmaf(skip, x, sum));
    }
    for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < p.N) p.h1[hrow + lane + 64 * i] = h[i];
}

// the last raw rows into the ring
template <int QT>
__global__ __launch_bounds__(256) void ssm_ring_kernel(SsmLayer p, int64_t T) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    const int64_t t = T - 1 - blockIdx.y;
    if (c < p.chan && t >= 0) p.conv[(p.p0 + t) % p.cap * p.chan + c] = load_q<QT>(p.xbc, t * p.xs + c);
}

template <int QT>
void run_prompt(ns_gpu* g, const SsmLayer& p, int64_t T, float* scratch) {
    float *u = scratch, *dt = scratch + std::min(T, PASS_ROWS) * p.chan;
    for (int64_t t0 = 0; t0 < T; t0 += PASS_ROWS) {
        const int n = (int) std::min(PASS_ROWS, T - t0);
        ssm_conv_kernel<QT><<<dim3((unsigned) ((std::max(p.chan, p.H) + 255) / 256), (unsigned) n), 256, 0, g->q>>>(p, t0, n, u, dt);
        ssm_scan_kernel<QT><<<(unsigned) (p.H * p.P), 64, 0, g->q>>>(p, t0, n, u, dt);
    }
    if (p.K > 1) ssm_ring_kernel<QT><<<dim3((unsigned) ((p.chan + 255) / 256), (unsigned) (p.K - 1)), 256, 0, g->q>>>(p, T);
}

}  // namespace

extern "C" {

int64_t ns_ssm_prompt_scratch(int64_t T, int64_t H, int64_t P, int64_t N, int64_t G, int64_t K) {
    if (T <= 0 || H <= 0 || P <= 0 || N <= 0 || G <= 0 || K <= 0) return 0;
    return std::min(T, PASS_ROWS) * (H * P + 2 * G * N + H);
}

int ns_ssm_prompt(ns_gpu* g, int qt, const void* xbc, int64_t xs, const void* dt, int64_t dts, const float* cw, const float* cb, const float* a,
                  const float* dtb, const float* d, float dt_lo, float dt_hi, float* conv, int64_t cap, int64_t p0, int64_t T, int64_t H,
                  int64_t P, int64_t N, int64_t G, int64_t K, const float* h0, float* h1, void* y, int64_t ys, float* scratch) {
    NS_TRY
    if (T <= 0) return 0;
    SsmLayer p{xbc, dt, xs, dts, cw, cb, a, dtb, d, dt_lo, dt_hi, conv, cap, p0, (int) H, (int) P, (int) N, (int) G, (int) K, 0, h0, h1, y, ys};
    if (ns_ssm_check("ns_ssm_prompt", g, qt, p, H, P, N, G, K, K - 1)) return -1;
    if (!scratch) return ns_fail("ns_ssm_prompt: a null buffer");
    p.chan = (int) (H * P + 2 * G * N);
    NS_HIP(hipSetDevice(g->dev));
    if (qt == 0) run_prompt<0>(g, p, T, scratch);
    else if (qt == 1) run_prompt<1>(g, p, T, scratch);
    else run_prompt<2>(g, p, T, scratch);
    NS_LAUNCHED("ssm_prompt");
    return 0;
    NS_CATCH
}

}  // extern "C"
