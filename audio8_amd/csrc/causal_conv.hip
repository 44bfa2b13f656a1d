// a8hip: short causal depthwise convolution over frames, channels-last, with its carried history and its gradient.
//
//   e = (state[b, 0 .. K-2], x[b, 0 .. T-1]);   pre[t] = bias + sum_k w[k] e[t + k];   y = act(pre);   state' = e[len .. len + K - 2]
//   g[t] = dy[t] act'(pre[t]);   de[j] = sum_k w[k] g[j - k] (+ dstate'[j - len]);   dw[k] = sum_{b,t} g[t] e[t + k];   dbias = sum g
//
// A lane owns a channel and walks frames with the last K inputs in registers, so an input is read once per span plus K - 1 frames of overlap.
#include "a8_seq.h"
#include "a8hip_internal.h"

namespace {

constexpr int CONV_SPAN = 16;                 // frames per thread

template <typename T> A8_DEV float conv_in(const a8_causal_conv_desc& d, int b, int j, int c, int len) {       // e[b, j, c]; 0 behind the end
    if (j < d.K - 1) return d.state ? to_f(((const T*)d.state)[((int64_t)b * (d.K - 1) + j) * d.C + c]) : 0.f;
    const int t = j - (d.K - 1);
    return t < len ? to_f(((const T*)d.x)[b * d.x_bs + t * d.x_ts + c]) : 0.f;
}

template <typename T, int K> __global__ __launch_bounds__(256) void conv_fwd_kernel(a8_causal_conv_desc d, int spans) {
    const int c = blockIdx.x * 64 + (threadIdx.x & 63);
    const int64_t s = (int64_t)blockIdx.y * 4 + (threadIdx.x >> 6);
    if (c >= d.C || s >= (int64_t)d.B * spans) return;
    const int b = (int)(s / spans), t0 = (int)(s % spans) * CONV_SPAN, len = seq_len(d.lengths, b, d.T);
    float w[K], e[K];
#pragma unroll
    for (int k = 0; k < K; ++k) w[k] = d.w[(int64_t)c * K + k];
    const float bias = d.bias ? d.bias[c] : 0.f;
#pragma unroll
    for (int k = 0; k < K - 1; ++k) e[k + 1] = conv_in<T>(d, b, t0 + k, c, len);
    for (int t = t0; t < min(t0 + CONV_SPAN, d.T); ++t) {
        float pre = bias;
#pragma unroll
        for (int k = 0; k < K - 1; ++k) e[k] = e[k + 1];
        e[K - 1] = conv_in<T>(d, b, t + K - 1, c, len);
#pragma unroll
        for (int k = 0; k < K; ++k) pre = fmaf(w[k], e[k], pre);
        const float y = d.act == A8_CONV_ACT_SILU ? silu_f(pre) : pre;
        ((T*)d.y)[((int64_t)b * d.T + t) * d.C + c] = from_f<T>(t < len ? y : 0.f);
    }
    if (d.state_out && t0 == 0)
        for (int j = 0; j < K - 1; ++j) ((T*)d.state_out)[((int64_t)b * (K - 1) + j) * d.C + c] = from_f<T>(conv_in<T>(d, b, len + j, c, len));
}

template <typename T, int K> __global__ __launch_bounds__(256) void conv_bwd_kernel(a8_causal_conv_desc d, int spans) {
    __shared__ float red[4][K + 1][64];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int c = blockIdx.x * 64 + lane, quads = (spans + 3) / 4;
    const int b = blockIdx.y / quads, span = (blockIdx.y % quads) * 4 + wv;
    float dw[K] = {}, db = 0.f;
    if (c < d.C && span < spans) {
        const int t0 = span * CONV_SPAN, t1 = min(t0 + CONV_SPAN, d.T), len = seq_len(d.lengths, b, d.T);
        float w[K], e[K], g[K];
#pragma unroll
        for (int k = 0; k < K; ++k) { w[k] = d.w[(int64_t)c * K + k]; g[k] = 0.f; }
        const float bias = d.bias ? d.bias[c] : 0.f;
#pragma unroll
        for (int k = 0; k < K - 1; ++k) e[k + 1] = conv_in<T>(d, b, t0 + k, c, len);
        // g runs K - 1 frames past the span's end, de[j] of j = t0 .. t1 - 1 + K - 1 lags it; the first span also owns the history's gradient
        for (int t = t0; t < t1 + K - 1; ++t) {
#pragma unroll
            for (int k = 0; k < K - 1; ++k) { e[k] = e[k + 1]; g[k] = g[k + 1]; }
            e[K - 1] = conv_in<T>(d, b, t + K - 1, c, len);
            float pre = bias;
#pragma unroll
            for (int k = 0; k < K; ++k) pre = fmaf(w[k], e[k], pre);
            float gt = t < len ? to_f(((const T*)d.dy)[b * d.dy_bs + t * d.dy_ts + c]) : 0.f;
            if (d.act == A8_CONV_ACT_SILU && t < len) gt *= silu_grad_f(pre);
            g[K - 1] = gt;                                            // g[k] = g of frame t - (K - 1) + k
            if (t < t1) {
                db += gt;
#pragma unroll
                for (int k = 0; k < K; ++k) dw[k] = fmaf(gt, e[k], dw[k]);
            }
            const int j = t - t0 < K - 1 ? -1 : t;                    // e index whose gradient is complete: frame t - (K - 1)
            if (j >= 0) {
                float de = 0.f;
#pragma unroll
                for (int k = 0; k < K; ++k) de = fmaf(w[K - 1 - k], g[k], de);
                const int tx = j - (K - 1);
                if (d.dstate_out && tx < len && tx >= len - (K - 1)) de += to_f(((const T*)d.dstate_out)[((int64_t)b * (K - 1) + tx + (K - 1) - len) * d.C + c]);
                if (d.dx) ((T*)d.dx)[((int64_t)b * d.T + tx) * d.C + c] = from_f<T>(tx < len ? de : 0.f);
            }
        }
    }
    if (span == 0 && c < d.C && d.dstate) {                           // de of the history: e indexes 0 .. K - 2
        const int len = seq_len(d.lengths, b, d.T);
        for (int j = 0; j < K - 1; ++j) {
            float de = 0.f;
            for (int t = 0; t <= min(j, len - 1); ++t) {              // frames t <= j read e[j] at tap j - t
                float pre = d.bias ? d.bias[c] : 0.f;
                for (int k = 0; k < K; ++k) pre = fmaf(d.w[(int64_t)c * K + k], conv_in<T>(d, b, t + k, c, len), pre);
                float gt = to_f(((const T*)d.dy)[b * d.dy_bs + t * d.dy_ts + c]);
                if (d.act == A8_CONV_ACT_SILU) gt *= silu_grad_f(pre);
                de = fmaf(d.w[(int64_t)c * K + j - t], gt, de);
            }
            if (d.dstate_out && j >= len) de += to_f(((const T*)d.dstate_out)[((int64_t)b * (K - 1) + j - len) * d.C + c]);
            ((T*)d.dstate)[((int64_t)b * (K - 1) + j) * d.C + c] = from_f<T>(de);
        }
    }
#pragma unroll
    for (int k = 0; k < K; ++k) red[wv][k][lane] = dw[k];
    red[wv][K][lane] = db;
    __syncthreads();
    for (int i = threadIdx.x; i < (K + 1) * 64; i += 256) {
        const int q = i >> 6, l = i & 63, cc = blockIdx.x * 64 + l;
        if (cc < d.C) d.partials[((int64_t)blockIdx.y * (K + 1) + q) * d.C + cc] = (red[0][q][l] + red[1][q][l]) + (red[2][q][l] + red[3][q][l]);
    }
}

template <typename T, int K> __global__ __launch_bounds__(256) void conv_step_kernel(a8_causal_conv_desc d) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)d.B * d.C) return;
    const int b = (int)(i / d.C), c = (int)(i % d.C);
    T* st = (T*)d.state_out + (int64_t)b * (K - 1) * d.C + c;
    T e[K];
#pragma unroll
    for (int k = 0; k < K - 1; ++k) e[k] = st[(int64_t)k * d.C];
    e[K - 1] = ((const T*)d.x)[b * d.x_bs + c];
    float pre = d.bias ? d.bias[c] : 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) pre = fmaf(d.w[(int64_t)c * K + k], to_f(e[k]), pre);
    ((T*)d.y)[i] = from_f<T>(d.act == A8_CONV_ACT_SILU ? silu_f(pre) : pre);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) st[(int64_t)k * d.C] = e[k + 1];
}

__global__ __launch_bounds__(256) void seq_reduce_kernel(A8SeqReduce r) {
    __shared__ float red[4][64];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int c = blockIdx.x * 64 + lane, q = blockIdx.y;
    float s = 0.f;
    if (c < r.C)
        for (int i = wv; i < r.rows; i += 4) s += r.in[((int64_t)i * r.planes + q) * r.C + c];
    red[wv][lane] = s;
    __syncthreads();
    if (wv == 0 && c < r.C) {
        s = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
        float* out = q < r.np ? r.major + (int64_t)c * r.np + q : r.minor[q - r.np] + c;
        const bool have = q < r.np ? r.major != nullptr : r.minor[q - r.np] != nullptr;
        const int add = q < r.np ? r.add_major : r.add_minor[q - r.np];
        if (have) *out = add ? *out + s : s;
    }
}

int conv_check(const a8_causal_conv_desc* d, const char* what) {
    A8_REQUIRE(d != nullptr && d->size == (int)sizeof(a8_causal_conv_desc), "%s: descriptor size %d, expected %d", what, d ? d->size : 0, (int)sizeof(a8_causal_conv_desc));
    A8_REQUIRE(d->dtype == A8_F32 || d->dtype == A8_BF16, "%s: bad dtype %d", what, d->dtype);
    A8_REQUIRE(d->B >= 0 && d->T >= 0 && d->C >= 1 && d->K >= 2 && d->K <= 4, "%s: bad sizes B=%d T=%d C=%d K=%d (2 to 4 taps)", what, d->B, d->T, d->C, d->K);
    A8_REQUIRE(d->act == A8_CONV_ACT_NONE || d->act == A8_CONV_ACT_SILU, "%s: unknown activation %d", what, d->act);
    A8_REQUIRE(d->w != nullptr, "%s: null weight", what);
    return A8_OK;
}

#define CONV_DISPATCH(KERNEL, GRID, STREAM, ...)                                                                                       \
    do {                                                                                                                               \
        if (d->dtype == A8_BF16) {                                                                                                     \
            if (d->K == 2) hipLaunchKernelGGL((KERNEL<bf16, 2>), GRID, dim3(256), 0, STREAM, __VA_ARGS__);                              \
            else if (d->K == 3) hipLaunchKernelGGL((KERNEL<bf16, 3>), GRID, dim3(256), 0, STREAM, __VA_ARGS__);                         \
            else hipLaunchKernelGGL((KERNEL<bf16, 4>), GRID, dim3(256), 0, STREAM, __VA_ARGS__);                                        \
        } else {                                                                                                                       \
            if (d->K == 2) hipLaunchKernelGGL((KERNEL<float, 2>), GRID, dim3(256), 0, STREAM, __VA_ARGS__);                             \
            else if (d->K == 3) hipLaunchKernelGGL((KERNEL<float, 3>), GRID, dim3(256), 0, STREAM, __VA_ARGS__);                        \
            else hipLaunchKernelGGL((KERNEL<float, 4>), GRID, dim3(256), 0, STREAM, __VA_ARGS__);                                       \
        }                                                                                                                              \
    } while (0)

int conv_rows(const a8_causal_conv_desc* d) { return d->B * cdiv(cdiv(d->T, CONV_SPAN), 4); }

}  // namespace

int a8i_seq_reduce(const A8SeqReduce& r, void* stream) {
    hipLaunchKernelGGL(seq_reduce_kernel, dim3(cdiv(r.C, 64), r.planes), dim3(256), 0, (hipStream_t)stream, r);
    return a8_check_launch("a8i_seq_reduce");
}

extern "C" int a8_causal_conv_fwd(const a8_causal_conv_desc* d, void* stream) {
    if (int e = conv_check(d, "a8_causal_conv_fwd")) return e;
    if (d->B == 0) return A8_OK;
    A8_REQUIRE((d->x && d->y) || d->T == 0, "a8_causal_conv_fwd: null x or y");
    A8_REQUIRE(d->state_out == nullptr || d->state_out != d->state, "a8_causal_conv_fwd: state_out may not be the state that is read");
    const int spans = d->T > 0 ? cdiv(d->T, CONV_SPAN) : 1;              // T = 0 still hands the history on
    CONV_DISPATCH(conv_fwd_kernel, dim3(cdiv(d->C, 64), cdiv((int64_t)d->B * spans, 4)), (hipStream_t)stream, *d, spans);
    return a8_check_launch("a8_causal_conv_fwd");
}

extern "C" int a8_causal_conv_bwd_partial_floats(const a8_causal_conv_desc* d, int64_t* floats) {
    if (int e = conv_check(d, "a8_causal_conv_bwd_partial_floats")) return e;
    A8_REQUIRE(floats != nullptr, "a8_causal_conv_bwd_partial_floats: null result");
    *floats = (int64_t)conv_rows(d) * (d->K + 1) * d->C;
    return A8_OK;
}

extern "C" int a8_causal_conv_bwd(const a8_causal_conv_desc* d, void* stream) {
    if (int e = conv_check(d, "a8_causal_conv_bwd")) return e;
    const int spans = cdiv(d->T, CONV_SPAN), rows = conv_rows(d);
    A8_REQUIRE((d->x && d->dy && d->partials) || rows == 0, "a8_causal_conv_bwd: null x, dy or partials");
    A8_REQUIRE(d->T > 0 || d->B == 0 || d->dstate == nullptr, "a8_causal_conv_bwd: a history's gradient needs T >= 1");
    A8_REQUIRE(rows <= 65535, "a8_causal_conv_bwd: B x T = %d x %d is too large", d->B, d->T);
    if (rows > 0) {
        CONV_DISPATCH(conv_bwd_kernel, dim3(cdiv(d->C, 64), rows), (hipStream_t)stream, *d, spans);
        if (int e = a8_check_launch("a8_causal_conv_bwd")) return e;
    }
    A8SeqReduce r = {d->partials, rows, d->K + 1, d->C, d->K, d->dw, {d->dbias}, d->add_dw, {d->add_dbias}};
    return a8i_seq_reduce(r, stream);
}

extern "C" int a8_causal_conv_step(const a8_causal_conv_desc* d, void* stream) {
    if (int e = conv_check(d, "a8_causal_conv_step")) return e;
    A8_REQUIRE(d->T == 1, "a8_causal_conv_step: one frame at a time (T = %d)", d->T);
    if (d->B == 0) return A8_OK;
    A8_REQUIRE(d->x && d->y && d->state_out, "a8_causal_conv_step: null x, y or state");
    CONV_DISPATCH(conv_step_kernel, dim3(cdiv((int64_t)d->B * d->C, 256)), (hipStream_t)stream, *d);
    return a8_check_launch("a8_causal_conv_step");
}
