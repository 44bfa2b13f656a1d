// a8hip: short causal depthwise convolution over frames, channels-last, with its carried history and its gradient.
//
//   e = (state[b, 0 .. K-2], x[b, 0 .. T-1]);   pre[t] = bias + sum_k w[k] e[t + k];   y = act(pre);   state' = e[len .. len + K - 2]
//   g[t] = dy[t] act'(pre[t]);   de[j] = sum_k w[k] g[j - k] (+ dstate'[j - len]);   dw[k] = sum_{b,t} g[t] e[t + k];   dbias = sum g
//
// Bound by HBM: x and y (backward: x, dy, dx) once.  A lane owns 4 channels (backward 2; 1 where width, strides or addresses do not allow it) and
// walks a span of frames with the last K inputs in registers: an input is read once per span plus K - 1 frames of overlap, which come from L2.  A
// wave is 64 such columns, the four waves of a block are consecutive spans of one utterance.  Short spans and narrow lanes win because they make
// waves: bf16 8 x 781 x 1536, K = 4, forward 8 channels x 16 frames 16.7 us, 4 x 16 14.5, 4 x 8 12.0 (38 MB: 3.2 TB/s; 64 utterances 66 us, 4.6 TB/s);
// backward 4 channels x 32 frames 27.2 us, 2 x 32 22.2, 2 x 16 19.6 but twice the partial sums (64 utterances 120 us against 111, 4.2 TB/s).
#include "a8_seq.h"
#include "a8hip_internal.h"

namespace {

constexpr int FWD_SPAN = 8, BWD_SPAN = 32;    // frames per wave

// V consecutive channels, moved as one access
template <typename T, int V> A8_DEV void ldv(float (&o)[V], const T* p) {
    struct __attribute__((aligned(V * sizeof(T)))) W { T v[V]; };
    const W w = *reinterpret_cast<const W*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = to_f(w.v[i]);
}
template <typename T, int V> A8_DEV void stv(T* p, const float (&o)[V]) {
    struct __attribute__((aligned(V * sizeof(T)))) W { T v[V]; } w;
#pragma unroll
    for (int i = 0; i < V; ++i) w.v[i] = from_f<T>(o[i]);
    *reinterpret_cast<W*>(p) = w;
}

// block and row of spans (quads per utterance) -> columns of V channels, utterance, first frame; the column of a lane past the width is the last one (its results are dropped)
struct Place { int c, b, t0, len; bool on; };
template <int V, int SPAN> A8_DEV Place place(const a8_causal_conv_desc& d, int cols, int quads, int64_t row) {
    Place q;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int cb = blockIdx.x % cols;
    q.b = (int)(row / quads);
    q.t0 = ((int)(row % quads) * 4 + wv) * SPAN;
    const int c = (cb * 64 + lane) * V;
    q.on = c < d.C;
    q.c = q.on ? c : d.C - V;
    q.len = seq_len(d.lengths, q.b, d.T);
    return q;
}
// e[b, j]: history, input, or zero behind the end; j < K - 1 + len is loaded, anything else not
template <typename T, int V> A8_DEV void conv_in(float (&o)[V], const a8_causal_conv_desc& d, const Place& q, int j) {
    const int t = j - (d.K - 1);
    if (t >= 0 && t < q.len) ldv<T, V>(o, (const T*)d.x + (q.b * d.x_bs + t * d.x_ts + q.c));
    else if (t < 0 && d.state) ldv<T, V>(o, (const T*)d.state + ((int64_t)q.b * (d.K - 1) + j) * d.C + q.c);
    else
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = 0.f;
}

template <typename T, int K, int V> __global__ __launch_bounds__(256) void conv_fwd_kernel(a8_causal_conv_desc d, int cols, int quads) {
    const Place q = place<V, FWD_SPAN>(d, cols, quads, blockIdx.x / cols);
    if (q.t0 >= d.T && !(q.t0 == 0)) return;                   // (a whole wave)
    float w[K][V], bias[V], e[K - 1][V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        bias[i] = d.bias ? d.bias[q.c + i] : 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) w[k][i] = d.w[(int64_t)(q.c + i) * K + k];
    }
#pragma unroll
    for (int k = 0; k < K - 1; ++k) conv_in<T, V>(e[k], d, q, q.t0 + k);
    const bool silu = d.act == A8_CONV_ACT_SILU;
    T* const y = (T*)d.y + ((int64_t)q.b * d.T + q.t0) * d.C + q.c;
    auto frame = [&](int s, const float (&x)[V]) {             // frame t0 + s, whose input is x
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float pre = fmaf(w[K - 1][i], x[i], bias[i]);
#pragma unroll
            for (int k = 0; k < K - 1; ++k) { pre = fmaf(w[k][i], e[k][i], pre); e[k][i] = k + 1 < K - 1 ? e[k + 1 < K - 1 ? k + 1 : 0][i] : x[i]; }
            o[i] = silu ? silu_f(pre) : pre;
        }
        return stv<T, V>(y + (int64_t)s * d.C, o);
    };
    const T* const x = (const T*)d.x + (q.b * d.x_bs + q.t0 * d.x_ts + q.c);
    if (q.t0 + FWD_SPAN <= q.len) {                            // a full span: 8 loads in flight at a time
#pragma unroll
        for (int s8 = 0; s8 < FWD_SPAN; s8 += 8) {
            float in[8][V];
#pragma unroll
            for (int s = 0; s < 8; ++s) ldv<T, V>(in[s], x + (s8 + s) * d.x_ts);
            if (q.on)
#pragma unroll
                for (int s = 0; s < 8; ++s) frame(s8 + s, in[s]);
        }
    } else if (q.on) {
        for (int s = 0; s < min(FWD_SPAN, d.T - q.t0); ++s) {
            float in[V] = {};
            if (q.t0 + s < q.len) { ldv<T, V>(in, x + s * d.x_ts); frame(s, in); }
            else stv<T, V>(y + (int64_t)s * d.C, in);
        }
    }
    if (d.state_out && q.t0 == 0 && q.on)
        for (int j = 0; j < K - 1; ++j) {
            float o[V];
            conv_in<T, V>(o, d, q, q.len + j);
            stv<T, V>((T*)d.state_out + ((int64_t)q.b * (K - 1) + j) * d.C + q.c, o);
        }
}

// MANY: more rows of spans than blocks per column, which walk them in turn (a template parameter: as one kernel, 64 x 781 x 1536 took 123 us against 107)
template <typename T, int K, int V, bool MANY> __global__ __launch_bounds__(256) void conv_bwd_kernel(a8_causal_conv_desc d, int cols, int quads, int64_t items) {
    __shared__ float red[4][K + 1][64 * V];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool silu = d.act == A8_CONV_ACT_SILU;
    const int slot = blockIdx.x / cols, slots = gridDim.x / cols;
    float dw[K][V] = {}, db[V] = {};
    for (int64_t row = slot; !MANY || row < items; row += slots) {
        const Place q = place<V, BWD_SPAN>(d, cols, quads, row);
        if (q.t0 < d.T) {
            const int t1 = min(q.t0 + BWD_SPAN, d.T);
            float w[K][V], bias[V], e[K][V], g[K][V] = {};         // e[k], g[k]: input and gradient before the activation of frame t - (K - 1) + k
#pragma unroll
            for (int i = 0; i < V; ++i) {
                bias[i] = d.bias ? d.bias[q.c + i] : 0.f;
#pragma unroll
                for (int k = 0; k < K; ++k) w[k][i] = d.w[(int64_t)(q.c + i) * K + k];
            }
#pragma unroll
            for (int k = 0; k < K - 1; ++k) conv_in<T, V>(e[k + 1], d, q, q.t0 + k);
            const T* const xp = (const T*)d.x + (q.b * d.x_bs + q.c);
            const T* const dp = (const T*)d.dy + (q.b * d.dy_bs + q.c);
            T* const dx = (T*)d.dx + (int64_t)q.b * d.T * d.C + q.c;
            auto frame = [&](int t, const float (&x)[V], const float (&dy)[V], bool own, bool valid) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
#pragma unroll
                    for (int k = 0; k < K - 1; ++k) { e[k][i] = e[k + 1][i]; g[k][i] = g[k + 1][i]; }
                    e[K - 1][i] = x[i];
                    float pre = bias[i];
#pragma unroll
                    for (int k = 0; k < K; ++k) pre = fmaf(w[k][i], e[k][i], pre);
                    const float gt = valid ? (silu ? dy[i] * silu_grad_f(pre) : dy[i]) : 0.f;
                    g[K - 1][i] = gt;
                    if (own) {
                        db[i] += gt;
#pragma unroll
                        for (int k = 0; k < K; ++k) dw[k][i] = fmaf(gt, e[k][i], dw[k][i]);
                    }
                }
            };
            auto emit = [&](int tx) {                              // the input gradient of frame tx, whose last tap was just taken in
                float de[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    de[i] = 0.f;
#pragma unroll
                    for (int k = 0; k < K; ++k) de[i] = fmaf(w[K - 1 - k][i], g[k][i], de[i]);
                }
                if (d.dstate_out && tx < q.len && tx >= q.len - (K - 1)) {
                    float ds[V];
                    ldv<T, V>(ds, (const T*)d.dstate_out + ((int64_t)q.b * (K - 1) + tx + (K - 1) - q.len) * d.C + q.c);
#pragma unroll
                    for (int i = 0; i < V; ++i) de[i] += ds[i];
                }
                if (tx >= q.len)
#pragma unroll
                    for (int i = 0; i < V; ++i) de[i] = 0.f;
                if (q.on && d.dx) stv<T, V>(dx + (int64_t)tx * d.C, de);
            };
            // g runs K - 1 frames past the span's end; the input gradient lags it by as many
            auto slow = [&](int t) {
                float x[V] = {}, dy[V] = {};
                const bool valid = t < q.len;
                if (valid) { ldv<T, V>(x, xp + t * d.x_ts); ldv<T, V>(dy, dp + t * d.dy_ts); }
                frame(t, x, dy, t < t1, valid);
                if (t - q.t0 >= K - 1) emit(t - (K - 1));
            };
            int t = q.t0;
            for (; t < min(q.t0 + K - 1, t1 + K - 1); ++t) slow(t);
            for (; t + 4 <= min(t1, q.len); t += 4) {              // four frames' loads in flight
                float x[4][V], dy[4][V];
#pragma unroll
                for (int s = 0; s < 4; ++s) { ldv<T, V>(x[s], xp + (t + s) * d.x_ts); ldv<T, V>(dy[s], dp + (t + s) * d.dy_ts); }
#pragma unroll
                for (int s = 0; s < 4; ++s) { frame(t + s, x[s], dy[s], true, true); emit(t + s - (K - 1)); }
            }
            for (; t < t1 + K - 1; ++t) slow(t);
        }
        if (q.t0 == 0 && q.on && d.dstate)                         // the history's gradient: e indexes 0 .. K - 2, read by frames t <= j at tap j - t
            for (int j = 0; j < K - 1; ++j)
                for (int i = 0; i < V; ++i) {
                    const int c = q.c + i;
                    float de = 0.f;
                    for (int t = 0; t <= min(j, q.len - 1); ++t) {
                        float pre = d.bias ? d.bias[c] : 0.f;
                        for (int k = 0; k < K; ++k) {
                            const int f = t + k - (K - 1);
                            const float v = f >= 0 ? to_f(((const T*)d.x)[q.b * d.x_bs + f * d.x_ts + c])
                                                   : d.state ? to_f(((const T*)d.state)[((int64_t)q.b * (K - 1) + t + k) * d.C + c]) : 0.f;
                            pre = fmaf(d.w[(int64_t)c * K + k], v, pre);
                        }
                        float gt = to_f(((const T*)d.dy)[q.b * d.dy_bs + t * d.dy_ts + c]);
                        if (silu) gt *= silu_grad_f(pre);
                        de = fmaf(d.w[(int64_t)c * K + j - t], gt, de);
                    }
                    if (d.dstate_out && j >= q.len) de += to_f(((const T*)d.dstate_out)[((int64_t)q.b * (K - 1) + j - q.len) * d.C + c]);
                    ((T*)d.dstate)[((int64_t)q.b * (K - 1) + j) * d.C + c] = from_f<T>(de);
                }
        if constexpr (!MANY) break;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int k = 0; k < K; ++k) red[wv][k][lane * V + i] = dw[k][i];
        red[wv][K][lane * V + i] = db[i];
    }
    __syncthreads();
    const int c0 = (blockIdx.x % cols) * 64 * V;
    for (int i = threadIdx.x; i < (K + 1) * 64 * V; i += 256) {
        const int p = i / (64 * V), l = i % (64 * V);
        if (c0 + l < d.C) d.partials[((int64_t)slot * (K + 1) + p) * d.C + c0 + l] = (red[0][p][l] + red[1][p][l]) + (red[2][p][l] + red[3][p][l]);
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

// 16 columns of one plane per block; the 16 waves take four rows at a time (a quarter of the lanes each), eight loads in flight, and meet in LDS.
__global__ __launch_bounds__(1024) void seq_reduce_kernel(A8SeqReduce r) {
    __shared__ float red[16][64];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int c = blockIdx.x * 16 + (lane & 15), q = blockIdx.y;
    const float* const in = r.in + (int64_t)q * r.C + min(c, r.C - 1);
    const int64_t pitch = (int64_t)r.planes * r.C;
    float s[8] = {};
    int i = wv * 4 + (lane >> 4);
    for (; i + 448 < r.rows; i += 512)
#pragma unroll
        for (int k = 0; k < 8; ++k) s[k] += in[(i + 64 * k) * pitch];
    for (; i < r.rows; i += 64) s[0] += in[i * pitch];
    red[wv][lane] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
    __syncthreads();
    if (threadIdx.x < 16 && c < r.C) {
        float t = 0.f;
        for (int k = 0; k < 64; ++k) t += red[k >> 2][(k & 3) * 16 + lane];
        float* out = q < r.np ? r.major + (int64_t)c * r.np + q : r.minor[q - r.np] + c;
        const bool have = q < r.np ? r.major != nullptr : r.minor[q - r.np] != nullptr;
        const int add = q < r.np ? r.add_major : r.add_minor[q - r.np];
        if (have) *out = add ? *out + t : t;
    }
}

int conv_check(const a8_causal_conv_desc* d, const char* what) {
    A8_REQUIRE(d != nullptr && d->size == (int)sizeof(a8_causal_conv_desc), "%s: descriptor size %d, expected %d", what, d ? d->size : 0, (int)sizeof(a8_causal_conv_desc));
    A8_REQUIRE(d->dtype == A8_F32 || d->dtype == A8_BF16, "%s: bad dtype %d", what, d->dtype);
    A8_REQUIRE(d->B >= 0 && d->T >= 0 && d->C >= 1 && d->K >= 2 && d->K <= 4, "%s: bad sizes B=%d T=%d C=%d K=%d (2 to 4 taps)", what, d->B, d->T, d->C, d->K);
    A8_REQUIRE(d->T < (1 << 30), "%s: T = %d is too large", what, d->T);           // (frame indices run up to a block's spans past the end)
    A8_REQUIRE(d->act == A8_CONV_ACT_NONE || d->act == A8_CONV_ACT_SILU, "%s: unknown activation %d", what, d->act);
    A8_REQUIRE(d->w != nullptr, "%s: null weight", what);
    return A8_OK;
}

bool multiple(const void* p, int bytes) { return ((uintptr_t)p % bytes) == 0; }
// whether V channels at a time are aligned everywhere: width, row and batch strides, base addresses
bool conv_vec(const a8_causal_conv_desc* d, int V, bool backward) {
    const int bytes = V * (d->dtype == A8_BF16 ? 2 : 4);
    bool ok = d->C % V == 0 && d->x_bs % V == 0 && d->x_ts % V == 0;
    for (const void* p : {d->x, d->state, (const void*)d->y, (const void*)d->state_out}) ok = ok && multiple(p, bytes);
    if (backward) {
        ok = ok && d->dy_bs % V == 0 && d->dy_ts % V == 0;
        for (const void* p : {d->dy, d->dstate_out, (const void*)d->dx, (const void*)d->dstate}) ok = ok && multiple(p, bytes);
    }
    return ok;
}
#define CONV_FWD(T, V) (d->K == 2 ? (conv_fwd_kernel<T, 2, V>) : d->K == 3 ? (conv_fwd_kernel<T, 3, V>) : (conv_fwd_kernel<T, 4, V>))
#define CONV_BWD(T, V, MANY) (d->K == 2 ? (conv_bwd_kernel<T, 2, V, MANY>) : d->K == 3 ? (conv_bwd_kernel<T, 3, V, MANY>) : (conv_bwd_kernel<T, 4, V, MANY>))
int conv_quads(const a8_causal_conv_desc* d, int span) { return cdiv(d->T > 0 ? d->T : 1, 4 * span); }        // blocks along an utterance (T = 0 still hands the history on)
// The backward's rows of spans, and the blocks per column that walk them: one each (8 x 781: 56), unless that is more than eight per CU and their partial
// sums (K + 1 floats per channel) would be more than twice the frames themselves, as with many utterances of a few frames; then as many as keep them
// below the frames (4096 x 1 x 1536: 126 -> 12 MB, 79 + 7 us against 76 + 39; 4096 x 8 x 768 stays at one each: 84 + 20 us against 113 + 17).
int64_t conv_items(const a8_causal_conv_desc* d) { return d->T > 0 ? (int64_t)d->B * conv_quads(d, BWD_SPAN) : 0; }
int conv_slots(const a8_causal_conv_desc* d) {
    const int cols = cdiv(d->C, 64);
    const int64_t most = std::max<int64_t>(cdiv(4096, cols), (int64_t)d->B * d->T / (2 * (d->K + 1)));
    return (int)std::min(conv_items(d) <= 2 * most ? conv_items(d) : most, (int64_t)std::max(1, (1 << 23) / cols));
}

}  // namespace

int a8i_seq_reduce(const A8SeqReduce& r, void* stream) {
    hipLaunchKernelGGL(seq_reduce_kernel, dim3(cdiv(r.C, 16), r.planes), dim3(1024), 0, (hipStream_t)stream, r);
    return a8_check_launch("a8i_seq_reduce");
}

extern "C" int a8_causal_conv_fwd(const a8_causal_conv_desc* d, void* stream) {
    if (int e = conv_check(d, "a8_causal_conv_fwd")) return e;
    if (d->B == 0) return A8_OK;
    A8_REQUIRE((d->x && d->y) || d->T == 0, "a8_causal_conv_fwd: null x or y");
    A8_REQUIRE(d->state_out == nullptr || d->state_out != d->state, "a8_causal_conv_fwd: state_out may not be the state that is read");
    A8_REQUIRE(!d->y || d->y != d->x, "a8_causal_conv_fwd: y may not be x");
    const bool bf = d->dtype == A8_BF16;
    const int V = conv_vec(d, 4, false) ? 4 : 1;
    const int cols = cdiv(d->C, 64 * V), quads = conv_quads(d, FWD_SPAN);
    A8_REQUIRE((int64_t)cols * d->B * quads < (1 << 24), "a8_causal_conv_fwd: B x T x C = %d x %d x %d is too large", d->B, d->T, d->C);
    auto kernel = bf ? (V == 4 ? CONV_FWD(bf16, 4) : CONV_FWD(bf16, 1))
                     : (V == 4 ? CONV_FWD(float, 4) : CONV_FWD(float, 1));
    hipLaunchKernelGGL(kernel, dim3(cols * d->B * quads), dim3(256), 0, (hipStream_t)stream, *d, cols, quads);
    return a8_check_launch("a8_causal_conv_fwd");
}

extern "C" int a8_causal_conv_bwd_partial_floats(const a8_causal_conv_desc* d, int64_t* floats) {
    if (int e = conv_check(d, "a8_causal_conv_bwd_partial_floats")) return e;
    A8_REQUIRE(floats != nullptr, "a8_causal_conv_bwd_partial_floats: null result");
    *floats = (int64_t)conv_slots(d) * (d->K + 1) * d->C;
    return A8_OK;
}

extern "C" int a8_causal_conv_bwd(const a8_causal_conv_desc* d, void* stream) {
    if (int e = conv_check(d, "a8_causal_conv_bwd")) return e;
    A8_REQUIRE(d->C < SEQ_REDUCE_MAX, "a8_causal_conv_bwd: C = %d is too large", d->C);
    const int rows = conv_slots(d);
    A8_REQUIRE((d->x && d->dy && d->partials) || rows == 0, "a8_causal_conv_bwd: null x, dy or partials");
    A8_REQUIRE((!d->dx || (d->dx != d->dy && d->dx != d->x)) && (!d->dstate || d->dstate != d->dstate_out), "a8_causal_conv_bwd: an output may not be an input");
    A8_REQUIRE(d->T > 0 || d->B == 0 || d->dstate == nullptr, "a8_causal_conv_bwd: a history's gradient needs T >= 1");
    if (rows > 0) {
        const bool bf = d->dtype == A8_BF16;
        const int V = conv_vec(d, 2, true) ? 2 : 1;
        const int cols = cdiv(d->C, 64 * V), quads = conv_quads(d, BWD_SPAN);
        const bool many = conv_items(d) > rows;
        auto kernel = many ? (bf ? (V == 2 ? CONV_BWD(bf16, 2, true) : CONV_BWD(bf16, 1, true)) : (V == 2 ? CONV_BWD(float, 2, true) : CONV_BWD(float, 1, true)))
                           : (bf ? (V == 2 ? CONV_BWD(bf16, 2, false) : CONV_BWD(bf16, 1, false)) : (V == 2 ? CONV_BWD(float, 2, false) : CONV_BWD(float, 1, false)));
        hipLaunchKernelGGL(kernel, dim3(cols * rows), dim3(256), 0, (hipStream_t)stream, *d, cols, quads, conv_items(d));
        if (int e = a8_check_launch("a8_causal_conv_bwd")) return e;
    }
    A8SeqReduce r = {d->partials, rows, d->K + 1, d->C, d->K, d->dw, {d->dbias}, d->add_dw, {d->add_dbias}};
    return a8i_seq_reduce(r, stream);
}

extern "C" int a8_causal_conv_step(const a8_causal_conv_desc* d, void* stream) {
    if (int e = conv_check(d, "a8_causal_conv_step")) return e;
    A8_REQUIRE(d->T == 1, "a8_causal_conv_step: one frame at a time (T = %d)", d->T);
    if (d->B == 0) return A8_OK;
    A8_REQUIRE((int64_t)d->B * d->C < (1 << 30), "a8_causal_conv_step: B x C = %d x %d is too large", d->B, d->C);
    A8_REQUIRE(d->x && d->y && d->state_out, "a8_causal_conv_step: null x, y or state");
    auto kernel = d->dtype == A8_BF16 ? (d->K == 2 ? conv_step_kernel<bf16, 2> : d->K == 3 ? conv_step_kernel<bf16, 3> : conv_step_kernel<bf16, 4>)
                                      : (d->K == 2 ? conv_step_kernel<float, 2> : d->K == 3 ? conv_step_kernel<float, 3> : conv_step_kernel<float, 4>);
    hipLaunchKernelGGL(kernel, dim3(cdiv((int64_t)d->B * d->C, 256)), dim3(256), 0, (hipStream_t)stream, *d);
    return a8_check_launch("a8_causal_conv_step");
}
