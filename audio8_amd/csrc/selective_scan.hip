// a8hip: selective state space scan, channels-last, forward, gradient and single-frame step.
//
//   D_t = softplus(dt + dt_bias);  h_t[n] = exp(D_t A[n]) h_{t-1}[n] + D_t u_t B_t[n];  y_t = sum_n C_t[n] h_t[n] + Dskip u_t;  out = y silu(z)
// per channel with N <= 32 states; B and C are shared by the channels of a group.  Adjoint, with g = dout silu(z) and c_t = exp(D_{t+1} A) q_{t+1}:
//   q_t = C_t g_t + c_t;   dC_t = sum_ch g h_t;   dB_t = sum_ch q D u;   du = D sum_n q B + Dskip g;
//   dD = u sum_n q B + sum_n A k_t,  k_t = exp(D_t A) q_t h_{t-1};   dA = sum_t k_t D_t;   d dt = dD sigmoid(dt + dt_bias)
// (c_{t-1} = exp(D_t A) q_t, so k_t = c_{t-1} h_{t-1}: the adjoint's own product is reused).
//
// Layout: a lane is a channel, a wave is 4 states of 64 channels, a block is ceil(N / 4) waves of the same 64 channels: the frame inputs are
// read along the channels (64 lanes, 128 B in bf16, any alignment), B and C are LDS broadcasts, no state is ever exchanged between lanes, and
// only the sums over states (y; q B, A k) cross waves, through LDS once per tile of 16 frames.  softplus / silu run once per (frame, channel),
// split over the block's waves, not once per state.
// Everything between the inputs and the outputs is f32: steps, decays, states, adjoints and all sums.
#include "a8_seq.h"
#include "a8hip_internal.h"

namespace {

constexpr int TT = 16;      // frames of a tile: a wave's 4 states x 16 frames of a and h live in registers in the backward
constexpr int CH = 64;      // channels of a block
constexpr int NS = 4;       // states of a wave

struct ScanArgs {
    a8_selective_scan_desc d;
    int cpg, tpg, tiles;               // channels and channel tiles per group, frame tiles of T
    float* part;                       // backward: [B][N + 2][D] partial dA planes, dD, ddt_bias
    float* part_b; float* part_c;      // backward: [tpg][B][T][G][N] partial dB, dC
};

struct Where { int b, g, ct, c0, ch; bool live; int64_t chan; int len; };
A8_DEV Where locate(const ScanArgs& p, int lane) {
    Where w;
    int i = blockIdx.x;
    w.ct = i % p.tpg; i /= p.tpg;
    w.g = i % p.d.G; w.b = i / p.d.G;
    const int c = w.ct * CH + lane;
    w.live = c < p.cpg;
    w.ch = w.g * p.cpg + min(c, p.cpg - 1);
    w.len = seq_len(p.d.lengths, w.b, p.d.T);
    return w;
}

template <typename T> A8_DEV float ldf(const void* p, int64_t i) { return to_f(((const T*)p)[i]); }

// B or C of one tile, one value per thread (TT x 4 NW values = the block's threads): frame tid / (4 NW), state tid % (4 NW)
template <typename T, int NW> A8_DEV float load_bc(const void* base, int64_t bs, int64_t ts, int64_t gs, const ScanArgs& p, const Where& w, int t0) {
    const int n = threadIdx.x % (NS * NW), t = t0 + threadIdx.x / (NS * NW);
    return t < w.len && n < p.d.N ? ldf<T>(base, w.b * bs + t * ts + w.g * gs + n) : 0.f;
}

template <typename T, int NW> __global__ __launch_bounds__(64 * NW) void scan_fwd_kernel(ScanArgs p) {
    constexpr int EP = TT / NW;                            // (frame, channel) elements of a tile per thread
    __shared__ float2 s_dx[TT][CH];                        // {D, D u}
    __shared__ __align__(16) float s_b[TT][NS * NW], s_c[TT][NS * NW];
    __shared__ float s_y[NW][TT][CH];
    const a8_selective_scan_desc& d = p.d;
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, n0 = wv * NS;
    const Where w = locate(p, lane);
    const float bias = d.dt_bias ? d.dt_bias[w.ch] : 0.f, skip = d.Dskip ? d.Dskip[w.ch] : 0.f;
    float A2[NS], h[NS];
#pragma unroll
    for (int n = 0; n < NS; ++n) {
        const bool has = n0 + n < d.N;
        A2[n] = has ? d.A[(int64_t)w.ch * d.N + n0 + n] * SEQ_LOG2E : 0.f;
        h[n] = has && d.h0 ? d.h0[((int64_t)w.b * d.D + w.ch) * d.N + n0 + n] : 0.f;
    }
    const int ntile = (w.len + TT - 1) / TT;
    float u[EP], dt[EP], z[EP], rb = 0.f, rc = 0.f;
    auto load = [&](int t0) {
#pragma unroll
        for (int j = 0; j < EP; ++j) {
            const int t = t0 + wv + NW * j;
            const bool in = t < w.len;
            u[j] = in ? ldf<T>(d.u, w.b * d.u_bs + t * d.u_ts + w.ch) : 0.f;
            dt[j] = in ? ldf<T>(d.dt, w.b * d.dt_bs + t * d.dt_ts + w.ch) : 0.f;
            z[j] = in && d.z ? ldf<T>(d.z, w.b * d.z_bs + t * d.z_ts + w.ch) : 0.f;
        }
        rb = load_bc<T, NW>(d.Bm, d.b_bs, d.b_ts, d.b_gs, p, w, t0);
        rc = load_bc<T, NW>(d.Cm, d.c_bs, d.c_ts, d.c_gs, p, w, t0);
    };
    if (ntile > 0) load(0);
    for (int i = 0; i < ntile; ++i) {
        const int t0 = i * TT;
        float cu[EP], cz[EP];
#pragma unroll
        for (int j = 0; j < EP; ++j) {
            const int t = wv + NW * j;
            const float raw = dt[j] + bias, D = t0 + t < w.len ? (d.softplus ? softplus_f(raw) : raw) : 0.f;
            s_dx[t][lane] = make_float2(D, D * u[j]);
            cu[j] = u[j]; cz[j] = z[j];
        }
        s_b[0][threadIdx.x] = rb;                          // ([TT][4 NW] flat)
        s_c[0][threadIdx.x] = rc;
        if (d.ckpt && w.live)
#pragma unroll
            for (int n = 0; n < NS; ++n)
                if (n0 + n < d.N) d.ckpt[(((int64_t)w.b * p.tiles + i) * d.N + n0 + n) * d.D + w.ch] = h[n];
        __syncthreads();
        if (i + 1 < ntile) load(t0 + TT);
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            const float2 dx = s_dx[t][lane];
            float y = 0.f;
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                h[n] = fmaf(__builtin_amdgcn_exp2f(dx.x * A2[n]), h[n], dx.y * s_b[t][n0 + n]);
                y = fmaf(s_c[t][n0 + n], h[n], y);
            }
            s_y[wv][t][lane] = y;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < EP; ++j) {
            const int t = wv + NW * j;
            float y = skip * cu[j];
#pragma unroll
            for (int v = 0; v < NW; ++v) y += s_y[v][t][lane];
            if (d.z) y *= silu_f(cz[j]);
            if (w.live && t0 + t < w.len) ((T*)d.y)[((int64_t)w.b * d.T + t0 + t) * d.D + w.ch] = from_f<T>(y);
        }
    }
    if (w.live) {
        for (int t = w.len + wv; t < d.T; t += NW) ((T*)d.y)[((int64_t)w.b * d.T + t) * d.D + w.ch] = from_f<T>(0.f);
        if (d.h_out)
#pragma unroll
            for (int n = 0; n < NS; ++n)
                if (n0 + n < d.N) d.h_out[((int64_t)w.b * d.D + w.ch) * d.N + n0 + n] = h[n];
    }
}

// Sum of 64 register values over the wave's 64 lanes, scattered: lane l returns the total of v[l].  Each step pairs lanes that differ in one
// index bit, adds, and keeps the half of the values whose index has the lane's bit: 63 adds instead of 64 x 6.  The upper two bits go
// through the half-wave and half-row register swaps (no select needed), the lower four through DPP (xor 8, mirror of 8, xor 2, xor 1).
template <int CTRL, int M> A8_DEV void scatter_step(float* v, bool upper) {
#pragma unroll
    for (int i = 0; i < M; ++i) {
        const float keep = upper ? v[i + M] : v[i], send = upper ? v[i] : v[i + M];
        v[i] = keep + dpp_f<CTRL>(send);
    }
}
A8_DEV float wave_sum_scatter64(float (&v)[64], int lane) {
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[i + 32]), false, false);
        v[i] = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[i]), __float_as_uint(v[i + 16]), false, false);
        v[i] = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
    scatter_step<0x128, 8>(v, lane & 8);          // row_ror:8
    scatter_step<0x141, 4>(v, lane & 4);          // row_half_mirror
    scatter_step<0x4E, 2>(v, lane & 2);           // quad_perm xor 2
    scatter_step<0xB1, 1>(v, lane & 1);           // quad_perm xor 1
    return v[0];
}

template <typename T, int NW> __global__ __launch_bounds__(64 * NW) void scan_bwd_kernel(ScanArgs p) {
    constexpr int EP = TT / NW;
    __shared__ float2 s_dx[TT][CH];                        // {D, D u}
    __shared__ float s_g[TT][CH];                          // dout silu(z)
    __shared__ __align__(16) float s_b[TT][NS * NW], s_c[TT][NS * NW];
    __shared__ float s_qb[NW][TT][CH], s_ak[NW][TT][CH], s_y[NW][TT][CH];
    const a8_selective_scan_desc& d = p.d;
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, n0 = wv * NS;
    const Where w = locate(p, lane);
    const float bias = d.dt_bias ? d.dt_bias[w.ch] : 0.f, skip = d.Dskip ? d.Dskip[w.ch] : 0.f;
    float A[NS], A2[NS], c[NS], dA[NS] = {};
#pragma unroll
    for (int n = 0; n < NS; ++n) {
        const bool has = n0 + n < d.N;
        A[n] = has ? d.A[(int64_t)w.ch * d.N + n0 + n] : 0.f;
        A2[n] = A[n] * SEQ_LOG2E;
        c[n] = has && w.live && d.dh_out ? d.dh_out[((int64_t)w.b * d.D + w.ch) * d.N + n0 + n] : 0.f;
    }
    float dskip = 0.f, dbias = 0.f;
    const int ntile = (w.len + TT - 1) / TT;
    float u[EP], dt[EP], z[EP], dy[EP], rb = 0.f, rc = 0.f, rh[NS] = {};
    auto load = [&](int i) {
#pragma unroll
        for (int j = 0; j < EP; ++j) {
            const int t = i * TT + wv + NW * j;
            const bool in = t < w.len && w.live;           // (an absent channel contributes nothing to dB and dC)
            u[j] = in ? ldf<T>(d.u, w.b * d.u_bs + t * d.u_ts + w.ch) : 0.f;
            dt[j] = in ? ldf<T>(d.dt, w.b * d.dt_bs + t * d.dt_ts + w.ch) : 0.f;
            z[j] = in && d.z ? ldf<T>(d.z, w.b * d.z_bs + t * d.z_ts + w.ch) : 0.f;
            dy[j] = in ? ldf<T>(d.dy, w.b * d.dy_bs + t * d.dy_ts + w.ch) : 0.f;
        }
        rb = load_bc<T, NW>(d.Bm, d.b_bs, d.b_ts, d.b_gs, p, w, i * TT);
        rc = load_bc<T, NW>(d.Cm, d.c_bs, d.c_ts, d.c_gs, p, w, i * TT);
#pragma unroll
        for (int n = 0; n < NS; ++n) rh[n] = w.live && n0 + n < d.N ? d.ckpt[(((int64_t)w.b * p.tiles + i) * d.N + n0 + n) * d.D + w.ch] : 0.f;
    };
    if (ntile > 0) load(ntile - 1);
    for (int i = ntile - 1; i >= 0; --i) {
        const int t0 = i * TT;
        float cu[EP], cr[EP], cz[EP], cdy[EP], a[TT][NS], h[TT + 1][NS];
#pragma unroll
        for (int j = 0; j < EP; ++j) {
            const int t = wv + NW * j;
            const float raw = dt[j] + bias, D = t0 + t < w.len ? (d.softplus ? softplus_f(raw) : raw) : 0.f;
            s_dx[t][lane] = make_float2(D, D * u[j]);
            s_g[t][lane] = d.z ? dy[j] * silu_f(z[j]) : dy[j];
            cu[j] = u[j]; cr[j] = raw; cz[j] = z[j]; cdy[j] = dy[j];
        }
        s_b[0][threadIdx.x] = rb;
        s_c[0][threadIdx.x] = rc;
#pragma unroll
        for (int n = 0; n < NS; ++n) h[0][n] = rh[n];
        __syncthreads();
        if (i > 0) load(i - 1);
#pragma unroll
        for (int t = 0; t < TT; ++t) {                     // the tile's states again, from the saved state before it
            const float2 dx = s_dx[t][lane];
            float y = 0.f;
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                a[t][n] = __builtin_amdgcn_exp2f(dx.x * A2[n]);
                h[t + 1][n] = fmaf(a[t][n], h[t][n], dx.y * s_b[t][n0 + n]);
                y = fmaf(s_c[t][n0 + n], h[t + 1][n], y);
            }
            if (d.z) s_y[wv][t][lane] = y;
        }
        float vb[TT * NS], vc[TT * NS];
#pragma unroll
        for (int t = TT - 1; t >= 0; --t) {
            const float2 dx = s_dx[t][lane];
            const float g = s_g[t][lane];
            float qb = 0.f, ak = 0.f;
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                const float q = fmaf(s_c[t][n0 + n], g, c[n]);
                vb[t * NS + n] = q * dx.y;
                vc[t * NS + n] = g * h[t + 1][n];
                qb = fmaf(q, s_b[t][n0 + n], qb);
                c[n] = a[t][n] * q;
                const float k = c[n] * h[t][n];
                ak = fmaf(A[n], k, ak);
                dA[n] = fmaf(k, dx.x, dA[n]);
            }
            s_qb[wv][t][lane] = qb;
            s_ak[wv][t][lane] = ak;
        }
        {
            const float sb = wave_sum_scatter64(vb, lane), sc = wave_sum_scatter64(vc, lane);
            const int t = t0 + (lane >> 2), n = n0 + (lane & 3);
            if (t < w.len && n < d.N) {
                const int64_t at = ((((int64_t)w.ct * d.B + w.b) * d.T + t) * d.G + w.g) * d.N + n;
                p.part_b[at] = sb;
                p.part_c[at] = sc;
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < EP; ++j) {
            const int t = wv + NW * j;
            const bool in = w.live && t0 + t < w.len;
            const float D = s_dx[t][lane].x, g = s_g[t][lane];
            float qb = 0.f, ak = 0.f, y = skip * cu[j];
#pragma unroll
            for (int v = 0; v < NW; ++v) { qb += s_qb[v][t][lane]; ak += s_ak[v][t][lane]; }
            const int64_t at = ((int64_t)w.b * d.T + t0 + t) * d.D + w.ch;
            float dd = fmaf(cu[j], qb, ak);
            if (d.softplus) dd *= sigmoid_f(cr[j]);
            if (in) {
                dskip = fmaf(g, cu[j], dskip);
                dbias += dd;
                ((T*)d.du)[at] = from_f<T>(fmaf(D, qb, skip * g));
                ((T*)d.ddt)[at] = from_f<T>(dd);
                if (d.z) {
#pragma unroll
                    for (int v = 0; v < NW; ++v) y += s_y[v][t][lane];
                    ((T*)d.dz)[at] = from_f<T>(cdy[j] * y * silu_grad_f(cz[j]));
                }
            }
        }
    }
    if (w.live)
        for (int t = w.len + wv; t < d.T; t += NW) {
            const int64_t at = ((int64_t)w.b * d.T + t) * d.D + w.ch;
            ((T*)d.du)[at] = from_f<T>(0.f);
            ((T*)d.ddt)[at] = from_f<T>(0.f);
            if (d.z) ((T*)d.dz)[at] = from_f<T>(0.f);
        }
    __syncthreads();                                       // (s_qb is read by the last tile's epilogue above)
    s_qb[wv][0][lane] = dskip;
    s_qb[wv][1][lane] = dbias;
    __syncthreads();
    float* const part = p.part + (int64_t)w.b * (d.N + 2) * d.D;
    if (w.live) {
#pragma unroll
        for (int n = 0; n < NS; ++n)
            if (n0 + n < d.N) {
                part[(int64_t)(n0 + n) * d.D + w.ch] = dA[n];
                if (d.dh0) d.dh0[((int64_t)w.b * d.D + w.ch) * d.N + n0 + n] = c[n];
            }
        if (wv == 0) {
            float s0 = 0.f, s1 = 0.f;
#pragma unroll
            for (int v = 0; v < NW; ++v) { s0 += s_qb[v][0][lane]; s1 += s_qb[v][1][lane]; }
            part[(int64_t)d.N * d.D + w.ch] = s0;
            part[(int64_t)(d.N + 1) * d.D + w.ch] = s1;
        }
    }
}

// dB, dC = the channel tiles' partial sums, in tile order; frames behind an utterance's end are zero
template <typename T> __global__ __launch_bounds__(256) void scan_bc_kernel(ScanArgs p) {
    const a8_selective_scan_desc& d = p.d;
    const int64_t row = (int64_t)d.G * d.N, total = (int64_t)d.B * d.T * row;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const int64_t bt = i / row;
    float sb = 0.f, sc = 0.f;
    if ((int)(bt % d.T) < seq_len(d.lengths, (int)(bt / d.T), d.T))
        for (int k = 0; k < p.tpg; ++k) { sb += p.part_b[k * total + i]; sc += p.part_c[k * total + i]; }
    ((T*)d.dBm)[i] = from_f<T>(sb);
    ((T*)d.dCm)[i] = from_f<T>(sc);
}

// One frame: 4 lanes per channel, 4 consecutive states per lane and round; the state is read and written once.
template <typename T> __global__ __launch_bounds__(256) void scan_step_kernel(ScanArgs p) {
    const a8_selective_scan_desc& d = p.d;
    const int b = blockIdx.y, c = blockIdx.x * 64 + (threadIdx.x >> 2), s4 = threadIdx.x & 3;
    const int ch = min(c, d.D - 1), g = ch / p.cpg;
    const float raw = ldf<T>(d.dt, b * d.dt_bs + ch) + (d.dt_bias ? d.dt_bias[ch] : 0.f);
    const float u = ldf<T>(d.u, b * d.u_bs + ch), D = d.softplus ? softplus_f(raw) : raw, x = D * u;
    float* const st = d.h_out + ((int64_t)b * d.D + ch) * d.N;
    const float* const A = d.A + (int64_t)ch * d.N;
    float y = 0.f;
    for (int n = s4 * 4; n < d.N; n += 16)
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (n + k < d.N) {
                const float h = fmaf(exp_fast(D * A[n + k]), st[n + k], x * ldf<T>(d.Bm, b * d.b_bs + g * d.b_gs + n + k));
                y = fmaf(ldf<T>(d.Cm, b * d.c_bs + g * d.c_gs + n + k), h, y);
                if (c < d.D) st[n + k] = h;
            }
    y += dpp_f<0xB1>(y);
    y += dpp_f<0x4E>(y);
    if (s4 == 0 && c < d.D) {
        if (d.Dskip) y = fmaf(d.Dskip[ch], u, y);
        if (d.z) y *= silu_f(ldf<T>(d.z, b * d.z_bs + ch));
        ((T*)d.y)[(int64_t)b * d.D + ch] = from_f<T>(y);
    }
}

int scan_check(const a8_selective_scan_desc* d, const char* what) {
    A8_REQUIRE(d != nullptr && d->size == (int)sizeof(a8_selective_scan_desc), "%s: descriptor size %d, expected %d", what, d ? d->size : 0, (int)sizeof(a8_selective_scan_desc));
    A8_REQUIRE(d->dtype == A8_F32 || d->dtype == A8_BF16, "%s: bad dtype %d", what, d->dtype);
    A8_REQUIRE(d->B >= 0 && d->T >= 0 && d->D >= 1 && d->N >= 1 && d->N <= 32, "%s: bad sizes B=%d T=%d D=%d N=%d (1 to 32 states)", what, d->B, d->T, d->D, d->N);
    A8_REQUIRE(d->G >= 1 && d->D % d->G == 0, "%s: %d channels do not split into %d groups", what, d->D, d->G);
    A8_REQUIRE(d->A != nullptr, "%s: null A", what);
    return A8_OK;
}
ScanArgs scan_args(const a8_selective_scan_desc* d) {
    ScanArgs p = {};
    p.d = *d;
    p.cpg = d->D / d->G;
    p.tpg = cdiv(p.cpg, CH);
    p.tiles = cdiv(d->T, TT);
    return p;
}
int64_t scan_blocks(const ScanArgs& p) { return (int64_t)p.d.B * p.d.G * p.tpg; }

#define SCAN_DISPATCH(KERNEL, STREAM)                                                                                                       \
    do {                                                                                                                                    \
        const dim3 grid((unsigned)scan_blocks(p));                                                                                          \
        const hipStream_t st = (hipStream_t)STREAM;                                                                                         \
        if (d->dtype == A8_BF16) {                                                                                                          \
            if (d->N <= 4) hipLaunchKernelGGL((KERNEL<bf16, 1>), grid, dim3(64), 0, st, p);                                                  \
            else if (d->N <= 8) hipLaunchKernelGGL((KERNEL<bf16, 2>), grid, dim3(128), 0, st, p);                                            \
            else if (d->N <= 16) hipLaunchKernelGGL((KERNEL<bf16, 4>), grid, dim3(256), 0, st, p);                                           \
            else hipLaunchKernelGGL((KERNEL<bf16, 8>), grid, dim3(512), 0, st, p);                                                           \
        } else {                                                                                                                            \
            if (d->N <= 4) hipLaunchKernelGGL((KERNEL<float, 1>), grid, dim3(64), 0, st, p);                                                 \
            else if (d->N <= 8) hipLaunchKernelGGL((KERNEL<float, 2>), grid, dim3(128), 0, st, p);                                           \
            else if (d->N <= 16) hipLaunchKernelGGL((KERNEL<float, 4>), grid, dim3(256), 0, st, p);                                          \
            else hipLaunchKernelGGL((KERNEL<float, 8>), grid, dim3(512), 0, st, p);                                                          \
        }                                                                                                                                   \
    } while (0)

}  // namespace

extern "C" int a8_selective_scan_workspace(const a8_selective_scan_desc* d, int backward, int64_t* ckpt_floats, int64_t* ws_floats) {
    if (int e = scan_check(d, "a8_selective_scan_workspace")) return e;
    A8_REQUIRE(ckpt_floats != nullptr && ws_floats != nullptr, "a8_selective_scan_workspace: null result");
    const ScanArgs p = scan_args(d);
    *ckpt_floats = (int64_t)d->B * p.tiles * d->N * d->D;
    *ws_floats = backward ? (int64_t)d->B * (d->N + 2) * d->D + 2 * (int64_t)p.tpg * d->B * d->T * d->G * d->N : 0;
    return A8_OK;
}

extern "C" int a8_selective_scan_fwd(const a8_selective_scan_desc* d, void* stream) {
    if (int e = scan_check(d, "a8_selective_scan_fwd")) return e;
    if (d->B == 0) return A8_OK;
    A8_REQUIRE(d->T == 0 || (d->u && d->dt && d->Bm && d->Cm && d->y), "a8_selective_scan_fwd: null u, dt, B, C or y");
    const ScanArgs p = scan_args(d);
    A8_REQUIRE(scan_blocks(p) < (1 << 22), "a8_selective_scan_fwd: B x D = %d x %d is too large", d->B, d->D);
    SCAN_DISPATCH(scan_fwd_kernel, stream);
    return a8_check_launch("a8_selective_scan_fwd");
}

extern "C" int a8_selective_scan_bwd(const a8_selective_scan_desc* d, void* stream) {
    if (int e = scan_check(d, "a8_selective_scan_bwd")) return e;
    ScanArgs p = scan_args(d);
    A8_REQUIRE(d->B == 0 || d->ws, "a8_selective_scan_bwd: null workspace");
    A8_REQUIRE(d->B == 0 || d->T == 0 || (d->u && d->dt && d->Bm && d->Cm && d->dy && d->ckpt && d->du && d->ddt && d->dBm && d->dCm && (d->dz || !d->z)),
               "a8_selective_scan_bwd: null operand");
    A8_REQUIRE(scan_blocks(p) < (1 << 22), "a8_selective_scan_bwd: B x D = %d x %d is too large", d->B, d->D);
    p.part = d->ws;
    p.part_b = p.part + (int64_t)d->B * (d->N + 2) * d->D;
    p.part_c = p.part_b + (int64_t)p.tpg * d->B * d->T * d->G * d->N;
    if (d->B > 0) {
        SCAN_DISPATCH(scan_bwd_kernel, stream);
        if (int e = a8_check_launch("a8_selective_scan_bwd")) return e;
        const int64_t total = (int64_t)d->B * d->T * d->G * d->N;
        if (total > 0) {
            const dim3 grid((unsigned)((total + 255) / 256));
            if (d->dtype == A8_BF16) hipLaunchKernelGGL((scan_bc_kernel<bf16>), grid, dim3(256), 0, (hipStream_t)stream, p);
            else hipLaunchKernelGGL((scan_bc_kernel<float>), grid, dim3(256), 0, (hipStream_t)stream, p);
            if (int e = a8_check_launch("a8_selective_scan_bwd")) return e;
        }
    }
    A8SeqReduce r = {p.part, d->B, d->N + 2, d->D, d->N, d->dA, {d->dD, d->ddt_bias}, d->add_dA, {d->add_dD, d->add_ddt_bias}};
    return a8i_seq_reduce(r, stream);
}

extern "C" int a8_selective_scan_step(const a8_selective_scan_desc* d, void* stream) {
    if (int e = scan_check(d, "a8_selective_scan_step")) return e;
    A8_REQUIRE(d->T == 1, "a8_selective_scan_step: one frame at a time (T = %d)", d->T);
    A8_REQUIRE(d->B <= 65535, "a8_selective_scan_step: B = %d is too large", d->B);
    if (d->B == 0) return A8_OK;
    A8_REQUIRE(d->u && d->dt && d->Bm && d->Cm && d->y && d->h_out, "a8_selective_scan_step: null u, dt, B, C, y or state");
    const ScanArgs p = scan_args(d);
    const dim3 grid(cdiv(d->D, 64), d->B);
    if (d->dtype == A8_BF16) hipLaunchKernelGGL((scan_step_kernel<bf16>), grid, dim3(256), 0, (hipStream_t)stream, p);
    else hipLaunchKernelGGL((scan_step_kernel<float>), grid, dim3(256), 0, (hipStream_t)stream, p);
    return a8_check_launch("a8_selective_scan_step");
}
