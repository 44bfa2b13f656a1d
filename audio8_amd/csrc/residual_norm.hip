// a8hip: the norms before and after a block, fused with the block's gate, its residual scale and the residual sum, forward and gradient.
//
//   p = N(o; pw, pb) (or o);  r = x + scale gate p;  n = N(r; w, b)      N: LayerNorm or RMS norm over the C channels of a row
// Gradient, from x, o, gate and the four row statistics (r is formed again in f32 instead of being read back rounded):
//   dR = dr + N'(dn w);  dx = dR;  dgate = dR scale p;  do = N'(dR scale gate pw);   N'(v) = rstd (v - mean(v) - hat mean(v hat)), RMS without mean(v)
//   dw = sum dn rhat, db = sum dn;  with E1 = sum dR gate ohat, E0 = sum dR gate:  dpw = scale E1, dpb = scale E0, dscale = pw E1 + pb E0
// (four column sums instead of five: p and dp are columns times ohat and dR gate).
//
// Bound by HBM.  A row is held in registers, 8 consecutive channels per lane and round, by one wave (forward up to 1024 channels, backward up to 512),
// by two (backward up to 1024) or by a block: every tensor is read and written once, statistics are exact two-pass in f32.  The backward walks many
// rows, the next row's loads in flight, the parameters in LDS, the column sums in registers.  bf16, both norms, a gate per utterance:
// 32 x 1499 x 1024 forward 83 us (393 MB, 4.8 TB/s), backward 142 us (589 MB, 4.1 TB/s), parameter gradients 13 us.
#include "a8_seq.h"
#include "a8hip_internal.h"

namespace {

enum { PLANE_W = 0, PLANE_B, PLANE_E1, PLANE_E0, PLANES };      // (rnorm_reduce_kernel takes them in pairs)

struct NormArgs { a8_residual_norm_desc d; int chunks, rows_per_chunk, vec; };

// 8 consecutive elements at p: 16-byte loads where the launch checked alignment and width, single elements below `left` otherwise
template <typename T> A8_DEV void ld8(float (&v)[8], const T* p, int vec, int left) {
    if (vec) {
        if constexpr (sizeof(T) == 2) {
            const bf16x8 r = *reinterpret_cast<const bf16x8*>(p);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = (float)r[k];
        } else {
            const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
            for (int k = 0; k < 4; ++k) { v[k] = a[k]; v[k + 4] = b[k]; }
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = k < left ? to_f(p[k]) : 0.f;
    }
}
template <typename T> A8_DEV void st8(T* p, const float (&v)[8], int vec, int left) {
    if (vec) {
        if constexpr (sizeof(T) == 2) {
            bf16x8 r;
#pragma unroll
            for (int k = 0; k < 8; ++k) r[k] = (bf16)v[k];
            *reinterpret_cast<bf16x8*>(p) = r;
        } else {
            *reinterpret_cast<f32x4*>(p) = (f32x4){v[0], v[1], v[2], v[3]};
            *reinterpret_cast<f32x4*>(p + 4) = (f32x4){v[4], v[5], v[6], v[7]};
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < left) p[k] = from_f<T>(v[k]);
    }
}

// sum over a row's threads: one wave, or RW waves through LDS (`red`: RW floats, reused by the next call behind its own barrier)
template <int RW> A8_DEV float row_sum(float v, float* red) {
    if constexpr (RW == 1) return wave_sum(v);
    else return block_sum<RW>(v, red);
}

// RW waves per row, NCH rounds of 8 channels per lane.  Blocks of 4 waves when RW = 1 (four rows at a time), else RW waves (one row).
template <typename T, int RW, int NCH> struct Row {
    static constexpr int NT = RW * 64, WAVES = RW == 1 ? 4 : RW;
    int C, vec, col[NCH];
    bool on[NCH];
    A8_DEV void init(int C_, int vec_) {
        C = C_; vec = vec_;
        const int tid = RW == 1 ? (threadIdx.x & 63) : threadIdx.x;
#pragma unroll
        for (int j = 0; j < NCH; ++j) { col[j] = (j * NT + tid) * 8; on[j] = col[j] < C; }
    }
    template <typename S> A8_DEV void load(float (&v)[NCH][8], const S* p) const {
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            if (on[j]) ld8<S>(v[j], p + col[j], vec, C - col[j]);
            else
#pragma unroll
                for (int k = 0; k < 8; ++k) v[j][k] = 0.f;
        }
    }
    template <typename S> A8_DEV void store(S* p, const float (&v)[NCH][8]) const {
#pragma unroll
        for (int j = 0; j < NCH; ++j)
            if (on[j]) st8<S>(p + col[j], v[j], vec, C - col[j]);
    }
    A8_DEV bool has(int j, int k) const { return vec ? on[j] : col[j] + k < C; }
};

template <int RW, int NCH, typename R> A8_DEV void stats(const R& row, const float (&v)[NCH][8], bool layer, float eps, float& mean, float& rstd, float* red) {
    mean = 0.f;
    const float inv = 1.0f / (float)row.C;
    if (layer) {
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
            for (int k = 0; k < 8; ++k) s += v[j][k];
        mean = row_sum<RW>(s, red) * inv;
    }
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < NCH; ++j)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float c = row.has(j, k) ? v[j][k] - mean : 0.f;
            q = fmaf(c, c, q);
        }
    rstd = 1.0f / sqrtf(fmaf(row_sum<RW>(q, red), inv, eps));
}

template <typename T, int RW, int NCH> __global__ __launch_bounds__(RW == 1 ? 256 : RW * 64) void rnorm_fwd_kernel(NormArgs p) {
    typedef Row<T, RW, NCH> R;
    __shared__ float red[R::WAVES];
    const a8_residual_norm_desc& d = p.d;
    R row;
    row.init(d.C, p.vec);
    const int rows = d.B * d.T;
    const int r = RW == 1 ? blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
    if (r >= rows) return;                                  // (a whole wave; RW > 1: the grid is exact)
    const bool layer = d.kind == A8_NORM_LAYER, lead = RW == 1 ? (threadIdx.x & 63) == 0 : threadIdx.x == 0;
    float o[NCH][8], x[NCH][8], v[NCH][8];
    row.load(o, (const T*)d.o + (int64_t)r * d.o_ld);
    row.load(x, (const T*)d.x + (int64_t)r * d.x_ld);
    if (d.post) {
        float mean, rstd;
        stats<RW, NCH>(row, o, layer, d.eps, mean, rstd, red);
        if (lead && d.stats) { d.stats[(int64_t)r] = mean; d.stats[(int64_t)rows + r] = rstd; }
        row.load(v, d.post_w);
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
            for (int k = 0; k < 8; ++k) o[j][k] = (o[j][k] - mean) * rstd * v[j][k];
        if (d.post_b) {
            row.load(v, d.post_b);
#pragma unroll
            for (int j = 0; j < NCH; ++j)
#pragma unroll
                for (int k = 0; k < 8; ++k) o[j][k] += v[j][k];
        }
    }
    if (d.gate) {
        row.load(v, (const T*)d.gate + (int64_t)(r / d.T) * d.g_bs + (d.gate_rows ? (int64_t)(r % d.T) * d.g_ts : 0));
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
            for (int k = 0; k < 8; ++k) o[j][k] *= v[j][k];
    }
    if (d.scale) {
        row.load(v, d.scale);
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
            for (int k = 0; k < 8; ++k) o[j][k] *= v[j][k];
    }
#pragma unroll
    for (int j = 0; j < NCH; ++j)
#pragma unroll
        for (int k = 0; k < 8; ++k) x[j][k] = row.has(j, k) ? x[j][k] + o[j][k] : 0.f;
    row.store((T*)d.r + (int64_t)r * d.C, x);
    if (d.n) {
        float mean, rstd;
        stats<RW, NCH>(row, x, layer, d.eps, mean, rstd, red);
        if (lead && d.stats) { d.stats[2 * (int64_t)rows + r] = mean; d.stats[3 * (int64_t)rows + r] = rstd; }
        row.load(v, d.w);
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
            for (int k = 0; k < 8; ++k) x[j][k] = (x[j][k] - mean) * rstd * v[j][k];
        if (d.b) {
            row.load(v, d.b);
#pragma unroll
            for (int j = 0; j < NCH; ++j)
#pragma unroll
                for (int k = 0; k < 8; ++k) x[j][k] += v[j][k];
        }
        row.store((T*)d.n + (int64_t)r * d.C, x);
    }
}

// 8 elements as loaded
template <typename T> struct Raw {
    T v[8];
    A8_DEV void load(const T* p, bool vec, int left) {
        if (vec) {
#pragma unroll
            for (int k = 0; k < (int)(8 * sizeof(T) / 16); ++k) reinterpret_cast<u32x4*>(v)[k] = reinterpret_cast<const u32x4*>(p)[k];
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = k < left ? p[k] : from_f<T>(0.f);
        }
    }
};

// two row sums at once.  Successive calls alternate between two `red`: a wave writes one only behind the barrier of the other's sum, in front of which
// every wave has read it, so a call has one barrier, and one that leaves the loads of the next row in flight.
template <int RW> A8_DEV void row_sum2(float& a, float& b, float2 (*red)[RW], int& turn) {
    a = wave_sum(a);
    b = wave_sum(b);
    if constexpr (RW > 1) {
        const int w = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) red[turn][w] = make_float2(a, b);
        lds_barrier();
        a = b = 0.f;
#pragma unroll
        for (int i = 0; i < RW; ++i) { a += red[turn][i].x; b += red[turn][i].y; }
        turn ^= 1;
    }
}

enum { GATE_NONE = 0, GATE_ROWS, GATE_UTT };
// one row as loaded
template <typename T, int NCH, bool GROWS> struct RawRow { Raw<T> o[NCH], x[NCH], dr[NCH], dn[NCH], g[GROWS ? NCH : 1]; float st[4]; };
// (the kind of gate is a template parameter for its registers: with all three in one kernel a row of 1024 took 314 and one wave per SIMD)
template <typename T, int RW, int NCH, bool VEC, int GATE> __global__ __launch_bounds__(RW == 1 ? 256 : RW * 64, VEC && RW <= 4 ? 3 : 1) void rnorm_bwd_kernel(NormArgs p) {
    typedef Row<T, RW, NCH> R;
    constexpr int W = R::NT * NCH * 8;                         // columns a row's threads cover
    // Rows in flight: two, where three waves per SIMD still hold them (32 x 1499 x 1024: 169 us with one row and two waves, 156 with one and three, 143 with two and three;
    // one wave per row, 32 x 2998 x 512: 127 us with one row, 270 with two and the spills of three waves).
    constexpr int AHEAD = RW == 1 || RW == 16 ? 1 : 2;
    __shared__ float2 red[2][RW];
    __shared__ __align__(16) float par[4][W];                  // scale, pw, pb, w (1, 1, 0, 1 where there is none); then the waves' column sums
    const a8_residual_norm_desc& d = p.d;
    int turn = 0;
    R row;
    row.init(d.C, VEC);
    const int rows = d.B * d.T, b = blockIdx.x / p.chunks, ck = blockIdx.x % p.chunks;
    const int ta = ck * p.rows_per_chunk, tb = min(ta + p.rows_per_chunk, d.T);
    const int wv = RW == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0, step = RW == 1 ? 4 : 1;
    constexpr bool gate_rows = GATE == GATE_ROWS;
    const bool layer = d.kind == A8_NORM_LAYER;
    for (int c = threadIdx.x; c < W; c += R::WAVES * 64) {
        const bool in = c < d.C;
        par[0][c] = in && d.scale ? d.scale[c] : 1.f;
        par[1][c] = in && d.post ? d.post_w[c] : 1.f;
        par[2][c] = in && d.post && d.post_b ? d.post_b[c] : 0.f;
        par[3][c] = in && d.w ? d.w[c] : 1.f;
    }
    __syncthreads();
    float acc[PLANES][NCH][8] = {};
    // the utterance's gate stays in registers, but not in the 128 of a block of 16 waves (32 x 187 x 8192: 246 us with it and its spills, 151 re-read)
    constexpr bool held = GATE == GATE_UTT && RW < 16;
    Raw<T> ug[GATE == GATE_UTT ? NCH : 1];
    auto load_ug = [&]() {
        if constexpr (GATE == GATE_UTT)
#pragma unroll
            for (int j = 0; j < NCH; ++j)
                if (row.on[j]) ug[j].load((const T*)d.gate + (int64_t)b * d.g_bs + row.col[j], VEC, d.C - row.col[j]);
    };
    if constexpr (held) load_ug();
    typedef RawRow<T, NCH, gate_rows> In;
    auto load = [&](In& in, int t) {
        const int64_t r = (int64_t)b * d.T + t;
#pragma unroll
        for (int j = 0; j < NCH; ++j)
            if (row.on[j]) {
                const int c = row.col[j], left = d.C - c;
                in.o[j].load((const T*)d.o + r * d.o_ld + c, VEC, left);
                if (d.dn) {
                    in.x[j].load((const T*)d.x + r * d.x_ld + c, VEC, left);
                    in.dn[j].load((const T*)d.dn + r * d.C + c, VEC, left);
                }
                if (d.dr) in.dr[j].load((const T*)d.dr + r * d.C + c, VEC, left);
                if constexpr (gate_rows) in.g[j].load((const T*)d.gate + (int64_t)b * d.g_bs + (int64_t)t * d.g_ts + c, VEC, left);
            }
#pragma unroll
        for (int k = 0; k < 4; ++k) in.st[k] = (k < 2 ? d.post != 0 : d.dn != nullptr) ? d.stats[k * (int64_t)rows + r] : k & 1;
    };
    auto walk = [&](In& in, int t) {
        if constexpr (GATE == GATE_UTT && !held) load_ug();
        auto gate_of = [&](int j, int k) { return gate_rows ? to_f(in.g[gate_rows ? j : 0].v[k]) : GATE == GATE_UTT ? to_f(ug[GATE == GATE_UTT ? j : 0].v[k]) : 1.f; };
        const int64_t r = (int64_t)b * d.T + t;
        float oh[NCH][8], g[gate_rows ? NCH : 1][8], h[NCH][8], v[NCH][8], dR[NCH][8];     // ohat (or o), the row's gate, rhat, scratch, dr then dR
        const float mo = in.st[0], so = in.st[1], mr = in.st[2], sr = in.st[3];
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            const float* const pc = &par[0][row.col[j]];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const bool on = row.has(j, k);
                const float xh = d.dn ? to_f(in.x[j].v[k]) : 0.f;
                oh[j][k] = on ? (to_f(in.o[j].v[k]) - mo) * so : 0.f;         // (mo = 0, so = 1 without a norm)
                const float gt = on ? gate_of(j, k) : 0.f;
                if constexpr (gate_rows) g[j][k] = gt;
                dR[j][k] = on && d.dr ? to_f(in.dr[j].v[k]) : 0.f;
                const float pp = fmaf(oh[j][k], pc[W + k], pc[2 * W + k]);
                h[j][k] = on && d.dn ? (fmaf(pc[k] * gt, pp, xh) - mr) * sr : 0.f;
                const float dn = on && d.dn ? to_f(in.dn[j].v[k]) : 0.f;
                acc[PLANE_W][j][k] = fmaf(dn, h[j][k], acc[PLANE_W][j][k]);
                acc[PLANE_B][j][k] += dn;
                v[j][k] = dn * pc[3 * W + k];
            }
        }
        if (t + AHEAD * step < tb) load(in, t + AHEAD * step);
        float s1 = 0.f, s2 = 0.f;
        const float inv = 1.0f / (float)d.C;
        if (d.dn) {
#pragma unroll
            for (int j = 0; j < NCH; ++j)
#pragma unroll
                for (int k = 0; k < 8; ++k) { s1 += v[j][k]; s2 = fmaf(v[j][k], h[j][k], s2); }
            row_sum2<RW>(s1, s2, red, turn);
            s1 = layer ? s1 * inv : 0.f;
            s2 *= inv;
#pragma unroll
            for (int j = 0; j < NCH; ++j)
#pragma unroll
                for (int k = 0; k < 8; ++k) dR[j][k] += row.has(j, k) ? sr * (v[j][k] - s1 - h[j][k] * s2) : 0.f;
        }
        row.store((T*)d.dx + r * d.C, dR);
        s1 = s2 = 0.f;
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            const float* const pc = &par[0][row.col[j]];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float pp = fmaf(oh[j][k], pc[W + k], pc[2 * W + k]), ds = dR[j][k] * pc[k];
                v[j][k] = ds * pp;                                          // the gate's gradient
                const float gt = gate_rows ? g[gate_rows ? j : 0][k] : row.has(j, k) ? gate_of(j, k) : 0.f;
                const float dg = gate_rows ? dR[j][k] * gt : dR[j][k];             // (a gate per utterance comes in at the end)
                acc[PLANE_E1][j][k] = fmaf(dg, oh[j][k], acc[PLANE_E1][j][k]);
                acc[PLANE_E0][j][k] += dg;
                h[j][k] = ds * gt * pc[W + k];                              // dp pw
                s1 += h[j][k];
                s2 = fmaf(h[j][k], oh[j][k], s2);
            }
        }
        if constexpr (gate_rows) row.store((T*)d.dgate + r * d.C, v);
        if (d.post) {
            row_sum2<RW>(s1, s2, red, turn);
            s1 = layer ? s1 * inv : 0.f;
            s2 *= inv;
#pragma unroll
            for (int j = 0; j < NCH; ++j)
#pragma unroll
                for (int k = 0; k < 8; ++k) h[j][k] = so * (h[j][k] - s1 - oh[j][k] * s2);
        }
        row.store((T*)d.d_o + r * d.C, h);
    };
    In in[AHEAD];
    const int t0 = ta + wv;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
        if (t0 + i * step < tb) load(in[i], t0 + i * step);
    for (int t = t0; t < tb; t += AHEAD * step) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            if (t + i * step < tb) walk(in[i], t + i * step);
    }
    // block totals [4 planes][C], and the utterance gate's gradient behind all blocks' planes.  Its terms per frame are dR scale (pw ohat + pb).
    float* const part = d.ws + (int64_t)blockIdx.x * PLANES * d.C;
    float* const partg = d.ws + (int64_t)gridDim.x * PLANES * d.C + (int64_t)blockIdx.x * d.C;
    constexpr bool utt = GATE == GATE_UTT;
    float gd[utt ? NCH : 1][8];
    if constexpr (utt && !held) load_ug();
    if constexpr (utt)
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            const float* const pc = &par[0][row.col[j]];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float gt = row.has(j, k) ? to_f(ug[j].v[k]) : 0.f;
                gd[j][k] = pc[k] * fmaf(pc[W + k], acc[PLANE_E1][j][k], pc[2 * W + k] * acc[PLANE_E0][j][k]);
                acc[PLANE_E1][j][k] *= gt;
                acc[PLANE_E0][j][k] *= gt;
            }
        }
    auto emit = [&](float* out, float (&v)[NCH][8]) {
        if constexpr (RW == 1) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < NCH; ++j)
#pragma unroll
                for (int k = 0; k < 8; ++k) par[wv][row.col[j] + k] = v[j][k];
            __syncthreads();
            for (int c = threadIdx.x; c < d.C; c += 256) out[c] = (par[0][c] + par[1][c]) + (par[2][c] + par[3][c]);
        } else {
            row.store(out, v);
        }
    };
#pragma unroll
    for (int q = 0; q < PLANES; ++q) emit(part + (int64_t)q * d.C, acc[q]);
    if constexpr (utt) emit(partg, gd);
}

// The blocks' column sums -> the five parameter gradients: the first 2 cdiv(C, 16) blocks, 16 columns and the two planes of one norm each; wave = plane x
// eighth of the rows, four rows and eight loads at a time.  The blocks behind them add up a gate per utterance's chunks: 1024 elements of dgate [B][C] each.
template <typename T> __global__ __launch_bounds__(1024) void rnorm_reduce_kernel(a8_residual_norm_desc d, int blocks, int chunks) {
    __shared__ float red[16][64];
    const int colblocks = (d.C + 15) / 16 * 2;
    if ((int)blockIdx.x >= colblocks) {
        const int64_t i = (int64_t)(blockIdx.x - colblocks) * 1024 + threadIdx.x;
        if (i >= (int64_t)d.B * d.C) return;
        const int64_t b = i / d.C, c = i % d.C;
        const float* const g = d.ws + (int64_t)blocks * PLANES * d.C + b * chunks * d.C + c;
        float s[8] = {};
        int k = 0;
        for (; k + 8 <= chunks; k += 8)
#pragma unroll
            for (int j = 0; j < 8; ++j) s[j] += g[(int64_t)(k + j) * d.C];
        for (; k < chunks; ++k) s[0] += g[(int64_t)k * d.C];
        ((T*)d.dgate)[i] = from_f<T>(((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7])));
        return;
    }
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, post = blockIdx.x & 1;
    const int c = (int)(blockIdx.x >> 1) * 16 + (lane & 15), cc = min(c, d.C - 1);
    const int64_t pitch = (int64_t)PLANES * d.C;
    const float* const in = d.ws + (int64_t)(2 * post + (wv & 1)) * d.C + cc;
    float s[8] = {};
    int i = (wv >> 1) * 4 + (lane >> 4);
    for (; i + 224 < blocks; i += 256)
#pragma unroll
        for (int k = 0; k < 8; ++k) s[k] += in[(i + 32 * k) * pitch];
    for (; i < blocks; i += 32) s[0] += in[i * pitch];
    red[wv][lane] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
    __syncthreads();
    if (threadIdx.x < 16 && c < d.C) {
        float t[2] = {};
#pragma unroll
        for (int w = 0; w < 16; ++w)
#pragma unroll
            for (int g = 0; g < 4; ++g) t[w & 1] += red[w][g * 16 + lane];
        auto put = [&](float* out, int add, float v) { if (out) out[c] = add ? out[c] + v : v; };
        if (post == 0) {
            put(d.dw, d.add_dw, t[0]);
            put(d.db, d.add_db, t[1]);
        } else {
            const float sc = d.scale ? d.scale[c] : 1.f, pw = d.post ? d.post_w[c] : 1.f, pb = d.post && d.post_b ? d.post_b[c] : 0.f;
            put(d.dpost_w, d.add_dpost_w, sc * t[0]);
            put(d.dpost_b, d.add_dpost_b, sc * t[1]);
            put(d.dscale, d.add_dscale, fmaf(pw, t[0], pb * t[1]));
        }
    }
}

int norm_check(const a8_residual_norm_desc* d, const char* what) {
    A8_REQUIRE(d != nullptr && d->size == (int)sizeof(a8_residual_norm_desc), "%s: descriptor size %d, expected %d", what, d ? d->size : 0, (int)sizeof(a8_residual_norm_desc));
    A8_REQUIRE(d->dtype == A8_F32 || d->dtype == A8_BF16, "%s: bad dtype %d", what, d->dtype);
    A8_REQUIRE(d->B >= 0 && d->T >= 0 && d->C >= 1 && d->C <= 8192, "%s: bad sizes B=%d T=%d C=%d (1 to 8192 channels)", what, d->B, d->T, d->C);
    const int row_threads = d->C <= 1024 ? 64 : d->C <= 2048 ? 256 : d->C <= 4096 ? 512 : 1024;       // (forward; a grid holds less than 2^32 threads)
    A8_REQUIRE(((int64_t)d->B * d->T + 4) * row_threads < (1ll << 32) && (int64_t)d->B * d->T < (1 << 30), "%s: B x T = %d x %d is too large", what, d->B, d->T);
    A8_REQUIRE(d->kind == A8_NORM_LAYER || d->kind == A8_NORM_RMS, "%s: unknown kind %d", what, d->kind);
    A8_REQUIRE(!d->post || d->post_w, "%s: null post weight", what);
    return A8_OK;
}
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
// 16-byte accesses: width, row strides and every base address a multiple of them
NormArgs norm_args(const a8_residual_norm_desc* d) {
    NormArgs p = {};
    p.d = *d;
    const void* ptrs[] = {d->x, d->o, d->gate, d->r, d->n, d->post_w, d->post_b, d->w, d->b, d->scale, d->dr, d->dn, d->dx, d->d_o, d->dgate, d->ws};
    p.vec = d->C % 8 == 0 && d->x_ld % 8 == 0 && d->o_ld % 8 == 0 && (!d->gate || (d->g_bs % 8 == 0 && (!d->gate_rows || d->g_ts % 8 == 0)));
    for (const void* q : ptrs) p.vec = p.vec && aligned16(q);
    // the backward's blocks: what the CUs hold at once, three waves per SIMD up to 2048 channels and one block per CU beyond, with at least 4 rows each
    const int resident = d->C <= 512 ? 768 : d->C <= 1024 ? 1536 : d->C <= 2048 ? 768 : 256;
    const int per_b = d->B > 0 ? std::max(1, resident / d->B) : 1;
    p.rows_per_chunk = d->T > 0 ? cdiv(d->T, per_b) : 1;
    if (p.rows_per_chunk < 4) p.rows_per_chunk = 4;
    p.chunks = d->T > 0 ? cdiv(d->T, p.rows_per_chunk) : 0;
    return p;
}

// Forward: a wave per row up to 1024 channels (four rows side by side), a block per row beyond.
#define NORM_FWD(T)                                                                                                              \
    (d->C <= 512 ? (rnorm_fwd_kernel<T, 1, 1>) : d->C <= 1024 ? (rnorm_fwd_kernel<T, 1, 2>) : d->C <= 2048 ? (rnorm_fwd_kernel<T, 4, 1>)    \
     : d->C <= 4096 ? (rnorm_fwd_kernel<T, 8, 1>) : (rnorm_fwd_kernel<T, 16, 1>))
// Backward: two waves per row from 513 on (a lane with 16 channels takes over 250 registers: 8 x 781 x 768 39 us against 28).
#define NORM_BWD(T, VEC, GATE)                                                                                                    \
    (d->C <= 512 ? (rnorm_bwd_kernel<T, 1, 1, VEC, GATE>) : d->C <= 1024 ? (rnorm_bwd_kernel<T, 2, 1, VEC, GATE>)                 \
     : d->C <= 2048 ? (rnorm_bwd_kernel<T, 4, 1, VEC, GATE>) : d->C <= 4096 ? (rnorm_bwd_kernel<T, 8, 1, VEC, GATE>) : (rnorm_bwd_kernel<T, 16, 1, VEC, GATE>))
#define NORM_GATE(T, VEC) (!d->gate ? NORM_BWD(T, VEC, GATE_NONE) : d->gate_rows ? NORM_BWD(T, VEC, GATE_ROWS) : NORM_BWD(T, VEC, GATE_UTT))

}  // namespace

extern "C" int a8_residual_norm_fwd(const a8_residual_norm_desc* d, void* stream) {
    if (int e = norm_check(d, "a8_residual_norm_fwd")) return e;
    if (d->B == 0 || d->T == 0) return A8_OK;
    A8_REQUIRE(d->x && d->o && d->r && (d->w || !d->n), "a8_residual_norm_fwd: null x, o, r or weight");
    const NormArgs p = norm_args(d);
    const int rows = d->B * d->T;
    auto kernel = d->dtype == A8_BF16 ? NORM_FWD(bf16) : NORM_FWD(float);
    hipLaunchKernelGGL(kernel, dim3(d->C <= 1024 ? cdiv(rows, 4) : rows), dim3(d->C <= 2048 ? 256 : d->C <= 4096 ? 512 : 1024), 0, (hipStream_t)stream, p);
    return a8_check_launch("a8_residual_norm_fwd");
}

extern "C" int a8_residual_norm_bwd_workspace(const a8_residual_norm_desc* d, int64_t* floats) {
    if (int e = norm_check(d, "a8_residual_norm_bwd_workspace")) return e;
    A8_REQUIRE(floats != nullptr, "a8_residual_norm_bwd_workspace: null result");
    *floats = (int64_t)d->B * norm_args(d).chunks * (PLANES + 1) * d->C;
    return A8_OK;
}

extern "C" int a8_residual_norm_bwd(const a8_residual_norm_desc* d, void* stream) {
    if (int e = norm_check(d, "a8_residual_norm_bwd")) return e;
    const NormArgs p = norm_args(d);
    const int blocks = d->B * p.chunks, threads = d->C <= 512 ? 256 : d->C <= 1024 ? 128 : d->C <= 2048 ? 256 : d->C <= 4096 ? 512 : 1024;
    const int64_t sums = 2 * cdiv(d->C, 16) + (d->gate && !d->gate_rows ? ((int64_t)d->B * d->C + 1023) / 1024 : 0);
    // (a grid holds less than 2^32 threads; a gate per utterance takes a block per utterance, and a thread per element of its gradient)
    A8_REQUIRE((int64_t)blocks * threads < (1ll << 32) && sums * 1024 < (1ll << 32), "a8_residual_norm_bwd: B x T x C = %d x %d x %d is too large", d->B, d->T, d->C);
    if (blocks > 0) {
        A8_REQUIRE(d->x && d->o && d->dx && d->d_o && d->ws && (d->dgate || !d->gate) && (d->stats || !(d->post || d->dn)) && (d->w || !d->dn),
                   "a8_residual_norm_bwd: null operand");
        auto kernel = d->dtype == A8_BF16 ? (p.vec ? NORM_GATE(bf16, true) : NORM_GATE(bf16, false)) : (p.vec ? NORM_GATE(float, true) : NORM_GATE(float, false));
        hipLaunchKernelGGL(kernel, dim3(blocks), dim3(threads), 0, (hipStream_t)stream, p);
        if (int e = a8_check_launch("a8_residual_norm_bwd")) return e;
    }
    const dim3 grid((unsigned)sums);
    if (d->dtype == A8_BF16) hipLaunchKernelGGL(rnorm_reduce_kernel<bf16>, grid, dim3(1024), 0, (hipStream_t)stream, *d, blocks, p.chunks);
    else hipLaunchKernelGGL(rnorm_reduce_kernel<float>, grid, dim3(1024), 0, (hipStream_t)stream, *d, blocks, p.chunks);
    return a8_check_launch("a8_residual_norm_bwd");
}
