// a8hip: the norms before and after a block, fused with the block's gate, its residual scale and the residual sum, forward and gradient.
//
//   p = N(o; pw, pb) (or o);  r = x + scale gate p;  n = N(r; w, b)      N: LayerNorm or RMS norm over the C channels of a row
// Gradient, from x, o, gate and the four row statistics (r is formed again in f32 instead of being read back rounded):
//   dR = dr + N'(dn w);  dx = dR;  dgate = dR scale p;  dscale = sum dR gate p;  dp = dR scale gate;  do = N'(dp pw)
//   dw = sum dn rhat, db = sum dn, dpw = sum dp ohat, dpb = sum dp;   N'(v) = rstd (v - mean(v) - hat mean(v hat)), RMS without mean(v)
//
// A row is held in registers by one wave (C <= 1024) or by a block (wider rows), 8 consecutive channels per lane and round: every tensor is
// read and written once, statistics are exact two-pass in f32, and the backward keeps its column sums in registers over all rows of its block.
#include "a8_seq.h"
#include "a8hip_internal.h"

namespace {

enum { PLANE_W = 0, PLANE_B, PLANE_PW, PLANE_PB, PLANE_SCALE, PLANES };

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

// v -> rstd (v - mean(v) - h mean(v h)), RMS without mean(v)
template <int RW, int NCH, typename R> A8_DEV void norm_back(const R& row, float (&v)[NCH][8], const float (&h)[NCH][8], bool layer, float rstd, float* red) {
    float s = 0.f, q = 0.f;
#pragma unroll
    for (int j = 0; j < NCH; ++j)
#pragma unroll
        for (int k = 0; k < 8; ++k) { s += v[j][k]; q = fmaf(v[j][k], h[j][k], q); }
    const float inv = 1.0f / (float)row.C;
    s = layer ? row_sum<RW>(s, red) * inv : 0.f;
    q = row_sum<RW>(q, red) * inv;
#pragma unroll
    for (int j = 0; j < NCH; ++j)
#pragma unroll
        for (int k = 0; k < 8; ++k) v[j][k] = rstd * (v[j][k] - s - h[j][k] * q);
}

template <typename T, int RW, int NCH> __global__ __launch_bounds__(RW == 1 ? 256 : RW * 64) void rnorm_bwd_kernel(NormArgs p) {
    typedef Row<T, RW, NCH> R;
    __shared__ float red[R::WAVES];
    __shared__ float comb[RW == 1 ? 4 * NCH * 512 : 1];
    const a8_residual_norm_desc& d = p.d;
    R row;
    row.init(d.C, p.vec);
    const int rows = d.B * d.T, b = blockIdx.x / p.chunks, ck = blockIdx.x % p.chunks;
    const int ta = ck * p.rows_per_chunk, tb = min(ta + p.rows_per_chunk, d.T);
    const int wv = RW == 1 ? threadIdx.x >> 6 : 0, step = RW == 1 ? 4 : 1;
    const bool layer = d.kind == A8_NORM_LAYER, gate_rows = d.gate && d.gate_rows;
    float acc[PLANES][NCH][8] = {}, accg[NCH][8] = {};
    for (int t = ta + wv; t < tb; t += step) {
        const int64_t r = (int64_t)b * d.T + t;
        float oh[NCH][8], s[NCH][8], v[NCH][8], h[NCH][8], dr[NCH][8];     // ohat (or o); scale x gate; scratch; rhat; dR
        row.load(oh, (const T*)d.o + r * d.o_ld);
        float rstd_o = 0.f;
        if (d.post) {
            const float mean = d.stats[r];
            rstd_o = d.stats[(int64_t)rows + r];
#pragma unroll
            for (int j = 0; j < NCH; ++j)
#pragma unroll
                for (int k = 0; k < 8; ++k) oh[j][k] = row.has(j, k) ? (oh[j][k] - mean) * rstd_o : 0.f;
        }
        float pp[NCH][8];                                                   // p
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
            for (int k = 0; k < 8; ++k) pp[j][k] = oh[j][k];
        if (d.post) {
            row.load(v, d.post_w);
#pragma unroll
            for (int j = 0; j < NCH; ++j)
#pragma unroll
                for (int k = 0; k < 8; ++k) pp[j][k] *= v[j][k];
            if (d.post_b) {
                row.load(v, d.post_b);
#pragma unroll
                for (int j = 0; j < NCH; ++j)
#pragma unroll
                    for (int k = 0; k < 8; ++k) pp[j][k] += v[j][k];
            }
        }
        float gt[NCH][8];
        if (d.gate) row.load(gt, (const T*)d.gate + (int64_t)b * d.g_bs + (gate_rows ? (int64_t)t * d.g_ts : 0));
        else
#pragma unroll
            for (int j = 0; j < NCH; ++j)
#pragma unroll
                for (int k = 0; k < 8; ++k) gt[j][k] = 1.f;
        if (d.scale) row.load(s, d.scale);
        else
#pragma unroll
            for (int j = 0; j < NCH; ++j)
#pragma unroll
                for (int k = 0; k < 8; ++k) s[j][k] = 1.f;
        if (d.dr) row.load(dr, (const T*)d.dr + r * d.C);
        else
#pragma unroll
            for (int j = 0; j < NCH; ++j)
#pragma unroll
                for (int k = 0; k < 8; ++k) dr[j][k] = 0.f;
        if (d.dn) {
            const float mean = d.stats[2 * (int64_t)rows + r], rstd = d.stats[3 * (int64_t)rows + r];
            row.load(h, (const T*)d.x + r * d.x_ld);
#pragma unroll
            for (int j = 0; j < NCH; ++j)
#pragma unroll
                for (int k = 0; k < 8; ++k) h[j][k] = row.has(j, k) ? (h[j][k] + s[j][k] * gt[j][k] * pp[j][k] - mean) * rstd : 0.f;
            float dn[NCH][8];
            row.load(dn, (const T*)d.dn + r * d.C);
            row.load(v, d.w);
#pragma unroll
            for (int j = 0; j < NCH; ++j)
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    acc[PLANE_W][j][k] = fmaf(dn[j][k], h[j][k], acc[PLANE_W][j][k]);
                    acc[PLANE_B][j][k] += dn[j][k];
                    dn[j][k] *= v[j][k];
                }
            norm_back<RW, NCH>(row, dn, h, layer, rstd, red);
#pragma unroll
            for (int j = 0; j < NCH; ++j)
#pragma unroll
                for (int k = 0; k < 8; ++k) dr[j][k] += row.has(j, k) ? dn[j][k] : 0.f;
        }
        row.store((T*)d.dx + r * d.C, dr);
        if (d.gate) {
#pragma unroll
            for (int j = 0; j < NCH; ++j)
#pragma unroll
                for (int k = 0; k < 8; ++k) { v[j][k] = dr[j][k] * s[j][k] * pp[j][k]; accg[j][k] += v[j][k]; }
            if (gate_rows) row.store((T*)d.dgate + r * d.C, v);
        }
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                acc[PLANE_SCALE][j][k] = fmaf(dr[j][k] * gt[j][k], pp[j][k], acc[PLANE_SCALE][j][k]);
                dr[j][k] *= s[j][k] * gt[j][k];                             // dp
                acc[PLANE_PW][j][k] = fmaf(dr[j][k], oh[j][k], acc[PLANE_PW][j][k]);
                acc[PLANE_PB][j][k] += dr[j][k];
            }
        if (d.post) {
            row.load(v, d.post_w);
#pragma unroll
            for (int j = 0; j < NCH; ++j)
#pragma unroll
                for (int k = 0; k < 8; ++k) dr[j][k] *= v[j][k];
            norm_back<RW, NCH>(row, dr, oh, layer, rstd_o, red);
        }
        row.store((T*)d.d_o + r * d.C, dr);
    }
    // block totals: the four waves' rows are joined through LDS when a row is one wave
    auto emit = [&](float* out, float (&v)[NCH][8]) {
        if constexpr (RW == 1) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < NCH; ++j)
#pragma unroll
                for (int k = 0; k < 8; ++k) comb[wv * NCH * 512 + row.col[j] + k] = v[j][k];
            __syncthreads();
            for (int c = threadIdx.x; c < d.C; c += 256)
                out[c] = (comb[c] + comb[NCH * 512 + c]) + (comb[2 * NCH * 512 + c] + comb[3 * NCH * 512 + c]);
        } else {
#pragma unroll
            for (int j = 0; j < NCH; ++j)
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (row.col[j] + k < d.C) out[row.col[j] + k] = v[j][k];
        }
    };
    float* const part = d.ws + (int64_t)blockIdx.x * PLANES * d.C;
#pragma unroll
    for (int q = 0; q < PLANES; ++q) emit(part + (int64_t)q * d.C, acc[q]);
    if (d.gate && !gate_rows) emit(d.ws + (int64_t)gridDim.x * PLANES * d.C + (int64_t)blockIdx.x * d.C, accg);
}

// dgate of a gate per utterance: the sum of the utterance's chunks
template <typename T> __global__ __launch_bounds__(256) void rnorm_gate_kernel(NormArgs p, const float* part) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)p.d.B * p.d.C) return;
    const int64_t b = i / p.d.C, c = i % p.d.C;
    float s = 0.f;
    for (int k = 0; k < p.chunks; ++k) s += part[(b * p.chunks + k) * p.d.C + c];
    ((T*)p.d.dgate)[i] = from_f<T>(s);
}

int norm_check(const a8_residual_norm_desc* d, const char* what) {
    A8_REQUIRE(d != nullptr && d->size == (int)sizeof(a8_residual_norm_desc), "%s: descriptor size %d, expected %d", what, d ? d->size : 0, (int)sizeof(a8_residual_norm_desc));
    A8_REQUIRE(d->dtype == A8_F32 || d->dtype == A8_BF16, "%s: bad dtype %d", what, d->dtype);
    A8_REQUIRE(d->B >= 0 && d->T >= 0 && d->C >= 1 && d->C <= 8192, "%s: bad sizes B=%d T=%d C=%d (1 to 8192 channels)", what, d->B, d->T, d->C);
    A8_REQUIRE((int64_t)d->B * d->T < (1 << 30), "%s: B x T = %d x %d is too large", what, d->B, d->T);
    A8_REQUIRE(d->kind == A8_NORM_LAYER || d->kind == A8_NORM_RMS, "%s: unknown kind %d", what, d->kind);
    A8_REQUIRE(!d->post || d->post_w, "%s: null post weight", what);
    return A8_OK;
}
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
// 16-byte accesses: width, row strides and every base address a multiple of them
NormArgs norm_args(const a8_residual_norm_desc* d) {
    NormArgs p = {};
    p.d = *d;
    const void* ptrs[] = {d->x, d->o, d->gate, d->r, d->n, d->post_w, d->post_b, d->w, d->b, d->scale, d->dr, d->dn, d->dx, d->d_o, d->dgate};
    p.vec = d->C % 8 == 0 && d->x_ld % 8 == 0 && d->o_ld % 8 == 0 && (!d->gate || (d->g_bs % 8 == 0 && (!d->gate_rows || d->g_ts % 8 == 0)));
    for (const void* q : ptrs) p.vec = p.vec && aligned16(q);
    const int per_b = d->B > 0 ? cdiv(512, d->B) : 1;        // about 512 blocks in all, at least 4 rows each
    p.rows_per_chunk = d->T > 0 ? cdiv(d->T, per_b) : 1;
    if (p.rows_per_chunk < 4) p.rows_per_chunk = 4;
    p.chunks = d->T > 0 ? cdiv(d->T, p.rows_per_chunk) : 0;
    return p;
}

#define NORM_DISPATCH(KERNEL, BLOCKS1, BLOCKSN)                                                                                     \
    do {                                                                                                                            \
        const hipStream_t st = (hipStream_t)stream;                                                                                 \
        const dim3 g1((unsigned)(BLOCKS1)), gn((unsigned)(BLOCKSN));                                                                \
        if (d->dtype == A8_BF16) {                                                                                                  \
            if (d->C <= 512) hipLaunchKernelGGL((KERNEL<bf16, 1, 1>), g1, dim3(256), 0, st, p);                                      \
            else if (d->C <= 1024) hipLaunchKernelGGL((KERNEL<bf16, 1, 2>), g1, dim3(256), 0, st, p);                                \
            else if (d->C <= 2048) hipLaunchKernelGGL((KERNEL<bf16, 4, 1>), gn, dim3(256), 0, st, p);                                \
            else if (d->C <= 4096) hipLaunchKernelGGL((KERNEL<bf16, 8, 1>), gn, dim3(512), 0, st, p);                                \
            else hipLaunchKernelGGL((KERNEL<bf16, 16, 1>), gn, dim3(1024), 0, st, p);                                                \
        } else {                                                                                                                    \
            if (d->C <= 512) hipLaunchKernelGGL((KERNEL<float, 1, 1>), g1, dim3(256), 0, st, p);                                     \
            else if (d->C <= 1024) hipLaunchKernelGGL((KERNEL<float, 1, 2>), g1, dim3(256), 0, st, p);                               \
            else if (d->C <= 2048) hipLaunchKernelGGL((KERNEL<float, 4, 1>), gn, dim3(256), 0, st, p);                               \
            else if (d->C <= 4096) hipLaunchKernelGGL((KERNEL<float, 8, 1>), gn, dim3(512), 0, st, p);                               \
            else hipLaunchKernelGGL((KERNEL<float, 16, 1>), gn, dim3(1024), 0, st, p);                                               \
        }                                                                                                                           \
    } while (0)

}  // namespace

extern "C" int a8_residual_norm_fwd(const a8_residual_norm_desc* d, void* stream) {
    if (int e = norm_check(d, "a8_residual_norm_fwd")) return e;
    if (d->B == 0 || d->T == 0) return A8_OK;
    A8_REQUIRE(d->x && d->o && d->r && (d->w || !d->n), "a8_residual_norm_fwd: null x, o, r or weight");
    const NormArgs p = norm_args(d);
    const int rows = d->B * d->T;
    NORM_DISPATCH(rnorm_fwd_kernel, cdiv(rows, 4), rows);
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
    const int blocks = d->B * p.chunks;
    if (blocks > 0) {
        A8_REQUIRE(d->x && d->o && d->dx && d->d_o && d->ws && (d->dgate || !d->gate) && (d->stats || !(d->post || d->dn)) && (d->w || !d->dn),
                   "a8_residual_norm_bwd: null operand");
        NORM_DISPATCH(rnorm_bwd_kernel, blocks, blocks);
        if (int e = a8_check_launch("a8_residual_norm_bwd")) return e;
    }
    if (d->gate && !d->gate_rows && d->B > 0) {
        const dim3 grid((unsigned)(((int64_t)d->B * d->C + 255) / 256));
        const float* part = d->ws + (int64_t)blocks * PLANES * d->C;
        if (d->dtype == A8_BF16) hipLaunchKernelGGL((rnorm_gate_kernel<bf16>), grid, dim3(256), 0, (hipStream_t)stream, p, part);
        else hipLaunchKernelGGL((rnorm_gate_kernel<float>), grid, dim3(256), 0, (hipStream_t)stream, p, part);
        if (int e = a8_check_launch("a8_residual_norm_bwd")) return e;
    }
    A8SeqReduce r = {d->ws, blocks, PLANES, d->C, 0, nullptr, {d->dw, d->db, d->dpost_w, d->dpost_b, d->dscale}, 0, {d->add_dw, d->add_db, d->add_dpost_w, d->add_dpost_b, d->add_dscale}};
    return a8i_seq_reduce(r, stream);
}
