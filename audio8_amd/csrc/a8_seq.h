// a8hip -- what the causal sequence kernels (causal_conv.hip, selective_scan.hip, residual_norm.hip) share.
#pragma once
#include "a8_common.h"

constexpr float SEQ_LOG2E = 1.4426950408889634f;

A8_DEV float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * SEQ_LOG2E); }
A8_DEV float sigmoid_f(float x) { return __builtin_amdgcn_rcpf(1.0f + exp_fast(-x)); }
A8_DEV float silu_f(float x) { return x * sigmoid_f(x); }
// d/dx [x s(x)] = s (1 + x (1 - s)).  1 - s(x) is taken as s(-x): the difference loses all its bits for large x.
A8_DEV float silu_grad_f(float x) {
    const float e = exp_fast(-fabsf(x)), r = __builtin_amdgcn_rcpf(1.0f + e);
    const float big = r, small = e * r;                       // s(|x|), s(-|x|)
    const float s = x >= 0.f ? big : small, c = x >= 0.f ? small : big;
    return s * fmaf(x, c, 1.0f);
}
// softplus(x) = max(x, 0) + log1p(e), e = exp(-|x|) in (0, 1].  log1p(e) = 2 atanh(s), s = e / (2 + e) <= 1/3, with 2 atanh(s) / s as a polynomial of
// degree 4 in s^2 (Chebyshev fit on [0, 1/9]: 4e-9 off, 7e-8 evaluated in f32): no 1 + e is rounded, so small step lengths keep their relative precision.
A8_DEV float softplus_f(float x) {
    const float e = exp_fast(-fabsf(x));
    const float s = e * __builtin_amdgcn_rcpf(2.0f + e), q = s * s;
    float r = 0.2817465662956238f;
    r = fmaf(r, q, 0.2796141803264618f);
    r = fmaf(r, q, 0.40024852752685547f);
    r = fmaf(r, q, 0.6666631698608398f);
    r = fmaf(r, q, 2.0f);
    return fmaf(s, r, fmaxf(x, 0.f));
}

// A block barrier for LDS only: __syncthreads also drains the wave's global loads and stores, which would put the latency of every prefetch and
// of every output store on the path of each tile.
A8_DEV void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// `planes` column sums over `rows` partial rows [rows][planes][C]: plane q < np goes to major[c * np + q] (a [C][np] matrix), plane np + i to
// minor[i][c]; null targets are skipped.  add = 1 accumulates.  Summed in a fixed order: the same inputs give the same bits.
struct A8SeqReduce {
    const float* in; int rows, planes, C, np;
    float* major; float* minor[2];
    int add_major, add_minor[2];
};
constexpr int SEQ_REDUCE_MAX = 1 << 26;      // C stays below: a block of 1024 threads per 16 columns, a grid of less than 2^32 (callers refuse before they launch)
int a8i_seq_reduce(const A8SeqReduce& r, void* stream);

// a descriptor's frame count of utterance b: lengths[b] clamped to [0, T]
A8_DEV int seq_len(const int32_t* lengths, int b, int T) { return lengths ? min(max(lengths[b], 0), T) : T; }
