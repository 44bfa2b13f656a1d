// a8hip: selective state space scan, channels-last, forward, gradient and single-frame step.
//
//   D_t = softplus(dt + dt_bias);  h_t[n] = exp(D_t A[n]) h_{t-1}[n] + D_t u_t B_t[n];  y_t = sum_n C_t[n] h_t[n] + Dskip u_t;  out = y silu(z)
// per channel with N <= 32 states; B and C are shared by the channels of a group.  Adjoint, with g = dout silu(z) and c_t = exp(D_{t+1} A) q_{t+1}:
//   q_t = C_t g_t + c_t;   dC_t = sum_ch g h_t;   dB_t = sum_ch q D u;   du = D sum_n q B + Dskip g;
//   dD = u sum_n q B + sum_n A k_t,  k_t = exp(D_t A) q_t h_{t-1};   dA = sum_t k_t D_t;   d dt = dD sigmoid(dt + dt_bias)
// (c_{t-1} = exp(D_t A) q_t, so k_t = c_{t-1} h_{t-1}: the adjoint's own product is reused).
//
// Layout: a lane is a channel, a wave is NS states of 64 channels, a block is ceil(N / NS) waves of the same 64 channels: the frame inputs are
// read along the channels (64 lanes, 128 B in bf16, any alignment), no state is ever exchanged between lanes, and only the sums over states
// (y; q B, A k) cross waves, through LDS once per tile of 16 frames.  softplus / silu run once per (frame, channel), split over the block's
// waves, not once per state.  A wave's B and C of a tile (16 NS values each) sit in NS VGPRs, the same 16 values in each row of 16 lanes: the
// row broadcast of a DPP operand hands them to the multiply for nothing (read as LDS broadcasts they took 32 16-byte reads per wave and tile).
// Everything between the inputs and the outputs is f32: steps, decays, states, adjoints and all sums.
#include "a8_seq.h"
#include "a8hip_internal.h"
#include <utility>

namespace {

constexpr int TT = 16;      // frames of a tile
constexpr int CH = 64;      // channels of a block
constexpr int FNS = 2;      // states of a wave, forward: 8 waves for 16 states, two per SIMD from one block (with 4: 1 x 781 x 1536 106 us against 88; no difference on a full card)
constexpr int BNS = 4;      // states of a wave, backward: 16 frames x 4 states of decays and of states live in registers

struct ScanArgs {
    a8_selective_scan_desc d;
    int cpg, tpg, tiles;               // channels and channel tiles per group, frame tiles of T
    int chunks, tpc;                   // frame chunks that run side by side, tiles per chunk
    float* ends;                       // chunks > 1: [B][chunks][N + 1][D] each chunk's own end state (backward: adjoint at its beginning) and sum of steps
    float* part;                       // backward: [B][chunks][N + 2][D] partial dA planes, dD, ddt_bias
    float* part_b; float* part_c;      // backward: [tpg][B][T][G][N] partial dB, dC
};

struct Where { int b, g, ct, ch, len, ck, i0, i1; bool live; };      // i0 .. i1: the chunk's tiles that hold valid frames
A8_DEV Where locate(const ScanArgs& p, int lane, int first_chunk, int nchunks) {
    Where w;
    int i = blockIdx.x;
    w.ct = i % p.tpg; i /= p.tpg;
    w.g = i % p.d.G; i /= p.d.G;
    w.ck = first_chunk + i % nchunks; w.b = i / nchunks;
    const int c = w.ct * CH + lane;
    w.live = c < p.cpg;
    w.ch = w.g * p.cpg + min(c, p.cpg - 1);
    w.len = seq_len(p.d.lengths, w.b, p.d.T);
    w.i0 = w.ck * p.tpc;
    w.i1 = min(w.i0 + p.tpc, (w.len + TT - 1) / TT);
    return w;
}

// row (b, t) of a strided input: a wave-uniform address, so that a load is one scalar base and one 32-bit lane offset
template <typename T> A8_DEV const T* row_of(const void* p, int64_t bs, int64_t ts, int b, int t) { return (const T*)p + (b * bs + t * ts); }

// The lane's byte offset in such a row, kept apart from the row's address: folded into it once, every access would need a 64-bit add of its own.
template <typename T> A8_DEV uint32_t lane_bytes(int ch) {
    uint32_t o = (uint32_t)ch * sizeof(T);
    asm volatile("" : "+v"(o));
    return o;
}
template <typename T> A8_DEV T ld_at(const T* row, uint32_t bytes) { return *(const T*)((const char*)row + bytes); }
template <typename T> A8_DEV void st_at(T* row, uint32_t bytes, T v) { *(T*)((char*)row + bytes) = v; }

// value I of the 16 that every row of 16 lanes holds in v, as a DPP operand
template <int I> A8_DEV float row_value(float v) { return dpp_f<0x150 + I>(v); }
template <int... I, typename F> A8_DEV void unroll_impl(std::integer_sequence<int, I...>, F f) { (f(std::integral_constant<int, I>()), ...); }
template <int N, typename F> A8_DEV void unroll(F f) { unroll_impl(std::make_integer_sequence<int, N>(), f); }

// The inputs of one tile as a thread holds them between their loads and their use a tile later.  Loads are unconditional: a frame behind the
// end reads the last valid one and is dropped where it is used, so nothing waits for a load before its time.
template <typename T, int NW, int NS, bool Z, bool DY> struct TileRegs {
    static constexpr int EP = TT / NW, BC = NS * NW;       // (frame, channel) elements per thread: frames wv, wv + NW, ...; states of the block
    T u[EP], dt[EP], z[Z ? EP : 1], dy[DY ? EP : 1], b, c;
    A8_DEV void load(const a8_selective_scan_desc& d, const Where& w, int wv, int t0) {
        const uint32_t at = lane_bytes<T>(w.ch);
#pragma unroll
        for (int j = 0; j < EP; ++j) {
            const int t = min(t0 + wv + NW * j, w.len - 1);
            u[j] = ld_at(row_of<T>(d.u, d.u_bs, d.u_ts, w.b, t), at);
            dt[j] = ld_at(row_of<T>(d.dt, d.dt_bs, d.dt_ts, w.b, t), at);
            if constexpr (Z) z[j] = ld_at(row_of<T>(d.z, d.z_bs, d.z_ts, w.b, t), at);
            if constexpr (DY) dy[j] = ld_at(row_of<T>(d.dy, d.dy_bs, d.dy_ts, w.b, t), at);
        }
        // B and C: one value per thread (at most: TT BC <= 64 NW), frame tid / BC, state tid % BC
        const int n = min((int)threadIdx.x % BC, d.N - 1), t = min(t0 + (int)threadIdx.x / BC, w.len - 1);
        b = ((const T*)d.Bm)[w.b * d.b_bs + t * d.b_ts + w.g * d.b_gs + n];
        c = ((const T*)d.Cm)[w.b * d.c_bs + t * d.c_ts + w.g * d.c_gs + n];
    }
    template <bool B = true, bool C = true> A8_DEV void stage_bc(const a8_selective_scan_desc& d, const Where& w, int t0, float* s_b, float* s_c) const {       // -> LDS [TT][BC]
        const int tid = threadIdx.x;
        if (TT * BC == 64 * NW || tid < TT * BC) {
            const bool in = tid % BC < d.N && t0 + tid / BC < w.len;
            if constexpr (B) s_b[tid] = in ? to_f(b) : 0.f;
            if constexpr (C) s_c[tid] = in ? to_f(c) : 0.f;
        }
    }
};
// a wave's values of an LDS tile [TT][BC]: v[k] holds frames 16 / NS * k .., frame (l & 15) / NS, state n0 + l % NS, in every row of 16 lanes
template <int NS, int BC> A8_DEV void wave_bc(float (&v)[NS], const float* s, int n0, int lane) {
#pragma unroll
    for (int k = 0; k < NS; ++k) v[k] = s[(16 / NS * k + (lane & 15) / NS) * BC + n0 + lane % NS];
}
// sum_n row value (I + n) of v * x[n], and its elementwise form x[n] += row value (I + n) of v * g: multiply-adds with the row broadcast in
// the DPP operand (the compiler folds it into multiplies only).  A DPP operand may not be read within two wait states of a VALU write of its register,
// which the compiler does not see here: one s_nop in front of the group covers a copy that it may have placed there.
#define A8_RB(op, acc, x, i) "v_" #op "_f32_dpp %" #acc ", %4, %" #x " row_newbcast:%" #i " row_mask:0xf bank_mask:0xf\n\t"
template <int I> A8_DEV void row_dot4x2(float (&y)[4], float v, const float (&x)[4][2]) {       // y[f] of 4 frames of 2 states
    asm("s_nop 1\n\t" A8_RB(mul, 0, 5, 13) A8_RB(mul, 1, 7, 15) A8_RB(mul, 2, 9, 17) A8_RB(mul, 3, 11, 19)
        A8_RB(fmac, 0, 6, 14) A8_RB(fmac, 1, 8, 16) A8_RB(fmac, 2, 10, 18) A8_RB(fmac, 3, 12, 20)
        : "=&v"(y[0]), "=&v"(y[1]), "=&v"(y[2]), "=&v"(y[3])
        : "v"(v), "v"(x[0][0]), "v"(x[0][1]), "v"(x[1][0]), "v"(x[1][1]), "v"(x[2][0]), "v"(x[2][1]), "v"(x[3][0]), "v"(x[3][1]),
          "n"(I), "n"(I + 1), "n"(I + 2), "n"(I + 3), "n"(I + 4), "n"(I + 5), "n"(I + 6), "n"(I + 7));
}
#undef A8_RB
#define A8_RM(o, x, i) "v_mul_f32_dpp %" #o ", %8, %" #x " row_newbcast:%" #i " row_mask:0xf bank_mask:0xf\n\t"
template <int I> A8_DEV void row_outer4x2(float (&o)[4][2], float v, float x0, float x1, float x2, float x3) {       // o[f][n] = row value (I + 2 f + n) of v * x_f
    asm("s_nop 1\n\t" A8_RM(0, 9, 13) A8_RM(1, 9, 14) A8_RM(2, 10, 15) A8_RM(3, 10, 16) A8_RM(4, 11, 17) A8_RM(5, 11, 18) A8_RM(6, 12, 19) A8_RM(7, 12, 20)
        : "=&v"(o[0][0]), "=&v"(o[0][1]), "=&v"(o[1][0]), "=&v"(o[1][1]), "=&v"(o[2][0]), "=&v"(o[2][1]), "=&v"(o[3][0]), "=&v"(o[3][1])
        : "v"(v), "v"(x0), "v"(x1), "v"(x2), "v"(x3), "n"(I), "n"(I + 1), "n"(I + 2), "n"(I + 3), "n"(I + 4), "n"(I + 5), "n"(I + 6), "n"(I + 7));
}
#undef A8_RM
template <int I> A8_DEV float row_dot(float v, const float (&x)[4]) {
    float acc;
    asm("s_nop 1\n\tv_mul_f32_dpp %0, %1, %2 row_newbcast:%6 row_mask:0xf bank_mask:0xf\n\tv_fmac_f32_dpp %0, %1, %3 row_newbcast:%7 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %1, %4 row_newbcast:%8 row_mask:0xf bank_mask:0xf\n\tv_fmac_f32_dpp %0, %1, %5 row_newbcast:%9 row_mask:0xf bank_mask:0xf"
        : "=&v"(acc) : "v"(v), "v"(x[0]), "v"(x[1]), "v"(x[2]), "v"(x[3]), "n"(I), "n"(I + 1), "n"(I + 2), "n"(I + 3));
    return acc;
}
template <int I> A8_DEV void row_axpy(float (&x)[4], float v, float g) {
    asm("s_nop 1\n\tv_fmac_f32_dpp %0, %4, %5 row_newbcast:%6 row_mask:0xf bank_mask:0xf\n\tv_fmac_f32_dpp %1, %4, %5 row_newbcast:%7 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %2, %4, %5 row_newbcast:%8 row_mask:0xf bank_mask:0xf\n\tv_fmac_f32_dpp %3, %4, %5 row_newbcast:%9 row_mask:0xf bank_mask:0xf"
        : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]) : "v"(v), "v"(g), "n"(I), "n"(I + 1), "n"(I + 2), "n"(I + 3));
}
// A as exp2 takes it, kept finite where A is -inf or its product is: a step of zero (frames behind the end) leaves such a state as it is, 0 x inf does not.
A8_DEV float log2_rate(float A) {
    const float r = A * SEQ_LOG2E;
    return r < -3.4028235e38f ? -3.4028235e38f : r;
}
// What a chunk makes of the state (adjoint) in front of it: exp2(x) v plus its own end e.  The factor of a whole chunk may be beyond f32 where the product is
// not (growing states, with a silent beginning or behind a chunk that decays): it is applied in two halves, and a state of zero stays zero.
A8_DEV float carry(float x, float v, float e) {
    const float f = __builtin_amdgcn_exp2f(0.5f * x);
    return v == 0.f ? e : fmaf(f, f * v, e);
}
// element (t, n) of wave_bc's values
template <int NS, int T_, int N_> A8_DEV float bc_at(const float (&v)[NS]) { return row_value<(T_ % (16 / NS)) * NS + N_>(v[T_ / (16 / NS)]); }

// The scan of one chunk, from the state that the chunks before it leave.  Bound by VALU issue: a state takes a multiply, an exp2 (two issue slots), a
// multiply and two multiply-adds, 24 cycles for 64 channels, and a (frame, channel) about 160 for softplus, silu, conversions and the sum over waves.
// bf16, N = 16, gated, states saved for the backward: 16 x 999 x 2048 180 us (524e6 states: 2.9e12 / s, VALU busy 78 % of the cycles, 0.39 GB at 2.2 TB/s),
// 8 x 781 x 1536 85 us (192 blocks leave a quarter of the CUs idle; chunks would cost what they win).
template <typename T, int NW, bool Z> __global__ __launch_bounds__(64 * NW) void scan_fwd_kernel(ScanArgs p) {
    constexpr int NS = FNS, EP = TT / NW, BC = NS * NW;
    __shared__ float2 s_dx[TT][CH];                        // {D, D u}
    __shared__ float s_b[TT * BC], s_c[TT * BC];
    __shared__ float s_y[NW][TT][CH];
    const a8_selective_scan_desc& d = p.d;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n0 = wv * NS;
    const Where w = locate(p, lane, 0, p.chunks);
    const float bias = d.dt_bias ? d.dt_bias[w.ch] : 0.f, skip = d.Dskip ? d.Dskip[w.ch] : 0.f;
    const bool sp = d.softplus != 0;
    float A2[NS], h[NS];
#pragma unroll
    for (int n = 0; n < NS; ++n) {
        const bool has = n0 + n < d.N;
        A2[n] = has ? log2_rate(d.A[(int64_t)w.ch * d.N + n0 + n]) : 0.f;
        h[n] = has && d.h0 ? d.h0[((int64_t)w.b * d.D + w.ch) * d.N + n0 + n] : 0.f;
    }
    for (int k = 0; k < w.ck; ++k) {                       // the states that the chunks before leave: at most a few dozen, each two loads away
        const float* const e = p.ends + ((int64_t)w.b * p.chunks + k) * (d.N + 1) * d.D + w.ch;
        const float s = e[(int64_t)d.N * d.D];
#pragma unroll
        for (int n = 0; n < NS; ++n)
            if (n0 + n < d.N) h[n] = carry(A2[n] * s, h[n], e[(int64_t)(n0 + n) * d.D]);
    }
    TileRegs<T, NW, NS, Z, false> nx, cu;                  // the next tile's inputs, this tile's u and z
    auto stage = [&](int t0) {                             // nx -> LDS
#pragma unroll
        for (int j = 0; j < EP; ++j) {
            const int t = wv + NW * j;
            const float raw = to_f(nx.dt[j]) + bias, s = sp ? softplus_f(raw) : raw, u = to_f(nx.u[j]);
            const bool in = t0 + t < w.len;
            s_dx[t][lane] = make_float2(in ? s : 0.f, in ? s * u : 0.f);
        }
        nx.stage_bc(d, w, t0, s_b, s_c);
    };
    if (w.i0 < w.i1) { nx.load(d, w, wv, w.i0 * TT); stage(w.i0 * TT); }
    for (int i = w.i0; i < w.i1; ++i) {
        const int t0 = i * TT;
        cu = nx;
        if (d.ckpt && w.live) {
            float* const ck = d.ckpt + (((int64_t)w.b * p.tiles + i) * d.N + n0) * d.D;
#pragma unroll
            for (int n = 0; n < NS; ++n)
                if (n0 + n < d.N) ck[(int64_t)n * d.D + w.ch] = h[n];
        }
        lds_barrier();
        if (i + 1 < w.i1) nx.load(d, w, wv, t0 + TT);
        float bv[NS], cv[NS];
        wave_bc<NS, BC>(bv, s_b, n0, lane);
        wave_bc<NS, BC>(cv, s_c, n0, lane);
        unroll<TT / 4>([&](auto qc) {
            constexpr int t4 = 4 * decltype(qc)::value;
            float hq[4][NS], y[4];
            float2 dx[4];
#pragma unroll
            for (int f = 0; f < 4; ++f) dx[f] = s_dx[t4 + f][lane];
            row_outer4x2<(t4 % 8) * 2>(hq, bv[t4 / 8], dx[0].y, dx[1].y, dx[2].y, dx[3].y);      // D u B, then the state in its place
#pragma unroll
            for (int f = 0; f < 4; ++f)
#pragma unroll
                for (int n = 0; n < NS; ++n) hq[f][n] = fmaf(__builtin_amdgcn_exp2f(dx[f].x * A2[n]), f ? hq[f ? f - 1 : 0][n] : h[n], hq[f][n]);
#pragma unroll
            for (int n = 0; n < NS; ++n) h[n] = hq[3][n];
            row_dot4x2<(t4 % 8) * 2>(y, cv[t4 / 8], hq);
#pragma unroll
            for (int f = 0; f < 4; ++f) s_y[wv][t4 + f][lane] = y[f];
        });
        lds_barrier();
        if (i + 1 < w.i1) stage(t0 + TT);                  // (the loads are a tile old; the stores below are not waited for)
        const uint32_t at = lane_bytes<T>(w.ch);
#pragma unroll
        for (int j = 0; j < EP; ++j) {
            const int t = wv + NW * j;
            float y = skip * to_f(cu.u[j]);
#pragma unroll
            for (int v = 0; v < NW; ++v) y += s_y[v][t][lane];
            if constexpr (Z) y *= silu_f(to_f(cu.z[j]));
            if (t0 + t < w.len && w.live) st_at((T*)d.y + ((int64_t)w.b * d.T + t0 + t) * d.D, at, from_f<T>(y));
        }
    }
    if (!w.live) return;
    for (int t = max(w.i0 * TT, w.len) + wv; t < min((w.i0 + p.tpc) * TT, d.T); t += NW) ((T*)d.y)[((int64_t)w.b * d.T + t) * d.D + w.ch] = from_f<T>(0.f);
    if (d.h_out && w.ck == p.chunks - 1)
#pragma unroll
        for (int n = 0; n < NS; ++n)
            if (n0 + n < d.N) d.h_out[((int64_t)w.b * d.D + w.ch) * d.N + n0 + n] = h[n];
}

// Each chunk's own end state (from zero) and the sum of its steps.  No output per frame, so the shared memory holds two tiles: while one is walked the
// next one is staged and the one after it requested, with one barrier per tile (1 x 48001 x 1536: 250 .. 278 us, VALU busy 88 %; as the kernel above without its output, two
// barriers, 340 us.  The kernel above gains nothing from the same form: its sums over states then allow only tiles of 8 frames, 97 us against 86 in one session at
// 8 x 781 x 1536).
template <typename T, int NW> __global__ __launch_bounds__(64 * NW) void scan_ends_kernel(ScanArgs p) {
    constexpr int NS = FNS, EP = TT / NW, BC = NS * NW;
    __shared__ float2 s_dx[2][TT][CH];
    __shared__ float s_b[2][TT * BC], s_sum[NW][CH];
    const a8_selective_scan_desc& d = p.d;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n0 = wv * NS;
    const Where w = locate(p, lane, 0, p.chunks - 1);
    const float bias = d.dt_bias ? d.dt_bias[w.ch] : 0.f;
    const bool sp = d.softplus != 0;
    float A2[NS], h[NS] = {}, sum = 0.f;
#pragma unroll
    for (int n = 0; n < NS; ++n) A2[n] = n0 + n < d.N ? log2_rate(d.A[(int64_t)w.ch * d.N + n0 + n]) : 0.f;
    TileRegs<T, NW, NS, false, false> nx;
    auto stage = [&](int i) {                              // (the tile behind the chunk's last one is staged like any other, and neither walked nor summed)
#pragma unroll
        for (int j = 0; j < EP; ++j) {
            const int t = wv + NW * j;
            const float raw = to_f(nx.dt[j]) + bias, s = sp ? softplus_f(raw) : raw, u = to_f(nx.u[j]);
            const bool in = i < w.i1 && i * TT + t < w.len;
            s_dx[i & 1][t][lane] = make_float2(in ? s : 0.f, in ? s * u : 0.f);
            sum += in ? s : 0.f;
        }
        nx.template stage_bc<true, false>(d, w, i * TT, s_b[i & 1], nullptr);
    };
    if (w.i0 < w.i1) {
        nx.load(d, w, wv, w.i0 * TT);
        stage(w.i0);
        nx.load(d, w, wv, (w.i0 + 1) * TT);
        lds_barrier();
    }
    for (int i = w.i0; i < w.i1; ++i) {
        const int q = i & 1;
        stage(i + 1);
        nx.load(d, w, wv, (i + 2) * TT);
        float bv[NS];
        wave_bc<NS, BC>(bv, s_b[q], n0, lane);
        unroll<TT / 4>([&](auto qc) {
            constexpr int t4 = 4 * decltype(qc)::value;
            float hq[4][NS];
            float2 dx[4];
#pragma unroll
            for (int f = 0; f < 4; ++f) dx[f] = s_dx[q][t4 + f][lane];
            row_outer4x2<(t4 % 8) * 2>(hq, bv[t4 / 8], dx[0].y, dx[1].y, dx[2].y, dx[3].y);
#pragma unroll
            for (int f = 0; f < 4; ++f)
#pragma unroll
                for (int n = 0; n < NS; ++n) h[n] = fmaf(__builtin_amdgcn_exp2f(dx[f].x * A2[n]), h[n], hq[f][n]);
        });
        lds_barrier();
    }
    s_sum[wv][lane] = sum;
    lds_barrier();
    if (!w.live) return;
    float* const e = p.ends + ((int64_t)w.b * p.chunks + w.ck) * (d.N + 1) * d.D + w.ch;
#pragma unroll
    for (int n = 0; n < NS; ++n)
        if (n0 + n < d.N) e[(int64_t)(n0 + n) * d.D] = h[n];
    if (wv == 0) {
        sum = 0.f;
#pragma unroll
        for (int v = 0; v < NW; ++v) sum += s_sum[v][lane];
        e[(int64_t)d.N * d.D] = sum;
    }
}

// Sums over a wave's 64 lanes of 64 values that come 16 at a time (4 frames x 4 states), scattered: lane l gets the total of value l.  A step pairs
// lanes that differ in one bit of the index, adds, and keeps the half of the values whose index has the lane's bit: one add per value left instead
// of six per value.  The bits that number a row's four banks of 4 lanes first (8 cycles per value left: the bank mask of the DPP add takes the place
// of a select), then the two inside a bank (two selects and an add: 12), then, with one value per 16 left, the rows through the half-wave and
// half-row register swaps (13).
template <int CTRL, int M> A8_DEV void scatter_step(float* v, bool upper) {
#pragma unroll
    for (int i = 0; i < M; ++i) {
        const float keep = upper ? v[i + M] : v[i], send = upper ? v[i] : v[i + M];
        v[i] = keep + dpp_f<CTRL>(send);
    }
}
#define A8_ROR8(a, b)                                                              \
    "v_add_f32_dpp %" #a ", %" #a ", %" #a " row_ror:8 row_mask:0xf bank_mask:0x3\n\t" \
    "v_add_f32_dpp %" #a ", %" #b ", %" #b " row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
#define A8_MIR8(a, b)                                                                      \
    "v_add_f32_dpp %" #a ", %" #a ", %" #a " row_half_mirror row_mask:0xf bank_mask:0x5\n\t" \
    "v_add_f32_dpp %" #a ", %" #b ", %" #b " row_half_mirror row_mask:0xf bank_mask:0xa\n\t"
A8_DEV float row_sum_scatter16(float (&v)[16], int lane) {      // lane l: the sum of v[l & 15] over its row
    // (the s_nops: two wait states between a VALU write and a DPP read of the register, on either side of what the compiler sees)
    asm("s_nop 1\n\t" A8_ROR8(0, 8) A8_ROR8(4, 12) A8_ROR8(1, 9) A8_ROR8(5, 13) A8_ROR8(2, 10) A8_ROR8(6, 14) A8_ROR8(3, 11) A8_ROR8(7, 15)
        A8_MIR8(0, 4) A8_MIR8(1, 5) A8_MIR8(2, 6) A8_MIR8(3, 7) "s_nop 1"
        : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3]), "+v"(v[4]), "+v"(v[5]), "+v"(v[6]), "+v"(v[7]),
          "+v"(v[8]), "+v"(v[9]), "+v"(v[10]), "+v"(v[11]), "+v"(v[12]), "+v"(v[13]), "+v"(v[14]), "+v"(v[15]));
    scatter_step<0x4E, 2>(v, lane & 2);           // quad_perm xor 2
    scatter_step<0xB1, 1>(v, lane & 1);           // quad_perm xor 1
    return v[0];
}
A8_DEV float rows_sum_scatter4(const float (&v)[4]) {           // row r: the sum of v[r] over the rows
    auto swap_add32 = [](float x, float y) {
        auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
        return __uint_as_float(s[0]) + __uint_as_float(s[1]);
    };
    const float lo = swap_add32(v[0], v[2]), hi = swap_add32(v[1], v[3]);
    auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(lo), __float_as_uint(hi), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// The gradient of one chunk, from the adjoint that the chunks behind it leave; tiles run backwards, each from its saved state.  Bound by VALU issue: per
// state the recurrence again (24 cycles), the adjoint with its five products (32), and its share of the two sums over channels (17); 256 registers and
// 76 KB of LDS allow two blocks of 16 states on a CU, two waves per SIMD.  bf16, N = 16, gated: 16 x 999 x 2048 457 us (1.1e12 states / s, VALU busy
// 78 %), 8 x 781 x 1536 142 + 33 us in 5 chunks.
template <typename T, int NW, bool Z> __global__ __launch_bounds__(64 * NW, NW >= 4 ? 2 : 1) void scan_bwd_kernel(ScanArgs p) {
    constexpr int NS = BNS, EP = TT / NW, BC = NS * NW;
    __shared__ float2 s_dxs[2][TT][CH];                    // {D, D u}, by tile parity
    __shared__ float s_gs[2][TT][CH];                      // dout silu(z)
    __shared__ float s_b[TT * BC], s_c[TT * BC];
    __shared__ float2 s_q[NW][TT][CH];                     // a wave's {sum q B, sum A k}
    __shared__ float s_y[Z ? NW : 1][TT][CH];
    const a8_selective_scan_desc& d = p.d;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n0 = wv * NS;
    const Where w = locate(p, lane, 0, p.chunks);
    const float bias = d.dt_bias ? d.dt_bias[w.ch] : 0.f, skip = d.Dskip ? d.Dskip[w.ch] : 0.f;
    const bool sp = d.softplus != 0;
    float A[NS], A2[NS], c[NS], dA[NS] = {};
#pragma unroll
    for (int n = 0; n < NS; ++n) {
        const bool has = n0 + n < d.N;
        A[n] = has ? d.A[(int64_t)w.ch * d.N + n0 + n] : 0.f;
        A2[n] = log2_rate(A[n]);
        c[n] = has && w.live && d.dh_out ? d.dh_out[((int64_t)w.b * d.D + w.ch) * d.N + n0 + n] : 0.f;
    }
    for (int k = p.chunks - 1; k > w.ck; --k) {            // the adjoint that the chunks behind leave
        const float* const e = p.ends + ((int64_t)w.b * p.chunks + k) * (d.N + 1) * d.D + w.ch;
        const float s = e[(int64_t)d.N * d.D];
#pragma unroll
        for (int n = 0; n < NS; ++n)
            if (n0 + n < d.N && w.live) c[n] = carry(A2[n] * s, c[n], e[(int64_t)(n0 + n) * d.D]);
    }
    float dskip = 0.f, dbias = 0.f;
    TileRegs<T, NW, NS, Z, true> nx, cu;
    float rh[NS] = {};
    auto load = [&](int i) {
        nx.load(d, w, wv, i * TT);
        const float* const ck = d.ckpt + (((int64_t)w.b * p.tiles + i) * d.N + n0) * d.D;
#pragma unroll
        for (int n = 0; n < NS; ++n) rh[n] = n0 + n < d.N ? ck[(int64_t)n * d.D + w.ch] : 0.f;
    };
    auto stage = [&](int t0) {
#pragma unroll
        for (int j = 0; j < EP; ++j) {
            const int t = wv + NW * j;
            const float raw = to_f(nx.dt[j]) + bias, s = sp ? softplus_f(raw) : raw, u = to_f(nx.u[j]);
            const bool in = t0 + t < w.len && w.live;      // (an absent channel contributes nothing to dB and dC)
            s_dxs[t0 / TT & 1][t][lane] = make_float2(in ? s : 0.f, in ? s * u : 0.f);
            float g = to_f(nx.dy[j]);
            if constexpr (Z) g *= silu_f(to_f(nx.z[j]));
            s_gs[t0 / TT & 1][t][lane] = in ? g : 0.f;
        }
        nx.stage_bc(d, w, t0, s_b, s_c);
    };
    if (w.i0 < w.i1) { load(w.i1 - 1); stage((w.i1 - 1) * TT); }
    for (int i = w.i1 - 1; i >= w.i0; --i) {
        const int t0 = i * TT;
        const float2 (&s_dx)[TT][CH] = s_dxs[i & 1];
        const float (&s_g)[TT][CH] = s_gs[i & 1];
        cu = nx;
        float a[TT][NS], h[TT + 1][NS], gb[4], gc[4];      // decays, states; dB's and dC's row sums of each 4 frames
#pragma unroll
        for (int n = 0; n < NS; ++n) h[0][n] = w.live ? rh[n] : 0.f;
        lds_barrier();
        if (i > w.i0) load(i - 1);
        float bv[NS], cv[NS];
        wave_bc<NS, BC>(bv, s_b, n0, lane);
        wave_bc<NS, BC>(cv, s_c, n0, lane);
        unroll<TT>([&](auto tc) {                         // the tile's states again, from the saved state before it
            constexpr int t = decltype(tc)::value;
            const float2 dx = s_dx[t][lane];
            unroll<NS>([&](auto nc) {
                constexpr int n = decltype(nc)::value;
                a[t][n] = __builtin_amdgcn_exp2f(dx.x * A2[n]);
                h[t + 1][n] = fmaf(a[t][n], h[t][n], dx.y * bc_at<NS, t, n>(bv));
            });
            if constexpr (Z) s_y[wv][t][lane] = row_dot<(t % 4) * 4>(cv[t / 4], h[t + 1]);
            if constexpr (t % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        });
        unroll<TT / 4>([&](auto qc) {                      // backwards, 4 frames at a time
            constexpr int t4 = TT - 4 - 4 * decltype(qc)::value;
            float vb[16], vc[16];
            unroll<4>([&](auto tc) {
                constexpr int t = t4 + 3 - decltype(tc)::value;
                const float2 dx = s_dx[t][lane];
                const float g = s_g[t][lane];
                row_axpy<(t % 4) * 4>(c, cv[t / 4], g);    // c is q_t here
                const float qb = row_dot<(t % 4) * 4>(bv[t / 4], c);
                float ak = 0.f;
#pragma unroll
                for (int n = 0; n < NS; ++n) {
                    vb[(t - t4) * 4 + n] = c[n] * dx.y;
                    vc[(t - t4) * 4 + n] = h[t + 1][n] * g;
                    c[n] *= a[t][n];
                    const float k = c[n] * h[t][n];
                    ak = fmaf(A[n], k, ak);
                    dA[n] = fmaf(k, dx.x, dA[n]);
                }
                s_q[wv][t][lane] = make_float2(qb, ak);
            });
            gb[t4 / 4] = row_sum_scatter16(vb, lane);
            gc[t4 / 4] = row_sum_scatter16(vc, lane);
            __builtin_amdgcn_sched_barrier(0);             // (read ahead of here, the next frames' inputs cost more registers than two waves per SIMD have)
        });
        const float sb = rows_sum_scatter4(gb), sc = rows_sum_scatter4(gc);
        lds_barrier();
        if (i > w.i0) stage(t0 - TT);
        {
            const int t = t0 + (lane >> 2), n = n0 + (lane & 3);
            if (t < w.len && n < d.N) {
                const int64_t at = ((((int64_t)w.ct * d.B + w.b) * d.T + t) * d.G + w.g) * d.N + n;
                p.part_b[at] = sb;
                p.part_c[at] = sc;
            }
        }
        const uint32_t at = lane_bytes<T>(w.ch);
#pragma unroll
        for (int j = 0; j < EP; ++j) {
            const int t = wv + NW * j;
            const float u = to_f(cu.u[j]), g = s_g[t][lane];
            float qb = 0.f, ak = 0.f, y = skip * u;
#pragma unroll
            for (int k = 0; k < NW; ++k) { const float2 q = s_q[k][t][lane]; qb += q.x; ak += q.y; }
            float dd = fmaf(u, qb, ak);
            if (sp) dd *= sigmoid_f(to_f(cu.dt[j]) + bias);
            float dz = 0.f;
            if constexpr (Z) {
#pragma unroll
                for (int k = 0; k < NW; ++k) y += s_y[k][t][lane];
                dz = to_f(cu.dy[j]) * y * silu_grad_f(to_f(cu.z[j]));
            }
            if (t0 + t < w.len && w.live) {
                const int64_t row = ((int64_t)w.b * d.T + t0 + t) * d.D;
                dskip = fmaf(g, u, dskip);
                dbias += dd;
                st_at((T*)d.du + row, at, from_f<T>(fmaf(s_dx[t][lane].x, qb, skip * g)));
                st_at((T*)d.ddt + row, at, from_f<T>(dd));
                if constexpr (Z) st_at((T*)d.dz + row, at, from_f<T>(dz));
            }
        }
    }
    if (w.live)
        for (int t = max(w.i0 * TT, w.len) + wv; t < min((w.i0 + p.tpc) * TT, d.T); t += NW) {
            const int64_t at = ((int64_t)w.b * d.T + t) * d.D + w.ch;
            ((T*)d.du)[at] = from_f<T>(0.f);
            ((T*)d.ddt)[at] = from_f<T>(0.f);
            if constexpr (Z) ((T*)d.dz)[at] = from_f<T>(0.f);
        }
    lds_barrier();                                         // (s_q is read by the last tile's epilogue above)
    s_q[wv][0][lane] = make_float2(dskip, dbias);
    lds_barrier();
    float* const part = p.part + ((int64_t)w.b * p.chunks + w.ck) * (d.N + 2) * d.D + w.ch;
    if (w.live) {
#pragma unroll
        for (int n = 0; n < NS; ++n)
            if (n0 + n < d.N) {
                part[(int64_t)(n0 + n) * d.D] = dA[n];
                if (d.dh0 && w.ck == 0) d.dh0[((int64_t)w.b * d.D + w.ch) * d.N + n0 + n] = c[n];
            }
        if (wv == 0) {
            float s0 = 0.f, s1 = 0.f;
#pragma unroll
            for (int k = 0; k < NW; ++k) { s0 += s_q[k][0][lane].x; s1 += s_q[k][0][lane].y; }
            part[(int64_t)d.N * d.D] = s0;
            part[(int64_t)(d.N + 1) * d.D] = s1;
        }
    }
}

// The adjoint at each chunk's beginning, from zero behind its end, and the sum of its steps: scan_ends_kernel backwards (8 x 781 x 1536: 33 us of 175).
template <typename T, int NW, bool Z> __global__ __launch_bounds__(64 * NW) void scan_back_ends_kernel(ScanArgs p) {
    constexpr int NS = BNS, EP = TT / NW, BC = NS * NW;
    __shared__ float2 s_dg[2][TT][CH];                     // {D, dout silu(z)}
    __shared__ float s_c[2][TT * BC], s_sum[NW][CH];
    const a8_selective_scan_desc& d = p.d;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n0 = wv * NS;
    const Where w = locate(p, lane, 1, p.chunks - 1);
    const float bias = d.dt_bias ? d.dt_bias[w.ch] : 0.f;
    const bool sp = d.softplus != 0;
    float A2[NS], c[NS] = {}, sum = 0.f;
#pragma unroll
    for (int n = 0; n < NS; ++n) A2[n] = n0 + n < d.N ? log2_rate(d.A[(int64_t)w.ch * d.N + n0 + n]) : 0.f;
    TileRegs<T, NW, NS, Z, true> nx;
    auto load = [&](int i) { nx.load(d, w, wv, max(i, 0) * TT); };
    auto stage = [&](int i) {                              // (the tile in front of the chunk's first one is neither walked nor summed)
#pragma unroll
        for (int j = 0; j < EP; ++j) {
            const int t = wv + NW * j;
            const float raw = to_f(nx.dt[j]) + bias, s = sp ? softplus_f(raw) : raw;
            const bool in = i >= w.i0 && i * TT + t < w.len;
            float g = to_f(nx.dy[j]);
            if constexpr (Z) g *= silu_f(to_f(nx.z[j]));
            s_dg[i & 1][t][lane] = make_float2(in ? s : 0.f, in ? g : 0.f);
            sum += in ? s : 0.f;
        }
        nx.template stage_bc<false, true>(d, w, i * TT, nullptr, s_c[i & 1]);
    };
    if (w.i0 < w.i1) {
        load(w.i1 - 1);
        stage(w.i1 - 1);
        load(w.i1 - 2);
        lds_barrier();
    }
    for (int i = w.i1 - 1; i >= w.i0; --i) {
        const int q = i & 1;
        stage(i - 1);
        load(i - 2);
        float cv[NS];
        wave_bc<NS, BC>(cv, s_c[q], n0, lane);
        unroll<TT>([&](auto tc) {
            constexpr int t = TT - 1 - decltype(tc)::value;
            const float2 dg = s_dg[q][t][lane];
            row_axpy<(t % 4) * 4>(c, cv[t / 4], dg.y);
#pragma unroll
            for (int n = 0; n < NS; ++n) c[n] *= __builtin_amdgcn_exp2f(dg.x * A2[n]);
        });
        lds_barrier();
    }
    s_sum[wv][lane] = sum;
    lds_barrier();
    if (!w.live) return;
    float* const e = p.ends + ((int64_t)w.b * p.chunks + w.ck) * (d.N + 1) * d.D + w.ch;
#pragma unroll
    for (int n = 0; n < NS; ++n)
        if (n0 + n < d.N) e[(int64_t)(n0 + n) * d.D] = c[n];
    if (wv == 0) {
        sum = 0.f;
#pragma unroll
        for (int v = 0; v < NW; ++v) sum += s_sum[v][lane];
        e[(int64_t)d.N * d.D] = sum;
    }
}

// dB, dC = the channel tiles' partial sums, in tile order; frames behind an utterance's end are zero.  Bound by HBM: the D / 64 tiles' sums, 8 bytes per
// frame, state and tile, are read once (8 x 781, 24 tiles, N = 16: 19 MB in 9.6 us; 16 x 999, 32 tiles: 65 MB in 20 us, 3.3 TB/s).
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

// One frame: 4 lanes per channel, 4 consecutive states per lane and round; the state is read and written once.  What a launch of one frame costs is
// latency, so every load is issued before the first use.  VEC: N % 4 = 0 and 16-byte aligned A and state.  bf16 32 x 1536, N = 16: 4.0 us, 6.8 MB.
template <typename T> A8_DEV float ldf(const void* p, int64_t i) { return to_f(((const T*)p)[i]); }
template <typename T, bool VEC> __global__ __launch_bounds__(256) void scan_step_kernel(ScanArgs p) {
    const a8_selective_scan_desc& d = p.d;
    const int b = blockIdx.y, c = blockIdx.x * 64 + (threadIdx.x >> 2), s4 = threadIdx.x & 3;
    const int ch = min(c, d.D - 1), g = ch / p.cpg;
    float* const st = d.h_out + ((int64_t)b * d.D + ch) * d.N;
    const float* const A = d.A + (int64_t)ch * d.N;
    const T* const Bp = (const T*)d.Bm + (b * d.b_bs + g * d.b_gs);
    const T* const Cp = (const T*)d.Cm + (b * d.c_bs + g * d.c_gs);
    const T rdt = ((const T*)d.dt)[b * d.dt_bs + ch], ru = ((const T*)d.u)[b * d.u_bs + ch];
    const T rz = d.z ? ((const T*)d.z)[b * d.z_bs + ch] : from_f<T>(0.f);
    const float bias = d.dt_bias ? d.dt_bias[ch] : 0.f, skip = d.Dskip ? d.Dskip[ch] : 0.f;
    float y = 0.f, D = 0.f, x = 0.f;
    for (int n = s4 * 4; n < d.N; n += 16) {
        float h[4], a[4], Bv[4], Cv[4];
        if constexpr (VEC) {
            const f32x4 hv = *reinterpret_cast<const f32x4*>(st + n), av = *reinterpret_cast<const f32x4*>(A + n);
#pragma unroll
            for (int k = 0; k < 4; ++k) { h[k] = hv[k]; a[k] = av[k]; Bv[k] = to_f(Bp[n + k]); Cv[k] = to_f(Cp[n + k]); }
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int m = min(n + k, d.N - 1);
                h[k] = st[m]; a[k] = A[m]; Bv[k] = to_f(Bp[m]); Cv[k] = n + k < d.N ? to_f(Cp[m]) : 0.f;
            }
        }
        if (n < 16) {                                      // (the first round; behind the loads)
            const float raw = to_f(rdt) + bias;
            D = d.softplus ? softplus_f(raw) : raw;
            x = D * to_f(ru);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            h[k] = fmaf(exp_fast(D * a[k]), h[k], x * Bv[k]);
            y = fmaf(Cv[k], VEC || n + k < d.N ? h[k] : 0.f, y);
        }
        if (c < d.D) {
            if constexpr (VEC) *reinterpret_cast<f32x4*>(st + n) = (f32x4){h[0], h[1], h[2], h[3]};
            else
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (n + k < d.N) st[n + k] = h[k];
        }
    }
    y += dpp_f<0xB1>(y);
    y += dpp_f<0x4E>(y);
    if (s4 == 0 && c < d.D) {
        y = fmaf(skip, to_f(ru), y);
        if (d.z) y *= silu_f(to_f(rz));
        ((T*)d.y)[(int64_t)b * d.D + ch] = from_f<T>(y);
    }
}

int scan_check(const a8_selective_scan_desc* d, const char* what) {
    A8_REQUIRE(d != nullptr && d->size == (int)sizeof(a8_selective_scan_desc), "%s: descriptor size %d, expected %d", what, d ? d->size : 0, (int)sizeof(a8_selective_scan_desc));
    A8_REQUIRE(d->dtype == A8_F32 || d->dtype == A8_BF16, "%s: bad dtype %d", what, d->dtype);
    A8_REQUIRE(d->B >= 0 && d->T >= 0 && d->D >= 1 && d->N >= 1 && d->N <= 32, "%s: bad sizes B=%d T=%d D=%d N=%d (1 to 32 states)", what, d->B, d->T, d->D, d->N);
    A8_REQUIRE(d->T < (1 << 30), "%s: T = %d is too large", what, d->T);           // (frame indices run up to three tiles past the end)
    A8_REQUIRE(d->G >= 1 && d->D % d->G == 0, "%s: %d channels do not split into %d groups", what, d->D, d->G);
    A8_REQUIRE(d->A != nullptr, "%s: null A", what);
    return A8_OK;
}
// Frame chunks.  A launch of n chunks takes as many tiles' time as a chunk has tiles, times the rounds of blocks that the 256 CUs hold: `part[k - 1]` is
// the time of a round with k blocks on a CU as a share of a full one, `extra` what the chunks' own ends (all but one chunk's) cost more, a hundredth per
// chunk what is left of first loads, partial sums and walks over earlier chunks.  Measured in one session, N = 16, kernels alone (us with one chunk / with
// the count taken here; to be compared with one another: the sweep holds one set of inputs, where a program's calls take turns):
//   forward   1 x 781 x 1536 83 / 26 (10), 4 x 781 86 / 58 (7), 8 x 781 90 / 90 (1; with 5: 90), 12 x 781 134 / 128 (7), 16 x 624 110 / 110 (1; with 2: 123),
//             8 x 999 x 2048 117 / 117 (1; with 3: 131), 16 x 999 178 / 178 (1; with 2: 221)
//   backward  1 x 781 x 1536 249 / 53 (10), 4 x 781 252 / 113 (5), 8 x 781 261 / 193 (5; with 7: 199), 12 x 781 344 / 275 (7), 16 x 624 285 / 281 (4),
//             8 x 999 x 2048 338 / 295 (2), 16 x 999 454 / 454 (1; with 2: 512)
// A chunk has at least 4 tiles.
int scan_chunks(float blocks, int tiles, const float* part, int resident, float extra) {
    int best = 1;
    float cost = 0.f;
    for (int n = 1; n == 1 || (n <= 32 && n * 4 <= tiles); ++n) {
        const int tpc = cdiv(tiles > 0 ? tiles : 1, n), m = cdiv(tiles > 0 ? tiles : 1, tpc);        // (the chunks that are left when each takes whole tiles)
        const int per_cu = (int)ceilf(blocks * m / 256.f);
        const int full = per_cu / resident, rest = per_cu % resident;
        const float c = (full + (rest ? part[rest - 1] : 0.f)) * tpc * (m > 1 ? 1.f + extra * (m - 1) / m + 0.01f * m : 1.f);
        if (n == 1 || c < cost) { best = n; cost = c; }
    }
    return best;
}
const float FWD_PART[3] = {0.44f, 0.74f, 1.f}, BWD_PART[2] = {0.69f, 1.f};
ScanArgs scan_args(const a8_selective_scan_desc* d, bool backward) {
    ScanArgs p = {};
    p.d = *d;
    p.cpg = d->D / d->G;
    p.tpg = cdiv(p.cpg, CH);
    p.tiles = cdiv(d->T, TT);
    const float blocks = (float)d->B * d->G * p.tpg;         // (in blocks of 16 states: fewer states, shorter blocks)
    p.chunks = backward ? scan_chunks(blocks * cdiv(d->N, BNS) / 4.f, p.tiles, BWD_PART, 2, 0.3f) : scan_chunks(blocks * cdiv(d->N, FNS) / 8.f, p.tiles, FWD_PART, 3, 0.9f);
    p.tpc = cdiv(p.tiles, p.chunks);
    p.chunks = p.tpc > 0 ? cdiv(p.tiles, p.tpc) : 1;         // (no empty chunks; T = 0: one without tiles)
    return p;
}
int64_t scan_blocks(const ScanArgs& p, int chunks) { return (int64_t)p.d.B * p.d.G * p.tpg * chunks; }
int64_t ends_floats(const ScanArgs& p) { return p.chunks > 1 ? (int64_t)p.d.B * p.chunks * (p.d.N + 1) * p.d.D : 0; }

#define FWD_WAVES(KERNEL, ...)                                                                                    \
    (waves <= 1 ? (KERNEL(1, __VA_ARGS__)) : waves <= 2 ? (KERNEL(2, __VA_ARGS__)) : waves <= 4 ? (KERNEL(4, __VA_ARGS__))      \
     : waves <= 8 ? (KERNEL(8, __VA_ARGS__)) : (KERNEL(16, __VA_ARGS__)))
#define FWD_KERNEL(NW, T, Z) scan_fwd_kernel<T, NW, Z>
#define ENDS_KERNEL(NW, T) scan_ends_kernel<T, NW>
#define BWD_WAVES(KERNEL, ...)                                                                                    \
    (waves <= 1 ? (KERNEL(1, __VA_ARGS__)) : waves <= 2 ? (KERNEL(2, __VA_ARGS__)) : waves <= 4 ? (KERNEL(4, __VA_ARGS__)) : (KERNEL(8, __VA_ARGS__)))
#define BWD_KERNEL(NW, T, Z) scan_bwd_kernel<T, NW, Z>
#define BACK_ENDS_KERNEL(NW, T, Z) scan_back_ends_kernel<T, NW, Z>

int launch_fwd(const ScanArgs& p, bool ends, hipStream_t st) {
    const int waves = cdiv(p.d.N, FNS);
    const bool bf = p.d.dtype == A8_BF16, z = p.d.z != nullptr;
    auto kernel = ends ? (bf ? FWD_WAVES(ENDS_KERNEL, bf16) : FWD_WAVES(ENDS_KERNEL, float))
                  : bf ? (z ? FWD_WAVES(FWD_KERNEL, bf16, true) : FWD_WAVES(FWD_KERNEL, bf16, false))
                       : (z ? FWD_WAVES(FWD_KERNEL, float, true) : FWD_WAVES(FWD_KERNEL, float, false));
    const int block = 64 * (waves <= 1 ? 1 : waves <= 2 ? 2 : waves <= 4 ? 4 : waves <= 8 ? 8 : 16);
    hipLaunchKernelGGL(kernel, dim3((unsigned)scan_blocks(p, ends ? p.chunks - 1 : p.chunks)), dim3(block), 0, st, p);
    return a8_check_launch("a8_selective_scan_fwd");
}
int launch_bwd(const ScanArgs& p, bool ends, hipStream_t st) {
    const int waves = cdiv(p.d.N, BNS);
    const bool bf = p.d.dtype == A8_BF16, z = p.d.z != nullptr;
    auto kernel = ends ? (bf ? (z ? BWD_WAVES(BACK_ENDS_KERNEL, bf16, true) : BWD_WAVES(BACK_ENDS_KERNEL, bf16, false))
                             : (z ? BWD_WAVES(BACK_ENDS_KERNEL, float, true) : BWD_WAVES(BACK_ENDS_KERNEL, float, false)))
                       : (bf ? (z ? BWD_WAVES(BWD_KERNEL, bf16, true) : BWD_WAVES(BWD_KERNEL, bf16, false))
                             : (z ? BWD_WAVES(BWD_KERNEL, float, true) : BWD_WAVES(BWD_KERNEL, float, false)));
    const int block = 64 * (waves <= 1 ? 1 : waves <= 2 ? 2 : waves <= 4 ? 4 : 8);
    hipLaunchKernelGGL(kernel, dim3((unsigned)scan_blocks(p, ends ? p.chunks - 1 : p.chunks)), dim3(block), 0, st, p);
    return a8_check_launch("a8_selective_scan_bwd");
}

}  // namespace

extern "C" int a8_selective_scan_workspace(const a8_selective_scan_desc* d, int backward, int64_t* ckpt_floats, int64_t* ws_floats) {
    if (int e = scan_check(d, "a8_selective_scan_workspace")) return e;
    A8_REQUIRE(ckpt_floats != nullptr && ws_floats != nullptr, "a8_selective_scan_workspace: null result");
    const ScanArgs p = scan_args(d, backward != 0);
    *ckpt_floats = (int64_t)d->B * p.tiles * d->N * d->D;
    *ws_floats = ends_floats(p);
    if (backward) *ws_floats += (int64_t)d->B * p.chunks * (d->N + 2) * d->D + 2 * (int64_t)p.tpg * d->B * d->T * d->G * d->N;
    return A8_OK;
}

extern "C" int a8_selective_scan_fwd(const a8_selective_scan_desc* d, void* stream) {
    if (int e = scan_check(d, "a8_selective_scan_fwd")) return e;
    if (d->B == 0) return A8_OK;
    A8_REQUIRE(d->T == 0 || (d->u && d->dt && d->Bm && d->Cm && d->y), "a8_selective_scan_fwd: null u, dt, B, C or y");
    A8_REQUIRE(!d->h_out || d->h_out != d->h0, "a8_selective_scan_fwd: h_out may not be the state that is read");
    ScanArgs p = scan_args(d, false);
    A8_REQUIRE(scan_blocks(p, p.chunks) < (1 << 21), "a8_selective_scan_fwd: B x D = %d x %d is too large", d->B, d->D);
    A8_REQUIRE(p.chunks == 1 || d->ws, "a8_selective_scan_fwd: null workspace");
    p.ends = d->ws;
    if (p.chunks > 1)
        if (int e = launch_fwd(p, true, (hipStream_t)stream)) return e;
    return launch_fwd(p, false, (hipStream_t)stream);
}

extern "C" int a8_selective_scan_bwd(const a8_selective_scan_desc* d, void* stream) {
    if (int e = scan_check(d, "a8_selective_scan_bwd")) return e;
    ScanArgs p = scan_args(d, true);
    A8_REQUIRE(d->D < SEQ_REDUCE_MAX, "a8_selective_scan_bwd: D = %d is too large", d->D);
    A8_REQUIRE(!d->dh0 || d->dh0 != d->dh_out, "a8_selective_scan_bwd: dh0 may not be the gradient that is read");
    A8_REQUIRE(d->B == 0 || d->ws, "a8_selective_scan_bwd: null workspace");
    A8_REQUIRE(d->B == 0 || d->T == 0 || (d->u && d->dt && d->Bm && d->Cm && d->dy && d->ckpt && d->du && d->ddt && d->dBm && d->dCm && (d->dz || !d->z)),
               "a8_selective_scan_bwd: null operand");
    A8_REQUIRE(scan_blocks(p, p.chunks) < (1 << 21), "a8_selective_scan_bwd: B x D = %d x %d is too large", d->B, d->D);
    const int64_t total = (int64_t)d->B * d->T * d->G * d->N;
    A8_REQUIRE(total < (1ll << 32) - 256, "a8_selective_scan_bwd: B x T x G x N = %d x %d x %d x %d is too large", d->B, d->T, d->G, d->N);
    p.ends = d->ws;
    p.part = p.ends + ends_floats(p);
    p.part_b = p.part + (int64_t)d->B * p.chunks * (d->N + 2) * d->D;
    p.part_c = p.part_b + (int64_t)p.tpg * d->B * d->T * d->G * d->N;
    if (d->B > 0) {
        if (p.chunks > 1)
            if (int e = launch_bwd(p, true, (hipStream_t)stream)) return e;
        if (int e = launch_bwd(p, false, (hipStream_t)stream)) return e;
        if (total > 0) {
            const dim3 grid((unsigned)((total + 255) / 256));
            if (d->dtype == A8_BF16) hipLaunchKernelGGL((scan_bc_kernel<bf16>), grid, dim3(256), 0, (hipStream_t)stream, p);
            else hipLaunchKernelGGL((scan_bc_kernel<float>), grid, dim3(256), 0, (hipStream_t)stream, p);
            if (int e = a8_check_launch("a8_selective_scan_bwd")) return e;
        }
    }
    A8SeqReduce r = {p.part, d->B * p.chunks, d->N + 2, d->D, d->N, d->dA, {d->dD, d->ddt_bias}, d->add_dA, {d->add_dD, d->add_ddt_bias}};
    return a8i_seq_reduce(r, stream);
}

extern "C" int a8_selective_scan_step(const a8_selective_scan_desc* d, void* stream) {
    if (int e = scan_check(d, "a8_selective_scan_step")) return e;
    A8_REQUIRE(d->T == 1, "a8_selective_scan_step: one frame at a time (T = %d)", d->T);
    A8_REQUIRE(d->B <= 65535, "a8_selective_scan_step: B = %d is too large", d->B);
    if (d->B == 0) return A8_OK;
    A8_REQUIRE(d->u && d->dt && d->Bm && d->Cm && d->y && d->h_out, "a8_selective_scan_step: null u, dt, B, C, y or state");
    const ScanArgs p = scan_args(d, false);
    const dim3 grid(cdiv(d->D, 64), d->B);
    const bool vec = d->N % 4 == 0 && ((uintptr_t)d->A | (uintptr_t)d->h_out) % 16 == 0;
    auto kernel = d->dtype == A8_BF16 ? (vec ? scan_step_kernel<bf16, true> : scan_step_kernel<bf16, false>)
                                      : (vec ? scan_step_kernel<float, true> : scan_step_kernel<float, false>);
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, (hipStream_t)stream, p);
    return a8_check_launch("a8_selective_scan_step");
}
