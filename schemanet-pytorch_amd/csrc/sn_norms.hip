// The end of a residual block and the norm before the next one (schemanet_blocks.h):
//     p = N_post(branch);  y = x + scale * sigmoid(gate) * p;  h = N_pre(y)
// and its backward pass, with u = dy + N_pre^T(dh) the whole gradient of y:
//     dx = u;   dgate = u scale p s (1 - s);   dp = u scale s;   dbranch = N_post^T(dp);      s = sigmoid(gate)
//     dscale = sum u s p;   dw_post = sum dp n1;  db_post = sum dp;  dw_pre = sum dh n2;  db_pre = sum dh     (n = the unit values)
//     N^T(d) = r (w d - mean(w d) - n mean(w d n))          (rms: without the first mean)
// Bound: HBM - forward reads x, branch, gate and writes y, h; backward reads those three and dy, dh and writes three gradients.
// Every element is read once and stays in registers: a row belongs to one wave (up to 512 columns, 8 or 4 a lane) or to up to
// eight of one workgroup, the means are two passes over registers (centred squares: no cancellation), the column sums of the
// backward pass are kept in registers over all rows of a workgroup, written once per workgroup and added in a fixed order by a
// second launch (no atomics).  The unit values are recomputed from the inputs and the forward pass's row statistics; y is not kept.
// What made it fast is loads that run one or two rows ahead in straight-line code (MODE below).
// Measured (the card copies at 5.13 TB/s): 32768 rows of 4096, bf16, rms with gate: forward 264 us (5.1 TB/s), backward 408 us
// (5.3 TB/s); 103424 rows of 256, fp32, LayerNorm with gate: forward 113 us (4.7 TB/s), backward 165 us (5.1 TB/s), a quarter of the
// rows padding and 8-bit checkpoints written and read: 130 us (3.9 TB/s) and 118 us (4.6 TB/s).
#include "sn_typed.h"

namespace {

using namespace sn;

constexpr int64_t kMostRows = 1ll << 48;  // (past any memory: sums of a few such numbers stay in 64 bits)
constexpr int kVectors = 5;              // column sums of the backward pass: pre weight, pre bias, scale, post weight, post bias

// all-reduce over the waves of the workgroup's row (up to 8; the buffers hold zeros for those that are not there); `slot` alternates
// between two LDS buffers, so one barrier is enough
template <bool MULTI> __device__ __forceinline__ float row_sum(float v, float *red, int &slot)
{
    v = sn_wave_sum(v);
    if constexpr (MULTI) {
        float *buf = red + slot * 16;
        if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
        __syncthreads();
        const float4 a = *reinterpret_cast<const float4 *>(buf), b = *reinterpret_cast<const float4 *>(buf + 4);
        v = ((a.x + a.y) + (a.z + a.w)) + ((b.x + b.y) + (b.z + b.w));
        slot ^= 1;
    }
    return v;
}
template <bool MULTI> __device__ __forceinline__ void row_sum2(float &p, float &q, float *red, int &slot)
{
    p = sn_wave_sum(p);
    q = sn_wave_sum(q);
    if constexpr (MULTI) {
        float *buf = red + slot * 16;
        if ((threadIdx.x & 63) == 0) { buf[threadIdx.x >> 6] = p; buf[8 + (threadIdx.x >> 6)] = q; }
        __syncthreads();
        const float4 a = *reinterpret_cast<const float4 *>(buf), b = *reinterpret_cast<const float4 *>(buf + 4);
        const float4 c = *reinterpret_cast<const float4 *>(buf + 8), d = *reinterpret_cast<const float4 *>(buf + 12);
        p = ((a.x + a.y) + (a.z + a.w)) + ((b.x + b.y) + (b.z + b.w));
        q = ((c.x + c.y) + (c.z + c.w)) + ((d.x + d.y) + (d.z + d.w));
        slot ^= 1;
    }
}

// 1 / (1 + exp(-z)).  bf16 and fp16 rows: the hardware's 2^x of the rounded product (off by 2^-24 |z| relative, far under a step of
// the result's type).  fp32 rows: with the product's rounding error as a first-order factor.  e: exp(-z)
template <int DT> __device__ __forceinline__ float sigmoid(float z, float &e)
{
    constexpr float L = 1.44269504088896340736f, Llo = 1.92596299112661746887e-8f, ln2 = 0.693147180559945309f;
    const float t = -z * L;
    e = __builtin_amdgcn_exp2f(t);
    if constexpr (DT == SN_F32) {
        const float lo = fmaf(-z, L, -t) - z * Llo;
        // (beyond 2^126 e may be infinite and the sigmoid is under 2^-126; under 2^-126 e no longer shows in 1 + e; an infinite z has no lo)
        e = fabsf(t) < 126.0f ? fmaf(e, lo * ln2, e) : e;
    }
    return __builtin_amdgcn_rcpf(1.0f + e);
}
template <int DT> __device__ __forceinline__ float sigmoid(float z)
{
    float e;
    return sigmoid<DT>(z, e);
}
// The backward pass needs s = sigmoid(z) and 1 - s, each to its own last bits: one register holds the smaller of the two, 1 - s = e s of
// an open gate (z > 0) as it is, s of a closed one with its sign turned; the other is one subtraction from 1 that cannot cancel.  (1 - s
// of a rounded s is off by 1e-3 of itself at z = 10 and zero from 17 on.  13 % more vector instructions in bf16, 8 % in fp32, no time: 32768
// rows of 4096, bf16, 406 us before and after; 103424 of 256, fp32, padded, from checkpoints, 119 and 120.)
template <int DT> __device__ __forceinline__ float gate_parts(float z, float &s)
{
    float e;
    s = sigmoid<DT>(z, e);
    float w = z > 0.0f ? e * s : -s;
    asm("" : "+v"(w));                       // (or the compiler keeps both in registers after all: 8 to 16 more, a wave less in places)
    return w;
}
__device__ __forceinline__ float gate_opened(float w) { return __float_as_int(w) < 0 ? -w : 1.0f - w; }
__device__ __forceinline__ float gate_closed(float w) { return __float_as_int(w) < 0 ? 1.0f + w : w; }

template <int EV, int CH> struct Row { float v[CH][EV]; };

// MULTI: the workgroup's 2 .. 8 waves have one row at a time; otherwise four rows side by side, each wave on its own
constexpr int block_of(bool multi) { return multi ? 512 : 256; }

template <int DT, int EV, int CH, bool MULTI>
struct Layout {
    static constexpr int kRows = MULTI ? 1 : 4;
    static constexpr int kWidth = 64 * EV * CH;                      // of one wave
    // turns a row is loaded ahead: two where the registers allow it.  fp32, 103424 rows of 256: forward 120 us with one, 110 with
    // two; backward 162 with one, 210 with two (a fourth of the waves less)
    static constexpr int kAheadForward = DT == SN_F32 && CH == 2 ? 1 : 2, kAheadBackward = DT == SN_F32 ? 1 : 2;
    static constexpr bool kTiny = EV == 4 && CH == 1 && !MULTI;      // rows under EV elements come here
};

// Rows are loaded one or two turns ahead of their use: the words of the next ones are on their way while this one is worked on.
template <int DT, int EV, int CH> struct Ahead { Raw<DT, EV> w[CH]; };

template <int DT, int EV, int CH, bool TINY>
__device__ __forceinline__ void issue_cols(Ahead<DT, EV, CH> &r, const void *base, int64_t row, int64_t stride, int col, int step, int E)
{
    const void *p = (const char *)base + row * stride * (DT == SN_F32 ? 4 : 2);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        if (!TINY || E >= EV) load_ahead<DT, EV>(r.w[c], p, col + c * step, E);
        else load_raw<DT, EV>(r.w[c], p, col + c * step, E);
    }
}
// tail: this wave holds columns beyond E (the same for all of its lanes)
template <int DT, int EV, int CH>
__device__ __forceinline__ void take_cols(Row<EV, CH> &r, const Ahead<DT, EV, CH> &a, int col, int step, int E, bool tail)
{
#pragma unroll
    for (int c = 0; c < CH; ++c) unpack<DT, EV>(r.v[c], a.w[c]);
    if (tail && E >= EV) {
#pragma unroll
        for (int c = 0; c < CH; ++c) turn_tail<EV>(r.v[c], tail_shift<EV>(col + c * step, E));
    }
}
// an 8-bit checkpoint's codes and exponents, ahead of their use (columns beyond the padded width: the last block again, cleared later)
template <int EV, int CH> struct AheadKept { uint32_t q[CH][EV / 4], e[CH]; };
template <int EV, int CH>
__device__ __forceinline__ void issue_kept(AheadKept<EV, CH> &r, const void *codes, const void *exps, int64_t row, int col, int step, int npad)
{
    const char *p = (const char *)codes + row * npad;
    const uint8_t *pe = (const uint8_t *)exps + row * (npad / 32);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int j = col + c * step < npad ? col + c * step : npad - EV;
        const uint32_t *src = (const uint32_t *)(p + j);
#pragma unroll
        for (int i = 0; i < EV / 4; ++i) r.q[c][i] = src[i];
        r.e[c] = pe[j / 32];
    }
}
template <int EV, int CH>
__device__ __forceinline__ void take_kept(Row<EV, CH> &r, const AheadKept<EV, CH> &a, int col, int step, int npad)
{
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        decode<EV>(r.v[c], a.q[c], a.e[c]);
        if (col + c * step >= npad) {
#pragma unroll
            for (int i = 0; i < EV; ++i) r.v[c][i] = 0.0f;
        }
    }
}
template <int DT, int EV, int CH>
__device__ __forceinline__ void store_cols(void *base, int64_t row, int col, int step, int E, const Row<EV, CH> &r)
{
    void *p = (char *)base + row * E * (DT == SN_F32 ? 4 : 2);
#pragma unroll
    for (int c = 0; c < CH; ++c) store_row<DT, EV>(p, col + c * step, E, r.v[c]);
}
template <int DT, int EV, int CH>
__device__ __forceinline__ void zero_cols(void *base, int64_t row, int col, int step, int E)
{
    Row<EV, CH> z;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < EV; ++i) z.v[c][i] = 0.0f;
    store_cols<DT, EV, CH>(base, row, col, step, E, z);
}
template <int PT, int EV, int CH>
__device__ __forceinline__ void load_param_as(Row<EV, CH> &r, const void *p, int col, int step, int E)
{
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        Raw<PT, EV> w;
        load_raw<PT, EV>(w, p, col + c * step, E);
        unpack<PT, EV>(r.v[c], w);
    }
}
// (columns beyond E get zeros)
template <int EV, int CH>
__device__ __forceinline__ void load_param(Row<EV, CH> &r, const void *p, int dtype, int col, int step, int E, float none)
{
    if (!p) {
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < EV; ++i) r.v[c][i] = none;
    } else if (dtype == SN_F32) {
        load_param_as<SN_F32, EV, CH>(r, p, col, step, E);
    } else if (dtype == SN_BF16) {
        load_param_as<SN_BF16, EV, CH>(r, p, col, step, E);
    } else {
        load_param_as<SN_F16, EV, CH>(r, p, col, step, E);
    }
}
// lanes of one block of 32 are neighbours; every lane of the wave takes part (features beyond E are zeros)
template <int EV, int CH>
__device__ __forceinline__ void store_checkpoint(void *codes, void *exps, int64_t row, int col, int step, int npad, const Row<EV, CH> &r)
{
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int j = col + c * step;
        const uint32_t e = block_exp(block_top<EV>(r.v[c]));
        uint32_t q[EV / 4];
        encode<EV>(q, r.v[c], e);
        if (j < npad) {
            uint32_t *dst = (uint32_t *)((char *)codes + row * npad + j);
#pragma unroll
            for (int i = 0; i < EV / 4; ++i) dst[i] = q[i];
            if ((j & 31) == 0) ((uint8_t *)exps)[row * (npad / 32) + j / 32] = (uint8_t)e;
        }
    }
}
// does row r count?  (wave-uniform: scalar arithmetic)
__device__ __forceinline__ bool row_counts(const sn_block_norms_args &a, int64_t row)
{
    if (row >= a.rows) return false;
    if (!a.n_valid) return true;
    const int64_t g = a.rows <= 0xFFFFFFFFll ? (int64_t)((uint32_t)row / (uint32_t)a.rows_per_graph) : row / a.rows_per_graph;
    return (int)(row - g * a.rows_per_graph) < a.n_valid[g];
}

// the first row from r on, in steps of turn, that counts (or one behind the last)
__device__ __forceinline__ int64_t next_row(const sn_block_norms_args &a, int64_t r, int64_t turn)
{
    if (a.n_valid)
        while (r < a.rows && !row_counts(a, r)) r += turn;
    return r;
}

struct NormStats { float mean, rstd; };

// mean and 1 / deviation of a row; elements beyond E do not count (they are zeros)
template <int EV, int CH, bool MULTI>
__device__ __forceinline__ NormStats statistics(const Row<EV, CH> &r, int col, int step, int E, bool tail, float inv_e, int rms, float eps, float *red, int &slot)
{
    NormStats s = {0.0f, 0.0f};
    if (!rms) {
        float t = 0.0f;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < EV; ++i) t += r.v[c][i];
        s.mean = row_sum<MULTI>(t, red, slot) * inv_e;
    }
    float q = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < EV; ++i) {
            const float d = r.v[c][i] - s.mean;
            q = !tail || col + c * step + i < E ? fmaf(d, d, q) : q;
        }
    s.rstd = 1.0f / sqrtf(row_sum<MULTI>(q, red, slot) * inv_e + eps);
    return s;
}

// MODE: 0 = the parts of the call are looked up at run time; otherwise the sum of those that are there: 1 the gate, 2 the norm after the
// block, 4 the norm before the next one.  The branches of mode 0 make the compiler wait for all loads and stores in flight where it needs
// the oldest row, the straight lines of the others do not (us, forward / backward, looked up and straight: bf16, 131072 rows of 1024, all
// parts 268 / 464 and 263 / 408, both norms 253 / 410 and 216 / 312, the second alone 215 / 357 and 191 / 309, the first alone 180 / 327
// and 141 / 242 (x is not read); 32768 rows of 4096, all parts 326 / 464 and 306 / 418; fp32, 103424 rows of 256, all parts 118 / 162 and
// 108 / 161; with 8-bit checkpoints measured for all parts only: that size padded, backward 145 and 134, bf16 129 and 105).  For the same reason rows that do not count are passed over by scalar arithmetic, and get their zeros in a loop of their own.
template <int DT, int EV, int CH, bool MULTI, int MODE, bool KEEP>
__global__ __launch_bounds__(block_of(MULTI)) void norms_forward_kernel(sn_block_norms_args a)
{
    using L = Layout<DT, EV, CH, MULTI>;
    constexpr bool ALL = MODE != 0;
    __shared__ __align__(16) float red[32];
    if constexpr (MULTI) {
        if (threadIdx.x < 32) red[threadIdx.x] = 0.0f;
        __syncthreads();
    }
    int slot = 0;
    const int group = MULTI ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = MULTI ? threadIdx.x : threadIdx.x & 63;
    const int E = a.width, step = (MULTI ? (int)blockDim.x : 64) * EV, col = t * EV, npad = (E + 31) & ~31;
    const float inv_e = 1.0f / (float)E;
    const bool gated = ALL ? MODE & 1 : a.gate != nullptr, post = ALL ? MODE & 2 : a.has_post != 0, pre = ALL ? MODE & 4 : a.has_pre != 0;
    const bool tail = __any(tail_shift<EV>(col + (CH - 1) * step, E) > 0);
    const int64_t turn = (int64_t)gridDim.x * L::kRows;

    struct Slot { Ahead<DT, EV, CH> x, f, z; };
    auto issue = [&](Slot &s, int64_t row) {
        issue_cols<DT, EV, CH, L::kTiny>(s.x, a.x, row, a.x_stride, col, step, E);
        issue_cols<DT, EV, CH, L::kTiny>(s.f, a.branch, row, a.branch_stride, col, step, E);
        if (gated) issue_cols<DT, EV, CH, L::kTiny>(s.z, a.gate, row, a.gate_stride, col, step, E);
    };
    const int64_t start = (int64_t)blockIdx.x * L::kRows + group;
    Slot s0, s1;
    int64_t ra = next_row(a, start, turn), rb = a.rows;
    if (ra < a.rows) {
        issue(s0, ra);
        rb = next_row(a, ra + turn, turn);
        if constexpr (L::kAheadForward == 2) issue(s1, rb < a.rows ? rb : ra);
    }
    Row<EV, CH> w1, b1, sc, w2, b2;
    load_param<EV, CH>(sc, a.scale, a.param_dtype, col, step, E, 1.0f);
    load_param<EV, CH>(w1, post ? a.post_weight : nullptr, a.param_dtype, col, step, E, 1.0f);
    load_param<EV, CH>(b1, post ? a.post_bias : nullptr, a.param_dtype, col, step, E, 0.0f);
    load_param<EV, CH>(w2, pre ? a.pre_weight : nullptr, a.param_dtype, col, step, E, 1.0f);
    load_param<EV, CH>(b2, pre ? a.pre_bias : nullptr, a.param_dtype, col, step, E, 0.0f);

    // row r out of s, which then takes row `after` (behind the last: r again, never used)
    auto work = [&](Slot &s, int64_t row, int64_t after) {
        Row<EV, CH> x, f, z;
        take_cols<DT, EV, CH>(x, s.x, col, step, E, tail);
        take_cols<DT, EV, CH>(f, s.f, col, step, E, tail);
        if (gated) take_cols<DT, EV, CH>(z, s.z, col, step, E, tail);
        issue(s, after < a.rows ? after : row);
        if constexpr (KEEP) {
            store_checkpoint<EV, CH>(a.x_codes, a.x_exps, row, col, step, npad, x);
            store_checkpoint<EV, CH>(a.branch_codes, a.branch_exps, row, col, step, npad, f);
            if (gated) store_checkpoint<EV, CH>(a.gate_codes, a.gate_exps, row, col, step, npad, z);
        }
        NormStats n1 = {0.0f, 1.0f}, n2 = {0.0f, 1.0f};
        if (post) n1 = statistics<EV, CH, MULTI>(f, col, step, E, tail, inv_e, a.rms, a.eps, red, slot);
        // (columns beyond E: inputs, weights and biases are zeros there, and so is y)
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < EV; ++i) {
                float p = f.v[c][i];
                if (post) p = fmaf((p - n1.mean) * n1.rstd, w1.v[c][i], b1.v[c][i]);
                if (gated) p *= sigmoid<DT>(z.v[c][i]);
                x.v[c][i] = fmaf(p, sc.v[c][i], x.v[c][i]);
            }
        store_cols<DT, EV, CH>(a.y, row, col, step, E, x);
        if (pre) {
            n2 = statistics<EV, CH, MULTI>(x, col, step, E, tail, inv_e, a.rms, a.eps, red, slot);
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < EV; ++i) x.v[c][i] = fmaf((x.v[c][i] - n2.mean) * n2.rstd, w2.v[c][i], b2.v[c][i]);
            store_cols<DT, EV, CH>(a.h, row, col, step, E, x);
        }
        if (a.stats && t == 0) *reinterpret_cast<float4 *>(a.stats + row * 4) = make_float4(n1.mean, n1.rstd, n2.mean, n2.rstd);
    };
    while (ra < a.rows) {
        if constexpr (L::kAheadForward == 2) {
            const int64_t rc = next_row(a, rb + turn, turn);
            work(s0, ra, rc);
            if (rb >= a.rows) break;
            const int64_t rd = next_row(a, rc + turn, turn);
            work(s1, rb, rd);
            ra = rc;
            rb = rd;
        } else {
            work(s0, ra, rb);
            ra = rb;
            rb = next_row(a, rb + turn, turn);
        }
    }
    if (a.n_valid) {
        for (int64_t row = start; row < a.rows; row += turn) {
            if (row_counts(a, row)) continue;
            zero_cols<DT, EV, CH>(a.y, row, col, step, E);
            if (pre) zero_cols<DT, EV, CH>(a.h, row, col, step, E);
        }
    }
}

template <int DT, int EV, int CH, bool MULTI, int MODE, bool KEPT>
__global__ __launch_bounds__(block_of(MULTI)) void norms_backward_kernel(sn_block_norms_args a, float *partial)
{
    using L = Layout<DT, EV, CH, MULTI>;
    constexpr bool ALL = MODE != 0;
    __shared__ __align__(16) float red[32];
    if constexpr (MULTI) {
        if (threadIdx.x < 32) red[threadIdx.x] = 0.0f;
        __syncthreads();
    }
    int slot = 0;
    const int group = MULTI ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = MULTI ? threadIdx.x : threadIdx.x & 63;
    const int E = a.width, step = (MULTI ? (int)blockDim.x : 64) * EV, col = t * EV, npad = (E + 31) & ~31;
    const float inv_e = 1.0f / (float)E;
    const bool gated = ALL ? MODE & 1 : KEPT ? a.gate_codes != nullptr : a.gate != nullptr;
    const bool post = ALL ? MODE & 2 : a.has_post != 0, has_dy = ALL || a.dy, has_dh = ALL ? MODE & 4 : a.dh != nullptr;
    const bool tail = __any(tail_shift<EV>(col + (CH - 1) * step, E) > 0);
    const int64_t turn = (int64_t)gridDim.x * L::kRows;

    struct Slot {
        Ahead<DT, EV, CH> x, f, z, dy, dh;
        AheadKept<EV, CH> kx, kf, kz;
        float4 st;
    };
    auto issue = [&](Slot &s, int64_t row) {
        if constexpr (KEPT) {
            issue_kept<EV, CH>(s.kx, a.x_codes, a.x_exps, row, col, step, npad);
            issue_kept<EV, CH>(s.kf, a.branch_codes, a.branch_exps, row, col, step, npad);
            if (gated) issue_kept<EV, CH>(s.kz, a.gate_codes, a.gate_exps, row, col, step, npad);
        } else {
            issue_cols<DT, EV, CH, L::kTiny>(s.x, a.x, row, a.x_stride, col, step, E);
            issue_cols<DT, EV, CH, L::kTiny>(s.f, a.branch, row, a.branch_stride, col, step, E);
            if (gated) issue_cols<DT, EV, CH, L::kTiny>(s.z, a.gate, row, a.gate_stride, col, step, E);
        }
        if (has_dy) issue_cols<DT, EV, CH, L::kTiny>(s.dy, a.dy, row, a.dy_stride, col, step, E);
        if (has_dh) issue_cols<DT, EV, CH, L::kTiny>(s.dh, a.dh, row, a.dh_stride, col, step, E);
        s.st = *reinterpret_cast<const float4 *>(a.stats + row * 4);
    };
    const int64_t start = (int64_t)blockIdx.x * L::kRows + group;
    Slot s0, s1;
    int64_t ra = next_row(a, start, turn), rb = a.rows;
    if (ra < a.rows) {
        issue(s0, ra);
        rb = next_row(a, ra + turn, turn);
        if constexpr (L::kAheadBackward == 2) issue(s1, rb < a.rows ? rb : ra);
    }
    Row<EV, CH> w1, b1, sc, w2;
    load_param<EV, CH>(sc, a.scale, a.param_dtype, col, step, E, 1.0f);
    load_param<EV, CH>(w1, post ? a.post_weight : nullptr, a.param_dtype, col, step, E, 1.0f);
    load_param<EV, CH>(b1, post ? a.post_bias : nullptr, a.param_dtype, col, step, E, 0.0f);
    load_param<EV, CH>(w2, has_dh ? a.pre_weight : nullptr, a.param_dtype, col, step, E, 1.0f);
    Row<EV, CH> sum[kVectors] = {};

    // row r out of s, which then takes row `after` (behind the last: r again, never used)
    auto work = [&](Slot &s, int64_t row, int64_t after) {
        Row<EV, CH> x, f, z, u = {}, d;
        if constexpr (KEPT) {
            take_kept<EV, CH>(x, s.kx, col, step, npad);
            take_kept<EV, CH>(f, s.kf, col, step, npad);
            if (gated) take_kept<EV, CH>(z, s.kz, col, step, npad);
        } else {
            take_cols<DT, EV, CH>(x, s.x, col, step, E, tail);
            take_cols<DT, EV, CH>(f, s.f, col, step, E, tail);
            if (gated) take_cols<DT, EV, CH>(z, s.z, col, step, E, tail);
        }
        if (has_dy) take_cols<DT, EV, CH>(u, s.dy, col, step, E, tail);
        if (has_dh) take_cols<DT, EV, CH>(d, s.dh, col, step, E, tail);
        const float4 st = s.st;
        issue(s, after < a.rows ? after : row);
        // f -> unit values of the post norm, z -> the gate's parts, x -> unit values of y.  Columns beyond E hold whatever the statistics make of
        // zeros: every use multiplies it by a weight or a gradient that is zero there, and no store takes it.
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < EV; ++i) {
                f.v[c][i] = (f.v[c][i] - st.x) * st.y;
                float p = fmaf(f.v[c][i], w1.v[c][i], b1.v[c][i]);
                if (gated) {
                    float open;
                    z.v[c][i] = gate_parts<DT>(z.v[c][i], open);
                    p *= open;
                }
                x.v[c][i] = (fmaf(p, sc.v[c][i], x.v[c][i]) - st.z) * st.w;
            }
        if (has_dh) {
            float m1 = 0.0f, m2 = 0.0f;
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < EV; ++i) {
                    sum[0].v[c][i] = fmaf(d.v[c][i], x.v[c][i], sum[0].v[c][i]);
                    sum[1].v[c][i] += d.v[c][i];
                    d.v[c][i] *= w2.v[c][i];
                    m1 += d.v[c][i];
                    m2 = fmaf(d.v[c][i], x.v[c][i], m2);
                }
            row_sum2<MULTI>(m1, m2, red, slot);
            m1 = a.rms ? 0.0f : m1 * inv_e;
            m2 *= inv_e;
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < EV; ++i) u.v[c][i] = fmaf(st.w, fmaf(-x.v[c][i], m2, d.v[c][i] - m1), u.v[c][i]);
        }
        if (ALL || a.dx) store_cols<DT, EV, CH>(a.dx, row, col, step, E, u);
        // d -> gradient of the gated product's p, x -> gradient of the gate
        float m1 = 0.0f, m2 = 0.0f;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < EV; ++i) {
                const float p = fmaf(f.v[c][i], w1.v[c][i], b1.v[c][i]);
                const float us = gated ? u.v[c][i] * gate_opened(z.v[c][i]) : u.v[c][i];
                sum[2].v[c][i] = fmaf(us, p, sum[2].v[c][i]);
                const float dp = us * sc.v[c][i];
                if (gated) x.v[c][i] = dp * p * gate_closed(z.v[c][i]);
                sum[3].v[c][i] = fmaf(dp, f.v[c][i], sum[3].v[c][i]);
                sum[4].v[c][i] += dp;
                d.v[c][i] = dp * w1.v[c][i];
                m1 += d.v[c][i];
                m2 = fmaf(d.v[c][i], f.v[c][i], m2);
            }
        if (gated && (ALL || a.dgate)) store_cols<DT, EV, CH>(a.dgate, row, col, step, E, x);
        if (post) {
            row_sum2<MULTI>(m1, m2, red, slot);
            m1 = a.rms ? 0.0f : m1 * inv_e;
            m2 *= inv_e;
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < EV; ++i) d.v[c][i] = st.y * fmaf(-f.v[c][i], m2, d.v[c][i] - m1);
        }
        if (ALL || a.dbranch) store_cols<DT, EV, CH>(a.dbranch, row, col, step, E, d);
    };
    while (ra < a.rows) {
        if constexpr (L::kAheadBackward == 2) {
            const int64_t rc = next_row(a, rb + turn, turn);
            work(s0, ra, rc);
            if (rb >= a.rows) break;
            const int64_t rd = next_row(a, rc + turn, turn);
            work(s1, rb, rd);
            ra = rc;
            rb = rd;
        } else {
            work(s0, ra, rb);
            ra = rb;
            rb = next_row(a, rb + turn, turn);
        }
    }
    if (a.n_valid) {
        for (int64_t row = start; row < a.rows; row += turn) {
            if (row_counts(a, row)) continue;
            if (a.dx) zero_cols<DT, EV, CH>(a.dx, row, col, step, E);
            if (a.dbranch) zero_cols<DT, EV, CH>(a.dbranch, row, col, step, E);
            if (a.dgate) zero_cols<DT, EV, CH>(a.dgate, row, col, step, E);
        }
    }
    if (partial) {
        // the workgroup's rows side by side are added here, one line of partial sums leaves for each workgroup
        float *dst = partial + (int64_t)blockIdx.x * kVectors * E;
        __shared__ float join[MULTI ? 1 : L::kRows * L::kWidth];
#pragma unroll
        for (int k = 0; k < kVectors; ++k) {
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < EV; ++i) {
                    const int j = col + c * step + i;
                    if constexpr (!MULTI) join[group * L::kWidth + j] = sum[k].v[c][i];
                    else if (j < E) dst[(int64_t)k * E + j] = sum[k].v[c][i];
                }
            if constexpr (!MULTI) {
                __syncthreads();
                for (int j = threadIdx.x; j < E; j += 256) {
                    float v = join[j];
#pragma unroll
                    for (int g = 1; g < L::kRows; ++g) v += join[g * L::kWidth + j];
                    dst[(int64_t)k * E + j] = v;
                }
                __syncthreads();
            }
        }
    }
}

struct ColumnOut { void *p[kVectors]; };

// column sums of the workgroups' partial rows in a fixed order: 32 columns, 32 slices of the parts side by side
__global__ __launch_bounds__(1024) void norms_columns_kernel(const float *partial, int parts, int E, ColumnOut out, int dtype)
{
    __shared__ float red[32][33];
    const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const int k = blockIdx.y, j = blockIdx.x * 32 + lane;
    if (!out.p[k]) return;
    float s = 0.0f;
    if (j < E) {
#pragma unroll 8
        for (int p = slice; p < parts; p += 32) s += partial[((int64_t)p * kVectors + k) * E + j];
    }
    red[slice][lane] = s;
    __syncthreads();
    s = red[lane][slice];                                    // now: lane = slice, slice = column
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) s += __shfl_xor(s, off, 32);
    const int c = blockIdx.x * 32 + slice;
    if (lane == 0 && c < E) store_any(out.p[k], dtype, c, s);
}

// Waves of a row: 8 elements a lane up to 4096 columns (16 waves with five column sums each would spill).  Up to 256 columns a lane
// takes 4: all lanes work and more waves are resident (bf16, 200000 rows forward / backward: 256 columns 108 / 212 us, with 8 a lane
// 152 / 230; 128 columns 104 / 193, with 8 a lane 152 / 227).
int waves_for(int E) { return (E + 511) / 512; }
int rows_per_block(int E) { return waves_for(E) > 1 ? 1 : 4; }
int backward_blocks(int64_t rows, int E)
{
    const int64_t turns = (rows + rows_per_block(E) - 1) / rows_per_block(E);
    // Workgroups take rows in turn (a stretch of rows for each: 32768 x 4096 bf16 693 us for 662, 103424 x 256 fp32 297 for 272).
    // As many as cover the loads, no more: each further one loads the parameters again, writes a line of column sums,
    // and has fewer rows to look ahead over.  Four workgroups of four waves a compute unit, about six waves of the wider rows (measured
    // with 1, 2, 3, 4, 6, 8 workgroups a compute unit: bf16 131072 x 1024 756 493 411 438 478 497 us; 65536 x 2048 413 447 500 486 488
    // 556; 32768 x 4096 420 434 465 465 500 541; fp32 32768 x 2048 405 430 446 436 462 454; one wave, fp32 200000 x 256 650 397 320 301
    // 355 322; bf16 200000 x 512 330 326 336 341 346 350).
    const int W = waves_for(E);
    const int64_t most = 256 * (W == 1 ? 4 : W > 6 ? 1 : 6 / W), each = (turns + most - 1) / most;
    return (int)((turns + each - 1) / each);                 // (the same number of turns for all but the last)
}

int check_args(const sn_block_norms_args *a, const char *who)
{
    SN_REQUIRE(a, SN_ERR_BAD_ARG, "%s: NULL arguments", who);
    SN_REQUIRE(a->struct_size == sizeof(sn_block_norms_args), SN_ERR_BAD_ARG, "%s: struct_size %u, the library's is %zu", who, a->struct_size,
               sizeof(sn_block_norms_args));
    SN_REQUIRE(a->dtype >= 0 && a->dtype <= 2 && a->param_dtype >= 0 && a->param_dtype <= 2, SN_ERR_BAD_ARG, "%s: unknown type", who);
    SN_REQUIRE(a->rows >= 0 && a->rows <= kMostRows, SN_ERR_BAD_ARG, "%s: rows %lld", who, (long long)a->rows);
    SN_REQUIRE(a->width >= 1 && a->width <= SN_BLOCK_NORMS_MAX_WIDTH, SN_ERR_UNSUPPORTED, "%s: width %d outside 1 .. 4096", who, a->width);
    SN_REQUIRE(!a->n_valid || (a->rows_per_graph > 0 && a->rows % a->rows_per_graph == 0), SN_ERR_BAD_ARG, "%s: rows_per_graph %d", who, a->rows_per_graph);
    SN_REQUIRE((!a->has_post || a->post_weight) && (!a->has_pre || a->pre_weight), SN_ERR_BAD_ARG, "%s: a norm without weight", who);
    return SN_OK;
}

// rest: whatever else a straight-line kernel takes for granted (without any norm there is none: index 1 of the tables is mode 0 too)
int mode_of(const sn_block_norms_args &a, const void *gate, bool rest) { return rest ? (gate ? 1 : 0) + (a.has_post ? 2 : 0) + (a.has_pre ? 4 : 0) : 0; }
#define SN_NORMS_MODES(kernel, kept) \
    {kernel<DT, EV, CH, MULTI, 0, kept>, kernel<DT, EV, CH, MULTI, 0, kept>, kernel<DT, EV, CH, MULTI, 2, kept>, kernel<DT, EV, CH, MULTI, 3, kept>, \
     kernel<DT, EV, CH, MULTI, 4, kept>, kernel<DT, EV, CH, MULTI, 5, kept>, kernel<DT, EV, CH, MULTI, 6, kept>, kernel<DT, EV, CH, MULTI, 7, kept>}

template <int DT, int EV, int CH, bool MULTI> int launch_forward(const sn_block_norms_args &a, hipStream_t st)
{
    using L = Layout<DT, EV, CH, MULTI>;
    // Workgroups a compute unit: eight of four waves, eight waves of the wider rows (measured with 1, 2, 3, 4, 8, 16 workgroups: bf16
    // 131072 x 1024 750 453 311 263 269 280 us; 65536 x 2048 394 275 288 287 286 308; 32768 x 4096 254 271 280 265 266 261).  Rows of one
    // wave, with 2, 4, 6, 8, 16: bf16 200000 x 256 133 111 109 110 107, 200000 x 512 202 208 207 208 205, 12544 x 256 14.4 13.7 13.8 15.1 16.3;
    // fp32 103424 x 256 125 101 125 110 111, a quarter of it padding 139 104 122 109 104, 103424 x 128 115 76 87 79 79, 12544 x 256 21.7 20.0
    // 19.4 21.6 22.1: for fp32 four are the better number by 4 to 9 %, eight is what all types take.
    const int W = waves_for(a.width);
    const int64_t turns = (a.rows + L::kRows - 1) / L::kRows, most = 256 * (MULTI ? (8 + W - 1) / W : 8), each = (turns + most - 1) / most;
    using Kernel = void (*)(sn_block_norms_args);
    static constexpr Kernel kernels[2][8] = {SN_NORMS_MODES(norms_forward_kernel, false), SN_NORMS_MODES(norms_forward_kernel, true)};
    const Kernel kernel = kernels[a.x_codes != nullptr][mode_of(a, a.gate, true)];
    hipLaunchKernelGGL(kernel, dim3((unsigned)((turns + each - 1) / each)), dim3(MULTI ? waves_for(a.width) * 64 : 256), 0, st, a);
    SN_CHECK_LAUNCH("sn_block_norms_forward");
    return SN_OK;
}
template <int DT, int EV, int CH, bool MULTI> int launch_backward(const sn_block_norms_args &a, hipStream_t st)
{
    const int blocks = backward_blocks(a.rows, a.width);
    const ColumnOut out = {{a.dpre_weight, a.dpre_bias, a.dscale, a.dpost_weight, a.dpost_bias}};
    bool columns = false;
    for (int k = 0; k < kVectors; ++k) columns |= out.p[k] != nullptr;
    float *partial = columns ? (float *)a.workspace : nullptr;
    const void *gate = a.x_codes ? a.gate_codes : a.gate;
    using Kernel = void (*)(sn_block_norms_args, float *);
    static constexpr Kernel kernels[2][8] = {SN_NORMS_MODES(norms_backward_kernel, false), SN_NORMS_MODES(norms_backward_kernel, true)};
    const bool rest = a.dy && (a.dh || !a.has_pre) && a.dx && a.dbranch && (!gate || a.dgate);
    const Kernel kernel = kernels[a.x_codes != nullptr][mode_of(a, gate, rest)];
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(MULTI ? waves_for(a.width) * 64 : 256), 0, st, a, partial);
    SN_CHECK_LAUNCH("sn_block_norms_backward");
    if (columns) {
        hipLaunchKernelGGL(norms_columns_kernel, dim3((a.width + 31) / 32, kVectors), dim3(1024), 0, st, partial, blocks, a.width, out, a.param_dtype);
        SN_CHECK_LAUNCH("sn_block_norms_backward (columns)");
    }
    return SN_OK;
}

template <bool FORWARD, int DT, int EV, int CH> int by_waves(const sn_block_norms_args &a, hipStream_t st)
{
    if constexpr (FORWARD) return waves_for(a.width) > 1 ? launch_forward<DT, EV, CH, true>(a, st) : launch_forward<DT, EV, CH, false>(a, st);
    else return waves_for(a.width) > 1 ? launch_backward<DT, EV, CH, true>(a, st) : launch_backward<DT, EV, CH, false>(a, st);
}
template <bool FORWARD, int DT> int by_width(const sn_block_norms_args &a, hipStream_t st)
{
    if (a.width <= 256) {
        if constexpr (FORWARD) return launch_forward<DT, 4, 1, false>(a, st);
        else return launch_backward<DT, 4, 1, false>(a, st);
    }
    if constexpr (DT == SN_F32) return by_waves<FORWARD, DT, 4, 2>(a, st);
    else return by_waves<FORWARD, DT, 8, 1>(a, st);
}
template <bool FORWARD> int by_type(const sn_block_norms_args &a, hipStream_t st)
{
    return a.dtype == SN_F32 ? by_width<FORWARD, SN_F32>(a, st) : a.dtype == SN_BF16 ? by_width<FORWARD, SN_BF16>(a, st) : by_width<FORWARD, SN_F16>(a, st);
}

}  // namespace

extern "C" int sn_block_norms_forward(const sn_block_norms_args *args, void *stream)
{
    const int rc = check_args(args, "sn_block_norms_forward");
    if (rc != SN_OK) return rc;
    const sn_block_norms_args &a = *args;
    if (a.rows == 0) return SN_OK;
    SN_REQUIRE(a.x && a.branch && a.y && (!a.has_pre || a.h), SN_ERR_BAD_ARG, "sn_block_norms_forward: NULL pointer");
    SN_REQUIRE(!a.x_codes || (a.x_exps && a.branch_codes && a.branch_exps && (!a.gate || (a.gate_codes && a.gate_exps))), SN_ERR_BAD_ARG,
               "sn_block_norms_forward: an incomplete set of checkpoint buffers");
    return by_type<true>(a, (hipStream_t)stream);
}

extern "C" size_t sn_block_norms_workspace(int64_t rows, int width)
{
    // (no rows: nothing to add up, and no workgroups to divide them among)
    if (rows < 1 || rows > kMostRows || width < 1 || width > SN_BLOCK_NORMS_MAX_WIDTH) return 0;
    return (size_t)backward_blocks(rows, width) * kVectors * width * sizeof(float);
}

extern "C" int sn_block_norms_backward(const sn_block_norms_args *args, void *stream)
{
    const int rc = check_args(args, "sn_block_norms_backward");
    if (rc != SN_OK) return rc;
    const sn_block_norms_args &a = *args;
    SN_REQUIRE(a.rows > 0, SN_ERR_BAD_ARG, "sn_block_norms_backward: no rows (the gradients of the parameters are zeros: the caller's)");
    SN_REQUIRE(a.stats && (a.dy || a.dh), SN_ERR_BAD_ARG, "sn_block_norms_backward: NULL pointer");
    SN_REQUIRE(!a.dh || a.has_pre, SN_ERR_BAD_ARG, "sn_block_norms_backward: a gradient of h without the norm before the next block");
    SN_REQUIRE(a.x_codes ? a.x_exps && a.branch_codes && a.branch_exps && (!a.gate_codes || a.gate_exps) : a.x && a.branch, SN_ERR_BAD_ARG,
               "sn_block_norms_backward: the inputs of the forward pass are missing");
    SN_REQUIRE(a.workspace && a.workspace_bytes >= sn_block_norms_workspace(a.rows, a.width), SN_ERR_WORKSPACE, "sn_block_norms_backward: workspace of %zu bytes",
               a.workspace_bytes);
    return by_type<false>(a, (hipStream_t)stream);
}
