// The end of a residual block and the norm before the next one (schemanet_blocks.h):
//     p = N_post(branch);  y = x + scale * sigmoid(gate) * p;  h = N_pre(y)
// and its backward pass, with u = dy + N_pre^T(dh) the whole gradient of y:
//     dx = u;   dgate = u scale p s (1 - s);   dp = u scale s;   dbranch = N_post^T(dp);      s = sigmoid(gate)
//     dscale = sum u s p;   dw_post = sum dp n1;  db_post = sum dp;  dw_pre = sum dh n2;  db_pre = sum dh     (n = the unit values)
//     N^T(d) = r (w d - mean(w d) - n mean(w d n))          (rms: without the first mean)
// Bound: HBM - forward reads x, branch, gate and writes y, h; backward reads those three and dy, dh and writes three gradients.
// Every element is read once and stays in registers: a row belongs to 64 .. 512 lanes (8 elements a lane), the means are two
// passes over registers (centred squares: no cancellation), the column sums of the backward pass are kept in registers over
// all rows of a workgroup, written once per workgroup and added in a fixed order by a second launch (no atomics).
// The unit values are recomputed from the inputs and the forward pass's row statistics; y is not kept.
#include "sn_typed.h"

namespace {

using namespace sn;

constexpr int kVectors = 5;              // column sums of the backward pass: pre weight, pre bias, scale, post weight, post bias

// all-reduce over the WAVES waves that hold one row; `slot` alternates between two LDS buffers, so one barrier is enough
template <int WAVES> __device__ __forceinline__ float row_sum(float v, float *red, int &slot, int wave_in_row, int group)
{
    v = sn_wave_sum(v);
    if constexpr (WAVES > 1) {
        float *buf = red + (slot * 16) + group * WAVES;
        if ((threadIdx.x & 63) == 0) buf[wave_in_row] = v;
        __syncthreads();
        v = buf[0];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) v += buf[i];
        slot ^= 1;
    }
    return v;
}
template <int WAVES> __device__ __forceinline__ void row_sum2(float &a, float &b, float *red, int &slot, int wave_in_row, int group)
{
    a = sn_wave_sum(a);
    b = sn_wave_sum(b);
    if constexpr (WAVES > 1) {
        float *ba = red + (slot * 16) + group * WAVES, *bb = ba + 32;
        if ((threadIdx.x & 63) == 0) { ba[wave_in_row] = a; bb[wave_in_row] = b; }
        __syncthreads();
        a = ba[0]; b = bb[0];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) { a += ba[i]; b += bb[i]; }
        slot ^= 1;
    }
}

// 1 / (1 + exp(-z)): one reciprocal with a Newton step; z under -80 gives exp(-80), NaN stays
__device__ __forceinline__ float sigmoid(float z)
{
    const float d = 1.0f + expf(z < -80.0f ? 80.0f : -z);
    const float r = __builtin_amdgcn_rcpf(d);
    return fmaf(fmaf(-d, r, 1.0f), r, r);
}

template <int EV, int CH> struct Row { float v[CH][EV]; };

constexpr int block_of(int waves) { return waves >= 4 ? waves * 64 : 256; }

template <int DT, int EV, int CH, int WAVES>
struct Layout {
    static constexpr int kThreads = WAVES * 64;                      // of one row
    static constexpr int kRows = WAVES >= 4 ? 1 : 4 / WAVES;         // rows of a workgroup at a time
    static constexpr int kBlock = kThreads * kRows;
    static constexpr int kStep = kThreads * EV;                      // columns of one chunk
    static constexpr int kWidth = kStep * CH;
};

template <int DT, int EV, int CH, int STEP>
__device__ __forceinline__ void load_cols(Row<EV, CH> &r, const void *base, int64_t row, int64_t stride, int col, int E)
{
    const void *p = (const char *)base + row * stride * (DT == SN_F32 ? 4 : 2);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        uint32_t w[words<DT, EV>()];
        load_raw<DT, EV>(w, p, col + c * STEP, E);
        unpack<DT, EV>(r.v[c], w);
    }
}
template <int DT, int EV, int CH, int STEP>
__device__ __forceinline__ void store_cols(void *base, int64_t row, int col, int E, const Row<EV, CH> &r)
{
    void *p = (char *)base + row * E * (DT == SN_F32 ? 4 : 2);
#pragma unroll
    for (int c = 0; c < CH; ++c) store_row<DT, EV>(p, col + c * STEP, E, r.v[c]);
}
template <int DT, int EV, int CH, int STEP>
__device__ __forceinline__ void zero_cols(void *base, int64_t row, int col, int E)
{
    Row<EV, CH> z;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < EV; ++i) z.v[c][i] = 0.0f;
    store_cols<DT, EV, CH, STEP>(base, row, col, E, z);
}
template <int PT, int EV, int CH, int STEP>
__device__ __forceinline__ void load_param_as(Row<EV, CH> &r, const void *p, int col, int E)
{
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        Raw<PT, EV> w;
        load_raw<PT, EV>(w, p, col + c * STEP, E);
        unpack<PT, EV>(r.v[c], w);
    }
}
// (columns beyond E get zeros)
template <int EV, int CH, int STEP>
__device__ __forceinline__ void load_param(Row<EV, CH> &r, const void *p, int dtype, int col, int E, float none)
{
    if (!p) {
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < EV; ++i) r.v[c][i] = none;
    } else if (dtype == SN_F32) {
        load_param_as<SN_F32, EV, CH, STEP>(r, p, col, E);
    } else if (dtype == SN_BF16) {
        load_param_as<SN_BF16, EV, CH, STEP>(r, p, col, E);
    } else {
        load_param_as<SN_F16, EV, CH, STEP>(r, p, col, E);
    }
}
// lanes of one block of 32 are neighbours; every lane of the wave takes part (features beyond E are zeros)
template <int EV, int CH, int STEP>
__device__ __forceinline__ void store_checkpoint(void *codes, void *exps, int64_t row, int col, int npad, const Row<EV, CH> &r)
{
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int j = col + c * STEP;
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
template <int EV, int CH, int STEP>
__device__ __forceinline__ void load_checkpoint(Row<EV, CH> &r, const void *codes, const void *exps, int64_t row, int col, int npad)
{
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int j = col + c * STEP;
        uint32_t q[EV / 4] = {}, e = 8u;
        if (j < npad) {
            const uint32_t *src = (const uint32_t *)((const char *)codes + row * npad + j);
#pragma unroll
            for (int i = 0; i < EV / 4; ++i) q[i] = src[i];
            e = ((const uint8_t *)exps)[row * (npad / 32) + j / 32];
        }
        decode<EV>(r.v[c], q, e);
    }
}

struct NormStats { float mean, rstd; };

// mean and 1 / deviation of a row; elements beyond E do not count (they are zeros)
template <int EV, int CH, int STEP, int WAVES>
__device__ __forceinline__ NormStats statistics(const Row<EV, CH> &r, int col, int E, float inv_e, int rms, float eps, float *red, int &slot, int wir, int group)
{
    NormStats s = {0.0f, 0.0f};
    if (!rms) {
        float t = 0.0f;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < EV; ++i) t += r.v[c][i];
        s.mean = row_sum<WAVES>(t, red, slot, wir, group) * inv_e;
    }
    float q = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < EV; ++i) {
            const float d = r.v[c][i] - s.mean;
            q = col + c * STEP + i < E ? fmaf(d, d, q) : q;
        }
    s.rstd = 1.0f / sqrtf(row_sum<WAVES>(q, red, slot, wir, group) * inv_e + eps);
    return s;
}

template <int DT, int EV, int CH, int WAVES>
__global__ __launch_bounds__(block_of(WAVES)) void norms_forward_kernel(sn_block_norms_args a)
{
    using L = Layout<DT, EV, CH, WAVES>;
    constexpr int STEP = L::kStep;
    __shared__ float red[64];
    int slot = 0;
    const int group = threadIdx.x / L::kThreads, t = threadIdx.x % L::kThreads, wir = t >> 6;
    const int E = a.width, col = t * EV, npad = (E + 31) & ~31;
    const float inv_e = 1.0f / (float)E;
    Row<EV, CH> w1, b1, sc, w2, b2;
    load_param<EV, CH, STEP>(sc, a.scale, a.param_dtype, col, E, 1.0f);
    load_param<EV, CH, STEP>(w1, a.has_post ? a.post_weight : nullptr, a.param_dtype, col, E, 1.0f);
    load_param<EV, CH, STEP>(b1, a.has_post ? a.post_bias : nullptr, a.param_dtype, col, E, 0.0f);
    load_param<EV, CH, STEP>(w2, a.has_pre ? a.pre_weight : nullptr, a.param_dtype, col, E, 1.0f);
    load_param<EV, CH, STEP>(b2, a.has_pre ? a.pre_bias : nullptr, a.param_dtype, col, E, 0.0f);

    // every wave of the workgroup makes the same number of turns: the row sums hold barriers
    for (int64_t first = (int64_t)blockIdx.x * L::kRows; first < a.rows; first += (int64_t)gridDim.x * L::kRows) {
        const int64_t row = first + group;
        bool live = row < a.rows;
        if (live && a.n_valid) {
            const int64_t g = row / a.rows_per_graph;
            if ((int)(row - g * a.rows_per_graph) >= a.n_valid[g]) {
                zero_cols<DT, EV, CH, STEP>(a.y, row, col, E);
                if (a.has_pre) zero_cols<DT, EV, CH, STEP>(a.h, row, col, E);
                live = false;
            }
        }
        if (WAVES == 1 && !live) continue;                   // (one wave a row: no barrier inside)
        Row<EV, CH> x = {}, f = {}, z = {};
        if (live) {
            load_cols<DT, EV, CH, STEP>(x, a.x, row, a.x_stride, col, E);
            load_cols<DT, EV, CH, STEP>(f, a.branch, row, a.branch_stride, col, E);
            if (a.gate) load_cols<DT, EV, CH, STEP>(z, a.gate, row, a.gate_stride, col, E);
            if (a.x_codes) {
                store_checkpoint<EV, CH, STEP>(a.x_codes, a.x_exps, row, col, npad, x);
                store_checkpoint<EV, CH, STEP>(a.branch_codes, a.branch_exps, row, col, npad, f);
                if (a.gate) store_checkpoint<EV, CH, STEP>(a.gate_codes, a.gate_exps, row, col, npad, z);
            }
        }
        NormStats s1 = {0.0f, 1.0f}, s2 = {0.0f, 1.0f};
        if (a.has_post) s1 = statistics<EV, CH, STEP, WAVES>(f, col, E, inv_e, a.rms, a.eps, red, slot, wir, group);
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < EV; ++i) {
                float p = f.v[c][i];
                if (a.has_post) p = fmaf((p - s1.mean) * s1.rstd, w1.v[c][i], b1.v[c][i]);
                if (a.gate) p *= sigmoid(z.v[c][i]);
                const float y = fmaf(p, sc.v[c][i], x.v[c][i]);
                x.v[c][i] = col + c * STEP + i < E ? y : 0.0f;
            }
        if (live) store_cols<DT, EV, CH, STEP>(a.y, row, col, E, x);
        if (a.has_pre) {
            s2 = statistics<EV, CH, STEP, WAVES>(x, col, E, inv_e, a.rms, a.eps, red, slot, wir, group);
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < EV; ++i) x.v[c][i] = fmaf((x.v[c][i] - s2.mean) * s2.rstd, w2.v[c][i], b2.v[c][i]);
            if (live) store_cols<DT, EV, CH, STEP>(a.h, row, col, E, x);
        }
        if (a.stats && live && t == 0) *reinterpret_cast<float4 *>(a.stats + row * 4) = make_float4(s1.mean, s1.rstd, s2.mean, s2.rstd);
    }
}

template <int DT, int EV, int CH, int WAVES, bool KEPT>
__global__ __launch_bounds__(block_of(WAVES)) void norms_backward_kernel(sn_block_norms_args a, float *partial)
{
    using L = Layout<DT, EV, CH, WAVES>;
    constexpr int STEP = L::kStep;
    __shared__ float red[64];
    int slot = 0;
    const int group = threadIdx.x / L::kThreads, t = threadIdx.x % L::kThreads, wir = t >> 6;
    const int E = a.width, col = t * EV, npad = (E + 31) & ~31;
    const float inv_e = 1.0f / (float)E;
    Row<EV, CH> w1, b1, sc, w2;
    load_param<EV, CH, STEP>(sc, a.scale, a.param_dtype, col, E, 1.0f);
    load_param<EV, CH, STEP>(w1, a.has_post ? a.post_weight : nullptr, a.param_dtype, col, E, 1.0f);
    load_param<EV, CH, STEP>(b1, a.has_post ? a.post_bias : nullptr, a.param_dtype, col, E, 0.0f);
    load_param<EV, CH, STEP>(w2, a.has_pre ? a.pre_weight : nullptr, a.param_dtype, col, E, 1.0f);
    Row<EV, CH> sum[kVectors] = {};

    for (int64_t first = (int64_t)blockIdx.x * L::kRows; first < a.rows; first += (int64_t)gridDim.x * L::kRows) {
        const int64_t row = first + group;
        bool live = row < a.rows;
        if (live && a.n_valid) {
            const int64_t g = row / a.rows_per_graph;
            if ((int)(row - g * a.rows_per_graph) >= a.n_valid[g]) {
                if (a.dx) zero_cols<DT, EV, CH, STEP>(a.dx, row, col, E);
                if (a.dbranch) zero_cols<DT, EV, CH, STEP>(a.dbranch, row, col, E);
                if (a.dgate) zero_cols<DT, EV, CH, STEP>(a.dgate, row, col, E);
                live = false;
            }
        }
        if (WAVES == 1 && !live) continue;
        Row<EV, CH> x = {}, f = {}, z = {}, u = {}, d = {};
        float4 st = make_float4(0.0f, 1.0f, 0.0f, 1.0f);
        if (live) {
            if constexpr (KEPT) {
                load_checkpoint<EV, CH, STEP>(x, a.x_codes, a.x_exps, row, col, npad);
                load_checkpoint<EV, CH, STEP>(f, a.branch_codes, a.branch_exps, row, col, npad);
                if (a.gate_codes) load_checkpoint<EV, CH, STEP>(z, a.gate_codes, a.gate_exps, row, col, npad);
            } else {
                load_cols<DT, EV, CH, STEP>(x, a.x, row, a.x_stride, col, E);
                load_cols<DT, EV, CH, STEP>(f, a.branch, row, a.branch_stride, col, E);
                if (a.gate) load_cols<DT, EV, CH, STEP>(z, a.gate, row, a.gate_stride, col, E);
            }
            if (a.dy) load_cols<DT, EV, CH, STEP>(u, a.dy, row, a.dy_stride, col, E);
            if (a.dh) load_cols<DT, EV, CH, STEP>(d, a.dh, row, a.dh_stride, col, E);
            st = *reinterpret_cast<const float4 *>(a.stats + row * 4);
        }
        const bool gated = KEPT ? a.gate_codes != nullptr : a.gate != nullptr;
        // f -> unit values of the post norm, z -> sigmoid, x -> unit values of y
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < EV; ++i) {
                const bool in = col + c * STEP + i < E;
                f.v[c][i] = in ? (f.v[c][i] - st.x) * st.y : 0.0f;
                const float p = fmaf(f.v[c][i], w1.v[c][i], b1.v[c][i]);
                if (gated) z.v[c][i] = sigmoid(z.v[c][i]);
                const float y = fmaf(gated ? p * z.v[c][i] : p, sc.v[c][i], x.v[c][i]);
                x.v[c][i] = in ? (y - st.z) * st.w : 0.0f;
            }
        if (a.dh) {
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
            row_sum2<WAVES>(m1, m2, red, slot, wir, group);
            m1 = a.rms ? 0.0f : m1 * inv_e;
            m2 *= inv_e;
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < EV; ++i) u.v[c][i] = fmaf(st.w, fmaf(-x.v[c][i], m2, d.v[c][i] - m1), u.v[c][i]);
        }
        if (a.dx && live) store_cols<DT, EV, CH, STEP>(a.dx, row, col, E, u);
        // d -> gradient of the gated product's p, x -> gradient of the gate
        float m1 = 0.0f, m2 = 0.0f;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < EV; ++i) {
                const bool in = col + c * STEP + i < E;
                const float p = fmaf(f.v[c][i], w1.v[c][i], b1.v[c][i]);
                const float s = gated ? z.v[c][i] : 1.0f, uu = in ? u.v[c][i] : 0.0f;
                const float us = uu * s;
                sum[2].v[c][i] = fmaf(us, p, sum[2].v[c][i]);
                const float dp = us * sc.v[c][i];
                x.v[c][i] = dp * p * (1.0f - s);
                sum[3].v[c][i] = fmaf(dp, f.v[c][i], sum[3].v[c][i]);
                sum[4].v[c][i] += dp;
                d.v[c][i] = dp * w1.v[c][i];
                m1 += d.v[c][i];
                m2 = fmaf(d.v[c][i], f.v[c][i], m2);
            }
        if (a.dgate && live) store_cols<DT, EV, CH, STEP>(a.dgate, row, col, E, x);
        if (a.has_post) {
            row_sum2<WAVES>(m1, m2, red, slot, wir, group);
            m1 = a.rms ? 0.0f : m1 * inv_e;
            m2 *= inv_e;
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < EV; ++i) d.v[c][i] = st.y * fmaf(-f.v[c][i], m2, d.v[c][i] - m1);
        }
        if (a.dbranch && live) store_cols<DT, EV, CH, STEP>(a.dbranch, row, col, E, d);
    }
    if (partial) {
        float *dst = partial + ((int64_t)blockIdx.x * L::kRows + group) * kVectors * E;
#pragma unroll
        for (int k = 0; k < kVectors; ++k)
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < EV; ++i) {
                    const int j = col + c * STEP + i;
                    if (j < E) dst[(int64_t)k * E + j] = sum[k].v[c][i];
                }
    }
}

struct ColumnOut { void *p[kVectors]; };

// column sums of the workgroups' partial rows, in order; 16 slices of the parts side by side
__global__ __launch_bounds__(1024) void norms_columns_kernel(const float *partial, int parts, int E, ColumnOut out, int dtype)
{
    __shared__ float red[16][64];
    const int lane = threadIdx.x & 63, slice = threadIdx.x >> 6;
    const int k = blockIdx.y, j = blockIdx.x * 64 + lane;
    if (!out.p[k]) return;
    const int per = (parts + 15) / 16, p0 = slice * per, p1 = p0 + per < parts ? p0 + per : parts;
    float s = 0.0f;
    if (j < E) {
#pragma unroll 8
        for (int p = p0; p < p1; ++p) s += partial[((int64_t)p * kVectors + k) * E + j];
    }
    red[slice][lane] = s;
    __syncthreads();
    if (slice == 0 && j < E) {
#pragma unroll
        for (int i = 1; i < 16; ++i) s += red[i][lane];
        store_any(out.p[k], dtype, j, s);
    }
}

// lanes of a row: 8 elements a lane up to 4096 columns (16 waves with five column sums each would spill); 4 a lane under 257 columns
int waves_for(int E)
{
    int w = 1;
    while (w * 512 < E) w *= 2;
    return w;
}
int rows_per_block(int E) { const int w = waves_for(E); return w >= 4 ? 1 : 4 / w; }
int backward_blocks(int64_t rows, int E)
{
    const int64_t turns = (rows + rows_per_block(E) - 1) / rows_per_block(E);
    const int64_t most = waves_for(E) <= 4 ? 1024 : 512;
    return (int)(turns < most ? turns : most);
}

int check_args(const sn_block_norms_args *a, const char *who)
{
    SN_REQUIRE(a, SN_ERR_BAD_ARG, "%s: NULL arguments", who);
    SN_REQUIRE(a->struct_size == sizeof(sn_block_norms_args), SN_ERR_BAD_ARG, "%s: struct_size %u, the library's is %zu", who, a->struct_size,
               sizeof(sn_block_norms_args));
    SN_REQUIRE(a->dtype >= 0 && a->dtype <= 2 && a->param_dtype >= 0 && a->param_dtype <= 2, SN_ERR_BAD_ARG, "%s: unknown type", who);
    SN_REQUIRE(a->rows >= 0, SN_ERR_BAD_ARG, "%s: rows %lld", who, (long long)a->rows);
    SN_REQUIRE(a->width >= 1 && a->width <= SN_BLOCK_NORMS_MAX_WIDTH, SN_ERR_UNSUPPORTED, "%s: width %d outside 1 .. 4096", who, a->width);
    SN_REQUIRE(!a->n_valid || (a->rows_per_graph > 0 && a->rows % a->rows_per_graph == 0), SN_ERR_BAD_ARG, "%s: rows_per_graph %d", who, a->rows_per_graph);
    SN_REQUIRE((!a->has_post || a->post_weight) && (!a->has_pre || a->pre_weight), SN_ERR_BAD_ARG, "%s: a norm without weight", who);
    return SN_OK;
}

template <int DT, int EV, int CH, int WAVES> int launch_forward(const sn_block_norms_args &a, hipStream_t st)
{
    using L = Layout<DT, EV, CH, WAVES>;
    const int64_t turns = (a.rows + L::kRows - 1) / L::kRows;
    const int64_t most = WAVES <= 4 ? 2048 : 1024;
    hipLaunchKernelGGL((norms_forward_kernel<DT, EV, CH, WAVES>), dim3((unsigned)(turns < most ? turns : most)), dim3(L::kBlock), 0, st, a);
    SN_CHECK_LAUNCH("sn_block_norms_forward");
    return SN_OK;
}
template <int DT, int EV, int CH, int WAVES> int launch_backward(const sn_block_norms_args &a, hipStream_t st)
{
    using L = Layout<DT, EV, CH, WAVES>;
    const int blocks = backward_blocks(a.rows, a.width);
    const ColumnOut out = {{a.dpre_weight, a.dpre_bias, a.dscale, a.dpost_weight, a.dpost_bias}};
    bool columns = false;
    for (int k = 0; k < kVectors; ++k) columns |= out.p[k] != nullptr;
    float *partial = columns ? (float *)a.workspace : nullptr;
    if (a.x_codes) hipLaunchKernelGGL((norms_backward_kernel<DT, EV, CH, WAVES, true>), dim3(blocks), dim3(L::kBlock), 0, st, a, partial);
    else hipLaunchKernelGGL((norms_backward_kernel<DT, EV, CH, WAVES, false>), dim3(blocks), dim3(L::kBlock), 0, st, a, partial);
    SN_CHECK_LAUNCH("sn_block_norms_backward");
    if (columns) {
        hipLaunchKernelGGL(norms_columns_kernel, dim3((a.width + 63) / 64, kVectors), dim3(1024), 0, st, partial, blocks * L::kRows, a.width, out, a.param_dtype);
        SN_CHECK_LAUNCH("sn_block_norms_backward (columns)");
    }
    return SN_OK;
}

template <bool FORWARD, int DT, int EV, int CH> int by_waves(const sn_block_norms_args &a, hipStream_t st)
{
    switch (waves_for(a.width)) {
#define SN_CASE(W) case W: if constexpr (FORWARD) return launch_forward<DT, EV, CH, W>(a, st); else return launch_backward<DT, EV, CH, W>(a, st);
        SN_CASE(1) SN_CASE(2) SN_CASE(4)
#undef SN_CASE
        default: if constexpr (FORWARD) return launch_forward<DT, EV, CH, 8>(a, st); else return launch_backward<DT, EV, CH, 8>(a, st);
    }
}
template <bool FORWARD, int DT> int by_width(const sn_block_norms_args &a, hipStream_t st)
{
    if (a.width <= 256) {
        if constexpr (FORWARD) return launch_forward<DT, 4, 1, 1>(a, st);
        else return launch_backward<DT, 4, 1, 1>(a, st);
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
    if (rows < 0 || width < 1 || width > SN_BLOCK_NORMS_MAX_WIDTH) return 0;
    return (size_t)backward_blocks(rows, width) * rows_per_block(width) * kVectors * width * sizeof(float);
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
