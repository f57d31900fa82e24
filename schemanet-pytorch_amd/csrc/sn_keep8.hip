// 8-bit checkpoints of activations (schemanet_blocks.h) and the weight gradient of a Linear layer from one.
//     s = 2^k, the smallest with max|x| < 127.5 s over 32 features;   q = rint(x / s);   kept = q s
//     dW[o, i] = sum_r dY[r, o] kept[r, i];    db[o] = sum_r dY[r, o]
// Scaling by a power of two is exact, |q| <= 127 fits bfloat16's significand: kept is exact in bf16, and the product needs no
// rounding of it.  dY goes in as bf16 pieces that add up to it (fp32: three of 8 bits, fp16: two, bf16: itself).
#include "sn_typed.h"

namespace {

using namespace sn;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kPackThreads = 256;

// HBM bound: one read of x, 1 + 1/32 bytes written per element; a lane holds 8 features, four lanes a block
template <int DT>
__global__ __launch_bounds__(kPackThreads) void checkpoint8_kernel(const void *x, int64_t rows, int n, int64_t stride, uint8_t *codes, uint8_t *exps)
{
    const int npad = (n + 31) & ~31, groups = npad / 8;
    const int64_t total = rows * groups, turn = (int64_t)gridDim.x * kPackThreads;
    for (int64_t i = (int64_t)blockIdx.x * kPackThreads + threadIdx.x; i - threadIdx.x % 64 < total; i += turn) {
        const bool in = i < total;
        const int64_t r = in ? (total <= 0xFFFFFFFFll ? (int64_t)((uint32_t)i / (uint32_t)groups) : i / groups) : 0;
        const int j = in ? (int)(i - r * groups) * 8 : npad;
        uint32_t w[words<DT, 8>()];
        float v[8];
        load_raw<DT, 8>(w, (const char *)x + r * stride * (DT == SN_F32 ? 4 : 2), j, in ? n : 0);
        unpack<DT, 8>(v, w);
        const uint32_t e = block_exp(block_top<8>(v));       // groups is a multiple of 4: the lanes of a block are one quad
        uint32_t q[2];
        encode<8>(q, v, e);
        if (in) {
            *reinterpret_cast<uint2 *>(codes + r * npad + j) = make_uint2(q[0], q[1]);
            if ((j & 31) == 0) exps[r * (npad / 32) + j / 32] = (uint8_t)e;
        }
    }
}

template <int DT>
__global__ __launch_bounds__(kPackThreads) void restore8_kernel(const uint8_t *codes, const uint8_t *exps, int64_t rows, int n, void *out)
{
    const int npad = (n + 31) & ~31, groups = (n + 7) / 8;
    const int64_t total = rows * groups, turn = (int64_t)gridDim.x * kPackThreads;
    for (int64_t i = (int64_t)blockIdx.x * kPackThreads + threadIdx.x; i < total; i += turn) {
        const int64_t r = total <= 0xFFFFFFFFll ? (int64_t)((uint32_t)i / (uint32_t)groups) : i / groups;
        const int j = (int)(i - r * groups) * 8;
        const uint2 c = *reinterpret_cast<const uint2 *>(codes + r * npad + j);
        const uint32_t q[2] = {c.x, c.y};
        float v[8];
        decode<8>(v, q, exps[r * (npad / 32) + j / 32]);
        store_row<DT, 8>((char *)out + r * n * (DT == SN_F32 ? 4 : 2), j, n, v);
    }
}

// ------------------------------------------------------------------------------------------
// dW: tiles of 128 x 128 outputs, 64 rows a step, four waves of 64 x 64 (2 x 2 MFMA 32x32x16).  Both operands lie with the
// summed index outermost, so a thread takes 8 rows of 4 columns, turns them in registers (the bf16 conversion pairs two ROWS
// into a word) and writes 8 consecutive k of one column to LDS as the matrix instruction wants them.
constexpr int kTile = 128, kStepRows = 64, kGradThreads = 256;
constexpr int kPlane = kTile * kStepRows;                   // bf16 elements of one operand piece in LDS (16 KiB)

// 16-byte chunk c (8 k) of column m: the eight chunks of a column are rotated so that both the writes (columns 4 apart) and the
// reads (neighbouring columns) of eight lanes fall on different banks
__device__ __forceinline__ int lds_at(int m, int c) { return m * kStepRows + ((c ^ ((m ^ (m >> 3)) & 7)) << 3); }

template <int DT> constexpr int pieces() { return DT == SN_F32 ? 3 : DT == SN_F16 ? 2 : 1; }

template <int DT>
__global__ __launch_bounds__(kGradThreads) void weight_grad8_kernel(const void *dy, int64_t dy_stride, const uint8_t *codes, const uint8_t *exps, int64_t rows,
                                                                    int out_f, int in_f, int rows_per_split, void *dw, void *db, int out_dtype, float *part_w,
                                                                    float *part_b)
{
    constexpr int P = pieces<DT>();
    extern __shared__ uint16_t lds[];                        // P pieces of dY, then kept
    uint16_t *const lb = lds + P * kPlane;
    const int tiles_i = (in_f + kTile - 1) / kTile;
    const int o0 = (blockIdx.x / tiles_i) * kTile, i0 = (blockIdx.x % tiles_i) * kTile;
    const int64_t r_begin = (int64_t)blockIdx.y * rows_per_split;
    const int64_t r_end = r_begin + rows_per_split < rows ? r_begin + rows_per_split : rows;
    const int npad = (in_f + 31) & ~31;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int cg = t & 31, kg = t >> 5;                      // columns 4 cg .. + 3, rows 8 kg .. + 7 of a step
    const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
    const bool sums = db && i0 == 0;

    f32x16 acc[2][2] = {};
    float bias[4] = {};
    uint32_t ra[8][words<DT, 4>()], rq[8], re[8];

    auto fetch = [&](int64_t r0) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int64_t r = r0 + kg * 8 + k;
            const bool in = r < r_end;
            load_raw<DT, 4>(ra[k], (const char *)dy + (in ? r : r_begin) * dy_stride * (DT == SN_F32 ? 4 : 2), o0 + 4 * cg, in ? out_f : 0);
            rq[k] = 0u;
            re[k] = 8u;
            if (in && i0 + 4 * cg < npad) {
                rq[k] = *reinterpret_cast<const uint32_t *>(codes + r * npad + i0 + 4 * cg);
                re[k] = exps[r * (npad / 32) + (i0 + 4 * cg) / 32];
            }
        }
    };
    auto stage = [&]() {
        float v[8][4];
#pragma unroll
        for (int k = 0; k < 8; ++k) unpack<DT, 4>(v[k], ra[k]);
        if (sums) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
#pragma unroll
                for (int j = 0; j < 4; ++j) bias[j] += v[k][j];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int at = lds_at(4 * cg + j, kg);
            uint32_t w[P][4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float a = v[2 * k][j], b = v[2 * k + 1][j];
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    w[p][k] = pack_bf16(a, b);
                    if (p + 1 < P) {                         // what the piece leaves is exact in fp32
                        a -= __uint_as_float(w[p][k] << 16);
                        b -= __uint_as_float(w[p][k] & 0xFFFF0000u);
                    }
                }
            }
#pragma unroll
            for (int p = 0; p < P; ++p) *reinterpret_cast<uint4 *>(lds + p * kPlane + at) = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint32_t q[1] = {rq[k]};
            decode<4>(v[k], q, re[k]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint4 w;
            w.x = pack_bf16(v[0][j], v[1][j]); w.y = pack_bf16(v[2][j], v[3][j]);
            w.z = pack_bf16(v[4][j], v[5][j]); w.w = pack_bf16(v[6][j], v[7][j]);
            *reinterpret_cast<uint4 *>(lb + lds_at(4 * cg + j, kg)) = w;
        }
    };

    if (r_begin < r_end) fetch(r_begin);
    for (int64_t r0 = r_begin; r0 < r_end; r0 += kStepRows) {
        stage();
        __syncthreads();
        if (r0 + kStepRows < r_end) fetch(r0 + kStepRows);
#pragma unroll
        for (int kk = 0; kk < kStepRows / 16; ++kk) {
            bf16x8 b[2];
#pragma unroll
            for (int n = 0; n < 2; ++n) b[n] = *reinterpret_cast<const bf16x8 *>(lb + lds_at(wn + n * 32 + (lane & 31), 2 * kk + (lane >> 5)));
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    const bf16x8 a = *reinterpret_cast<const bf16x8 *>(lds + p * kPlane + lds_at(wm + m * 32 + (lane & 31), 2 * kk + (lane >> 5)));
#pragma unroll
                    for (int n = 0; n < 2; ++n) acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b[n], acc[m][n], 0, 0, 0);
                }
        }
        __syncthreads();
    }

    // C of the 32x32 instruction: column lane & 31, row (i & 3) + 8 (i >> 2) + 4 (lane >> 5)
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int o = o0 + wm + m * 32 + (i & 3) + 8 * (i >> 2) + 4 * (lane >> 5), c = i0 + wn + n * 32 + (lane & 31);
                if (o < out_f && c < in_f) {
                    if (part_w) part_w[((int64_t)blockIdx.y * out_f + o) * in_f + c] = acc[m][n][i];
                    else store_any(dw, out_dtype, (int64_t)o * in_f + c, acc[m][n][i]);
                }
            }
    if (sums) {
        float *red = reinterpret_cast<float *>(lds);         // [8 row groups][128 columns]
#pragma unroll
        for (int j = 0; j < 4; ++j) red[kg * kTile + 4 * cg + j] = bias[j];
        __syncthreads();
        if (t < kTile && o0 + t < out_f) {
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) s += red[k * kTile + t];
            if (part_b) part_b[(int64_t)blockIdx.y * out_f + o0 + t] = s;
            else store_any(db, out_dtype, o0 + t, s);
        }
    }
}

// the splits' partial results, added in order: 4 elements a thread; the last blocks take db
__global__ __launch_bounds__(256) void weight_grad8_join_kernel(const float *part_w, const float *part_b, int splits, int64_t cells, int out_f, void *dw, void *db,
                                                                int out_dtype)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < cells) {
        float s = 0.0f;
#pragma unroll 8
        for (int p = 0; p < splits; ++p) s += part_w[(int64_t)p * cells + i];
        store_any(dw, out_dtype, i, s);
    } else if (db && i - cells < out_f) {
        float s = 0.0f;
        for (int p = 0; p < splits; ++p) s += part_b[(int64_t)p * out_f + (i - cells)];
        store_any(db, out_dtype, i - cells, s);
    }
}

// splits of the summed rows: enough workgroups for two on each of the 256 compute units, at least 256 rows a split
struct Split { int n, rows; };
Split split_rows(int64_t rows, int out_f, int in_f)
{
    const int64_t tiles = (int64_t)((out_f + kTile - 1) / kTile) * ((in_f + kTile - 1) / kTile);
    int64_t n = 512 / tiles;
    const int64_t most = (rows + 255) / 256;
    n = n < 1 ? 1 : n;
    n = n > most ? most : n;
    n = n < 1 ? 1 : n;
    int64_t per = (rows + n - 1) / n;
    per = (per + kStepRows - 1) / kStepRows * kStepRows;
    per = per < kStepRows ? kStepRows : per;
    n = rows ? (rows + per - 1) / per : 1;
    return Split{(int)n, (int)per};
}

template <int DT>
int launch_grad(const void *dy, int64_t dy_stride, const void *codes, const void *exps, int64_t rows, int out_f, int in_f, void *dw, void *db, int out_dtype,
                void *workspace, hipStream_t st)
{
    const Split sp = split_rows(rows, out_f, in_f);
    const int64_t tiles = (int64_t)((out_f + kTile - 1) / kTile) * ((in_f + kTile - 1) / kTile), cells = (int64_t)out_f * in_f;
    float *part_w = sp.n > 1 ? (float *)workspace : nullptr, *part_b = sp.n > 1 ? part_w + sp.n * cells : nullptr;
    const size_t lds = (size_t)(pieces<DT>() + 1) * kPlane * 2;
    const int rc = sn_ensure_dynamic_lds((const void *)weight_grad8_kernel<DT>, lds, "sn_checkpoint8_weight_grad");
    if (rc != SN_OK) return rc;
    hipLaunchKernelGGL(weight_grad8_kernel<DT>, dim3((unsigned)tiles, sp.n), dim3(kGradThreads), lds, st, dy, dy_stride, (const uint8_t *)codes, (const uint8_t *)exps,
                       rows, out_f, in_f, sp.rows, dw, db, out_dtype, part_w, part_b);
    SN_CHECK_LAUNCH("sn_checkpoint8_weight_grad");
    if (sp.n > 1) {
        hipLaunchKernelGGL(weight_grad8_join_kernel, dim3((unsigned)((cells + (db ? out_f : 0) + 255) / 256)), dim3(256), 0, st, part_w, part_b, sp.n, cells, out_f,
                           dw, db, out_dtype);
        SN_CHECK_LAUNCH("sn_checkpoint8_weight_grad (join)");
    }
    return SN_OK;
}

unsigned pack_blocks(int64_t total)
{
    const int64_t b = (total + kPackThreads - 1) / kPackThreads;
    return (unsigned)(b < 4096 ? b : 4096);
}

}  // namespace

extern "C" int sn_checkpoint8(const void *x, int dtype, int64_t rows, int n, int64_t row_stride, void *codes, void *exps, void *stream)
{
    SN_REQUIRE(rows >= 0 && n >= 1 && n <= (1 << 30) && dtype >= 0 && dtype <= 2, SN_ERR_BAD_ARG, "sn_checkpoint8: bad rows=%lld n=%d type=%d", (long long)rows, n, dtype);
    if (rows == 0) return SN_OK;
    SN_REQUIRE(x && codes && exps, SN_ERR_BAD_ARG, "sn_checkpoint8: NULL pointer");
    const int64_t total = rows * (((int64_t)n + 31) / 32 * 4);
    const dim3 grid(pack_blocks(total)), block(kPackThreads);
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == SN_F32) hipLaunchKernelGGL(checkpoint8_kernel<SN_F32>, grid, block, 0, st, x, rows, n, row_stride, (uint8_t *)codes, (uint8_t *)exps);
    else if (dtype == SN_BF16) hipLaunchKernelGGL(checkpoint8_kernel<SN_BF16>, grid, block, 0, st, x, rows, n, row_stride, (uint8_t *)codes, (uint8_t *)exps);
    else hipLaunchKernelGGL(checkpoint8_kernel<SN_F16>, grid, block, 0, st, x, rows, n, row_stride, (uint8_t *)codes, (uint8_t *)exps);
    SN_CHECK_LAUNCH("sn_checkpoint8");
    return SN_OK;
}

extern "C" int sn_checkpoint8_restore(const void *codes, const void *exps, int64_t rows, int n, void *out, int dtype, void *stream)
{
    SN_REQUIRE(rows >= 0 && n >= 1 && n <= (1 << 30) && dtype >= 0 && dtype <= 2, SN_ERR_BAD_ARG, "sn_checkpoint8_restore: bad rows=%lld n=%d type=%d", (long long)rows, n,
               dtype);
    if (rows == 0) return SN_OK;
    SN_REQUIRE(out && codes && exps, SN_ERR_BAD_ARG, "sn_checkpoint8_restore: NULL pointer");
    const dim3 grid(pack_blocks(rows * (((int64_t)n + 7) / 8))), block(kPackThreads);
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == SN_F32) hipLaunchKernelGGL(restore8_kernel<SN_F32>, grid, block, 0, st, (const uint8_t *)codes, (const uint8_t *)exps, rows, n, out);
    else if (dtype == SN_BF16) hipLaunchKernelGGL(restore8_kernel<SN_BF16>, grid, block, 0, st, (const uint8_t *)codes, (const uint8_t *)exps, rows, n, out);
    else hipLaunchKernelGGL(restore8_kernel<SN_F16>, grid, block, 0, st, (const uint8_t *)codes, (const uint8_t *)exps, rows, n, out);
    SN_CHECK_LAUNCH("sn_checkpoint8_restore");
    return SN_OK;
}

extern "C" size_t sn_checkpoint8_weight_grad_workspace(int64_t rows, int out_features, int in_features, int dy_dtype)
{
    if (rows < 0 || out_features < 1 || in_features < 1 || dy_dtype < 0 || dy_dtype > 2) return 0;
    const Split sp = split_rows(rows, out_features, in_features);
    return sp.n > 1 ? (size_t)sp.n * ((size_t)out_features * in_features + out_features) * sizeof(float) : 16;
}

extern "C" int sn_checkpoint8_weight_grad(const void *dy, int dy_dtype, int64_t dy_row_stride, const void *codes, const void *exps, int64_t rows, int out_features,
                                          int in_features, void *dw, void *db, int out_dtype, void *workspace, size_t workspace_bytes, void *stream)
{
    SN_REQUIRE(rows > 0 && out_features >= 1 && in_features >= 1, SN_ERR_BAD_ARG, "sn_checkpoint8_weight_grad: bad rows=%lld out=%d in=%d", (long long)rows,
               out_features, in_features);
    SN_REQUIRE(dy_dtype >= 0 && dy_dtype <= 2 && out_dtype >= 0 && out_dtype <= 2, SN_ERR_BAD_ARG, "sn_checkpoint8_weight_grad: unknown type");
    SN_REQUIRE(out_features <= (1 << 20) && in_features <= (1 << 20) && rows < (1ll << 31), SN_ERR_UNSUPPORTED, "sn_checkpoint8_weight_grad: too large");
    SN_REQUIRE(dy && codes && exps && dw, SN_ERR_BAD_ARG, "sn_checkpoint8_weight_grad: NULL pointer");
    SN_REQUIRE(workspace && workspace_bytes >= sn_checkpoint8_weight_grad_workspace(rows, out_features, in_features, dy_dtype), SN_ERR_WORKSPACE,
               "sn_checkpoint8_weight_grad: workspace of %zu bytes", workspace_bytes);
    const hipStream_t st = (hipStream_t)stream;
    if (dy_dtype == SN_F32) return launch_grad<SN_F32>(dy, dy_row_stride, codes, exps, rows, out_features, in_features, dw, db, out_dtype, workspace, st);
    if (dy_dtype == SN_BF16) return launch_grad<SN_BF16>(dy, dy_row_stride, codes, exps, rows, out_features, in_features, dw, db, out_dtype, workspace, st);
    return launch_grad<SN_F16>(dy, dy_row_stride, codes, exps, rows, out_features, in_features, dw, db, out_dtype, workspace, st);
}
