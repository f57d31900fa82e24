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
constexpr int kMostSide = 1 << 20;               // of a weight gradient: features and summed rows
constexpr int64_t kMostRows = (1ll << 31) - 1;

// HBM bound: one read of x, 1 + 1/32 bytes written per element; a lane holds 8 features, four lanes a block.  32768 rows of 2048, bf16:
// 36 us, 5.6 TB/s
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

// HBM bound: 16 bytes of the result a lane (fp32 32 bytes, 16-bit types 8: slower both at 12544 rows of 256, 4.9 -> 5.4 us and 3.5 -> 4.3, and at
// 32768 rows of 2048, 69 -> 94 and 31.8 -> 34.3; the same codes again, from the caches).  Codes of their own each time: 6.0 and 3.9 us, 68 and
// 40; the latter, bf16, is 5.1 TB/s
template <int DT>
__global__ __launch_bounds__(kPackThreads) void restore8_kernel(const uint8_t *codes, const uint8_t *exps, int64_t rows, int n, void *out)
{
    constexpr int EV = DT == SN_F32 ? 4 : 8;
    const int npad = (n + 31) & ~31, groups = (n + EV - 1) / EV;
    const int64_t total = rows * groups, turn = (int64_t)gridDim.x * kPackThreads;
    for (int64_t i = (int64_t)blockIdx.x * kPackThreads + threadIdx.x; i < total; i += turn) {
        const int64_t r = total <= 0xFFFFFFFFll ? (int64_t)((uint32_t)i / (uint32_t)groups) : i / groups;
        const int j = (int)(i - r * groups) * EV;
        const uint32_t *src = reinterpret_cast<const uint32_t *>(codes + r * npad + j);
        uint32_t q[EV / 4];
#pragma unroll
        for (int k = 0; k < EV / 4; ++k) q[k] = src[k];
        float v[EV];
        decode<EV>(v, q, exps[r * (npad / 32) + j / 32]);
        if constexpr (DT == SN_F16) {                        // a value from 65024 on was kept as 65536: to fp16's largest, not to infinity (NaN stays)
#pragma unroll
            for (int k = 0; k < EV; ++k) v[k] = fabsf(v[k]) > 65504.0f ? copysignf(65504.0f, v[k]) : v[k];
        }
        store_row<DT, EV>((char *)out + r * n * (DT == SN_F32 ? 4 : 2), j, n, v);
    }
}

// ------------------------------------------------------------------------------------------
// dW: a workgroup owns TILE x TILE outputs of one split of the summed rows, BK rows a step, MFMA 32x32x16 on wave tiles of
// 128 x 64 (TILE 256) or 64 x 32 (TILE 128) of eight waves.  Both operands lie with the summed index outermost, so a
// staging thread takes 8 rows of UC columns, turns them in registers (the bf16 conversion pairs two ROWS into a word) and
// writes 8 consecutive rows of one column to LDS, as the matrix instruction wants them.  Half of the waves stage dY, the other
// half the kept codes; two LDS buffers, one barrier a step; the dY waves stage before their products and the code waves after
// them, so that on every SIMD the vector work of one wave runs under the matrix instructions of the other; priorities keep that
// order (code waves multiply first: 1061 -> 1040 us at the size below).
// Bound: the matrix pipe with the vector work beside it (64 codes are 160 vector instructions a step, a third of the issue slots).
// 32768 rows of 2048 -> 8192, bf16: 1040 us, 1057 TFLOP/s; the library's product of the same operands, both in bf16, takes 937 us.
// fp32 gradients (three products): 32768 rows of 2048 -> 2048 698 us, 394 TFLOP/s (1.18 PFLOP/s of matrix work), fp16 485 us.
// Small sizes are bound by a few steps' latency: 12544 rows of 256 -> 256, fp32: 14 us and 5 us for the joining of 49 splits.
typedef uint32_t u32;

template <int V> struct Type { static constexpr int value = V; };
template <int DT> constexpr int pieces() { return DT == SN_F32 ? 3 : DT == SN_F16 ? 2 : 1; }

template <int DT, int TILE> struct Grad {
    static constexpr int P = pieces<DT>();
    static constexpr int BK = TILE == 128 || P == 1 ? 64 : 32;       // rows of a step: two buffers of P + 1 pieces in 128 KiB
    static constexpr int UC = TILE == 256 && P == 1 ? 8 : 4; // columns of a staging thread
    static constexpr int kWaves = 8, kThreads = kWaves * 64;
    static constexpr int kPlane = TILE * BK;                 // bf16 elements of one piece
    static constexpr int kBuffer = (P + 1) * kPlane;
    static constexpr int kGroups = TILE / UC;                // column groups
    static constexpr int MT = TILE == 256 ? 4 : 2, NT = TILE == 256 ? 2 : 1;     // 32 x 32 products of a wave
    static constexpr int kBlocks = TILE / 32;                // checkpoint blocks of a row of the tile
    static constexpr int kKg = 64 / kGroups > 0 ? 64 / kGroups : 1;      // row groups of a staging wave
    static constexpr int JR = 64 / (kKg * kBlocks);          // rows of a group whose exponents one register of the wave holds
    static_assert(kGroups * (BK / 8) * 2 == kThreads, "half of the threads stage each operand");
    static_assert(JR == 4 || JR == 8, "a wave's exponents in one or two registers");
};

// 16-byte chunk c (8 rows) of column m.  The chunks of a column are rotated so that the writes (columns UC apart) and the reads
// (neighbouring columns) of eight lanes fall on different banks (BK 32: the writes on half of them)
template <int BK> __device__ __forceinline__ int lds_at(int m, int c)
{
    if constexpr (BK == 64) return m * BK + ((c ^ ((m ^ (m >> 3)) & 7)) << 3);
    else return m * BK + ((c ^ (((m >> 1) ^ (m >> 3)) & 3)) << 3);
}

template <int DT, int NW> __device__ __forceinline__ float element(const u32 (&w)[NW], int j)
{
    if constexpr (DT == SN_F32) return __uint_as_float(w[j]);
    else return (float)__builtin_bit_cast(_Float16, (uint16_t)(w[j / 2] >> (16 * (j & 1))));
}

// SMALL: sizes under one tile or one step, rows too far apart for 32-bit offsets - every load is tested.  Otherwise none is: the last
// tile of a row or column of tiles and the last step of a split are moved back to where they are whole; outputs that two tiles
// share come out of both with the same bits, rows that a split has had already are cleared from dY before they are staged.
template <int DT, int TILE, bool SMALL>
__global__ __launch_bounds__((Grad<DT, TILE>::kThreads), 2) void weight_grad8_kernel(const void *dy, int64_t dy_stride, const uint8_t *codes, const uint8_t *exps,
                                                                                 int64_t rows, int out_f, int in_f, int splits, int rows_per_split, void *dw,
                                                                                 void *db, int out_dtype, float *part_w, float *part_b)
{
    using G = Grad<DT, TILE>;
    constexpr int P = G::P, BK = G::BK, UC = G::UC, SIZE = DT == SN_F32 ? 4 : 2;
    extern __shared__ uint16_t lds[];
    // the workgroups of one XCD (every eighth) take neighbouring tiles of the same rows: they share panels in its L2
    const int tiles_i = (in_f + TILE - 1) / TILE, tiles = tiles_i * ((out_f + TILE - 1) / TILE), total = tiles * splits;
    const int xcd = blockIdx.x & 7, each = total >> 3, rest = total & 7;
    const int work = xcd * each + (xcd < rest ? xcd : rest) + (int)(blockIdx.x >> 3);
    const int split = work / tiles, tile = work - split * tiles;
    const int npad = (in_f + 31) & ~31, nblk = npad >> 5;
    int o0 = (tile / tiles_i) * TILE, i0 = (tile % tiles_i) * TILE;
    if constexpr (!SMALL) {
        o0 = o0 + TILE <= out_f ? o0 : out_f - TILE;
        i0 = i0 + TILE <= npad ? i0 : npad - TILE;
    }
    const int64_t r_begin = (int64_t)split * rows_per_split;
    const int64_t r_end = r_begin + rows_per_split < rows ? r_begin + rows_per_split : rows;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const bool role_x = wave >= G::kWaves / 2;               // stages the kept codes
    const int unit = role_x ? t - G::kThreads / 2 : t;
    const int cg = unit % G::kGroups, kg = unit / G::kGroups;
    const int wm = (wave & 1) * (TILE / 2), wn = (wave >> 1) * (TILE / 4);
    const bool sums = db && i0 == 0;

    f32x16 acc[G::MT][G::NT] = {};
    float bias[UC] = {};
    u32 raw[8][UC * SIZE / 4];                               // dY, or (the first words) codes
    u32 ex[8 / G::JR];

    // exponents: one or two loads for the wave's rows and blocks, handed round by lane
    const int ex_b = i0 / 32 + lane % G::kBlocks;
    const int ex_row = (kg - lane / G::kGroups + lane / (G::kBlocks * G::JR)) * 8 + (lane / G::kBlocks) % G::JR;
    // a scalar row address and a 32-bit offset of the lane
    const u32 lane_off = role_x ? (u32)(kg * 8 * npad + UC * cg) : (u32)(kg * 8 * (int)dy_stride + UC * cg) * SIZE;
    const u32 ex_off = (u32)(ex_row * nblk + ex_b);
    auto fetch = [&](int64_t r0) {
        if constexpr (!SMALL) {
            r0 = r0 + BK <= r_end ? r0 : r_end - BK;
            if (!role_x) {
                const char *const base = (const char *)dy + (r0 * dy_stride + o0) * SIZE;
#pragma unroll
                for (int k = 0; k < 8; ++k) load_words<UC * SIZE / 4>(raw[k], base + k * dy_stride * SIZE + lane_off);
            } else {
                const uint8_t *const base = codes + r0 * npad + i0, *const ebase = exps + r0 * nblk;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const u32 *src = (const u32 *)(base + k * npad + lane_off);
#pragma unroll
                    for (int q = 0; q < UC / 4; ++q) raw[k][q] = src[q];
                }
#pragma unroll
                for (int q = 0; q < 8 / G::JR; ++q) ex[q] = (ebase + q * G::JR * nblk)[ex_off];
            }
        } else if (!role_x) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int64_t r = r0 + kg * 8 + k;
                const bool in = r < r_end;
                load_raw<DT, UC>(raw[k], (const char *)dy + (in ? r : r_begin) * dy_stride * SIZE, o0 + UC * cg, in ? out_f : 0);
            }
        } else {
            const int j = i0 + UC * cg;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int64_t r = r0 + kg * 8 + k;
                const bool in = r < r_end && j < npad;
                const u32 *src = (const u32 *)(codes + (in ? r * npad + j : 0));
#pragma unroll
                for (int q = 0; q < UC / 4; ++q) raw[k][q] = in ? src[q] : 0u;
            }
#pragma unroll
            for (int q = 0; q < 8 / G::JR; ++q) {
                const int64_t r = r0 + ex_row + q * G::JR;
                ex[q] = r < r_end && ex_b < nblk ? exps[r * nblk + ex_b] : 8u;
            }
        }
    };
    auto stage = [&](uint16_t *buf, int64_t r0) {
        if (!role_x) {
            if (!SMALL && r0 + BK > r_end) {                 // (the rows before r0 of a step that was moved back)
                const int had = (int)(r0 + BK - r_end) - kg * 8;
#pragma unroll
                for (int k = 0; k < 8; ++k)
#pragma unroll
                    for (int q = 0; q < UC * SIZE / 4; ++q) raw[k][q] = k < had ? 0u : raw[k][q];
            }
            if (sums) {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    float v[UC];
                    unpack<DT, UC>(v, raw[k]);
#pragma unroll
                    for (int j = 0; j < UC; ++j) bias[j] += v[j];
                }
            }
#pragma unroll
            for (int j = 0; j < UC; ++j) {
                const int at = lds_at<BK>(UC * cg + j, kg);
                u32 w[P][4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if constexpr (DT == SN_BF16) {           // already bf16: two rows' halves into a word
                        w[0][k] = (j & 1) ? __builtin_amdgcn_perm(raw[2 * k + 1][j / 2], raw[2 * k][j / 2], 0x07060302u)
                                          : __builtin_amdgcn_perm(raw[2 * k + 1][j / 2], raw[2 * k][j / 2], 0x05040100u);
                    } else {
                        float a = element<DT>(raw[2 * k], j), b = element<DT>(raw[2 * k + 1], j);
#pragma unroll
                        for (int p = 0; p < P; ++p) {
                            w[p][k] = pack_bf16(a, b);
                            if (p + 1 < P) {                 // what the piece leaves is exact in fp32
                                a -= __uint_as_float(w[p][k] << 16);
                                b -= __uint_as_float(w[p][k] & 0xFFFF0000u);
                            }
                        }
                    }
                }
#pragma unroll
                for (int p = 0; p < P; ++p) *reinterpret_cast<uint4 *>(buf + p * G::kPlane + at) = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
            }
        } else {
            uint16_t *const bx = buf + P * G::kPlane;
            const int from = ((lane / G::kGroups) * G::JR) * G::kBlocks + (cg * UC) / 32;
            float step[8];
#pragma unroll
            for (int q = 0; q < 8 / G::JR; ++q) {
                const int held = __float_as_int(block_step(ex[q]));
#pragma unroll
                for (int k = 0; k < G::JR; ++k) step[q * G::JR + k] = __int_as_float(__builtin_amdgcn_ds_bpermute((from + k * G::kBlocks) * 4, held));
            }
#pragma unroll
            for (int j = 0; j < UC; ++j) {
                u32 w[4];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    w[k] = pack_bf16((float)(int8_t)(raw[2 * k][j / 4] >> (8 * (j & 3))) * step[2 * k],
                                     (float)(int8_t)(raw[2 * k + 1][j / 4] >> (8 * (j & 3))) * step[2 * k + 1]);
                *reinterpret_cast<uint4 *>(bx + lds_at<BK>(UC * cg + j, kg)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    };
    // operands of one group of 16 rows are read while the previous group multiplies (P = 1; more pieces: their products are long enough)
    constexpr int KK = BK / 16, AHEAD = P == 1 ? 2 : 1;
    auto multiply = [&](const uint16_t *buf) {
        const uint16_t *const bx = buf + P * G::kPlane;
        bf16x8 a[AHEAD][G::MT][P], b[AHEAD][G::NT];
        auto read = [&](int kk, int s) {
#pragma unroll
            for (int n = 0; n < G::NT; ++n) b[s][n] = *reinterpret_cast<const bf16x8 *>(bx + lds_at<BK>(wn + n * 32 + (lane & 31), 2 * kk + (lane >> 5)));
#pragma unroll
            for (int m = 0; m < G::MT; ++m)
#pragma unroll
                for (int p = 0; p < P; ++p)
                    a[s][m][p] = *reinterpret_cast<const bf16x8 *>(buf + p * G::kPlane + lds_at<BK>(wm + m * 32 + (lane & 31), 2 * kk + (lane >> 5)));
        };
        if constexpr (AHEAD == 2) read(0, 0);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            const int s = kk % AHEAD;
            if constexpr (AHEAD == 1) read(kk, 0);
            else if (kk + 1 < KK) read(kk + 1, (kk + 1) % AHEAD);
#pragma unroll
            for (int m = 0; m < G::MT; ++m)
#pragma unroll
                for (int p = 0; p < P; ++p)
#pragma unroll
                    for (int n = 0; n < G::NT; ++n) acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[s][m][p], b[s][n], acc[m][n], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);               // (or the compiler reads all groups at once and spills)
        }
    };

    // Turn t multiplies step t out of one buffer and stages step t + 1 into the other (the first turn only stages); one copy of each part
    // in the code: the kernel is small enough to be fetched in the time that a few steps take.  (Every split has rows.)
    fetch(r_begin);
    int cur = 1;
    for (int64_t r0 = r_begin - BK; r0 < r_end; r0 += BK, cur ^= 1) {
        uint16_t *const here = lds + cur * G::kBuffer, *const next = lds + (cur ^ 1) * G::kBuffer;
        const bool more = r0 + BK < r_end, after = r0 + 2 * BK < r_end;
        if (!role_x) {
            if (more) stage(next, r0 + BK);
            if (after) fetch(r0 + 2 * BK);
        }
        if (r0 >= r_begin) {
            if (role_x) __builtin_amdgcn_s_setprio(2);
            else __builtin_amdgcn_s_setprio(1);
            multiply(here);
            __builtin_amdgcn_s_setprio(0);
        }
        if (role_x) {
            if (more) stage(next, r0 + BK);
            if (after) fetch(r0 + 2 * BK);
        }
        __syncthreads();
    }

    // C of the 32x32 instruction: column lane & 31, row (i & 3) + 8 (i >> 2) + 4 (lane >> 5).  One run of stores for each place and type:
    // (a choice for every element was half of the kernel's code and, cold, a fifth of its time at 12544 rows of 256)
    auto write = [&](auto type, void *to) {
        constexpr int OT = decltype(type)::value;
#pragma unroll
        for (int n = 0; n < G::NT; ++n) {
            const int c = i0 + wn + n * 32 + (lane & 31);
            if (c < in_f) {
#pragma unroll
                for (int m = 0; m < G::MT; ++m) {
                    const int o = o0 + wm + m * 32 + 4 * (lane >> 5);
                    char *p = (char *)to + ((int64_t)o * in_f + c) * (OT == SN_F32 ? 4 : 2);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int r = (i & 3) + 8 * (i >> 2);
                        if (!SMALL || o + r < out_f) store_one<OT>(p + (int64_t)r * in_f * (OT == SN_F32 ? 4 : 2), 0, acc[m][n][i]);
                    }
                }
            }
        }
    };
    if (part_w || out_dtype == SN_F32) write(Type<SN_F32>(), part_w ? (void *)(part_w + (int64_t)split * out_f * in_f) : dw);
    else if (out_dtype == SN_BF16) write(Type<SN_BF16>(), dw);
    else write(Type<SN_F16>(), dw);
    if (sums) {                                              // (the last turn ended with a barrier: LDS is free)
        float *red = reinterpret_cast<float *>(lds);         // [BK / 8 row groups][TILE columns]
        if (!role_x) {
#pragma unroll
            for (int j = 0; j < UC; ++j) red[kg * TILE + UC * cg + j] = bias[j];
        }
        __syncthreads();
        if (t < TILE && o0 + t < out_f) {
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < BK / 8; ++k) s += red[k * TILE + t];
            if (part_b) part_b[(int64_t)split * out_f + o0 + t] = s;
            else store_any(db, out_dtype, o0 + t, s);
        }
    }
}

// the splits' partial results: 4 cells a thread, the splits dealt to four groups of threads, added in a fixed order.  The cells of
// dW and db lie behind one another (part_b = part_w + splits * cells of dW); a thread's four never span both.
__global__ __launch_bounds__(256) void weight_grad8_join_kernel(const float *part_w, const float *part_b, int splits, int64_t cells, int out_f, void *dw, void *db,
                                                                int out_dtype)
{
    __shared__ float4 red[4][64];
    const int q = threadIdx.x & 63, group = threadIdx.x >> 6;
    const int64_t quads = (cells + 3) / 4, i = (int64_t)blockIdx.x * 64 + q;
    const bool bias = i >= quads;
    const int64_t c = bias ? (i - quads) * 4 : i * 4, n = bias ? out_f : cells;
    const float *src = bias ? part_b : part_w;
    float s[4] = {};
    if (c < n && (!bias || db)) {
#pragma unroll 4
        for (int p = group; p < splits; p += 4) {
            u32 w[4];
            load_raw<SN_F32, 4>(w, src + p * n + c, 0, n - c < 4 ? (int)(n - c) : 4);
#pragma unroll
            for (int k = 0; k < 4; ++k) s[k] += __uint_as_float(w[k]);
        }
    }
    red[group][q] = make_float4(s[0], s[1], s[2], s[3]);
    __syncthreads();
    if (group == 0 && c < n && (!bias || db)) {
        const float4 a = red[1][q], b = red[2][q], d = red[3][q];
        const float v[4] = {(s[0] + a.x) + (b.x + d.x), (s[1] + a.y) + (b.y + d.y), (s[2] + a.z) + (b.z + d.z), (s[3] + a.w) + (b.w + d.w)};
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (c + k < n) store_any(bias ? db : dw, out_dtype, c + k, v[k]);
    }
}

int64_t tiles_of(int out_f, int in_f, int tile) { return (int64_t)((out_f + tile - 1) / tile) * ((in_f + tile - 1) / tile); }

// Tile and splits of the summed rows.  The large tile where at least 4 of them, times splits, give each of the 256 compute units one
// with 512 rows or more (32768 rows, bf16: 1024 x 1024 131 us on small tiles, 98 on large ones; 512 x 512 42.0, 41.6; 8192 rows of 512 x 1024
// 32.0, 37.4), the small one otherwise; then 512 small or 256 large workgroups (fewer leave units idle, more write partial sums: bf16,
// 1024 x 1024, 512 workgroups of the large tile 117 us, 128 of them 140), at least 256 rows a split.
// The rule comes from bf16, whose small workgroup takes 64 KB of LDS: two to a compute unit.  fp16's takes 96 KB and fp32's 128, one to a
// unit: their 512 run in two rounds and write twice the partial sums that 256 would (us with 256 | 512 small workgroups, joining included,
// bf16, fp16, fp32: 20000 rows of 512 -> 512 30.2 | 29.6, 39.1 | 43.3, 47.7 | 51.7; 8192 of 512 -> 1024 29.0 | 28.6, 35.5 | 39.1, 41.2 | 47.1;
// 32768 of 256 -> 256 22.2 | 26.0, 25.4 | 32.4, 28.1 | 36.6; 4999 of 387 -> 1000 22.3 | 25.2, 26.3 | 31.3, 29.8 | 34.9; 12544 of 256 -> 256
// 18.0 | 18.0, 19.8 | 19.6, 22.0 | 21.3).
struct Split { int tile, n, rows; bool small; };
Split split_rows(int64_t rows, int out_f, int in_f, int64_t dy_stride)
{
    Split s;
    const int npad = (in_f + 31) & ~31;
    s.small = rows < 64 || out_f < 128 || npad < 128 || dy_stride >= (1 << 22) || npad >= (1 << 22);
    const int64_t large = tiles_of(out_f, in_f, 256);
    s.tile = !s.small && out_f >= 256 && npad >= 256 && large >= 4 && rows * large >= 256 * 512 ? 256 : 128;
    const int64_t tiles = tiles_of(out_f, in_f, s.tile);
    int64_t n = (s.tile == 256 ? 256 : 512) / tiles;
    const int64_t most = (rows + 255) / 256;
    n = n > most ? most : n;
    n = n < 1 ? 1 : n;
    int64_t per = (rows + n - 1) / n;
    per = (per + 63) / 64 * 64;
    s.rows = (int)(per < 64 ? 64 : per);
    s.n = rows ? (int)((rows + s.rows - 1) / s.rows) : 1;
    return s;
}

template <int DT, int TILE, bool SMALL>
int launch_tile(const Split &sp, const void *dy, int64_t dy_stride, const void *codes, const void *exps, int64_t rows, int out_f, int in_f, void *dw, void *db,
                int out_dtype, float *part_w, float *part_b, hipStream_t st)
{
    using G = Grad<DT, TILE>;
    const size_t lds = (size_t)2 * G::kBuffer * 2;
    const int rc = sn_ensure_dynamic_lds((const void *)weight_grad8_kernel<DT, TILE, SMALL>, lds, "sn_checkpoint8_weight_grad");
    if (rc != SN_OK) return rc;
    hipLaunchKernelGGL((weight_grad8_kernel<DT, TILE, SMALL>), dim3((unsigned)(tiles_of(out_f, in_f, TILE) * sp.n)), dim3(G::kThreads), lds, st, dy, dy_stride,
                       (const uint8_t *)codes, (const uint8_t *)exps, rows, out_f, in_f, sp.n, sp.rows, dw, db, out_dtype, part_w, part_b);
    SN_CHECK_LAUNCH("sn_checkpoint8_weight_grad");
    return SN_OK;
}

template <int DT>
int launch_grad(const void *dy, int64_t dy_stride, const void *codes, const void *exps, int64_t rows, int out_f, int in_f, void *dw, void *db, int out_dtype,
                void *workspace, hipStream_t st)
{
    const Split sp = split_rows(rows, out_f, in_f, dy_stride);
    const int64_t cells = (int64_t)out_f * in_f;
    float *part_w = sp.n > 1 ? (float *)workspace : nullptr, *part_b = sp.n > 1 ? part_w + sp.n * cells : nullptr;
    const auto launch = sp.small ? launch_tile<DT, 128, true> : sp.tile == 256 ? launch_tile<DT, 256, false> : launch_tile<DT, 128, false>;
    const int rc = launch(sp, dy, dy_stride, codes, exps, rows, out_f, in_f, dw, db, out_dtype, part_w, part_b, st);
    if (rc != SN_OK || sp.n == 1) return rc;
    const int64_t quads = (cells + 3) / 4 + (db ? (out_f + 3) / 4 : 0);
    hipLaunchKernelGGL(weight_grad8_join_kernel, dim3((unsigned)((quads + 63) / 64)), dim3(256), 0, st, part_w, part_b, sp.n, cells, out_f, dw, db, out_dtype);
    SN_CHECK_LAUNCH("sn_checkpoint8_weight_grad (join)");
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
    const int ev = dtype == SN_F32 ? 4 : 8;
    const dim3 grid(pack_blocks(rows * (((int64_t)n + ev - 1) / ev))), block(kPackThreads);
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == SN_F32) hipLaunchKernelGGL(restore8_kernel<SN_F32>, grid, block, 0, st, (const uint8_t *)codes, (const uint8_t *)exps, rows, n, out);
    else if (dtype == SN_BF16) hipLaunchKernelGGL(restore8_kernel<SN_BF16>, grid, block, 0, st, (const uint8_t *)codes, (const uint8_t *)exps, rows, n, out);
    else hipLaunchKernelGGL(restore8_kernel<SN_F16>, grid, block, 0, st, (const uint8_t *)codes, (const uint8_t *)exps, rows, n, out);
    SN_CHECK_LAUNCH("sn_checkpoint8_restore");
    return SN_OK;
}

extern "C" size_t sn_checkpoint8_weight_grad_workspace(int64_t rows, int out_features, int in_features, int dy_dtype)
{
    if (rows < 0 || rows > kMostRows || out_features < 1 || out_features > kMostSide || in_features < 1 || in_features > kMostSide || dy_dtype < 0 || dy_dtype > 2) return 0;
    // (the stride of dy decides between two splits: room for either)
    const int n = split_rows(rows, out_features, in_features, out_features).n, far = split_rows(rows, out_features, in_features, 1 << 22).n;
    const int most = n > far ? n : far;
    return most > 1 ? (size_t)most * ((size_t)out_features * in_features + out_features) * sizeof(float) : 16;
}

extern "C" int sn_checkpoint8_weight_grad(const void *dy, int dy_dtype, int64_t dy_row_stride, const void *codes, const void *exps, int64_t rows, int out_features,
                                          int in_features, void *dw, void *db, int out_dtype, void *workspace, size_t workspace_bytes, void *stream)
{
    SN_REQUIRE(rows > 0 && out_features >= 1 && in_features >= 1, SN_ERR_BAD_ARG, "sn_checkpoint8_weight_grad: bad rows=%lld out=%d in=%d", (long long)rows,
               out_features, in_features);
    SN_REQUIRE(dy_dtype >= 0 && dy_dtype <= 2 && out_dtype >= 0 && out_dtype <= 2, SN_ERR_BAD_ARG, "sn_checkpoint8_weight_grad: unknown type");
    SN_REQUIRE(out_features <= kMostSide && in_features <= kMostSide && rows <= kMostRows, SN_ERR_UNSUPPORTED, "sn_checkpoint8_weight_grad: too large");
    SN_REQUIRE(dy && codes && exps && dw, SN_ERR_BAD_ARG, "sn_checkpoint8_weight_grad: NULL pointer");
    SN_REQUIRE(workspace && workspace_bytes >= sn_checkpoint8_weight_grad_workspace(rows, out_features, in_features, dy_dtype), SN_ERR_WORKSPACE,
               "sn_checkpoint8_weight_grad: workspace of %zu bytes", workspace_bytes);
    const hipStream_t st = (hipStream_t)stream;
    if (dy_dtype == SN_F32) return launch_grad<SN_F32>(dy, dy_row_stride, codes, exps, rows, out_features, in_features, dw, db, out_dtype, workspace, st);
    if (dy_dtype == SN_BF16) return launch_grad<SN_BF16>(dy, dy_row_stride, codes, exps, rows, out_features, in_features, dw, db, out_dtype, workspace, st);
    return launch_grad<SN_F16>(dy, dy_row_stride, codes, exps, rows, out_features, in_features, dw, db, out_dtype, workspace, st);
}
