// Log probabilities of given tokens, with entropy and the top alternatives (schemanet_blocks.h).
//     d_j = x_j - max x;  s = sum exp(d);  t = sum exp(d) d;   log p_j = d_j - log s;   H = log s - t / s
//     grad_j = g (delta_jt - p_j) - g_H p_j (log p_j + H)
// Bound: HBM - forward reads the logits once (running max, s and t per lane, joined at the end; the top list is kept beside
// them), backward reads them once and writes the gradient.  A row belongs to one wave (up to kWaveRow entries), to the four
// waves of a workgroup, or - few rows - to up to 64 workgroups whose partial results a second launch joins.
//
// Top list: a wave keeps its k best (value, index) sorted across its lanes, lane j the j-th.  A group of elements is looked at
// again only if one of them beats the k-th; an insertion is one ballot (its place) and one shift by a lane.  Order: larger value
// first, lower index among equals.  Lists are joined in pairs: an element's place in the join is its own plus the number of
// the partner's that come before it (binary search).
#include "sn_typed.h"

namespace {

using namespace sn;

constexpr int kScoreThreads = 256, kScoreWaves = 4;
constexpr int64_t kWaveRow = 2048;       // entries of a row that one wave takes
constexpr int kMaxSplits = 64;
constexpr float kLog2e = 1.44269504088896340736f;
// stands for any distance beyond it where it is multiplied by exp(d): exp(-10^4) = 0 in fp32, and 0 times an infinite d must stay 0
constexpr float kFar = -1.0e4f;
constexpr int kNone = 0x7FFFFFFF;

struct Soft { float m, s, t; };

// exp(d) for d <= 0 from the hardware's 2^x
__device__ __forceinline__ float exp_fast(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

// two partial sums of one row; an empty one has m = -inf, s = t = 0.  NaN in s stays.
__device__ __forceinline__ Soft join(Soft a, Soft b)
{
    Soft r;
    r.m = fmaxf(a.m, b.m);
    const float base = r.m == -INFINITY ? 0.0f : r.m;
    const float da = a.m - base, db = b.m - base, fa = exp_fast(da), fb = exp_fast(db);
    r.s = a.s * fa + b.s * fb;
    r.t = (a.t + a.s * fmaxf(da, kFar)) * fa + (b.t + b.s * fmaxf(db, kFar)) * fb;
    return r;
}
__device__ __forceinline__ Soft wave_join(Soft a)
{
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        Soft b;
        b.m = __shfl_xor(a.m, off, 64);
        b.s = __shfl_xor(a.s, off, 64);
        b.t = __shfl_xor(a.t, off, 64);
        // the same order on both sides: every lane ends with the same bits
        a = (threadIdx.x & off) ? join(b, a) : join(a, b);
    }
    return a;
}

__device__ __forceinline__ bool before(float va, int ia, float vb, int ib) { return va > vb || (va == vb && ia < ib); }

// sorted list of a wave
struct TopList {
    float v;
    int i;
    float last_v;         // the k-th entry, in every lane
    int last_i;
    __device__ __forceinline__ void reset() { v = -INFINITY; i = kNone; last_v = -INFINITY; last_i = kNone; }
    // (nv, ni): the same in every lane, before the k-th entry
    __device__ __forceinline__ void insert(float nv, int ni, int k)
    {
        const int lane = threadIdx.x & 63;
        const int pos = __popcll(__ballot(before(v, i, nv, ni)));
        const float up_v = __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x138, 0xF, 0xF, false));     // wave_shr:1
        const int up_i = __builtin_amdgcn_update_dpp(0, i, 0x138, 0xF, 0xF, false);
        v = lane > pos ? up_v : lane == pos ? nv : v;
        i = lane > pos ? up_i : lane == pos ? ni : i;
        last_v = SN_READLANE_F32(v, k - 1);
        last_i = __builtin_amdgcn_readlane(i, k - 1);
    }
    __device__ __forceinline__ void offer(float x, int ix, int k)
    {
        uint64_t b = __ballot(before(x, ix, last_v, last_i));
        while (b) {
            const int l = __builtin_ctzll(b);
            const float nv = SN_READLANE_F32(x, l);
            const int ni = __builtin_amdgcn_readlane(ix, l);
            insert(nv, ni, k);
            b = __ballot(before(x, ix, last_v, last_i) && (threadIdx.x & 63) > l);
        }
    }
};

// the wave's share (segments w, w + nw, ...) of entries c0 .. c1 - 1 of a row
template <int DT, bool TOP>
__device__ __forceinline__ void scan(const void *row, int64_t c0, int64_t c1, int w, int nw, Soft &soft, TopList &top, int k)
{
    constexpr int EV = DT == SN_F32 ? 4 : 8, PER = 2, SEG = 64 * EV * PER;
    const int lane = threadIdx.x & 63;
    const char *base = (const char *)row + c0 * (DT == SN_F32 ? 4 : 2);
    const int n = (int)(c1 - c0);
    const uint32_t fill = DT == SN_F32 ? 0xFF800000u : DT == SN_BF16 ? 0xFF80u : 0xFC00u;      // -inf
    for (int s0 = w * SEG; s0 < n; s0 += nw * SEG) {
        float x[PER][EV];
#pragma unroll
        for (int c = 0; c < PER; ++c) {
            uint32_t raw[words<DT, EV>()];
            load_raw<DT, EV>(raw, base, s0 + (c * 64 + lane) * EV, n, fill);
            unpack<DT, EV>(x[c], raw);
        }
        float m = x[0][0];
#pragma unroll
        for (int c = 0; c < PER; ++c)
#pragma unroll
            for (int e = 0; e < EV; ++e) m = fmaxf(m, x[c][e]);
        const float mx = fmaxf(m, soft.m);
        if (mx > soft.m) {
            const float d = soft.m - mx, f = exp_fast(d);
            soft.t = (soft.t + soft.s * fmaxf(d, kFar)) * f;
            soft.s *= f;
            soft.m = mx;
        }
        const float ref = soft.m == -INFINITY ? 0.0f : soft.m;
#pragma unroll
        for (int c = 0; c < PER; ++c)
#pragma unroll
            for (int e = 0; e < EV; ++e) {
                const float d = x[c][e] - ref, p = exp_fast(d);
                soft.s += p;
                soft.t = fmaf(p, fmaxf(d, kFar), soft.t);
            }
        if constexpr (TOP) {
            if (__any(m > top.last_v) || top.last_i == kNone) {
#pragma unroll
                for (int c = 0; c < PER; ++c)
#pragma unroll
                    for (int e = 0; e < EV; ++e) {
                        const int j = s0 + (c * 64 + lane) * EV + e;
                        top.offer(j < n ? x[c][e] : -INFINITY, j < n ? (int)c0 + j : kNone, k);
                    }
            }
        }
    }
}

struct ScoreArgs {
    const void *logits;
    int64_t rows, n, stride;
    const int64_t *target;
    int64_t ignore;
    int k, splits;
    int64_t per_split;
    float *log_probs, *entropy, *stats, *top_lp;
    int64_t *top_ids;
    float *part;          // [rows, splits, 3 + 2 k]: m, s, t, values, indexes
};

template <int DT> __device__ __forceinline__ void write_row(const ScoreArgs &a, int64_t row, Soft s)
{
    const float ls = logf(s.s);
    const float h = s.s == 0.0f ? 0.0f : ls - s.t / s.s;
    const int64_t tg = a.target[row];
    float lp = 0.0f;
    if (tg != a.ignore) {
        if (tg < 0 || tg >= a.n) lp = __uint_as_float(0x7FC00000u);
        else lp = s.s == 0.0f ? -INFINITY : (load_one<DT>((const char *)a.logits + row * a.stride * (DT == SN_F32 ? 4 : 2), tg) - s.m) - ls;
    }
    a.log_probs[row] = lp;
    a.entropy[row] = h;
    a.stats[row * 3] = s.m;
    a.stats[row * 3 + 1] = s.s;
    a.stats[row * 3 + 2] = h;
}
__device__ __forceinline__ void write_top(const ScoreArgs &a, int64_t row, int j, float v, int i, Soft s)
{
    const float ls = logf(s.s);
    a.top_lp[row * a.k + j] = s.s == 0.0f ? -INFINITY : i == kNone ? __uint_as_float(0x7FC00000u) : (v - s.m) - ls;
    a.top_ids[row * a.k + j] = i == kNone ? -1 : i;
}

// `lists` sorted lists of k in src -> one, in pairs; both buffers hold lists * k entries.  Every thread of the workgroup calls.
// -> the buffer that holds the result
struct Entry { float v; int i; };
__device__ Entry *join_lists(Entry *src, Entry *dst, int lists, int k)
{
    while (lists > 1) {
        const int total = lists * k;
        for (int e = threadIdx.x; e < total; e += blockDim.x) {
            const int l = e / k, j = e - l * k;
            const Entry me = src[e];
            int pos = j;
            if ((l ^ 1) < lists) {
                const Entry *o = src + (l ^ 1) * k;
                int lo = 0, hi = k;                          // how many of the partner's come before this one
                while (lo < hi) {
                    const int mid = (lo + hi) >> 1;
                    // (entries that were never filled are equal: those of the lower list first)
                    const bool b = before(o[mid].v, o[mid].i, me.v, me.i) || (o[mid].v == me.v && o[mid].i == me.i && (l & 1));
                    if (b) lo = mid + 1; else hi = mid;
                }
                pos += lo;
            }
            if (pos < k) dst[(l >> 1) * k + pos] = me;
        }
        __syncthreads();
        Entry *const swap = src;
        src = dst;
        dst = swap;
        lists = (lists + 1) >> 1;
    }
    return src;
}

// one wave a row
template <int DT, bool TOP>
__global__ __launch_bounds__(kScoreThreads) void scores_wave_kernel(ScoreArgs a)
{
    const int lane = threadIdx.x & 63;
    const int64_t turn = (int64_t)gridDim.x * kScoreWaves;
    for (int64_t row = (int64_t)blockIdx.x * kScoreWaves + (threadIdx.x >> 6); row < a.rows; row += turn) {
        Soft soft = {-INFINITY, 0.0f, 0.0f};
        TopList top;
        top.reset();
        scan<DT, TOP>((const char *)a.logits + row * a.stride * (DT == SN_F32 ? 4 : 2), 0, a.n, 0, 1, soft, top, a.k);
        soft = wave_join(soft);
        if (lane == 0) write_row<DT>(a, row, soft);
        if (TOP && lane < a.k) write_top(a, row, lane, top.v, top.i, soft);
    }
}

// four waves a row or a split of one
template <int DT, bool TOP>
__global__ __launch_bounds__(kScoreThreads) void scores_group_kernel(ScoreArgs a)
{
    __shared__ Soft part[kScoreWaves];
    __shared__ Entry lists[2][TOP ? kScoreWaves * SN_SCORES_MAX_TOP : 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = blockIdx.x / a.splits;
    const int split = (int)(blockIdx.x - row * a.splits);
    const int64_t c0 = split * a.per_split, c1 = c0 + a.per_split < a.n ? c0 + a.per_split : a.n;
    Soft soft = {-INFINITY, 0.0f, 0.0f};
    TopList top;
    top.reset();
    if (c0 < c1) scan<DT, TOP>((const char *)a.logits + row * a.stride * (DT == SN_F32 ? 4 : 2), c0, c1, wave, kScoreWaves, soft, top, a.k);
    soft = wave_join(soft);
    if (lane == 0) part[wave] = soft;
    if (TOP && lane < a.k) lists[0][wave * a.k + lane] = Entry{top.v, top.i};
    __syncthreads();
    soft = join(join(part[0], part[1]), join(part[2], part[3]));
    const Entry *best = nullptr;
    if constexpr (TOP) best = join_lists(lists[0], lists[1], kScoreWaves, a.k);
    if (a.splits == 1) {
        if (threadIdx.x == 0) write_row<DT>(a, row, soft);
        if (TOP && (int)threadIdx.x < a.k) write_top(a, row, threadIdx.x, best[threadIdx.x].v, best[threadIdx.x].i, soft);
    } else {
        float *dst = a.part + (row * a.splits + split) * (3 + 2 * a.k);
        if (threadIdx.x == 0) { dst[0] = soft.m; dst[1] = soft.s; dst[2] = soft.t; }
        if (TOP && (int)threadIdx.x < a.k) {
            dst[3 + threadIdx.x] = best[threadIdx.x].v;
            dst[3 + a.k + threadIdx.x] = __int_as_float(best[threadIdx.x].i);
        }
    }
}

// the splits of a row, one workgroup a row; two buffers of splits * k entries in LDS
template <int DT, bool TOP>
__global__ __launch_bounds__(kScoreThreads) void scores_join_kernel(ScoreArgs a)
{
    extern __shared__ Entry buffers[];
    __shared__ Soft all;
    const int64_t row = blockIdx.x;
    const float *src = a.part + row * a.splits * (3 + 2 * a.k);
    if (threadIdx.x < 64) {
        Soft s = {-INFINITY, 0.0f, 0.0f};
        if ((int)threadIdx.x < a.splits) {
            const float *p = src + threadIdx.x * (3 + 2 * a.k);
            s = Soft{p[0], p[1], p[2]};
        }
        s = wave_join(s);
        if (threadIdx.x == 0) { all = s; write_row<DT>(a, row, s); }
    }
    if constexpr (TOP) {
        for (int e = threadIdx.x; e < a.splits * a.k; e += kScoreThreads) {
            const int l = e / a.k, j = e - l * a.k;
            const float *p = src + l * (3 + 2 * a.k) + 3;
            buffers[e] = Entry{p[j], __float_as_int(p[a.k + j])};
        }
        __syncthreads();
        const Entry *best = join_lists(buffers, buffers + a.splits * a.k, a.splits, a.k);
        if ((int)threadIdx.x < a.k) write_top(a, row, threadIdx.x, best[threadIdx.x].v, best[threadIdx.x].i, all);
    }
}

// ------------------------------------------------------------------------------------------ backward
struct ScoreGradArgs {
    const void *logits;
    int64_t rows, n, stride;
    const int64_t *target;
    int64_t ignore;
    const float *stats, *g_lp, *g_h;
    void *grad;
};

template <int DT>
__global__ __launch_bounds__(kScoreThreads) void scores_backward_kernel(ScoreGradArgs a, int64_t pieces, int64_t per_piece)
{
    constexpr int EV = DT == SN_F32 ? 4 : 8, SIZE = DT == SN_F32 ? 4 : 2;
    const int64_t row = blockIdx.x / pieces, c0 = (blockIdx.x - row * pieces) * per_piece;
    const int n = (int)(c0 + per_piece < a.n ? per_piece : a.n - c0);
    const float m = a.stats[row * 3], s = a.stats[row * 3 + 1], h = a.stats[row * 3 + 2];
    const int64_t tg = a.target[row];
    const bool used = tg != a.ignore;
    const float g = used && a.g_lp ? a.g_lp[row] : 0.0f, gh = a.g_h ? a.g_h[row] : 0.0f;
    const char *src = (const char *)a.logits + (row * a.stride + c0) * SIZE;
    char *dst = (char *)a.grad + (row * a.n + c0) * SIZE;
    const bool none = s == 0.0f;                             // a row without a distribution
    const bool wrong = used && (tg < 0 || tg >= a.n);
    const float ls = logf(s), inv = 1.0f / s;
    const int at = used && !wrong && tg >= c0 && tg < c0 + n ? (int)(tg - c0) : -1;
    for (int j = threadIdx.x * EV; j < n; j += kScoreThreads * EV) {
        uint32_t raw[words<DT, EV>()];
        float x[EV];
        load_raw<DT, EV>(raw, src, j, n);
        unpack<DT, EV>(x, raw);
#pragma unroll
        for (int e = 0; e < EV; ++e) {
            const float d = x[e] - m;
            float p = __builtin_amdgcn_exp2f(d * kLog2e);
            if constexpr (DT == SN_F32) {
                // the product's rounding error and log2 e's own, as a first-order factor: 2^-24 |d| would show in 32-bit gradients
                const float hi = d * kLog2e;
                const float lo = fmaf(d, kLog2e, -hi) + d * 1.92596299112661746887e-8f;
                p = d > -100.0f ? fmaf(p, lo * 0.693147180559945309f, p) : p;
            }
            p *= inv;
            const float lg = fmaxf(d - ls, kFar);
            x[e] = -p * fmaf(gh, lg + h, g);
            if (j + e == at) x[e] += g;
            if (none) x[e] = 0.0f;
            if (wrong) x[e] = __uint_as_float(0x7FC00000u);
        }
        store_row<DT, EV>(dst, j, n, x);
    }
}

int splits_for(int64_t rows, int64_t n)
{
    if (n <= kWaveRow || rows <= 0) return 1;
    int64_t s = 1024 / rows;                                 // four workgroups for each compute unit
    const int64_t most = (n + 4095) / 4096;
    s = s > most ? most : s;
    s = s > kMaxSplits ? kMaxSplits : s;
    return (int)(s < 1 ? 1 : s);
}

template <int DT, bool TOP> int launch_scores(ScoreArgs &a, hipStream_t st)
{
    if (a.n <= kWaveRow) {
        const int64_t blocks = (a.rows + kScoreWaves - 1) / kScoreWaves;
        hipLaunchKernelGGL((scores_wave_kernel<DT, TOP>), dim3((unsigned)(blocks < 16384 ? blocks : 16384)), dim3(kScoreThreads), 0, st, a);
        SN_CHECK_LAUNCH("sn_label_log_probs");
        return SN_OK;
    }
    hipLaunchKernelGGL((scores_group_kernel<DT, TOP>), dim3((unsigned)(a.rows * a.splits)), dim3(kScoreThreads), 0, st, a);
    SN_CHECK_LAUNCH("sn_label_log_probs");
    if (a.splits > 1) {
        const size_t lds = TOP ? (size_t)2 * a.splits * a.k * sizeof(Entry) : 0;
        const int rc = sn_ensure_dynamic_lds((const void *)scores_join_kernel<DT, TOP>, lds, "sn_label_log_probs");
        if (rc != SN_OK) return rc;
        hipLaunchKernelGGL((scores_join_kernel<DT, TOP>), dim3((unsigned)a.rows), dim3(kScoreThreads), lds, st, a);
        SN_CHECK_LAUNCH("sn_label_log_probs (join)");
    }
    return SN_OK;
}

int check_scores(const char *who, const void *logits, int dtype, int64_t rows, int64_t n, const int64_t *target)
{
    SN_REQUIRE(rows >= 0 && n >= 1 && dtype >= 0 && dtype <= 2, SN_ERR_BAD_ARG, "%s: bad rows=%lld n=%lld type=%d", who, (long long)rows, (long long)n, dtype);
    SN_REQUIRE(rows < (1ll << 24) && n < (1ll << 30), SN_ERR_UNSUPPORTED, "%s: rows under 2^24 and entries under 2^30", who);
    SN_REQUIRE(rows == 0 || (logits && target), SN_ERR_BAD_ARG, "%s: NULL pointer", who);
    return SN_OK;
}

}  // namespace

extern "C" size_t sn_label_log_probs_workspace(int64_t rows, int64_t n, int k)
{
    if (rows < 0 || n < 1 || k < 0 || k > SN_SCORES_MAX_TOP) return 0;
    const int s = splits_for(rows, n);
    return s > 1 ? (size_t)rows * s * (3 + 2 * k) * sizeof(float) : 16;
}

extern "C" int sn_label_log_probs(const void *logits, int dtype, int64_t rows, int64_t n, int64_t row_stride, const int64_t *target, int64_t ignore_index, int k,
                                  float *log_probs, float *entropy, float *stats, float *top_log_probs, int64_t *top_ids, void *workspace, size_t workspace_bytes,
                                  void *stream)
{
    const int rc = check_scores("sn_label_log_probs", logits, dtype, rows, n, target);
    if (rc != SN_OK) return rc;
    SN_REQUIRE(k >= 0 && k <= SN_SCORES_MAX_TOP && k <= n, SN_ERR_BAD_ARG, "sn_label_log_probs: %d alternatives of %lld entries (at most %d)", k, (long long)n,
               SN_SCORES_MAX_TOP);
    if (rows == 0) return SN_OK;
    SN_REQUIRE(log_probs && entropy && stats && (k == 0 || (top_log_probs && top_ids)), SN_ERR_BAD_ARG, "sn_label_log_probs: NULL pointer");
    SN_REQUIRE(workspace && workspace_bytes >= sn_label_log_probs_workspace(rows, n, k), SN_ERR_WORKSPACE, "sn_label_log_probs: workspace of %zu bytes", workspace_bytes);
    ScoreArgs a = {logits, rows, n, row_stride, target, ignore_index, k, splits_for(rows, n), 0, log_probs, entropy, stats, top_log_probs, top_ids, (float *)workspace};
    a.per_split = ((n + a.splits - 1) / a.splits + 7) / 8 * 8;
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == SN_F32) return k ? launch_scores<SN_F32, true>(a, st) : launch_scores<SN_F32, false>(a, st);
    if (dtype == SN_BF16) return k ? launch_scores<SN_BF16, true>(a, st) : launch_scores<SN_BF16, false>(a, st);
    return k ? launch_scores<SN_F16, true>(a, st) : launch_scores<SN_F16, false>(a, st);
}

extern "C" int sn_label_log_probs_backward(const void *logits, int dtype, int64_t rows, int64_t n, int64_t row_stride, const int64_t *target, int64_t ignore_index,
                                           const float *stats, const float *g_log_probs, const float *g_entropy, void *grad, void *stream)
{
    const int rc = check_scores("sn_label_log_probs_backward", logits, dtype, rows, n, target);
    if (rc != SN_OK) return rc;
    if (rows == 0) return SN_OK;
    SN_REQUIRE(stats && grad && (g_log_probs || g_entropy), SN_ERR_BAD_ARG, "sn_label_log_probs_backward: NULL pointer");
    const ScoreGradArgs a = {logits, rows, n, row_stride, target, ignore_index, stats, g_log_probs, g_entropy, grad};
    const int64_t per = 8192, pieces = (n + per - 1) / per;
    SN_REQUIRE(rows * pieces < (1ll << 31), SN_ERR_UNSUPPORTED, "sn_label_log_probs_backward: too large");
    const dim3 grid((unsigned)(rows * pieces)), block(kScoreThreads);
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == SN_F32) hipLaunchKernelGGL(scores_backward_kernel<SN_F32>, grid, block, 0, st, a, pieces, per);
    else if (dtype == SN_BF16) hipLaunchKernelGGL(scores_backward_kernel<SN_BF16>, grid, block, 0, st, a, pieces, per);
    else hipLaunchKernelGGL(scores_backward_kernel<SN_F16>, grid, block, 0, st, a, pieces, per);
    SN_CHECK_LAUNCH("sn_label_log_probs_backward");
    return SN_OK;
}
