// Log probabilities of given tokens, with entropy and the top alternatives (schemanet_blocks.h).
//     d_j = x_j - max x;  s = sum exp(d);  t = sum exp(d) d;   log p_j = d_j - log s;   H = log s - t / s
//     grad_j = g (delta_jt - p_j) - g_H p_j (log p_j + H)
// Bound: HBM - forward reads the logits once (running max, s and t per lane, joined at the end; the top list is kept beside
// them), backward reads them once and writes the gradient.  A row belongs to one wave, to the four
// waves of a workgroup, or - few rows - to up to 64 workgroups whose partial results a second launch joins.
// Measured (the card copies at 5.13 TB/s): 4096 rows of 32769, bf16: forward and backward pass 82 + 85 us of kernels (805 MB, 4.8 TB/s);
// 16 rows of 131072, bf16, 20 alternatives: 10.6 + 5.8 us; one row of 1000, fp32, 5 alternatives: 5.3 us (3.4 without them): latency.
//
// Top list: a wave keeps its k best (value, index) sorted across its lanes, lane j the j-th.  A group of 1024 elements is looked at again
// only if one of them beats the k-th: a few candidates are inserted one by one (one ballot for the place, one shift by a lane),
// more are gathered, sorted and merged at once (absorb).  Order: larger value first, lower index among equals, as one 64-bit
// number.
#include "sn_typed.h"

namespace {

using namespace sn;

constexpr int kScoreThreads = 256, kScoreWaves = 4;
constexpr int kMaxSplits = 64;
constexpr float kLog2e = 1.44269504088896340736f;
// stands for any distance beyond it where it is multiplied by exp(d): exp(-10^4) = 0 in fp32, and 0 times an infinite d must stay 0
constexpr float kFar = -1.0e4f;
constexpr float kLowest = -3.402823466e38f;

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

// An entry as one number that orders like (value, then the lower index): the value's bits turned so that they order as an unsigned
// number, over the index's complement.  -0 counts as 0.  kNone: an entry that was never filled; no logit at -inf enters a list.
typedef uint64_t Key;
constexpr Key kNone = 0x007FFFFF00000000ull;                 // (-inf, -1)
__device__ __forceinline__ Key key_of(float v, int i)
{
    const uint32_t b = __float_as_uint(v + 0.0f);
    return ((Key)(b ^ ((uint32_t)((int)b >> 31) | 0x80000000u)) << 32) | (uint32_t)~i;
}
__device__ __forceinline__ float key_value(Key k)
{
    const uint32_t b = (uint32_t)(k >> 32);
    return __uint_as_float(b ^ ((uint32_t)((int)~b >> 31) | 0x80000000u));
}
__device__ __forceinline__ int key_index(Key k) { return (int)~(uint32_t)k; }
__device__ __forceinline__ Key lane_key(Key k, int lane)
{
    return ((Key)(uint32_t)__builtin_amdgcn_readlane((int)(k >> 32), lane) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)k, lane);
}

// value of lane ^ STRIDE without LDS: quad permutations, mirrors and rotations of 16 lanes, swaps of 16 and 32
template <int STRIDE> __device__ __forceinline__ uint32_t lane_xor(uint32_t v)
{
    if constexpr (STRIDE == 1) return SN_DPP_U32(v, 0xB1);
    else if constexpr (STRIDE == 2) return SN_DPP_U32(v, 0x4E);
    else if constexpr (STRIDE == 4) return SN_DPP_U32(SN_DPP_U32(v, 0x1B), 0x141);      // 3 - i in the quad, then 7 - i in the half row
    else if constexpr (STRIDE == 8) return SN_DPP_U32(v, 0x128);                        // row_ror:8
    else if constexpr (STRIDE == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return (threadIdx.x & 16) ? r[0] : r[1];
    } else {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return (threadIdx.x & 32) ? r[0] : r[1];
    }
}
__device__ __forceinline__ float other_lane(float v, float o, bool first) { return first ? fmaxf(v, o) : fminf(v, o); }
__device__ __forceinline__ Key other_lane(Key v, Key o, bool first) { return (o > v) == first ? o : v; }
template <int STRIDE> __device__ __forceinline__ float lane_xor(float v) { return __uint_as_float(lane_xor<STRIDE>(__float_as_uint(v))); }
template <int STRIDE> __device__ __forceinline__ Key lane_xor(Key v)
{
    return ((Key)lane_xor<STRIDE>((uint32_t)(v >> 32)) << 32) | lane_xor<STRIDE>((uint32_t)v);
}
template <int SIZE, int STRIDE, class T> __device__ __forceinline__ void sort_merge(T &v, int lane)
{
    // the lower lane of a pair keeps the larger one in the blocks that are sorted downwards
    const bool first = ((lane & STRIDE) == 0) == ((lane & SIZE) == 0 || SIZE == 64);
    v = other_lane(v, lane_xor<STRIDE>(v), first);
    if constexpr (STRIDE > 1) sort_merge<SIZE, STRIDE / 2>(v, lane);
}
// the wave's 64 numbers (no NaN) in order, lane 0 the largest: bitonic
template <class T> __device__ __forceinline__ void wave_sort(T &v)
{
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));           // (the 21 lane masks are made here, not kept in scalar registers over the caller's loop)
    sort_merge<2, 1>(v, lane);
    sort_merge<4, 2>(v, lane);
    sort_merge<8, 4>(v, lane);
    sort_merge<16, 8>(v, lane);
    sort_merge<32, 16>(v, lane);
    sort_merge<64, 32>(v, lane);
}

// sorted list of a wave
struct TopList {
    Key key, last;        // this lane's entry; the k-th entry, in every lane
    float last_v;
    __device__ __forceinline__ void reset() { key = last = kNone; last_v = -INFINITY; }
    __device__ __forceinline__ void set_last(int k)
    {
        last = lane_key(key, k - 1);
        last_v = key_value(last);
    }
    // n: the same in every lane, before the k-th entry
    __device__ __forceinline__ void insert(Key n, int k)
    {
        const int lane = threadIdx.x & 63;
        const int pos = __popcll(__ballot(key > n));
        const uint32_t up_hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(key >> 32), 0x138, 0xF, 0xF, false);        // wave_shr:1
        const uint32_t up_lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)key, 0x138, 0xF, 0xF, false);
        key = lane > pos ? ((Key)up_hi << 32) | up_lo : lane == pos ? n : key;
        set_last(k);
    }
    __device__ __forceinline__ void offer(float x, int i, int k)
    {
        const Key mine = key_of(x, i);
        uint64_t b = __ballot(x >= last_v && mine > last && x > -INFINITY);      // (NaN: not)
        while (b) {
            const int l = __builtin_ctzll(b);
            insert(lane_key(mine, l), k);
            b &= b - 1;
            b &= __ballot(mine > last);
        }
    }
};

__device__ __forceinline__ uint32_t ordered(float v)
{
    const uint32_t b = __float_as_uint(v);
    return b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t o) { return __uint_as_float(o ^ ((uint32_t)((int)~o >> 31) | 0x80000000u)); }
__device__ __forceinline__ int lanes_below(uint64_t m) { return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0)); }
template <int N> __device__ __forceinline__ int count_from(const float (&x)[N], float bound)
{
    int count = 0;
#pragma unroll
    for (int u = 0; u < N; ++u) count += __popcll(__ballot(x[u] >= bound));
    return count;
}

// The list's new state after N elements a lane (x, their indexes index(u), all behind those it has seen).  Candidates are the elements from
// a bound on: what lies above the last entry of a full list; until it is full, the k-th largest of the 64 lanes' maxima (at least k
// elements reach it) or, with fewer lanes above -inf, all elements there.  More than 64 of them: the bound is raised by bisection over the values' bits to the largest that k elements
// reach; where that still leaves more than 64 - equal values - those above it and the first of the equal ones by index (EV elements of
// a lane lie behind one another).  The candidates are gathered, sorted and merged with the list (larger of entry i and entry
// 63 - i of the other, then the last merge of the sort).  room: 64 entries of LDS of this wave
template <int EV, int N, class Index> __device__ __forceinline__ void absorb(TopList &top, const float (&x)[N], float lane_max, Index index, int k, Key *room)
{
    const int lane = threadIdx.x & 63;
    const bool full = top.last != kNone, empty = lane_key(top.key, 0) == kNone;
    float b = lane_max;
    uint32_t low;
    if (!full) {
        wave_sort(b);
        low = ordered(fmaxf(SN_READLANE_F32(b, k - 1), kLowest));                // (never an entry at -inf)
    } else {
        low = ordered(top.last_v) + 1;
    }
    int count = count_from(x, unordered(low));
    if (!empty && count <= 4) {
#pragma unroll
        for (int u = 0; u < N; ++u) top.offer(x[u], index(u), k);
        return;
    }
    if (count > 64) {
        uint32_t high = ordered(sn_wave_max(lane_max)) + 1;                       // under k elements reach it
        while (high - low > 1 && count > 64) {
            const uint32_t mid = low + (high - low) / 2;
            const int c = count_from(x, unordered(mid));
            if (c >= k) { low = mid; count = c; } else high = mid;
        }
    }
    const float bound = unordered(low);
    const bool equal = count > 64;                           // the bound's own value goes last
    int at = 0;
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const bool in = equal ? x[u] > bound : x[u] >= bound;
        const uint64_t m = __ballot(in);
        if (in) room[at + lanes_below(m)] = key_of(x[u], index(u));
        at += __popcll(m);
    }
    if (equal) {
#pragma unroll
        for (int c = 0; c < N / EV; ++c) {
            int before = at, all = 0;
#pragma unroll
            for (int e = 0; e < EV; ++e) {
                const uint64_t m = __ballot(x[c * EV + e] == bound);
                before += lanes_below(m);
                all += __popcll(m);
            }
#pragma unroll
            for (int e = 0; e < EV; ++e) {
                const bool in = x[c * EV + e] == bound;
                if (in && before < 64) room[before] = key_of(bound, index(c * EV + e));
                before += in;
            }
            at += all;
        }
        count = 64;
    }
    __builtin_amdgcn_wave_barrier();                         // (one wave's LDS operations stay in order)
    Key fresh = lane < count ? room[lane] : kNone;
    wave_sort(fresh);
    if (!empty) {
        const Key back = ((Key)(uint32_t)__shfl((int)(fresh >> 32), 63 - lane, 64) << 32) | (uint32_t)__shfl((int)(uint32_t)fresh, 63 - lane, 64);
        fresh = back > top.key ? back : top.key;
        sort_merge<64, 32>(fresh, lane);
    }
    top.key = lane < k ? fresh : kNone;
    top.set_last(k);
}

// the wave's share (segments w, w + nw, ...) of entries c0 .. c1 - 1 of a row
template <int DT, bool TOP>
__device__ __forceinline__ void scan(const void *row, int64_t c0, int64_t c1, int w, int nw, Soft &soft, TopList &top, int k, Key *room)
{
    constexpr int EV = DT == SN_F32 ? 4 : 8, PER = 16 / EV, SEG = 64 * 16;
    const int lane = threadIdx.x & 63;
    const char *base = (const char *)row + c0 * (DT == SN_F32 ? 4 : 2);
    const int n = (int)(c1 - c0);
    const uint32_t fill = DT == SN_F32 ? 0xFF800000u : DT == SN_BF16 ? 0xFF80u : 0xFC00u;      // -inf
    for (int s0 = w * SEG; s0 < n; s0 += nw * SEG) {
        float x[16];
#pragma unroll
        for (int c = 0; c < PER; ++c) {
            uint32_t raw[words<DT, EV>()];
            load_raw<DT, EV>(raw, base, s0 + (c * 64 + lane) * EV, n, fill);
            float part[EV];
            unpack<DT, EV>(part, raw);
#pragma unroll
            for (int e = 0; e < EV; ++e) x[c * EV + e] = part[e];
        }
        float m = x[0];
#pragma unroll
        for (int u = 1; u < 16; ++u) m = fmaxf(m, x[u]);
        const float mx = fmaxf(m, soft.m);
        if (mx > soft.m) {
            const float d = soft.m - mx, f = exp_fast(d);
            soft.t = (soft.t + soft.s * fmaxf(d, kFar)) * f;
            soft.s *= f;
            soft.m = mx;
        }
        const float ref = soft.m == -INFINITY ? 0.0f : soft.m;
#pragma unroll
        for (int u = 0; u < 16; ++u) {
            const float d = x[u] - ref, p = exp_fast(d);
            soft.s += p;
            soft.t = fmaf(p, fmaxf(d, kFar), soft.t);
        }
        if constexpr (TOP) {
            auto index = [&](int u) { return (int)c0 + s0 + ((u / EV) * 64 + lane) * EV + u % EV; };
            // (m is NaN only where every element of the lane is: none of them is a candidate)
            if (__any(m > top.last_v)) absorb<EV>(top, x, m == m ? m : -INFINITY, index, k, room);
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
    float *part;          // [rows, splits, 4 + 2 k]: m, s, t, nothing, keys
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
    if (a.stats) {
        a.stats[row * 3] = s.m;
        a.stats[row * 3 + 1] = s.s;
        a.stats[row * 3 + 2] = h;
    }
}
// the row's list, entry j by lane j of one wave (every lane of it calls; lanes from k on: kNone).  A row without NaN that has fewer than k
// entries above -inf: the rest are its entries at -inf, the lowest index first - nearly all others are, so the first few hundred
// hold enough.
template <int DT> __device__ __forceinline__ void write_top(const ScoreArgs &a, int64_t row, Key key, Soft s)
{
    const int lane = threadIdx.x & 63;
    const float ls = logf(s.s);
    const bool nan = s.s != s.s;
    float v = key_value(key);
    int i = key_index(key);
    int have = __popcll(__ballot(lane < a.k && key != kNone));
    if (have < a.k && !nan) {
        const void *p = (const char *)a.logits + row * a.stride * (DT == SN_F32 ? 4 : 2);
        for (int64_t j0 = 0; have < a.k && j0 < a.n; j0 += 64) {
            const bool masked = j0 + lane < a.n && load_one<DT>(p, j0 + lane) == -INFINITY;
            const uint64_t m = __ballot(masked);
            const int want = lane - have;                    // this lane takes the want-th of them
            int seen = 0;
            for (uint64_t r = m; r && seen < a.k - have; r &= r - 1, ++seen)
                if (seen == want) i = (int)j0 + __builtin_ctzll(r);
            have += __popcll(m);
        }
    }
    if (lane < a.k) {
        a.top_lp[row * a.k + lane] = nan ? __uint_as_float(0x7FC00000u) : v == -INFINITY ? -INFINITY : (v - s.m) - ls;
        a.top_ids[row * a.k + lane] = i;
    }
}

// `lists` sorted lists of k in src -> one, in pairs: an entry's place in the join is its own plus the number of the partner's that
// come before it.  Both buffers hold lists * k entries.  Every thread of the workgroup calls.  -> the buffer that holds the result
__device__ __forceinline__ Key *join_lists(Key *src, Key *dst, int lists, int k)
{
    while (lists > 1) {
        const int total = lists * k;
        for (int e = threadIdx.x; e < total; e += blockDim.x) {
            const int l = e / k, j = e - l * k;
            const Key me = src[e];
            int pos = j;
            if ((l ^ 1) < lists) {
                const Key *o = src + (l ^ 1) * k;
                int lo = 0, hi = k;
                while (lo < hi) {
                    const int mid = (lo + hi) >> 1;
                    // (only entries that were never filled are equal: those of the lower list first)
                    if (o[mid] > me || (o[mid] == me && (l & 1))) lo = mid + 1; else hi = mid;
                }
                pos += lo;
            }
            if (pos < k) dst[(l >> 1) * k + pos] = me;
        }
        __syncthreads();
        Key *const swap = src;
        src = dst;
        dst = swap;
        lists = (lists + 1) >> 1;
    }
    return src;
}

// The k best of `lists` (at most 64) sorted lists of k in src, lane j of wave 0 the j-th: with j = ceil(k / lists), the ceil(k / j)-th
// largest of the lists' j-th entries is a bound that k entries reach; those that do, if they are at most 64, are sorted by one wave,
// otherwise the lists are joined in pairs.  Every thread of the workgroup calls, after a barrier behind the writing of src.
struct Select { float bound; int counts[kScoreWaves]; Key room[64]; };
__device__ __forceinline__ Key best_of_lists(Key *src, Key *other, int lists, int k, Select &sh)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, total = lists * k;
    const int j = (k + lists - 1) / lists;
    // (every wave finds the bound: no barrier for it)
    float b = lane < lists ? key_value(src[lane * k + j - 1]) : -INFINITY;
    wave_sort(b);
    b = __shfl(b, (k + j - 1) / j - 1, 64);
    int count = 0;
    for (int e = threadIdx.x; e < total; e += kScoreThreads) {
        const Key q = src[e];
        count += q != kNone && key_value(q) >= b;
    }
    int upto = count;                                        // exclusive sum over the workgroup
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int o = __shfl_up(upto, off, 64);
        upto += lane >= off ? o : 0;
    }
    if (lane == 63) sh.counts[wave] = upto;
    __syncthreads();
    int all = 0, place = upto - count;
#pragma unroll
    for (int w = 0; w < kScoreWaves; ++w) {
        place += w < wave ? sh.counts[w] : 0;
        all += sh.counts[w];
    }
    if (all > 64) {
        const Key *best = join_lists(src, other, lists, k);
        return lane < k ? best[lane] : kNone;
    }
    for (int e = threadIdx.x; e < total; e += kScoreThreads) {
        const Key q = src[e];
        if (q != kNone && key_value(q) >= b) sh.room[place++] = q;
    }
    __syncthreads();
    Key mine = lane < all ? sh.room[lane] : kNone;
    if (wave == 0) wave_sort(mine);
    return lane < k ? mine : kNone;
}

// one wave a row
template <int DT, bool TOP>
__global__ __launch_bounds__(kScoreThreads) void scores_wave_kernel(ScoreArgs a)
{
    __shared__ Key room[TOP ? kScoreWaves : 1][TOP ? 64 : 1];
    const int lane = threadIdx.x & 63;
    const int64_t turn = (int64_t)gridDim.x * kScoreWaves;
    for (int64_t row = (int64_t)blockIdx.x * kScoreWaves + (threadIdx.x >> 6); row < a.rows; row += turn) {
        Soft soft = {-INFINITY, 0.0f, 0.0f};
        TopList top;
        top.reset();
        scan<DT, TOP>((const char *)a.logits + row * a.stride * (DT == SN_F32 ? 4 : 2), 0, a.n, 0, 1, soft, top, a.k, room[TOP ? threadIdx.x >> 6 : 0]);
        soft = wave_join(soft);
        if (lane == 0) write_row<DT>(a, row, soft);
        if constexpr (TOP) write_top<DT>(a, row, top.key, soft);
    }
}

// four waves a row or a split of one
template <int DT, bool TOP>
__global__ __launch_bounds__(kScoreThreads) void scores_group_kernel(ScoreArgs a)
{
    __shared__ Soft part[kScoreWaves];
    __shared__ Key lists[2][TOP ? kScoreWaves * SN_SCORES_MAX_TOP : 1];
    __shared__ Select select;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = blockIdx.x / a.splits;
    const int split = (int)(blockIdx.x - row * a.splits);
    const int64_t c0 = split * a.per_split, c1 = c0 + a.per_split < a.n ? c0 + a.per_split : a.n;
    Soft soft = {-INFINITY, 0.0f, 0.0f};
    TopList top;
    top.reset();
    if (c0 < c1) scan<DT, TOP>((const char *)a.logits + row * a.stride * (DT == SN_F32 ? 4 : 2), c0, c1, wave, kScoreWaves, soft, top, a.k, lists[1] + (TOP ? wave * 64 : 0));
    soft = wave_join(soft);
    if (lane == 0) part[wave] = soft;
    if (TOP && lane < a.k) lists[0][wave * a.k + lane] = top.key;
    __syncthreads();
    soft = join(join(part[0], part[1]), join(part[2], part[3]));
    Key best = kNone;
    if constexpr (TOP) best = best_of_lists(lists[0], lists[1], kScoreWaves, a.k, select);
    if (wave != 0) return;
    if (a.splits == 1) {
        if (lane == 0) write_row<DT>(a, row, soft);
        if constexpr (TOP) write_top<DT>(a, row, best, soft);
    } else {
        float *dst = a.part + (row * a.splits + split) * (4 + 2 * a.k);
        if (lane == 0) { dst[0] = soft.m; dst[1] = soft.s; dst[2] = soft.t; }
        if (TOP && lane < a.k) reinterpret_cast<Key *>(dst + 4)[lane] = best;
    }
}

// the splits of a row, one workgroup a row; two buffers of splits * k entries in LDS
template <int DT, bool TOP>
__global__ __launch_bounds__(kScoreThreads) void scores_join_kernel(ScoreArgs a)
{
    extern __shared__ Key buffers[];
    __shared__ Select select;
    const int64_t row = blockIdx.x;
    const int lane = threadIdx.x & 63, size = 4 + 2 * a.k;
    const float *src = a.part + row * a.splits * size;
    if constexpr (TOP) {
        for (int e = threadIdx.x; e < a.splits * a.k; e += kScoreThreads) {
            const int l = e / a.k;
            buffers[e] = reinterpret_cast<const Key *>(src + l * size + 4)[e - l * a.k];
        }
    }
    Soft s = {-INFINITY, 0.0f, 0.0f};
    if (lane < a.splits) {
        const float *p = src + lane * size;
        s = Soft{p[0], p[1], p[2]};
    }
    s = wave_join(s);
    if (threadIdx.x == 0) write_row<DT>(a, row, s);
    if constexpr (TOP) {
        __syncthreads();
        const Key best = best_of_lists(buffers, buffers + a.splits * a.k, a.splits, a.k, select);
        if (threadIdx.x < 64) write_top<DT>(a, row, best, s);
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
    const bool wrong = used && (tg < 0 || tg >= a.n);
    if (!wrong && (s == 0.0f || (g == 0.0f && gh == 0.0f))) {        // a row without a distribution, or without a part in the loss: not read
        const float zeros[EV] = {};
        for (int j = threadIdx.x * EV; j < n; j += kScoreThreads * EV) store_row<DT, EV>(dst, j, n, zeros);
        return;
    }
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
            if (wrong) x[e] = __uint_as_float(0x7FC00000u);
        }
        store_row<DT, EV>(dst, j, n, x);
    }
}

// One wave a row: short rows, and longer ones where there are waves enough (us, wave against workgroup, bf16, without | with 5
// alternatives: 256 x 2048 4.0, 3.8 | 8.4, 8.1; 256 x 4096 5.0, 3.9 | 13.2, 8.1; 1024 x 4096 5.2, 5.6 | 13.4, 13.1; 2048 x 8192 10.3,
// 10.6 | 23.7, 28.0; 4096 x 16384 26.5, 28.5 | 50.2, 67.8; 4096 x 32769 49.0, 47.2 | 76.0, 99.8; 2048 x 131072 133, 101 | 171, 142).  The rule is
// made for calls without alternatives: with them many rows of 16385 entries and more, up to somewhere under 131072, would do better by wave,
// which keeps one list instead of four (4096 x 32769: 76 us, they take 100; with 20 alternatives 109 and 128).
bool wave_a_row(int64_t rows, int64_t n) { return n <= 2048 || (rows >= 2048 && n <= 16384); }
// Workgroups a row: one up to 8192 entries (one row of 8192: 3.8 us, in two parts and joined 6.0), else four for each compute unit of
// 4096 entries or more (16 x 131072, bf16, 20 alternatives: parts of 4096 15.5 us, 8192 16.2, 16384 21.0, 2048 17.9)
int splits_for(int64_t rows, int64_t n)
{
    if (n <= 8192 || rows <= 0 || wave_a_row(rows, n)) return 1;
    int64_t s = 1024 / rows;
    const int64_t most = (n + 4095) / 4096;
    s = s > most ? most : s;
    s = s > kMaxSplits ? kMaxSplits : s;
    return (int)(s < 1 ? 1 : s);
}

template <int DT, bool TOP> int launch_scores(ScoreArgs &a, hipStream_t st)
{
    if (wave_a_row(a.rows, a.n)) {
        const int64_t blocks = (a.rows + kScoreWaves - 1) / kScoreWaves;
        hipLaunchKernelGGL((scores_wave_kernel<DT, TOP>), dim3((unsigned)(blocks < 16384 ? blocks : 16384)), dim3(kScoreThreads), 0, st, a);
        SN_CHECK_LAUNCH("sn_label_log_probs");
        return SN_OK;
    }
    hipLaunchKernelGGL((scores_group_kernel<DT, TOP>), dim3((unsigned)(a.rows * a.splits)), dim3(kScoreThreads), 0, st, a);
    SN_CHECK_LAUNCH("sn_label_log_probs");
    if (a.splits > 1) {
        const size_t lds = TOP ? (size_t)2 * a.splits * a.k * sizeof(Key) : 0;
        const int rc = sn_ensure_dynamic_lds((const void *)scores_join_kernel<DT, TOP>, lds + sizeof(Select), "sn_label_log_probs");
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
    return s > 1 ? (size_t)rows * s * (4 + 2 * k) * sizeof(float) : 0;
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
    SN_REQUIRE(log_probs && entropy && (k == 0 || (top_log_probs && top_ids)), SN_ERR_BAD_ARG, "sn_label_log_probs: NULL pointer");
    SN_REQUIRE(splits_for(rows, n) == 1 || (workspace && workspace_bytes >= sn_label_log_probs_workspace(rows, n, k)), SN_ERR_WORKSPACE, "sn_label_log_probs: workspace of %zu bytes", workspace_bytes);
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
    // (pieces of a row, us for 4096 x 32768 bf16: 2048 118, 4096 104, 8192 99, 16384 102, 32768 107)
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
