// Loads and stores of fp32 / bf16 / fp16 rows as fp32 registers, and the 8-bit checkpoint of 32 features.
// A lane moves EV consecutive elements with one access of up to 16 bytes; the address needs the element's own alignment only
// (the target's unaligned access mode: rows of an odd length start anywhere), the last, partial group of a row is moved
// element by element.
#pragma once

#include "sn_common.h"
#include "schemanet_blocks.h"

namespace sn {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float bf16_to_f32(uint32_t u) { return __uint_as_float(u << 16); }
// two floats -> two bf16 in one word, round to nearest even (v_cvt_pk_bf16_f32)
__device__ __forceinline__ uint32_t pack_bf16(float a, float b)
{
    const f32x2 v = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}

// dwords of EV elements
template <int DT, int EV> constexpr int words() { return EV * (DT == SN_F32 ? 4 : 2) / 4; }

template <int DT, int EV> using Raw = uint32_t[words<DT, EV>()];
typedef uint32_t sn_u32x4 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t sn_u32x2 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t sn_u32x1 __attribute__((aligned(2)));

template <int NW> __device__ __forceinline__ void load_words(uint32_t (&w)[NW], const void *p)
{
    static_assert(NW == 4 || NW == 2 || NW == 1 || NW == 8, "16-, 8- or 4-byte accesses");
    if constexpr (NW == 8) {
        const sn_u32x4 a = *reinterpret_cast<const sn_u32x4 *>(p), b = *reinterpret_cast<const sn_u32x4 *>((const char *)p + 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) { w[i] = a[i]; w[4 + i] = b[i]; }
    } else if constexpr (NW == 4) {
        const sn_u32x4 a = *reinterpret_cast<const sn_u32x4 *>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = a[i];
    } else if constexpr (NW == 2) {
        const sn_u32x2 a = *reinterpret_cast<const sn_u32x2 *>(p);
        w[0] = a[0]; w[1] = a[1];
    } else {
        w[0] = *reinterpret_cast<const sn_u32x1 *>(p);
    }
}
template <int NW> __device__ __forceinline__ void store_words(void *p, const uint32_t (&w)[NW])
{
    if constexpr (NW == 8) {
        *reinterpret_cast<sn_u32x4 *>(p) = sn_u32x4{w[0], w[1], w[2], w[3]};
        *reinterpret_cast<sn_u32x4 *>((char *)p + 16) = sn_u32x4{w[4], w[5], w[6], w[7]};
    } else if constexpr (NW == 4) {
        *reinterpret_cast<sn_u32x4 *>(p) = sn_u32x4{w[0], w[1], w[2], w[3]};
    } else if constexpr (NW == 2) {
        *reinterpret_cast<sn_u32x2 *>(p) = sn_u32x2{w[0], w[1]};
    } else {
        *reinterpret_cast<sn_u32x1 *>(p) = w[0];
    }
}

// raw words of EV elements <-> floats
template <int DT, int EV> __device__ __forceinline__ void unpack(float (&v)[EV], const Raw<DT, EV> &w)
{
    if constexpr (DT == SN_F32) {
#pragma unroll
        for (int i = 0; i < EV; ++i) v[i] = __uint_as_float(w[i]);
    } else if constexpr (DT == SN_BF16) {
#pragma unroll
        for (int i = 0; i < EV / 2; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    } else {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int i = 0; i < EV / 2; ++i) {
            const h2 h = __builtin_bit_cast(h2, w[i]);
            v[2 * i] = (float)h[0];
            v[2 * i + 1] = (float)h[1];
        }
    }
}
template <int DT, int EV> __device__ __forceinline__ void pack(Raw<DT, EV> &w, const float (&v)[EV])
{
    if constexpr (DT == SN_F32) {
#pragma unroll
        for (int i = 0; i < EV; ++i) w[i] = __float_as_uint(v[i]);
    } else if constexpr (DT == SN_BF16) {
#pragma unroll
        for (int i = 0; i < EV / 2; ++i) w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
    } else {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int i = 0; i < EV / 2; ++i) {
            const h2 h = {(_Float16)v[2 * i], (_Float16)v[2 * i + 1]};
            w[i] = __builtin_bit_cast(uint32_t, h);
        }
    }
}

template <int DT> __device__ __forceinline__ float load_one(const void *p, int64_t i)
{
    if constexpr (DT == SN_F32) return ((const float *)p)[i];
    else if constexpr (DT == SN_BF16) return bf16_to_f32(((const uint16_t *)p)[i]);
    else return (float)((const _Float16 *)p)[i];
}
template <int DT> __device__ __forceinline__ void store_one(void *p, int64_t i, float v)
{
    if constexpr (DT == SN_F32) ((float *)p)[i] = v;
    else if constexpr (DT == SN_BF16) ((uint16_t *)p)[i] = (uint16_t)(pack_bf16(v, 0.0f) & 0xFFFFu);
    else ((_Float16 *)p)[i] = (_Float16)v;
}
// the type as a (uniform) run-time value: gradients of parameters
__device__ __forceinline__ void store_any(void *p, int dtype, int64_t i, float v)
{
    if (dtype == SN_F32) store_one<SN_F32>(p, i, v);
    else if (dtype == SN_BF16) store_one<SN_BF16>(p, i, v);
    else store_one<SN_F16>(p, i, v);
}

// elements i .. i + EV - 1 of a row of n; `fill` beyond its end
template <int DT, int EV> __device__ __forceinline__ void load_raw(Raw<DT, EV> &w, const void *row, int i, int n, uint32_t fill = 0u)
{
    const char *p = (const char *)row + (int64_t)i * (DT == SN_F32 ? 4 : 2);
    if (i + EV <= n) {
        load_words<words<DT, EV>()>(w, p);
    } else if constexpr (DT == SN_F32) {
#pragma unroll
        for (int e = 0; e < EV; ++e) w[e] = i + e < n ? ((const uint32_t *)p)[e] : fill;
    } else {
#pragma unroll
        for (int e = 0; e < EV / 2; ++e) {
            const uint32_t lo = i + 2 * e < n ? (uint32_t)((const uint16_t *)p)[2 * e] : (fill & 0xFFFFu);
            const uint32_t hi = i + 2 * e + 1 < n ? (uint32_t)((const uint16_t *)p)[2 * e + 1] : (fill & 0xFFFFu);
            w[e] = lo | (hi << 16);
        }
    }
}
// The same without a test that a load would wait behind (for loads that run ahead of their use): the last group of a row is read
// from EV elements before the row's end (n >= EV) and turned into place when it is unpacked.
template <int EV> __device__ __forceinline__ int tail_shift(int i, int n) { return i + EV <= n ? 0 : (i >= n ? EV : i + EV - n); }
template <int DT, int EV> __device__ __forceinline__ void load_ahead(Raw<DT, EV> &w, const void *row, int i, int n)
{
    const int at = i + EV <= n ? i : n - EV;
    load_words<words<DT, EV>()>(w, (const char *)row + (int64_t)at * (DT == SN_F32 ? 4 : 2));
}
template <int EV> __device__ __forceinline__ void turn_tail(float (&v)[EV], int shift)
{
#pragma unroll
    for (int s = 1; s <= EV; s *= 2)
#pragma unroll
        for (int e = 0; e < EV; ++e) v[e] = (shift & s) ? (e + s < EV ? v[e + s] : 0.0f) : v[e];
}
template <int DT, int EV> __device__ __forceinline__ void store_row(void *row, int i, int n, const float (&v)[EV])
{
    char *p = (char *)row + (int64_t)i * (DT == SN_F32 ? 4 : 2);
    if (i + EV <= n) {
        uint32_t w[words<DT, EV>()];
        pack<DT, EV>(w, v);
        store_words<words<DT, EV>()>(p, w);
    } else {
#pragma unroll
        for (int e = 0; e < EV; ++e)
            if (i + e < n) store_one<DT>(p, e, v[e]);
    }
}

// ---- 8-bit checkpoints (schemanet_blocks.h): 32 / EV neighbouring lanes hold one block of 32 features
// |v| as bits orders like the magnitude, and NaN sorts above inf
template <int EV> __device__ __forceinline__ uint32_t block_top(const float (&v)[EV])
{
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < EV; ++i) {
        const uint32_t a = __float_as_uint(v[i]) & 0x7FFFFFFFu;
        top = a > top ? a : top;
    }
    static_assert(EV == 4 || EV == 8, "a lane holds 4 or 8 features of a block");
    auto both = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
    top = both(top, SN_DPP_U32(top, 0xB1));                // quad_perm [1,0,3,2]
    top = both(top, SN_DPP_U32(top, 0x4E));                // quad_perm [2,3,0,1]
    if constexpr (EV == 4) top = both(top, SN_DPP_U32(top, 0x141));      // row_half_mirror: the other quad of eight lanes
    return top;
}
// exponent byte: 0x10000 carries into the exponent field when the mantissa is 127.5 / 64 or more
__device__ __forceinline__ uint32_t block_exp(uint32_t top)
{
    if (top >= 0x7F800000u) return 255u;
    const uint32_t e = (top + 0x10000u) >> 23;
    return e < 8u ? 8u : (e > 254u ? 254u : e);
}
// 2^(133 - e) and 2^(e - 133) (NaN for the mark 255)
__device__ __forceinline__ float block_inverse(uint32_t e) { return __uint_as_float((260u - e) << 23); }
__device__ __forceinline__ float block_step(uint32_t e) { return e == 255u ? __uint_as_float(0x7FC00000u) : __uint_as_float((e - 6u) << 23); }
template <int EV> __device__ __forceinline__ void encode(uint32_t (&codes)[EV / 4], const float (&v)[EV], uint32_t e)
{
    const float inv = block_inverse(e);
#pragma unroll
    for (int i = 0; i < EV / 4; ++i) {
        codes[i] = 0u;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            // (a block marked 255 holds NaN or inf: whatever is stored, the restored value is code * NaN)
            const float q = __builtin_amdgcn_fmed3f(rintf(v[4 * i + j] * inv), -127.0f, 127.0f);
            codes[i] |= ((uint32_t)(int)q & 0xFFu) << (8 * j);
        }
    }
}
template <int EV> __device__ __forceinline__ void decode(float (&v)[EV], const uint32_t (&codes)[EV / 4], uint32_t e)
{
    const float step = block_step(e);
#pragma unroll
    for (int i = 0; i < EV; ++i) v[i] = (float)(int8_t)(codes[i / 4] >> (8 * (i & 3))) * step;
}

}  // namespace sn
