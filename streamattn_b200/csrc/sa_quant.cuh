// 8-bit KV caches: the row format, the conversions of both code types and the launch descriptors
// of the kernels that write rows and read them back.
//
// A row is D codes and one scale byte e (scale 2^(e - 127), 255 = NaN); the K and the V byte of a
// token lie side by side, head-major: pair index = outer * so + head * sh + token.
#pragma once

#include "sa_common.cuh"

namespace sa {

constexpr int kMinScaleByte = 27;   // 2^-100: 1 / scale and x / scale stay clear of the ends of fp32
constexpr int kNanScaleByte = 255;

// The smallest e with amax <= top * 2^(e - 127), from the bits of amax >= 0: with amax =
// m * 2^(x - 127), 1 <= m < 2, and top = t * 2^k, it is x - k, and one more where m > t
// (t = 1.75, k = 8 for e4m3's 448; t = 127/64, k = 6 for int8's 127).  Integer arithmetic: exact.
template <int CODE> __device__ __forceinline__ int scale_byte(uint32_t amax_bits)
{
    constexpr uint32_t kTopMantissa = CODE == kCodeE4M3 ? 0x600000u : 0x7e0000u;
    constexpr int kTopExponent = CODE == kCodeE4M3 ? 8 : 6;
    const int x = static_cast<int>(amax_bits >> 23);
    const int e = x - kTopExponent + ((amax_bits & 0x7fffffu) > kTopMantissa ? 1 : 0);
    return x == 255 ? kNanScaleByte : max(e, kMinScaleByte);
}

// 2^(e - 127) for e in [1, 254]; NaN for 255, and 0 for the byte 0, which no writer here produces.
__device__ __forceinline__ float scale_value(int e)
{
    return __uint_as_float(e == kNanScaleByte ? 0x7fffffffu : static_cast<uint32_t>(e) << 23);
}

// 2^(127 - e) for e in [27, 253].
__device__ __forceinline__ float inverse_scale(int e) { return __uint_as_float(static_cast<uint32_t>(254 - e) << 23); }

// Four values, already divided by the scale, to four codes (first value in the lowest byte).
template <int CODE> __device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d)
{
    if constexpr (CODE == kCodeE4M3) {
        uint16_t lo, hi;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
        return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
    } else {
        // |value| <= 127 by the choice of the scale: nothing saturates.
        const uint32_t ab = __byte_perm(__float2int_rn(a), __float2int_rn(b), 0x0040);
        const uint32_t cd = __byte_perm(__float2int_rn(c), __float2int_rn(d), 0x0040);
        return __byte_perm(ab, cd, 0x5410);
    }
}

// Four e4m3 codes to two pairs of halves (exact: 4 significant bits, |code| <= 448).
__device__ __forceinline__ void e4m3x4_to_halves(uint32_t x, uint32_t &lo, uint32_t &hi)
{
    asm("{\n\t.reg .b16 a, b;\n\t"
        "mov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(x));
}

// Four codes to two pairs of halves.  int8: with the sign bit flipped a byte is x + 128, and the
// half whose high byte is 0x64 and low byte u is exactly 1024 + u, so subtracting 1152 leaves x.
template <int CODE> __device__ __forceinline__ void decode4(uint32_t codes, uint32_t &lo, uint32_t &hi)
{
    if constexpr (CODE == kCodeE4M3) {
        e4m3x4_to_halves(codes, lo, hi);
    } else {
        const uint32_t u = codes ^ 0x80808080u;
        const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));  // 1152
        uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
        __half2 x = __hsub2(*reinterpret_cast<__half2 *>(&a), bias);
        __half2 y = __hsub2(*reinterpret_cast<__half2 *>(&b), bias);
        lo = *reinterpret_cast<uint32_t *>(&x);
        hi = *reinterpret_cast<uint32_t *>(&y);
    }
}

template <int CODE> __device__ __forceinline__ float decode1(uint8_t code)
{
    if constexpr (CODE == kCodeE4M3) {
        uint32_t h, unused;
        e4m3x4_to_halves(code, h, unused);
        return __low2float(*reinterpret_cast<const __half2 *>(&h));
    } else {
        return static_cast<float>(static_cast<int8_t>(code));
    }
}

// An element of a cache read next to queries of type T.
template <typename T, int CODE> struct CacheElem {
    using type = uint8_t;
    __device__ __forceinline__ static float to_float(uint8_t x) { return decode1<CODE>(x); }
};
template <typename T> struct CacheElem<T, kCodeNone> {
    using type = T;
    __device__ __forceinline__ static float to_float(T x) { return Elem<T>::to_float(x); }
};

// Where the rows of a cache lie.
struct QuantCache {
    uint8_t *key;
    uint8_t *value;
    uint8_t *scales;
    int kv_heads, head_dim;
    int capacity;                     // tokens a row can hold (< 2^31)
    int64_t so, sn, sh;               // codes: outer (row or page), token (or slot), head
    int64_t scale_so, scale_sh;       // pairs: outer, head (a token is one pair)
    const void *page_table;           // null: contiguous
    int table_i64;
    int max_pages, page_size;
    int page_shift;                   // log2(page_size), or -1
    int64_t num_pages;
};

// Token `pos` (in [0, capacity)) of row b: its code and pair offsets for head 0; false where its
// page id names no page.
__device__ __forceinline__ bool locate_token(const QuantCache &c, int b, int pos, int64_t &code_off, int64_t &pair_off)
{
    int64_t outer = b;
    int tok = pos;
    if (c.page_table != nullptr) {
        const int lp = c.page_shift >= 0 ? pos >> c.page_shift : pos / c.page_size;
        tok = pos - lp * c.page_size;
        outer = load_index(c.page_table, c.table_i64, static_cast<int64_t>(b) * c.max_pages + lp);
        if (outer < 0 || outer >= c.num_pages) return false;
    }
    code_off = outer * c.so + tok * c.sn;
    pair_off = outer * c.scale_so + tok;
    return true;
}

// n / d for n < 2^31 by a multiplication: with 2^(s-1) < d <= 2^s and m = ceil(2^(31+s) / d), which fits 32 bits,
// floor(n m / 2^(31+s)) = floor(n / d) because m d exceeds 2^(31+s) by less than d <= 2^s.
struct FastDiv {
    unsigned d, magic;
    int shift;  // s - 1; -1: d == 1
    FastDiv() = default;
    explicit FastDiv(unsigned divisor) : d(divisor), magic(0), shift(-1)
    {
        while (shift < 30 && (1u << (shift + 1)) < d) ++shift;
        if (shift >= 0) magic = static_cast<unsigned>(((1ull << (32 + shift)) + d - 1) / d);
    }
    __device__ __forceinline__ unsigned divide(unsigned n) const { return shift < 0 ? n : __umulhi(n, magic) >> shift; }
};

struct QuantizeParams {
    QuantCache cache;
    const void *k_new;
    const void *v_new;
    int64_t new_sb, new_st, new_sh;
    int tokens, batch;
    const void *positions;
    int pos_i64, pos_shared;
    const void *counts;               // null: tokens
    int counts_i64;
    void *lens_out;
    const void *cos;
    const void *sin;
    int64_t rope_sb, rope_st;
    const void *q_in;
    void *q_out;
    int q_heads;
    int64_t qi_sb, qi_st, qi_sh, qo_sb, qo_st, qo_sh;
    int *status;
    int heads_fastest;                // order in which a row's (token, head) units are taken
    int kv_blocks;                    // CTAs of one batch row that write K/V; the others move the query
    FastDiv kv_div, q_div;            // by the index of a unit that varies fastest
};

struct DequantizeParams {
    QuantCache cache;
    void *k_out;
    void *v_out;
    int64_t out_sb, out_st, out_sh;
    int tokens, batch;
    const void *starts;               // null: 0
    int starts_i64;
    const void *counts;               // null: tokens
    int counts_i64;
    int *status;
    int heads_fastest;
    FastDiv div;
};

// `vector`: head_dim is a multiple of 16, addresses allow 8-element accesses, and every stride but the batch row's fits 32 bits.
cudaError_t launch_quantize(QuantizeParams p, int code, int dtype, bool vector, cudaStream_t stream);
cudaError_t launch_dequantize(DequantizeParams p, int code, int dtype, bool vector, cudaStream_t stream);

}  // namespace sa
