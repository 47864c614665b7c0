// Rows of an 8-bit KV cache: quantise new K/V rows (after rotating K) into a contiguous or paged
// cache, and read rows back.  The format is described in sa_quant.cuh.
//
// Both are one pass over the data and bound by memory: D * (element + 1) + 1 bytes a row.  A unit is
// the K and the V row of one (token, head); D / 16 lanes (rounded up to a power of two) share it,
// 8 elements of either half of the row each, so 16-bit rows move in 16-byte and codes in 8-byte
// pieces, the maximum of a row is a few shuffles, and the two scale bytes of a token leave in one
// 2-byte store.  A thread requests all that it reads before it writes anything.  Rows that do not allow
// such accesses (D no multiple of 16, odd strides) take one warp a unit with single-element accesses.
//
// Measured (bytes as above against the time): 8 x 4096 tokens x 2 heads, D64, bf16 with rotation and 16 query heads to
// e4m3 31.0 us, 5.4 TB/s; 13 ragged rows of up to 8190 tokens x 8 heads, D128, fp16 to int8 in token-major pages 80 to 82 us,
// 5.3 TB/s; read back: ragged 8 x 65536 x 2, D64, pages of 16 46 to 50 us (the lengths are drawn), 5.4 to 5.9 TB/s;
// 3 x 32768 x 8, D128, int8 to fp16 91.6 us, 6.6 TB/s.  One token a row (8 rows, 2 + 16 heads): 6.0 us, the launch and one
// chain of position, page id and rows.  8 x 4096 x 2 heads without rotation: D48 7.4 us written and 5.2 read in pieces,
// D40 29.8 and 13.1 by single elements, which nothing but being right was asked of.
// What made the difference: pieces of both halves of a row in one lane, so that rotation needs no other lane and each
// unit costs half the index arithmetic; it halved the writes.  Putting the page id's look-up behind the row loads gained
// nothing.
#include <algorithm>

#include "sa_quant.cuh"

namespace sa {
namespace {

constexpr int kThreads = 256;
constexpr int kScalarUnits = 2;  // units a warp of the scalar kernels takes
constexpr int kMaxLaneElems = 8; // scalar form: elements of a row a lane holds (head_dim <= 256)

__device__ __forceinline__ void wait_for_stream()
{
    // Let the next kernel of the stream be scheduled early, and hold this one, before its first
    // global access, until everything launched before it has completed.
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Eight consecutive elements as they lie in memory, and as floats.
template <typename T> struct Eight;
template <> struct Eight<float> {
    float4 a, b;
    // Bits of the largest magnitude (a NaN is larger than an infinity, an infinity larger than a number).
    __device__ __forceinline__ uint32_t top() const
    {
        float x[8];
        get(x);
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
        return m;
    }
    __device__ __forceinline__ void load(const float *p)
    {
        a = reinterpret_cast<const float4 *>(p)[0];
        b = reinterpret_cast<const float4 *>(p)[1];
    }
    __device__ __forceinline__ void get(float (&x)[8]) const
    {
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    }
    __device__ __forceinline__ static void store(float *p, const float (&x)[8])
    {
        reinterpret_cast<float4 *>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4 *>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    }
};
template <typename T> struct Eight {
    uint4 a;
    __device__ __forceinline__ uint32_t top() const  // two 16-bit patterns at a time: their order is that of the magnitudes
    {
        const uint32_t m = __vmaxu2(__vmaxu2(a.x & 0x7fff7fffu, a.y & 0x7fff7fffu), __vmaxu2(a.z & 0x7fff7fffu, a.w & 0x7fff7fffu));
        const uint16_t pattern = static_cast<uint16_t>(max(m & 0xffffu, m >> 16));
        return __float_as_uint(Elem<T>::to_float(*reinterpret_cast<const T *>(&pattern)));
    }
    __device__ __forceinline__ void load(const T *p) { a = *reinterpret_cast<const uint4 *>(p); }
    __device__ __forceinline__ void get(float (&x)[8]) const
    {
        const T *e = reinterpret_cast<const T *>(&a);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = Elem<T>::to_float(e[i]);
    }
    __device__ __forceinline__ static void store(T *p, const float (&x)[8])
    {
        uint4 v;
        T *e = reinterpret_cast<T *>(&v);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = Elem<T>::from_float(x[i]);
        *reinterpret_cast<uint4 *>(p) = v;
    }
};

// x * cos + rotate_half(x) * sin in fp32; `partner` is the element half a row away, `low` says that
// x lies in the row's first half.  Products of 16-bit inputs are exact in fp32, so the sum is the
// only rounding; fp32 inputs round each product (no contraction), as the same tensor expression does.
__device__ __forceinline__ float rotate(float x, float partner, bool low, float cos, float sin)
{
    return __fadd_rn(__fmul_rn(x, cos), __fmul_rn(low ? -partner : partner, sin));
}

// Where one batch row's new tokens go.  `ok`: they fit the cache.
struct RowPlace {
    int start, count;
    bool ok;
};

__device__ __forceinline__ int clipped_count(const void *counts, int counts_i64, int b, int tokens)
{
    if (counts == nullptr) return tokens;
    const int64_t n = load_index(counts, counts_i64, b);
    return static_cast<int>(n < 0 ? 0 : (n < tokens ? n : tokens));
}

__device__ __forceinline__ RowPlace row_place(const QuantizeParams &p, int b)
{
    RowPlace r;
    const int64_t start = load_index(p.positions, p.pos_i64, p.pos_shared ? 0 : b);
    r.count = clipped_count(p.counts, p.counts_i64, b, p.tokens);
    r.ok = start >= 0 && start <= p.cache.capacity - r.count;
    r.start = r.ok ? static_cast<int>(start) : 0;
    return r;
}

__device__ __forceinline__ void report(int *status, int bits)
{
    if (status != nullptr) atomicOr(status, bits);
}

__device__ __forceinline__ void put_length(const QuantizeParams &p, int b, const RowPlace &r)
{
    if (p.pos_i64) static_cast<int64_t *>(p.lens_out)[b] = static_cast<int64_t>(r.start) + r.count;
    else static_cast<int32_t *>(p.lens_out)[b] = r.start + r.count;
}

// unit -> (token, head), the inner one of the two varying fastest.
__device__ __forceinline__ void unit_of(unsigned unit, const FastDiv &inner, int heads_fastest, int &t, int &h)
{
    const unsigned outer_index = inner.divide(unit), inner_index = unit - outer_index * inner.d;
    t = static_cast<int>(heads_fastest ? outer_index : inner_index);
    h = static_cast<int>(heads_fastest ? inner_index : outer_index);
}

// Offset i * stride for strides that fit 32 bits (the vector kernels; the host checks): one instruction.
__device__ __forceinline__ int64_t at(int i, int64_t stride) { return static_cast<int64_t>(i) * static_cast<int>(stride); }

// Token `pos` of row b for the vector kernels: code and pair offsets of head 0; false where its page id names no page.
__device__ __forceinline__ bool place_token(const QuantCache &c, int b, int pos, int64_t &code_off, int64_t &pair_off)
{
    if (c.page_table == nullptr) {
        code_off = b * c.so + at(pos, c.sn);
        pair_off = b * c.scale_so + pos;
        return true;
    }
    const int lp = c.page_shift >= 0 ? pos >> c.page_shift : pos / c.page_size;
    const int slot = pos - lp * c.page_size;
    const int64_t page = load_index(c.page_table, c.table_i64, static_cast<int64_t>(b) * c.max_pages + lp);
    if (page < 0 || page >= c.num_pages) return false;
    code_off = at(static_cast<int>(page), c.so) + at(slot, c.sn);
    pair_off = at(static_cast<int>(page), c.scale_so) + slot;
    return true;
}

// Codes of eight values of a row with scale byte e.
template <int CODE> __device__ __forceinline__ uint2 encode8(const float (&x)[8], int e)
{
    const float inv = inverse_scale(e);
    uint2 codes;
    if constexpr (CODE == kCodeE4M3) {
        codes.x = encode4<CODE>(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
        codes.y = encode4<CODE>(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv);
    } else {
        // x * inv is exact and at most 127 in magnitude; added to 1.5 * 2^23 it is rounded to an integer, halves to
        // even, whose two's complement is the sum's lowest byte.
        uint32_t y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = __float_as_uint(__fmaf_rn(x[i], inv, 12582912.0f));
        codes.x = __byte_perm(__byte_perm(y[0], y[1], 0x0040), __byte_perm(y[2], y[3], 0x0040), 0x5410);
        codes.y = __byte_perm(__byte_perm(y[4], y[5], 0x0040), __byte_perm(y[6], y[7], 0x0040), 0x5410);
    }
    return e == kNanScaleByte ? make_uint2(0u, 0u) : codes;
}

// The two pieces of a row a lane holds: elements d .. d + 7 of each half of the row, so that the lanes of a row read
// consecutive pieces and every element finds the one it is rotated with in the same lane.
template <typename T> struct Halves {
    Eight<T> lo, hi;
    __device__ __forceinline__ void load(const T *row, int half)
    {
        lo.load(row);
        hi.load(row + half);
    }
    __device__ __forceinline__ void get(float (&x)[8], float (&y)[8]) const
    {
        lo.get(x);
        hi.get(y);
    }
    __device__ __forceinline__ void turned(const Halves &cos, const Halves &sin, float (&x)[8], float (&y)[8]) const
    {
        float a[8], b[8], c[8], s[8];
        get(a, b);
        cos.lo.get(c);
        sin.lo.get(s);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = rotate(a[i], b[i], true, c[i], s[i]);
        cos.hi.get(c);
        sin.hi.get(s);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = rotate(b[i], a[i], false, c[i], s[i]);
    }
};

// 16-bit rows: registers for five CTAs an SM with rotation (48; 64 and four without the bound, which takes 3 % more for
// the chunk above), for six without (40; five take 3 % more for the prompts).
template <typename T, int CODE, bool ROPE>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? (ROPE ? 5 : 6) : 1) quantize_vector_kernel(const __grid_constant__ QuantizeParams p, int lane_shift)
{
    wait_for_stream();
    const int b = blockIdx.y;
    const int half = p.cache.head_dim >> 1;
    const int lanes = 1 << lane_shift;
    const int d = (threadIdx.x & (lanes - 1)) * 8;
    const bool in_row = d < half;
    const bool is_query = static_cast<int>(blockIdx.x) >= p.kv_blocks;
    const unsigned first = (blockIdx.x - (is_query ? p.kv_blocks : 0)) * (kThreads >> lane_shift);  // the CTA's first unit
    const unsigned unit = first + (threadIdx.x >> lane_shift);
    const FastDiv &div = is_query ? p.q_div : p.kv_div;
    int t, h;
    unit_of(unit, div, p.heads_fastest, t, h);
    const T *cos = static_cast<const T *>(p.cos) + b * p.rope_sb + at(t, p.rope_st) + d;
    const T *sin = static_cast<const T *>(p.sin) + b * p.rope_sb + at(t, p.rope_st) + d;
    Halves<T> c, s;
    float x[8], y[8];

    if (is_query) {
        if (unit >= static_cast<unsigned>(p.tokens) * p.q_heads || !in_row) return;
        Halves<T> q;
        q.load(static_cast<const T *>(p.q_in) + b * p.qi_sb + at(t, p.qi_st) + at(h, p.qi_sh) + d, half);
        if (ROPE) {
            c.load(cos, half);
            s.load(sin, half);
            q.turned(c, s, x, y);
        } else {
            q.get(x, y);
        }
        T *out = static_cast<T *>(p.q_out) + b * p.qo_sb + at(t, p.qo_st) + at(h, p.qo_sh) + d;
        Eight<T>::store(out, x);
        Eight<T>::store(out + half, y);
        return;
    }

    const RowPlace place = row_place(p, b);
    const bool alone = p.kv_blocks == 1;  // the only CTA that reads this row's position: it may also replace it
    if (!place.ok && threadIdx.x == 0) report(p.status, SA_DEV_BAD_POSITION);
    if (!alone && p.heads_fastest && div.divide(first) >= static_cast<unsigned>(place.count)) return;  // padding
    // Everything that is read - rows, angles, page id - is requested before anything is written.
    const bool mine = place.ok && unit < static_cast<unsigned>(p.tokens) * p.cache.kv_heads && t < place.count && in_row;
    Halves<T> k, v;
    int64_t code_off = 0, pair_off = 0;
    bool there = true;  // the token's page
    uint32_t e = 0;     // scale bytes of K and V, side by side
    if (mine) {
        const int64_t src = b * p.new_sb + at(t, p.new_st) + at(h, p.new_sh) + d;
        k.load(static_cast<const T *>(p.k_new) + src, half);
        v.load(static_cast<const T *>(p.v_new) + src, half);
        if (ROPE) {
            c.load(cos, half);
            s.load(sin, half);
        }
        there = place_token(p.cache, b, place.start + t, code_off, pair_off);
        uint32_t k_top = 0;
        if (ROPE) {
            k.turned(c, s, x, y);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                k_top = max(k_top, max(__float_as_uint(x[i]) & 0x7fffffffu, __float_as_uint(y[i]) & 0x7fffffffu));
        } else {
            k.get(x, y);
            k_top = max(k.lo.top(), k.hi.top());
        }
        e = scale_byte<CODE>(k_top) | (scale_byte<CODE>(max(v.lo.top(), v.hi.top())) << 16);
    }
    // The scale byte grows with the largest magnitude: a row's byte is the largest of its lanes' bytes.
    for (int o = lanes >> 1; o > 0; o >>= 1) e = __vmaxu2(e, __shfl_xor_sync(0xffffffffu, e, o));
    if (mine && there) {
        const int ek = e & 0xffffu, ev = e >> 16;
        uint8_t *key = p.cache.key + code_off + at(h, p.cache.sh) + d, *value = p.cache.value + code_off + at(h, p.cache.sh) + d;
        *reinterpret_cast<uint2 *>(key) = encode8<CODE>(x, ek);
        *reinterpret_cast<uint2 *>(key + half) = encode8<CODE>(y, ek);
        v.get(x, y);
        *reinterpret_cast<uint2 *>(value) = encode8<CODE>(x, ev);
        *reinterpret_cast<uint2 *>(value + half) = encode8<CODE>(y, ev);
        if (d == 0)
            reinterpret_cast<uint16_t *>(p.cache.scales)[pair_off + at(h, p.cache.scale_sh)] = static_cast<uint16_t>(ek | (ev << 8));
    } else if (mine && d == 0) {
        report(p.status, SA_DEV_BAD_PAGE);
    }
    if (alone && p.lens_out != nullptr) {
        const bool bad = __syncthreads_or(!there) || !place.ok;  // and: every thread has read its position
        if (threadIdx.x == 0 && !bad) put_length(p, b, place);
    }
}

// One warp a unit, single-element accesses: any head_dim up to 256, any stride.
template <typename T, int CODE>
__global__ void __launch_bounds__(kThreads) quantize_scalar_kernel(const __grid_constant__ QuantizeParams p)
{
    wait_for_stream();
    const int b = blockIdx.y;
    const int dim = p.cache.head_dim, half = dim >> 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int kWarps = kThreads / 32;
    const bool rope = p.cos != nullptr;
    const bool is_query = static_cast<int>(blockIdx.x) >= p.kv_blocks;
    // The query's CTAs must not read the position: another CTA may be replacing it.
    const RowPlace place = is_query ? RowPlace{0, p.tokens, true} : row_place(p, b);
    const int heads = is_query ? p.q_heads : p.cache.kv_heads;
    const unsigned total = static_cast<unsigned>(p.tokens) * heads;
    const unsigned first = (blockIdx.x - (is_query ? p.kv_blocks : 0)) * kWarps * kScalarUnits + warp;
    if (!is_query && !place.ok && threadIdx.x == 0) report(p.status, SA_DEV_BAD_POSITION);
    bool bad = !place.ok;

    for (int u = 0; u < kScalarUnits; ++u) {
        const unsigned unit = first + u * kWarps;
        int t, h;
        unit_of(unit, is_query ? p.q_div : p.kv_div, p.heads_fastest, t, h);
        if (unit >= total || t >= place.count) continue;        // warp-uniform, like everything down to the stores
        const T *cos_row = static_cast<const T *>(p.cos) + b * p.rope_sb + t * p.rope_st;
        const T *sin_row = static_cast<const T *>(p.sin) + b * p.rope_sb + t * p.rope_st;
        auto element = [&](const T *row, int d, bool turn) {
            float x = Elem<T>::to_float(row[d]);
            if (turn) x = rotate(x, Elem<T>::to_float(row[d < half ? d + half : d - half]), d < half,
                                 Elem<T>::to_float(cos_row[d]), Elem<T>::to_float(sin_row[d]));
            return x;
        };
        if (is_query) {
            const T *src = static_cast<const T *>(p.q_in) + b * p.qi_sb + t * p.qi_st + h * p.qi_sh;
            T *dst = static_cast<T *>(p.q_out) + b * p.qo_sb + t * p.qo_st + h * p.qo_sh;
            for (int d = lane; d < dim; d += 32) dst[d] = Elem<T>::from_float(element(src, d, rope));
            continue;
        }
        if (!place.ok) continue;
        int64_t code_off, pair_off;
        if (!locate_token(p.cache, b, place.start + t, code_off, pair_off)) {
            if (lane == 0) report(p.status, SA_DEV_BAD_PAGE);
            bad = true;
            continue;
        }
        const int64_t src = b * p.new_sb + t * p.new_st + h * p.new_sh;
        int e[2];
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const T *row = static_cast<const T *>(which ? p.v_new : p.k_new) + src;
            uint8_t *dst = (which ? p.cache.value : p.cache.key) + code_off + h * p.cache.sh;
            float x[kMaxLaneElems];
            uint32_t amax = 0;
#pragma unroll
            for (int i = 0; i < kMaxLaneElems; ++i) {
                const int d = lane + 32 * i;
                x[i] = d < dim ? element(row, d, rope && which == 0) : 0.0f;
                amax = max(amax, __float_as_uint(x[i]) & 0x7fffffffu);
            }
            amax = __reduce_max_sync(0xffffffffu, amax);
            e[which] = scale_byte<CODE>(amax);
            const float inv = inverse_scale(e[which]);
#pragma unroll
            for (int i = 0; i < kMaxLaneElems; ++i) {
                const int d = lane + 32 * i;
                if (d < dim)
                    dst[d] = e[which] == kNanScaleByte ? 0 : static_cast<uint8_t>(encode4<CODE>(x[i] * inv, 0.0f, 0.0f, 0.0f));
            }
        }
        if (lane == 0)
            reinterpret_cast<uint16_t *>(p.cache.scales)[pair_off + h * p.cache.scale_sh] =
                static_cast<uint16_t>(e[0] | (e[1] << 8));
    }
    if (!is_query && p.lens_out != nullptr && p.kv_blocks == 1) {  // as above
        bad = __syncthreads_or(bad);
        if (threadIdx.x == 0 && !bad) put_length(p, b, place);
    }
}

// Rows whose tokens were written by several CTAs: the lengths, after all of them, where every page of the range exists.
__global__ void __launch_bounds__(128) quantize_lengths_kernel(const __grid_constant__ QuantizeParams p)
{
    wait_for_stream();
    const int b = blockIdx.x;
    const RowPlace r = row_place(p, b);
    bool bad = !r.ok;
    if (r.ok && p.cache.page_table != nullptr && r.count > 0) {
        const int first = r.start / p.cache.page_size, last = (r.start + r.count - 1) / p.cache.page_size;
        for (int lp = first + threadIdx.x; lp <= last; lp += blockDim.x) {
            const int64_t page = load_index(p.cache.page_table, p.cache.table_i64, static_cast<int64_t>(b) * p.cache.max_pages + lp);
            bad = bad || page < 0 || page >= p.cache.num_pages;
        }
    }
    bad = __syncthreads_or(bad);
    if (threadIdx.x == 0 && !bad) put_length(p, b, r);
}

template <typename T, int CODE>
__global__ void __launch_bounds__(kThreads) dequantize_vector_kernel(const __grid_constant__ DequantizeParams p, int lane_shift)
{
    wait_for_stream();
    const int b = blockIdx.y;
    const int half = p.cache.head_dim >> 1;
    const int d = (threadIdx.x & ((1 << lane_shift) - 1)) * 8;
    const unsigned unit = blockIdx.x * (kThreads >> lane_shift) + (threadIdx.x >> lane_shift);
    int t, h;
    unit_of(unit, p.div, p.heads_fastest, t, h);
    const int64_t pos = (p.starts == nullptr ? 0 : load_index(p.starts, p.starts_i64, b)) + t;
    const int count = clipped_count(p.counts, p.counts_i64, b, p.tokens);
    if (unit >= static_cast<unsigned>(p.tokens) * p.cache.kv_heads || t >= count || d >= half) return;
    int64_t code_off, pair_off;
    int bad = 0;
    if (pos < 0 || pos >= p.cache.capacity) bad = SA_DEV_BAD_POSITION;
    else if (!place_token(p.cache, b, static_cast<int>(pos), code_off, pair_off)) bad = SA_DEV_BAD_PAGE;
    if (bad != 0) {
        if (d == 0) report(p.status, bad);
        return;
    }
    code_off += at(h, p.cache.sh) + d;
    const uint32_t pair = reinterpret_cast<const uint16_t *>(p.cache.scales)[pair_off + at(h, p.cache.scale_sh)];
    uint2 codes[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        codes[0][i] = *reinterpret_cast<const uint2 *>(p.cache.key + code_off + i * half);
        codes[1][i] = *reinterpret_cast<const uint2 *>(p.cache.value + code_off + i * half);
    }
    const int64_t to = b * p.out_sb + at(t, p.out_st) + at(h, p.out_sh) + d;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const float scale = scale_value(which ? pair >> 8 : pair & 0xffu);
        T *row = static_cast<T *>(which ? p.v_out : p.k_out) + to;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float x[8];
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                uint32_t lo, hi;
                decode4<CODE>(w ? codes[which][i].y : codes[which][i].x, lo, hi);
                const float2 a = __half22float2(*reinterpret_cast<__half2 *>(&lo));
                const float2 c = __half22float2(*reinterpret_cast<__half2 *>(&hi));
                x[4 * w] = a.x * scale; x[4 * w + 1] = a.y * scale;
                x[4 * w + 2] = c.x * scale; x[4 * w + 3] = c.y * scale;
            }
            Eight<T>::store(row + i * half, x);
        }
    }
}

// One warp a unit, single-element accesses.
template <typename T, int CODE>
__global__ void __launch_bounds__(kThreads) dequantize_scalar_kernel(const __grid_constant__ DequantizeParams p)
{
    wait_for_stream();
    const int b = blockIdx.y;
    const int lane = threadIdx.x & 31;
    constexpr int kWarps = kThreads / 32;
    const int64_t start = p.starts == nullptr ? 0 : load_index(p.starts, p.starts_i64, b);
    const int count = clipped_count(p.counts, p.counts_i64, b, p.tokens);
    const unsigned total = static_cast<unsigned>(p.tokens) * p.cache.kv_heads;
    for (int u = 0; u < kScalarUnits; ++u) {
        const unsigned unit = (blockIdx.x * kScalarUnits + u) * kWarps + (threadIdx.x >> 5);
        int t, h;
        unit_of(unit, p.div, p.heads_fastest, t, h);
        if (unit >= total || t >= count) continue;
        const int64_t pos = start + t;
        int64_t code_off, pair_off;
        int bad = 0;
        if (pos < 0 || pos >= p.cache.capacity) bad = SA_DEV_BAD_POSITION;
        else if (!locate_token(p.cache, b, static_cast<int>(pos), code_off, pair_off)) bad = SA_DEV_BAD_PAGE;
        if (bad != 0) {
            if (lane == 0) report(p.status, bad);
            continue;
        }
        code_off += h * p.cache.sh;
        const uint32_t pair = reinterpret_cast<const uint16_t *>(p.cache.scales)[pair_off + h * p.cache.scale_sh];
        const float sk = scale_value(pair & 0xffu), sv = scale_value(pair >> 8);
        const int64_t to = b * p.out_sb + t * p.out_st + h * p.out_sh;
        for (int i = lane; i < p.cache.head_dim; i += 32) {
            static_cast<T *>(p.k_out)[to + i] = Elem<T>::from_float(decode1<CODE>(p.cache.key[code_off + i]) * sk);
            static_cast<T *>(p.v_out)[to + i] = Elem<T>::from_float(decode1<CODE>(p.cache.value[code_off + i]) * sv);
        }
    }
}

int lane_shift_of(int dim)
{
    int shift = 0;
    while ((16 << shift) < dim) ++shift;
    return shift;
}

struct Launch {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    Launch(dim3 grid, int threads, cudaStream_t stream)
    {
        cfg.gridDim = grid;
        cfg.blockDim = dim3(threads);
        cfg.stream = stream;
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
    }
};

unsigned blocks_for(int64_t units, int per_block)
{
    return static_cast<unsigned>((units + per_block - 1) / per_block);
}

template <typename T, int CODE> cudaError_t quantize_typed(QuantizeParams p, bool vector, cudaStream_t stream)
{
    const int shift = vector ? lane_shift_of(p.cache.head_dim) : 5;
    const int per_block = (kThreads >> shift) * (vector ? 1 : kScalarUnits);
    p.kv_div = FastDiv(p.heads_fastest ? p.cache.kv_heads : p.tokens);
    p.q_div = FastDiv(p.heads_fastest ? std::max(p.q_heads, 1) : p.tokens);
    p.kv_blocks = static_cast<int>(blocks_for(static_cast<int64_t>(p.tokens) * p.cache.kv_heads, per_block));
    const unsigned q_blocks = p.q_in != nullptr ? blocks_for(static_cast<int64_t>(p.tokens) * p.q_heads, per_block) : 0;
    Launch rows(dim3(p.kv_blocks + q_blocks, p.batch), kThreads, stream);
    cudaError_t err;
    if (!vector) err = cudaLaunchKernelEx(&rows.cfg, quantize_scalar_kernel<T, CODE>, p);
    else if (p.cos != nullptr) err = cudaLaunchKernelEx(&rows.cfg, quantize_vector_kernel<T, CODE, true>, p, shift);
    else err = cudaLaunchKernelEx(&rows.cfg, quantize_vector_kernel<T, CODE, false>, p, shift);
    if (err != cudaSuccess || p.lens_out == nullptr || p.kv_blocks == 1) return err;
    Launch lengths(dim3(p.batch), 128, stream);
    return cudaLaunchKernelEx(&lengths.cfg, quantize_lengths_kernel, p);
}

template <typename T, int CODE> cudaError_t dequantize_typed(DequantizeParams p, bool vector, cudaStream_t stream)
{
    const int shift = vector ? lane_shift_of(p.cache.head_dim) : 5;
    p.div = FastDiv(p.heads_fastest ? p.cache.kv_heads : p.tokens);
    Launch rows(dim3(blocks_for(static_cast<int64_t>(p.tokens) * p.cache.kv_heads, (kThreads >> shift) * (vector ? 1 : kScalarUnits)), p.batch),
                kThreads, stream);
    return vector ? cudaLaunchKernelEx(&rows.cfg, dequantize_vector_kernel<T, CODE>, p, shift)
                  : cudaLaunchKernelEx(&rows.cfg, dequantize_scalar_kernel<T, CODE>, p);
}

}  // namespace

cudaError_t launch_quantize(QuantizeParams p, int code, int dtype, bool vector, cudaStream_t stream)
{
    const bool e4m3 = code == kCodeE4M3;
    if (dtype == SA_DTYPE_BF16)
        return e4m3 ? quantize_typed<__nv_bfloat16, kCodeE4M3>(p, vector, stream)
                    : quantize_typed<__nv_bfloat16, kCodeInt8>(p, vector, stream);
    if (dtype == SA_DTYPE_F16)
        return e4m3 ? quantize_typed<__half, kCodeE4M3>(p, vector, stream)
                    : quantize_typed<__half, kCodeInt8>(p, vector, stream);
    return e4m3 ? quantize_typed<float, kCodeE4M3>(p, vector, stream)
                : quantize_typed<float, kCodeInt8>(p, vector, stream);
}

cudaError_t launch_dequantize(DequantizeParams p, int code, int dtype, bool vector, cudaStream_t stream)
{
    const bool e4m3 = code == kCodeE4M3;
    if (dtype == SA_DTYPE_BF16)
        return e4m3 ? dequantize_typed<__nv_bfloat16, kCodeE4M3>(p, vector, stream)
                    : dequantize_typed<__nv_bfloat16, kCodeInt8>(p, vector, stream);
    if (dtype == SA_DTYPE_F16)
        return e4m3 ? dequantize_typed<__half, kCodeE4M3>(p, vector, stream)
                    : dequantize_typed<__half, kCodeInt8>(p, vector, stream);
    return e4m3 ? dequantize_typed<float, kCodeE4M3>(p, vector, stream)
                : dequantize_typed<float, kCodeInt8>(p, vector, stream);
}

}  // namespace sa
