// What the streaming kernel does with a tile of an 8-bit cache: the query's operand registers, the
// products and the online softmax of one warp.  Used by stream_decode_kernel (sa_stream_kernel.cuh),
// which moves the tiles.
//
//   S^T[token, head] = K q^T          tokens on the M rows of the tensor-core instructions, heads on N
//   O^T[dim, head]  += V^T P^T
//
// q is multiplied by the power of two that brings its largest element to [2^14, 2^15) and becomes fp16: exact for
// all but elements some 2^28 times smaller than that one.  The codes of K and of V are converted to fp16, in which
// either type of them is exact, and the products accumulate in fp32.
// e4m3   There is an instruction with e4m3 operands, but on this GPU it executes as conversions and fp16 products:
//        measured 10 instructions and 16 cycles of the tensor pipe for its 16 x 8 x 32, where two fp16
//        instructions take the same.
// int8   The 8-bit integer instruction is native and needs no conversion of K, but it wants the query in bytes: two of
//        them hold every element to a step of 2^-16 of the largest, which loses the small elements of a
//        query that has a few large ones, however small the K channels under those are.
// P V uses fp16 for p too: it has a far larger range than two bytes hold (the tail of a long row may carry all of
// its weight at 2^-20 of the maximum a token).
//
// Every score is then multiplied by the token's K scale, 2^(e - 127 - k_down) exactly, and row_scale puts the powers
// of two right that the query took and k_down left out.  The products are below 2^31, the codes times their scale below
// 2^128, so scores at 2^-24 (k_down = 24) of the products stay finite for every finite K.
//
// p times the V scale is rounded to fp16 (2^-11; the denominator sums p in fp32).  It is taken relative to the largest such
// product so far, 2^(score - max + e - v_exp + lift + 15) <= 2^15 with v_exp the largest V byte so far and lift, a head's
// own, what the row's products stay below 2^15 by: at the top of fp16's range, where a small p or a small row of V keeps
// its eleven bits down to 2^-20 of the largest product and a part of them to 2^-30, however large the V rows are that
// hardly count (down to 2^-100).  `room` is at least what the products stay below the bound by.  While it is below kFreeRoom,
// as in any row whose V scales are of one order, lift is 0 and the tiles are not searched for their largest product; room
// may then be up to kFreeRoom too large, which lift leaves out.  Beside a form that knew v_exp alone, in which 2^26 between
// the V rows cost bits and 2^40 the smaller rows, this costs 1 % on long rows, 3 % on short ones and 4 to 6 % with 9 to 16
// heads.  The products are made before the branch: scores that change in it, for lift to go into their exponent, hold up
// every tile's exponentials, another 2 to 6 %.
//
// What bounds it (8 rows x 2 KV heads x 65536 tokens unless said otherwise): at D64 the instructions between two tiles as much
// as memory: 27.0 to 27.9 us (boxes differ), 4.9 to 5.05 TB/s, of which 5 us are launch, first tile and merge; 29.4 in pages of
// 64, 33.4 of 16.  Groups of 9 to 16 heads do both products twice per conversion and are bound by issue: 35.2 us.  int8 takes 30.8 and 38.6 us there: a
// word of codes becomes halves in five instructions against two.  At D128 a warp has one tile in flight, so what it
// computes adds to the wait for the next: 50.3 us e4m3, 5.4 TB/s, 55 int8, and 62 and 69 with 16 heads; with 8 KV heads of 4 and
// 1M tokens 336 and 347 us, 6.4 and 6.2 TB/s (int8 by integer products, which lost small elements of the query: 325).  What
// made the difference at first, at that D64 shape (its codes drawn uniformly): heads on M, tokens on N and one tile in four
// used 36.7 us; tokens on M (no padded rows) 33; e4m3 as fp16 instead of e4m3 instructions 29.4; scales as floats
// once a token, places once a tile, the rescale skipped while the maximum stands 27.2; instances by where the tokens
// lie 24.9.
#pragma once

#include <type_traits>
#include <utility>

#include "sa_quant.cuh"
#include "sa_stream.cuh"

namespace sa {
namespace {

// Shared-memory loads at a register plus a constant, which the instruction adds itself.
template <int OFFSET> __device__ __forceinline__ uint4 lds128(uint32_t addr)
{
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4 + %5];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(addr), "n"(OFFSET)
                 : "memory");
    return v;
}

template <int OFFSET> __device__ __forceinline__ uint2 lds64(uint32_t addr)
{
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2 + %3];" : "=r"(v.x), "=r"(v.y) : "r"(addr), "n"(OFFSET) : "memory");
    return v;
}

template <int OFFSET> __device__ __forceinline__ uint32_t lds32(uint32_t addr)
{
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1 + %2];" : "=r"(v) : "r"(addr), "n"(OFFSET) : "memory");
    return v;
}

template <int OFFSET> __device__ __forceinline__ float2 lds_float2(uint32_t addr)
{
    float2 v;
    asm volatile("ld.shared.v2.f32 {%0, %1}, [%2 + %3];" : "=f"(v.x), "=f"(v.y) : "r"(addr), "n"(OFFSET) : "memory");
    return v;
}

__device__ __forceinline__ void sts_float4(uint32_t addr, float a, float b, float c, float d)
{
    asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}

__device__ __forceinline__ void sts128_zero(uint32_t addr)
{
    asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(addr), "r"(0) : "memory");
}

// f(std::integral_constant<int, 0>) ... f(std::integral_constant<int, N - 1>): an unrolled loop whose index
// is a constant expression.
template <int N, typename F, int... I> __device__ __forceinline__ void unrolled(F &&f, std::integer_sequence<int, I...>)
{
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F> __device__ __forceinline__ void unrolled(F &&f)
{
    unrolled<N>(static_cast<F &&>(f), std::make_integer_sequence<int, N>{});
}

// FIRST: c is the product alone, not added to.
template <bool FIRST>
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    if constexpr (FIRST)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Four 8 x 16-byte matrices; lane i gives the address of row i % 8 of matrix i / 8.
template <int OFFSET> __device__ __forceinline__ void load_matrices(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4 + %5];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr), "n"(OFFSET)
                 : "memory");
}

// Transposes an 8 x 8 matrix of halves, two of a row's elements a lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t x)
{
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

__device__ __forceinline__ uint32_t pack_halves(float lo, float hi)
{
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}

// Which tokens a lane meets.  A 16-token tile's rows r and r + 8 are the neighbours tile_token(r) and
// tile_token(r) ^ 1, and lane (g, t4)'s columns 2 t4, 2 t4 + 1 of the second product are the four tokens
// 4 t4 .. 4 t4 + 3 in an order that depends on t4.  Both are chosen so that no two lanes of a load phase meet
// in a bank under the copies' swizzle: for D = 64 a 128-byte line holds two tokens and its 16-byte pieces are
// permuted with bits 1-2 of the token, for D = 128 with bits 0-2.
template <int D> __device__ __forceinline__ int token_flip(int t4) { return D == 64 ? (t4 ^ (t4 >> 1)) & 1 : t4 & 2; }
template <int D> __device__ __forceinline__ int tile_token(int r) { return 4 * (r >> 1) + (((r & 1) * 3) ^ token_flip<D>(r >> 1)); }

// Byte offset of 16-byte piece `chunk` of tile row `row`.
template <int D> __device__ __forceinline__ uint32_t piece(int row, int chunk)
{
    return row * D + ((D == 64 ? chunk ^ ((row >> 1) & 3) : chunk ^ (row & 7)) << 4);
}

constexpr float kFreeRoom = 8.0f;

// Powers of two by which p is raised when the products of p and V scale stay 2^room below their bound.
__device__ __forceinline__ float lift_of(float room) { return fmaxf(floorf(fminf(room, kFreeRoom + 100.0f)) - kFreeRoom, 0.0f); }

template <typename T, int D, bool ROWS16, int CODE> struct QuantWarp {
    static constexpr int TILE_N = kQuantTileTokens;  // two tokens' scales a lane
    static constexpr int NH = ROWS16 ? 2 : 1;     // groups of eight heads
    static constexpr int MT = TILE_N / 16;        // 16-token tiles
    static constexpr int KS = D / 32;             // k-steps of 32 dimensions
    static constexpr int DT = D / 16;             // output tiles

    // Operand registers of a k-step: two of each of its two instructions.
    uint32_t q[NH][KS][4];
    int k_down;                  // (warp) powers of two left out of the K scales, as the exponent field of a float
    float row_scale[NH][2];      // heads 2 t4 and 2 t4 + 1: what turns the products into base-2 scores
    float m[NH][2], l[NH][2];    // running maximum (in the products' unit) and this lane's part of the sum, of 2^lift p
    float room[NH][2];           // see above
    bool lifted;                 // (warp) room is kFreeRoom or more for one of the heads
    float o[NH][DT][4];          // in units of 2^(v_exp - 142 - lift)
    int v_exp;                   // largest scale byte of V so far, at least 16
    bool has_nan;                // a NaN scale was met: the result is NaN
    int nan_heads;               // bit 2 nh + h: the query of that head holds a NaN or an infinity, and its result is NaN

    // Query rows of `group` heads from head0 on; lane (g, t4) holds columns of head g of each eight.
    __device__ __forceinline__ void begin(const T *q0, int64_t stride, int group, float scale_log2, int g, int t4)
    {
        v_exp = 16;
        has_nan = false;
        nan_heads = 0;
        lifted = false;
        int up[NH];  // exponent of the factor of head g of each eight, in [-113, 140]
#pragma unroll
        for (int nh = 0; nh < NH; ++nh) {
            const bool ok = nh * 8 + g < group;
            const T *row = q0 + (nh * 8 + g) * stride;
            float x[KS][8];
            uint32_t amax = 0;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const int col = 32 * ks + 4 * t4 + (e >> 2) * 16 + (e & 2);
                    const uint32_t w = ok ? *reinterpret_cast<const uint32_t *>(row + col) : 0u;
                    const T *pair = reinterpret_cast<const T *>(&w);
                    x[ks][e] = Elem<T>::to_float(pair[0]);
                    x[ks][e + 1] = Elem<T>::to_float(pair[1]);
                    amax = max(amax, max(__float_as_uint(x[ks][e]) & 0x7fffffffu, __float_as_uint(x[ks][e + 1]) & 0x7fffffffu));
                }
            }
            amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            // m and l stay finite, as for NaN scales, so that no merge takes the state for an empty one.
            const bool finite = amax < 0x7f800000u;
            if (!finite) {
                amax = 0;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[ks][i] = 0.0f;
            }
            up[nh] = amax < (1u << 23) ? 0 : 14 + 127 - static_cast<int>(amax >> 23);  // (subnormal numbers count as zeros)
            const int up_half = up[nh] / 2;  // the factor in two steps: as one it might pass fp32's range
            const float f0 = __uint_as_float(static_cast<uint32_t>(127 + up_half) << 23);
            const float f1 = __uint_as_float(static_cast<uint32_t>(127 + up[nh] - up_half) << 23);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int i = 0; i < 8; ++i) x[ks][i] = x[ks][i] * f0 * f1;
            // A 32-bit word of K codes c0 .. c3 becomes the halves c0 c1 and c2 c3; a lane's word 4 t4 .. of the first
            // 16 bytes of a k-step meets the lane's word of the second 16 bytes in one instruction each.
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                q[nh][ks][0] = pack_halves(x[ks][0], x[ks][1]);
                q[nh][ks][1] = pack_halves(x[ks][4], x[ks][5]);
                q[nh][ks][2] = pack_halves(x[ks][2], x[ks][3]);
                q[nh][ks][3] = pack_halves(x[ks][6], x[ks][7]);
            }
            nan_heads |= (__shfl_sync(0xffffffffu, finite ? 0 : 1, 8 * t4) | __shfl_sync(0xffffffffu, finite ? 0 : 2, 8 * t4 + 4)) << (2 * nh);
            m[nh][0] = m[nh][1] = -INFINITY;
            l[nh][0] = l[nh][1] = 0.0f;
            room[nh][0] = room[nh][1] = INFINITY;
#pragma unroll
            for (int i = 0; i < DT; ++i) o[nh][i][0] = o[nh][i][1] = o[nh][i][2] = o[nh][i][3] = 0.0f;
        }
        // 24, and less only where a query of 2^90 or more would bring row_scale to the end of fp32's range.
        int down = 24;
#pragma unroll
        for (int nh = 0; nh < NH; ++nh) down = min(down, 100 + up[nh]);
        down = max(__reduce_min_sync(0xffffffffu, down), 0);
        k_down = down << 23;
#pragma unroll
        for (int nh = 0; nh < NH; ++nh) {
            const float scale = scale_log2 * __uint_as_float(static_cast<uint32_t>(127 + down - up[nh]) << 23);
            row_scale[nh][0] = __shfl_sync(0xffffffffu, scale, 8 * t4);
            row_scale[nh][1] = __shfl_sync(0xffffffffu, scale, 8 * t4 + 4);
        }
    }

    // One tile: codes at kb and vb, scale pairs at sb, room for TILE_N float pairs at fb (shared memory).
    // Tokens from n_valid on, and those of the fragments in `bad` (1 << frag_shift tokens each), are not there.
    __device__ __forceinline__ void tile(uint32_t kb, uint32_t vb, uint32_t sb, uint32_t fb, int n_valid, unsigned bad,
                                         int frag_shift, int lane, int g, int t4)
    {
        const bool partial = n_valid < TILE_N || bad != 0u;
        auto valid = [&](int tok) { return tok < n_valid && ((bad >> (tok >> frag_shift)) & 1u) == 0u; };

        // The scale bytes become floats once a token: K's 2^k_down too small, V's relative to the unit.  Tokens that are not
        // there get zeros, and so do their V codes: what the buffers hold for them is stale.
        uint32_t pairs = lds32<0>(sb + lane * 4);
        if (partial) {
            if (!valid(2 * lane)) pairs &= 0xffff0000u;
            if (!valid(2 * lane + 1)) pairs &= 0x0000ffffu;
            for (int i = lane; i < TILE_N * (D / 16); i += 32)
                if (!valid(i / (D / 16))) sts128_zero(vb + i * 16);
        }
        const uint32_t nan_bytes = __vcmpeq4(pairs, 0xffffffffu);
        pairs &= ~nan_bytes;
        const uint32_t my_top = max((pairs >> 8) & 0xffu, pairs >> 24);
        int top = static_cast<int>(__reduce_max_sync(0xffffffffu, nan_bytes != 0u ? 256u : my_top));
        if (top == 256) {
            has_nan = true;
            top = static_cast<int>(__reduce_max_sync(0xffffffffu, my_top));
        }
        const int old_exp = v_exp;
        v_exp = max(v_exp, top);
        const int off = (142 - v_exp) * (1 << 23);
        sts_float4(fb + lane * 16, __int_as_float(max(static_cast<int>((pairs << 23) & 0x7f800000u) - k_down, 0)),
                   __int_as_float(max(static_cast<int>((pairs << 15) & 0x7f800000u) + off, 0)),
                   __int_as_float(max(static_cast<int>((pairs << 7) & 0x7f800000u) - k_down, 0)),
                   __int_as_float(max(static_cast<int>((pairs >> 1) & 0x7f800000u) + off, 0)));
        __syncwarp();

        // Every 16-token tile has the same swizzle, so a lane's places in it are computed once a tile.
        const int row_g = tile_token<D>(g);
        const uint32_t f0 = fb + row_g * 8, f1 = fb + (row_g ^ 1) * 8;
        // K, matrix loads: matrices 0 and 2 are rows 0-7 of a 16-token tile, 1 and 3 rows 8-15; 0 and 1 are the first
        // 16 bytes of a k-step, 2 and 3 the second.
        const uint32_t k_at = piece<D>(tile_token<D>(lane & 7) ^ ((lane >> 3) & 1), lane >> 4);
        // V: the tokens of the lane's columns are tok, tok ^ 3 | tok ^ 1, tok ^ 2; D/8 bytes of each.
        const int tok = 4 * t4 + token_flip<D>(t4);
        uint32_t v_at[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int row = tok ^ (c == 0 ? 0 : c == 1 ? 3 : c == 2 ? 1 : 2);
            v_at[c] = vb + (D == 128 ? piece<D>(row, g) : piece<D>(row, g >> 1) + (g & 1) * 8);
        }

        float s[MT][NH][4];
        float v_weight[MT][2];
        uint32_t k_from[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) k_from[ks] = kb + (k_at ^ (ks << 5));
        unrolled<MT>([&](auto mt_c) {
            constexpr int mt = decltype(mt_c)::value;
            unrolled<KS>([&](auto ks_c) {
                constexpr int ks = decltype(ks_c)::value;
                uint32_t a[4];
                load_matrices<mt * 16 * D>(k_from[ks], a);
                uint32_t x[4], y[4];  // halves 0, 1 and 2, 3 of each word
#pragma unroll
                for (int i = 0; i < 4; ++i) decode4<CODE>(a[i], x[i], y[i]);
#pragma unroll
                for (int nh = 0; nh < NH; ++nh) {
                    mma_f16<ks == 0>(s[mt][nh], x[0], x[1], x[2], x[3], q[nh][ks][0], q[nh][ks][1]);
                    mma_f16<false>(s[mt][nh], y[0], y[1], y[2], y[3], q[nh][ks][2], q[nh][ks][3]);
                }
            });
            const float2 kv0 = lds_float2<mt * 128>(f0), kv1 = lds_float2<mt * 128>(f1);
            v_weight[mt][0] = kv0.y;
            v_weight[mt][1] = kv1.y;
#pragma unroll
            for (int nh = 0; nh < NH; ++nh) {
                s[mt][nh][0] *= kv0.x;
                s[mt][nh][1] *= kv0.x;
                s[mt][nh][2] *= kv1.x;
                s[mt][nh][3] *= kv1.x;
            }
        });
        if (partial) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                const bool ok0 = valid(mt * 16 + row_g), ok1 = valid(mt * 16 + (row_g ^ 1));
#pragma unroll
                for (int nh = 0; nh < NH; ++nh) {
                    if (!ok0) s[mt][nh][0] = s[mt][nh][1] = -INFINITY;
                    if (!ok1) s[mt][nh][2] = s[mt][nh][3] = -INFINITY;
                }
            }
        }

        // Online softmax.  The running maximum is subtracted before row_scale is applied, so that the largest p
        // is exactly 1 however large the scores are (fma(s, scale, -max * scale) makes it 2^(rounding of the product)).
        float alpha[NH][2], sum[NH][2];
        bool same = v_exp == old_exp && !lifted;
#pragma unroll
        for (int nh = 0; nh < NH; ++nh) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float x = -INFINITY;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) x = fmaxf(x, fmaxf(s[mt][nh][h], s[mt][nh][2 + h]));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                same = same && !(x > m[nh][h]);
                x = fmaxf(m[nh][h], x);
                const float sub = x == -INFINITY ? 0.0f : x;
                alpha[nh][h] = (m[nh][h] - sub) * row_scale[nh][h];  // -inf for the first tokens
                m[nh][h] = x;
                // The scores become p times the V scale, before it is known whether the sums so far have to be rescaled.
                sum[nh][h] = 0.0f;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const float p0 = exp2f((s[mt][nh][h] - sub) * row_scale[nh][h]), p1 = exp2f((s[mt][nh][2 + h] - sub) * row_scale[nh][h]);
                    sum[nh][h] += p0 + p1;
                    s[mt][nh][h] = p0 * v_weight[mt][0];
                    s[mt][nh][2 + h] = p1 * v_weight[mt][1];
                }
            }
        }
        if (!__all_sync(0xffffffffu, same)) {  // a new maximum or unit, or lift is in use: after a row's first tiles rarely
            const float rise = static_cast<float>(v_exp - old_exp);
            bool free = true;
#pragma unroll
            for (int nh = 0; nh < NH; ++nh)
#pragma unroll
                for (int h = 0; h < 2; ++h) free = free && room[nh][h] - alpha[nh][h] + rise < kFreeRoom;
            if (!__all_sync(0xffffffffu, free)) {
                lifted = find_room(s, sum, alpha, rise);
            } else {
#pragma unroll
                for (int nh = 0; nh < NH; ++nh)
#pragma unroll
                    for (int h = 0; h < 2; ++h) room[nh][h] = room[nh][h] - alpha[nh][h] + rise;
            }
#pragma unroll
            for (int nh = 0; nh < NH; ++nh) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    l[nh][h] *= exp2f(alpha[nh][h]);
                    alpha[nh][h] = exp2f(alpha[nh][h] - rise);
                }
#pragma unroll
                for (int i = 0; i < DT; ++i) {
                    o[nh][i][0] *= alpha[nh][0];
                    o[nh][i][1] *= alpha[nh][1];
                    o[nh][i][2] *= alpha[nh][0];
                    o[nh][i][3] *= alpha[nh][1];
                }
            }
        }

#pragma unroll
        for (int nh = 0; nh < NH; ++nh) {
            l[nh][0] += sum[nh][0];
            l[nh][1] += sum[nh][1];
        }
        unrolled<MT>([&](auto mt_c) {
            constexpr int mt = decltype(mt_c)::value;
            uint32_t b[NH][2];
#pragma unroll
            for (int nh = 0; nh < NH; ++nh) {
                b[nh][0] = transpose8(pack_halves(s[mt][nh][0], s[mt][nh][1]));
                b[nh][1] = transpose8(pack_halves(s[mt][nh][2], s[mt][nh][3]));
            }
            // The lane's D/8 bytes of its four tokens; two tokens are interleaved byte by byte, so that one
            // conversion yields one operand register.  Byte 2 i is row g of output tile i, byte 2 i + 1 row g + 8.
            uint32_t v[4][D / 32];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                if constexpr (D == 128) {
                    const uint4 x = lds128<mt * 16 * D>(v_at[c]);
                    v[c][0] = x.x; v[c][1] = x.y; v[c][2] = x.z; v[c][3] = x.w;
                } else {
                    const uint2 x = lds64<mt * 16 * D>(v_at[c]);
                    v[c][0] = x.x; v[c][1] = x.y;
                }
            }
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                uint32_t a[2][4];
                decode4<CODE>(__byte_perm(v[0][i], v[1][i], 0x5140), a[0][0], a[0][1]);
                decode4<CODE>(__byte_perm(v[0][i], v[1][i], 0x7362), a[1][0], a[1][1]);
                decode4<CODE>(__byte_perm(v[2][i], v[3][i], 0x5140), a[0][2], a[0][3]);
                decode4<CODE>(__byte_perm(v[2][i], v[3][i], 0x7362), a[1][2], a[1][3]);
#pragma unroll
                for (int nh = 0; nh < NH; ++nh) {
                    mma_f16<false>(o[nh][2 * i], a[0][0], a[0][1], a[0][2], a[0][3], b[nh][0], b[nh][1]);
                    mma_f16<false>(o[nh][2 * i + 1], a[1][0], a[1][1], a[1][2], a[1][3], b[nh][0], b[nh][1]);
                }
            }
        });
    }

    // Finds how far the tile's largest products w = p * (V scale) lie below their bound 2^15.  Where that leaves room they and
    // the tile's sums of p are raised, and `fall`, by which the sums so far are scaled, takes the change of lift in.
    // Whether one of the heads has kFreeRoom or more.
    __device__ __forceinline__ bool find_room(float (&w)[MT][NH][4], float (&sum)[NH][2], float (&fall)[NH][2], float rise)
    {
        bool any = false;
#pragma unroll
        for (int nh = 0; nh < NH; ++nh) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float x = 0.0f;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) x = fmaxf(x, fmaxf(w[mt][nh][h], w[mt][nh][2 + h]));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                const float before = lift_of(room[nh][h]);
                room[nh][h] = fminf(room[nh][h] - fall[nh][h] + rise, static_cast<float>(142 - (__float_as_int(x) >> 23)));
                const float lift = lift_of(room[nh][h]), up = exp2f(lift);
                sum[nh][h] *= up;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    w[mt][nh][h] *= up;
                    w[mt][nh][2 + h] *= up;
                }
                fall[nh][h] += lift - before;
                any = any || room[nh][h] >= kFreeRoom;
            }
        }
        return __any_sync(0xffffffffu, any);
    }

    // The warp's state into its area: rows of `stride` floats, (o[D], m, l), m in base-2 scores.
    __device__ __forceinline__ void store(float *area, int stride, int g, int t4)
    {
        const float unit = __uint_as_float(static_cast<uint32_t>(v_exp - 15) << 23);  // 2^(v_exp - 142)
#pragma unroll
        for (int nh = 0; nh < NH; ++nh) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float sum = l[nh][h];
                sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                const float lower = lifted ? exp2f(-lift_of(room[nh][h])) : 1.0f;
                float *row = area + (nh * 8 + 2 * t4 + h) * stride;
#pragma unroll
                for (int i = 0; i < DT; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        row[g * (D / 8) + 2 * i + e] = has_nan || ((nan_heads >> (2 * nh + h)) & 1) ? __uint_as_float(0x7fffffffu) : o[nh][i][2 * e + h] * lower * unit;
                if (g == 0) {
                    row[D] = m[nh][h] * row_scale[nh][h];
                    row[D + 1] = sum * lower;
                }
            }
        }
    }
};

}  // namespace
}  // namespace sa
