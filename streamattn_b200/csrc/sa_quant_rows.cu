// Rows of an 8-bit KV cache: quantise new K/V rows (after rotating K) into a contiguous or paged
// cache, and read rows back.  The format is described in sa_quant.cuh.
//
// Both are one pass over the data and bound by memory: D * (element + 1) + 1 bytes a row.  A unit is
// the K and the V row of one (token, head); ceil(D / 8) lanes (rounded up to a power of two) share
// it, 8 elements each, so 16-bit rows move in 16-byte and codes in 8-byte pieces, the maximum of a
// row is a few shuffles, and the two scale bytes of a token leave in one 2-byte store.  Every
// thread requests all of its kUnits units before it looks at the first.  Rows that do not allow
// such accesses (odd sizes, odd strides) take one warp a unit with single-element accesses.
#include "sa_quant.cuh"

namespace sa {
namespace {

constexpr int kThreads = 256;
constexpr int kUnits = 4;        // units a lane group has in flight
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

// Writes position + count of row b where every page of the range exists (whole CTA; `bad` is the
// CTA's own shared flag).
__device__ __forceinline__ void store_length(const QuantizeParams &p, int b, const RowPlace &r, int *bad)
{
    if (threadIdx.x == 0) *bad = r.ok ? 0 : 1;
    __syncthreads();  // and: every thread of the CTA has read its position
    if (r.ok && p.cache.page_table != nullptr && r.count > 0) {
        const int first = r.start / p.cache.page_size, last = (r.start + r.count - 1) / p.cache.page_size;
        for (int lp = first + threadIdx.x; lp <= last; lp += blockDim.x) {
            const int64_t page = load_index(p.cache.page_table, p.cache.table_i64, static_cast<int64_t>(b) * p.cache.max_pages + lp);
            if (page < 0 || page >= p.cache.num_pages) *bad = 1;
        }
    }
    __syncthreads();
    if (threadIdx.x == 0 && *bad == 0) {
        if (p.pos_i64) static_cast<int64_t *>(p.lens_out)[b] = static_cast<int64_t>(r.start) + r.count;
        else static_cast<int32_t *>(p.lens_out)[b] = r.start + r.count;
    }
}

// unit -> (token, head)
__device__ __forceinline__ void unit_of(unsigned unit, unsigned heads, unsigned tokens, int heads_fastest, int &t, int &h)
{
    const unsigned inner = heads_fastest ? heads : tokens;
    const unsigned outer_index = unit / inner, inner_index = unit - outer_index * inner;
    t = static_cast<int>(heads_fastest ? outer_index : inner_index);
    h = static_cast<int>(heads_fastest ? inner_index : outer_index);
}

// One K or V row of a unit, eight elements a lane: scale byte from the maximum over the `lanes`
// lanes that share the row, then the codes.
template <int CODE> __device__ __forceinline__ int quantize_eight(const float (&x)[8], int lanes, uint2 &codes)
{
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = max(amax, __float_as_uint(x[i]) & 0x7fffffffu);  // a NaN is the largest
    for (int o = lanes >> 1; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const int e = scale_byte<CODE>(amax);
    const float inv = inverse_scale(e);
    codes.x = encode4<CODE>(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
    codes.y = encode4<CODE>(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv);
    if (e == kNanScaleByte) codes = make_uint2(0u, 0u);
    return e;
}

template <typename T, int CODE>
__global__ void __launch_bounds__(kThreads) quantize_vector_kernel(const __grid_constant__ QuantizeParams p, int lanes)
{
    __shared__ int bad;
    wait_for_stream();
    const int b = blockIdx.y;
    const int dim = p.cache.head_dim, half = dim >> 1;
    const int groups = kThreads / lanes;             // units the CTA handles at a time
    const int group = threadIdx.x / lanes;
    const int d = (threadIdx.x - group * lanes) * 8;
    const bool in_row = d < dim;
    const bool rope = p.cos != nullptr;
    const T *cos_b = static_cast<const T *>(p.cos) + b * p.rope_sb;
    const T *sin_b = static_cast<const T *>(p.sin) + b * p.rope_sb;

    if (static_cast<int>(blockIdx.x) >= p.kv_blocks) {  // query rows
        const int count = clipped_count(p.counts, p.counts_i64, b, p.tokens);
        const unsigned total = static_cast<unsigned>(p.tokens) * p.q_heads;
        const unsigned first = (blockIdx.x - p.kv_blocks) * groups * kUnits + group;
        for (int u = 0; u < kUnits; ++u) {
            const unsigned unit = first + u * groups;
            int t, h;
            unit_of(unit, p.q_heads, p.tokens, p.heads_fastest, t, h);
            if (unit >= total || t >= count || !in_row) continue;
            const T *src = static_cast<const T *>(p.q_in) + b * p.qi_sb + t * p.qi_st + h * p.qi_sh;
            Eight<T> raw;
            raw.load(src + d);
            float x[8];
            raw.get(x);
            if (rope) {
                float y[8], c[8], s[8];
                raw.load(src + (d < half ? d + half : d - half));
                raw.get(y);
                raw.load(cos_b + t * p.rope_st + d);
                raw.get(c);
                raw.load(sin_b + t * p.rope_st + d);
                raw.get(s);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = rotate(x[i], y[i], d < half, c[i], s[i]);
            }
            Eight<T>::store(static_cast<T *>(p.q_out) + b * p.qo_sb + t * p.qo_st + h * p.qo_sh + d, x);
        }
        return;
    }

    const RowPlace place = row_place(p, b);
    if (!place.ok && threadIdx.x == 0) report(p.status, SA_DEV_BAD_POSITION);
    const unsigned total = static_cast<unsigned>(p.tokens) * p.cache.kv_heads;   // < 2^30: the host checks
    const unsigned first = blockIdx.x * groups * kUnits + group;
    Eight<T> k[kUnits], v[kUnits], partner[kUnits];
    int t[kUnits], h[kUnits];
    bool active[kUnits];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        const unsigned unit = first + u * groups;
        unit_of(unit, p.cache.kv_heads, p.tokens, p.heads_fastest, t[u], h[u]);
        active[u] = place.ok && unit < total && t[u] < place.count;
        if (active[u] && in_row) {
            const int64_t src = b * p.new_sb + t[u] * p.new_st + h[u] * p.new_sh;
            k[u].load(static_cast<const T *>(p.k_new) + src + d);
            v[u].load(static_cast<const T *>(p.v_new) + src + d);
            if (rope) partner[u].load(static_cast<const T *>(p.k_new) + src + (d < half ? d + half : d - half));
        }
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        float x[8], y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = y[i] = 0.0f;   // lanes without a part of the row
        if (active[u] && in_row) {
            k[u].get(x);
            v[u].get(y);
            if (rope) {
                float other[8], c[8], s[8];
                Eight<T> raw;
                partner[u].get(other);
                raw.load(cos_b + t[u] * p.rope_st + d);
                raw.get(c);
                raw.load(sin_b + t[u] * p.rope_st + d);
                raw.get(s);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = rotate(x[i], other[i], d < half, c[i], s[i]);
            }
        }
        uint2 k_codes, v_codes;
        const int ek = quantize_eight<CODE>(x, lanes, k_codes);   // all lanes: shuffles inside
        const int ev = quantize_eight<CODE>(y, lanes, v_codes);
        if (!active[u] || !in_row) continue;
        int64_t code_off, pair_off;
        if (!locate_token(p.cache, b, place.start + t[u], code_off, pair_off)) {
            if (d == 0) report(p.status, SA_DEV_BAD_PAGE);
            continue;
        }
        code_off += h[u] * p.cache.sh + d;
        *reinterpret_cast<uint2 *>(p.cache.key + code_off) = k_codes;
        *reinterpret_cast<uint2 *>(p.cache.value + code_off) = v_codes;
        if (d == 0)
            reinterpret_cast<uint16_t *>(p.cache.scales)[pair_off + h[u] * p.cache.scale_sh] =
                static_cast<uint16_t>(ek | (ev << 8));
    }
    // The only CTA that reads this row's position may also replace it.
    if (p.lens_out != nullptr && p.kv_blocks == 1) store_length(p, b, place, &bad);
}

// One warp a unit, single-element accesses: any head_dim up to 256, any stride.
template <typename T, int CODE>
__global__ void __launch_bounds__(kThreads) quantize_scalar_kernel(const __grid_constant__ QuantizeParams p)
{
    __shared__ int bad;
    wait_for_stream();
    const int b = blockIdx.y;
    const int dim = p.cache.head_dim, half = dim >> 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int kWarps = kThreads / 32;
    const bool rope = p.cos != nullptr;
    const bool is_query = static_cast<int>(blockIdx.x) >= p.kv_blocks;
    // The query's CTAs must not read the position: another CTA may be replacing it.
    const RowPlace place = is_query ? RowPlace{0, clipped_count(p.counts, p.counts_i64, b, p.tokens), true} : row_place(p, b);
    const int heads = is_query ? p.q_heads : p.cache.kv_heads;
    const unsigned total = static_cast<unsigned>(p.tokens) * heads;
    const unsigned first = (blockIdx.x - (is_query ? p.kv_blocks : 0)) * kWarps * kUnits + warp;
    if (!is_query && !place.ok && threadIdx.x == 0) report(p.status, SA_DEV_BAD_POSITION);

    for (int u = 0; u < kUnits; ++u) {
        const unsigned unit = first + u * kWarps;
        int t, h;
        unit_of(unit, heads, p.tokens, p.heads_fastest, t, h);
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
    if (!is_query && p.lens_out != nullptr && p.kv_blocks == 1) store_length(p, b, place, &bad);
}

// Rows whose tokens were written by several CTAs: the lengths, after all of them.
__global__ void __launch_bounds__(128) quantize_lengths_kernel(const __grid_constant__ QuantizeParams p)
{
    __shared__ int bad;
    wait_for_stream();
    store_length(p, blockIdx.x, row_place(p, blockIdx.x), &bad);
}

template <typename T, int CODE, bool VECTOR>
__global__ void __launch_bounds__(kThreads) dequantize_kernel(const __grid_constant__ DequantizeParams p, int lanes)
{
    wait_for_stream();
    const int b = blockIdx.y;
    const int dim = p.cache.head_dim;
    const int groups = kThreads / lanes;
    const int group = threadIdx.x / lanes;
    const int d = (threadIdx.x - group * lanes) * (VECTOR ? 8 : 1);
    const int64_t start = p.starts == nullptr ? 0 : load_index(p.starts, p.starts_i64, b);
    const int count = clipped_count(p.counts, p.counts_i64, b, p.tokens);
    const unsigned total = static_cast<unsigned>(p.tokens) * p.cache.kv_heads;   // < 2^30: the host checks
    const unsigned first = blockIdx.x * groups * kUnits + group;
    uint2 k[kUnits], v[kUnits];
    uint32_t pair[kUnits];
    int64_t from[kUnits], to[kUnits];   // code offset of the unit's row (-1: nothing to do), output offset
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        const unsigned unit = first + u * groups;
        int t, h;
        unit_of(unit, p.cache.kv_heads, p.tokens, p.heads_fastest, t, h);
        from[u] = -1;
        if (unit >= total || t >= count || d >= dim) continue;
        const int64_t pos = start + t;
        int64_t code_off, pair_off;
        if (pos < 0 || pos >= p.cache.capacity) {
            if (d == 0) report(p.status, SA_DEV_BAD_POSITION);
        } else if (!locate_token(p.cache, b, static_cast<int>(pos), code_off, pair_off)) {
            if (d == 0) report(p.status, SA_DEV_BAD_PAGE);
        } else {
            from[u] = code_off + h * p.cache.sh;
            to[u] = b * p.out_sb + t * p.out_st + h * p.out_sh;
            pair[u] = reinterpret_cast<const uint16_t *>(p.cache.scales)[pair_off + h * p.cache.scale_sh];
            if (VECTOR) {
                k[u] = *reinterpret_cast<const uint2 *>(p.cache.key + from[u] + d);
                v[u] = *reinterpret_cast<const uint2 *>(p.cache.value + from[u] + d);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        if (from[u] < 0) continue;
        const float sk = scale_value(pair[u] & 0xffu), sv = scale_value(pair[u] >> 8);
        T *k_row = static_cast<T *>(p.k_out) + to[u], *v_row = static_cast<T *>(p.v_out) + to[u];
        if (VECTOR) {
            auto put = [&](uint2 codes, float scale, T *row) {
                float x[8];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t lo, hi;
                    decode4<CODE>(i ? codes.y : codes.x, lo, hi);
                    const float2 a = __half22float2(*reinterpret_cast<__half2 *>(&lo));
                    const float2 c = __half22float2(*reinterpret_cast<__half2 *>(&hi));
                    x[4 * i] = a.x * scale; x[4 * i + 1] = a.y * scale;
                    x[4 * i + 2] = c.x * scale; x[4 * i + 3] = c.y * scale;
                }
                Eight<T>::store(row + d, x);
            };
            put(k[u], sk, k_row);
            put(v[u], sv, v_row);
        } else {
            for (int i = d; i < dim; i += lanes) {
                k_row[i] = Elem<T>::from_float(decode1<CODE>(p.cache.key[from[u] + i]) * sk);
                v_row[i] = Elem<T>::from_float(decode1<CODE>(p.cache.value[from[u] + i]) * sv);
            }
        }
    }
}

int lanes_per_row(int dim)
{
    int lanes = 1;
    while (lanes * 8 < dim) lanes <<= 1;
    return lanes;
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

unsigned blocks_for(int64_t units, int groups)
{
    const int64_t per_block = static_cast<int64_t>(groups) * kUnits;
    return static_cast<unsigned>((units + per_block - 1) / per_block);
}

template <typename T, int CODE> cudaError_t quantize_typed(QuantizeParams p, bool vector, cudaStream_t stream)
{
    const int lanes = vector ? lanes_per_row(p.cache.head_dim) : 32;
    const int groups = kThreads / lanes;
    p.kv_blocks = static_cast<int>(blocks_for(static_cast<int64_t>(p.tokens) * p.cache.kv_heads, groups));
    const unsigned q_blocks = p.q_in != nullptr ? blocks_for(static_cast<int64_t>(p.tokens) * p.q_heads, groups) : 0;
    Launch rows(dim3(p.kv_blocks + q_blocks, p.batch), kThreads, stream);
    cudaError_t err = vector ? cudaLaunchKernelEx(&rows.cfg, quantize_vector_kernel<T, CODE>, p, lanes)
                             : cudaLaunchKernelEx(&rows.cfg, quantize_scalar_kernel<T, CODE>, p);
    if (err != cudaSuccess || p.lens_out == nullptr || p.kv_blocks == 1) return err;
    Launch lengths(dim3(p.batch), 128, stream);
    return cudaLaunchKernelEx(&lengths.cfg, quantize_lengths_kernel, p);
}

template <typename T, int CODE> cudaError_t dequantize_typed(const DequantizeParams &p, bool vector, cudaStream_t stream)
{
    const int lanes = vector ? lanes_per_row(p.cache.head_dim) : 32;
    const unsigned blocks = blocks_for(static_cast<int64_t>(p.tokens) * p.cache.kv_heads, kThreads / lanes);
    Launch rows(dim3(blocks, p.batch), kThreads, stream);
    return vector ? cudaLaunchKernelEx(&rows.cfg, dequantize_kernel<T, CODE, true>, p, lanes)
                  : cudaLaunchKernelEx(&rows.cfg, dequantize_kernel<T, CODE, false>, p, lanes);
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
