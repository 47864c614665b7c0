// The streaming decode kernel over 16-bit caches, and the host side of every form of it.
#include "sa_stream_kernel.cuh"

namespace sa {

#ifdef SA_TIMELINE
// Instrumented builds only: where the kernels write their per-CTA time stamps (16 words per CTA).
unsigned long long *g_timeline = nullptr;
extern "C" __attribute__((visibility("default"))) void sa_debug_timeline(void *ptr)
{
    g_timeline = static_cast<unsigned long long *>(ptr);
}
#endif

int stream_kv_split(int group)
{
    for (int s = 1; s <= group; ++s)
        if (group % s == 0 && group / s <= 16) return s;
    return 0;
}

int stream_tile_tokens(int head_dim, bool quant) { return quant ? kQuantTileTokens : kTileBytes / (head_dim * 2); }

int stream_stages(int head_dim, bool rows16, bool quant) { return stages_of(head_dim, rows16, quant); }

size_t stream_smem_bytes(int head_dim, bool rows16, int stages, int batch, bool quant, bool solo)
{
    const size_t warps = kStreamWarps;
    const size_t bars = (warps * stages * 8 + 15) / 16 * 16;
    // Per-warp (o, m, l) areas plus (16-bit caches) the context-parallel staging rows (8-byte words).
    const size_t states = (solo ? 2 * warps : warps + (quant ? 0 : 2)) * (rows16 ? 16 : 8) * (head_dim + 2) * 4;
    const size_t scratch = warps * 32 * 6 * 4;  // merges: 6 floats per thread
    // A stage: K and V tile, for 8-bit caches with the tile's scale bytes.
    const size_t stage = quant ? static_cast<size_t>(kQuantTileTokens) * (2 * head_dim + 2) : 2 * kTileBytes;
    const size_t floats = quant ? warps * kQuantTileTokens * 8 : 0;
    return 1024 + warps * stages * stage + floats + bars + states + scratch + (2 * static_cast<size_t>(batch) + 1) * 4 + 16;
}

cudaError_t launch_stream(const Problem &p, const StreamGeometry &geo, const CpFuse &cp, cudaStream_t stream)
{
    StreamParams sp;
    sp.q = p.q;
    sp.q_sb = p.q_sb;
    sp.q_sh = p.q_sh;
    sp.out = p.out;
    sp.out_mode = p.out_mode;
    sp.partials = p.ws.partials;
    sp.counters = p.ws.counters;
    sp.pool = p.ws.counters + static_cast<size_t>(p.batch) * p.q_heads;
    sp.status = p.ws.status;
    sp.trace = p.trace;
    sp.batch = p.batch;
    sp.q_heads = p.q_heads;
    sp.kv_heads = p.kv_heads * geo.kv_split;
    sp.group = p.q_heads / sp.kv_heads;
    sp.kv_split = geo.kv_split;
    sp.scale_log2 = kLog2e / sqrtf(static_cast<float>(p.head_dim));
    sp.frag_tokens = geo.frag_tokens;
    sp.frags_per_tile = geo.frags_per_tile;
    sp.frags_per_unit = geo.frags_per_unit;
    auto log2i = [](int x) { int s = 0; while ((1 << s) < x) ++s; return s; };
    sp.frag_shift = log2i(geo.frag_tokens);
    sp.fpt_shift = log2i(geo.frags_per_tile);
    sp.fpu_shift = log2i(geo.frags_per_unit);
    sp.tok_dim = geo.tok_dim;
    // A row subset makes the rows' tile counts differ (rows left out have none).
    sp.uniform_tiles = p.seq.num_rows >= 0 ? -1 : geo.uniform_tiles;
    sp.schedule = geo.schedule;
    // More pairs than CTAs: slices cut by warps, which need room for two states a warp - up to 8 query heads a KV head, and at
    // D128 up to some 2800 rows.
    sp.solo = p.quant.code != kCodeNone && sp.group <= 8 && static_cast<int64_t>(p.batch) * sp.kv_heads > geo.num_ctas &&
              stream_smem_bytes(p.head_dim, false, stages_of(p.head_dim, false, true), p.batch, true, true) <= kStreamSmemLimit;
    sp.wait_ns = p.wait_ns;
    sp.first_merges = geo.first_merges;
    sp.seq = p.seq;
    sp.quant = p.quant;
    sp.key = p.k;
    sp.value = p.v;
    sp.cp = cp;
#ifdef SA_TIMELINE
    sp.timeline = g_timeline;
#endif
    if (p.quant.code == kCodeE4M3) return launch_stream_e4m3(geo.map_k, geo.map_v, sp, p.dtype, p.head_dim, geo.num_ctas, stream);
    if (p.quant.code == kCodeInt8) return launch_stream_int8(geo.map_k, geo.map_v, sp, p.dtype, p.head_dim, geo.num_ctas, stream);
    return launch_code<kCodeNone>(geo.map_k, geo.map_v, sp, p.dtype, p.head_dim, geo.num_ctas, stream);
}

}  // namespace sa
