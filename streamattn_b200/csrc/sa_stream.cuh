// Host-side description of one launch of the streaming (TMA + tensor core) kernel.
#pragma once

#include "sa_common.cuh"

namespace sa {

#ifndef SA_STREAM_WARPS
#define SA_STREAM_WARPS 8
#endif
constexpr int kStreamWarps = SA_STREAM_WARPS;    // each with its own ring of tiles
#ifndef SA_STREAM_STAGES
#define SA_STREAM_STAGES 1
#endif
constexpr int kStreamStages = SA_STREAM_STAGES;  // 16 KB K+V tiles in flight per warp
#ifndef SA_QW64
#define SA_QW64 8
#define SA_QT64 64
#define SA_QS64 2
#endif
#ifndef SA_QW128
#define SA_QW128 8
#define SA_QT128 64
#define SA_QS128 1
#endif
__host__ __device__ constexpr int quant_tile_tokens(int head_dim) { return head_dim == 64 ? SA_QT64 : SA_QT128; }  // 8-bit caches: 8 KB (D64) or 16 KB (D128) of codes a tile

constexpr int warps_of(int head_dim, bool rows16, bool quant) { return !quant ? kStreamWarps : rows16 ? 8 : head_dim == 64 ? SA_QW64 : SA_QW128; }

// Tiles in flight per warp (the state areas of 16 head rows at D128 leave room for fewer).
constexpr int stages_of(int head_dim, bool rows16, bool quant)
{
    if (quant) return rows16 ? 8192 / (quant_tile_tokens(head_dim) * head_dim) : head_dim == 64 ? SA_QS64 : SA_QS128;
    return (head_dim == 128 && rows16 && kStreamStages > 2) ? 2 : kStreamStages;
}

constexpr int kCpMaxWorld = SA_CP_MAX_WORLD;
constexpr int kCpFuseWorld = 8;  // ranks the fused decode+exchange launch supports (one NVSwitch box)

// How the CTAs that share one (row, kv head) pair divide its tiles (pairs with at least four
// CTAs each; otherwise the tile list is cut into equal slices regardless of pair boundaries).
enum StreamSchedule : int {
    kScheduleBlocked = 0,  // one contiguous slice per CTA
    kScheduleCyclic = 1,   // tiles dealt round-robin to the pair's warps
    kScheduleClaims = 2,   // first tiles round-robin, then one claim per tile from a device counter
};

// Context-parallel exchange fused into the decode launch: where the ranks' gather buffers are.
//   gather[2][world][rows][D+2] of 64-bit words (step << 32 | float bits); gather_words_per_parity counts words.
struct CpFuse {
    int world;  // 0 = not a context-parallel launch
    int rank;
    uint32_t step;
    uint64_t bases[kCpMaxWorld];
    unsigned long long gather_words_per_parity;
    void *final_out;  // [batch, q_heads, D] in the query dtype
};

struct StreamGeometry {
    CUtensorMap map_k;
    CUtensorMap map_v;
    int frag_tokens;     // rows of one TMA box
    int frags_per_tile;  // boxes per 8 KB tile
    int frags_per_unit;  // boxes per page / seed block
    int tok_dim;         // TMA coordinate carrying the token index (1 or 2)
    int uniform_tiles;   // tiles per row if all rows are equally long, else -1
    int num_ctas;
    int kv_split;        // groups of more than 16 query heads: virtual KV heads per physical one (else 1)
    int schedule;        // how the CTAs of one (row, kv head) pair share its tiles (kSchedule*)
    int first_merges;    // a pair's first CTA merges its split states (grids of at most one CTA per SM); else a ticket elects the last arriver
};

// Smallest s with group % s == 0 and group / s <= 16 (0 if there is none): a KV head with more
// than 16 query heads is served as s virtual KV heads that read the same K/V rows.
int stream_kv_split(int group);
int stream_tile_tokens(int head_dim, bool quant);
int stream_stages(int head_dim, bool rows16, bool quant);
size_t stream_smem_bytes(int head_dim, bool rows16, int stages, int batch, bool quant);
constexpr size_t kStreamSmemLimit = 227 * 1024 - 64;

// The instances over 8-bit caches, in translation units of their own.
struct StreamParams;
cudaError_t launch_stream_e4m3(const CUtensorMap &mk, const CUtensorMap &mv, const StreamParams &sp, int dtype, int head_dim,
                               int ctas, cudaStream_t stream);
cudaError_t launch_stream_int8(const CUtensorMap &mk, const CUtensorMap &mv, const StreamParams &sp, int dtype, int head_dim,
                               int ctas, cudaStream_t stream);
cudaError_t launch_stream(const Problem &p, const StreamGeometry &geo, const CpFuse &cp, cudaStream_t stream);

}  // namespace sa
