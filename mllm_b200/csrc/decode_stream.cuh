// The argument block and the plan of the even-split decode (decode_stream.cu), shared with the shared-prefix
// decode (shared_prefix.cu).
#pragma once

#include "common.cuh"
#include "host_util.h"
#include "kv_layout.cuh"

namespace mllm_b200 {

constexpr int kMaxGroup = 8;       // query heads per kv head (the N side of the MMAs)

constexpr int kPlanPer = 0, kPlanPair = 1, kPlanSingle = 2, kPlanHead = 3;

struct StreamArgs {
    const __nv_bfloat16* q;        // [B, H, D]
    const int32_t* kv_lens;        // [B]
    __nv_bfloat16* out;            // [B, H * D]
    float* part_o;                 // parts: rows of D floats ...
    float* part_lse;               // ... and log2 of their weights
    int* plan;                     // [kPlanHead + B * Hkv]: what the kernels work out for one another (kPlan*), then
                                   // the first tile of every pair that has any
    int B, H, Hkv, n_rep, max_len;
    int ctas;                      // two per SM
    int direct;                    // the bound on the lengths says that every pair gets a CTA of its own
    float scale_log2;
    KvLayout lay;
    // shared prefix: rows before first_row are the prefix kernel's, which leaves plan[kPlanPair] parts of every query
    // row of the first pair_seqs sequences, plan[kPlanSingle] of the others', at row prefix_base of the parts:
    // [part][kv head][sequence][head of the group]
    int first_row;
    int shared;                    // there is a prefix, and its kernel let this grid in
    int pair_seqs;
    int64_t prefix_base;
    // The prefix kernel waits for all that ran before the call, then publishes `ticket` here, a number of this call only;
    // whoever reads it back is ordered behind that wait.  The joining kernel clears it, for a graph's next replay.
    unsigned long long* ready;
    unsigned long long ticket;
};

__device__ __forceinline__ void publish_ticket(const StreamArgs& a) {
    asm volatile("st.release.gpu.global.u64 [%0], %1;" ::"l"(a.ready), "l"(a.ticket) : "memory");
}

__device__ __forceinline__ bool ticket_published(const StreamArgs& a) {
    unsigned long long t;
    asm volatile("ld.acquire.gpu.global.u64 %0, [%1];" : "=l"(t) : "l"(a.ready) : "memory");
    return t == a.ticket;
}

// Rows [first_row, len) of a sequence in tiles of TILE cache rows.  A length outside [0, max_len] is recorded and
// clamped; a sequence shorter than the prefix (an empty one too) has no rows here, and no prefix either.
struct SeqTiles {
    int len, first_tile, tiles;
    bool short_len;
};

template <int TILE>
__device__ __forceinline__ SeqTiles seq_tiles(const StreamArgs& a, int b) {
    SeqTiles s;
    int len = a.kv_lens[b];
    if (len < 0 || len > a.max_len || (len > 0 && len < a.first_row)) {
        record_error(kErrBadLength);
        len = len < 0 ? 0 : min(len, a.max_len);
    }
    s.short_len = len < a.first_row;
    s.len = len;
    s.first_tile = a.first_row / TILE;
    s.tiles = len > a.first_row ? (len + TILE - 1) / TILE - s.first_tile : 0;
    return s;
}

// Tiles of all pairs, and those of the longest (the lanes of a full warp, lane given); the host has checked that the most
// there can be plus a grid fits 31 bits.
template <int TILE>
__device__ __forceinline__ int total_tiles(const StreamArgs& a, int lane, int* longest = nullptr) {
    int n = 0, top = 0;
    for (int b = lane; b < a.B; b += 32) {
        const int t = seq_tiles<TILE>(a, b).tiles;
        n += t;
        top = max(top, t);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        n += __shfl_xor_sync(0xffffffffu, n, o);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    if (longest) *longest = top;
    return n * a.Hkv;
}

// Small calls: where every pair can have a CTA and the longest is a few tiles, CTA i takes pair i, nothing is cut and
// nothing is left to join.  Measured against cutting (one sequence, 4 kv heads of 64, tiles of 128 rows): 1 tile 3.6 us
// against 6.1, 5 tiles 6.4 against 7.3, 8 tiles 8.5 against 7.3; for 16 sequences still 8.6 against 8.7 at 8.  The rule is
// on the tiles there are, so that a longer bound gives the same bits; where the bound itself is that short, the host leaves
// the joining kernel out.
constexpr int kDirectTiles = 6;

__host__ __device__ __forceinline__ bool direct_pairs(int64_t pairs, int longest, int ctas, int shared) {
    return !shared && pairs <= ctas && longest <= kDirectTiles;
}

// CTAs the tiles are dealt to: two per SM, which stay; behind a prefix kernel up to four times as many, so that the SMs
// that become free first take more of them (with two per SM, the ones that had to wait for a prefix CTA's SM ended
// last), but only where each has a few tiles.  It follows from the tiles there are, not from a bound on them: a graph
// captured for longer sequences gives the same bits.
constexpr int kSharedWaves = 4;
constexpr int kWaveTiles = 4;

__host__ __device__ __forceinline__ int stream_ctas(int64_t tiles, int ctas, int shared) {
    int64_t n = ctas;
    if (shared) {
        const int64_t waves = tiles / kWaveTiles < (int64_t)kSharedWaves * ctas ? tiles / kWaveTiles
                                                                                : (int64_t)kSharedWaves * ctas;
        if (waves > n) n = waves;
    }
    if (n > tiles) n = tiles;
    return n < 1 ? 1 : (int)n;
}

__device__ __forceinline__ int tiles_per_cta(const StreamArgs& a, int total) {
    const int n = stream_ctas(total, a.ctas, a.shared);
    return max((total + n - 1) / n, 1);
}

// The CTAs whose stretches hold a pair's tiles, from its first tile p0 on the line of tiles: first .. first + count - 1.
// `ctas` is the most there can be, which the workspace has slots for.  False where p0 is not a place on that line: it was
// never written, since the CTA that the pair begins in gave up a wait, and the workspace may hold anything there.
__host__ __device__ __forceinline__ bool own_parts(int p0, int tiles, int per, int ctas, int* first, int* count) {
    *first = *count = 0;
    if (tiles == 0) return true;
    const int64_t last = ((int64_t)p0 + tiles - 1) / per;
    if (p0 < 0 || last >= ctas) return false;
    *first = p0 / per;
    *count = (int)last - *first + 1;
    return true;
}

// CTAs that the tiles may be dealt to: those that the workspace has slots for.
__host__ __device__ __forceinline__ int most_ctas(int ctas, int shared) { return shared ? kSharedWaves * ctas : ctas; }

// The workspace: the ticket, `part_rows` rows of D floats, their weights, the plan.
// Rows of parts the even-split decode writes: two slots a CTA, and with a shared prefix one per pair.
size_t stream_part_rows(int n_rep, int batch, int num_kv_heads, bool shared);
size_t stream_workspace_bytes(int D, size_t part_rows, int batch, int num_kv_heads);
void stream_place(StreamArgs& a, void* workspace, int D, size_t part_rows);

struct Kv8View;

// Runs the split and the combine kernel over a bf16 paged cache, or an 8-bit one.
int launch_stream_bf16(StreamArgs& a, int head_dim, const CUtensorMap& tmK, const CUtensorMap& tmV, int num_sms,
                       cudaStream_t s);
int launch_stream_kv8(StreamArgs& a, int head_dim, const mllm_paged_kv8* kv, const Kv8View& view, int num_sms,
                      cudaStream_t s);

}  // namespace mllm_b200
