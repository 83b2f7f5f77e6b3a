// Decode attention for a batch whose sequences share their first rows (a system prompt, a document).
//
// With P shared rows the plain decode reads them once per sequence.  Here the query rows of all sequences of one
// kv head meet the prefix together: a [B * n_rep, D] x [D, P] product per kv head, which reads the prefix once and
// is work for the tensor cores; every sequence's own rows go through the even-split decode (decode_stream.cu), and
// its combine kernel joins the parts of both by their maxima and sums.
//
// prefix_kernel: one CTA per (kv head, block of query rows, stretch of the prefix); the machinery is that of the
// prefill kernel (tcgen05.mma M = 128, scores and O in tensor memory, one softmax thread per row, TMA ring with
// separate K and V barriers), without a causal bound and in two forms:
//   a pair of query tiles: 256 query rows share every K/V tile.  For batches of more than 128 rows, where the tensor
//       and exponential work per K/V byte is what bounds.
//   a single query tile (a small batch, or the odd tile of a large one): the two softmax groups take alternate K/V
//       tiles, each with its own running maximum, sum and O, and are joined at the end.  With few rows the kernel is
//       bound by the K/V bytes; alternating keeps one tile's products running under the other's softmax.
// A query tile holds floor(128 / n_rep) sequences with their n_rep heads, fetched by one TMA box
// {64 columns, n_rep heads, sequences}; rows behind them are never looked at.  Warps without a valid row skip
// their softmax.  The stretches are dealt out by what a K/V tile costs each form.
// A stretch leaves one normalised fp32 row and log2 weight per query row.  The rows of a tile are contiguous in the
// parts; they go through shared memory (the tiles are done with by then), because a thread holds a whole row in tensor
// memory and 32 threads storing 16 bytes of 32 rows at a time took 4 us of a 16 us kernel.
// The rows of the last K/V tile behind the prefix are other rows of the block: K's are masked, V's read as zero
// through a tensor map that ends with the prefix, so that their contents cannot matter.
// Over an 8-bit cache four more warps fetch the rows and store them as the exact bf16 values where TMA would have put
// them; all else is the same, and so are the bits of a stretch's results.  For a pair that hides behind the softmax (128 sequences
// behind 8192 rows: 61 us, bf16 59), a single tile's pace it sets (4 behind 32700: 53 us, bf16 41).
//
// P is bf16 for the second product (A and B of an MMA have one type, and V is bf16); sums and O are fp32.
#include <algorithm>
#include <atomic>
#include <chrono>
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "decode_stream.cuh"
#include "host_util.h"
#include "kv8.cuh"
#include "kv_layout.cuh"
#include "tcgen05.cuh"

namespace mllm_b200 {
namespace {

constexpr int kBM = 128;            // query rows per tile
constexpr int kBN = 128;            // cache rows per K/V tile
// Threads: {producer, MMA, 2 idle warps}, softmax group 0, softmax group 1, for an 8-bit cache the converting warps.
// The register split of the prefill kernel: 128 x 72 + 256 x 216 = 384 x 168; with converting warps 256 x 56 +
// 256 x 200 = 512 x 128.
template <bool k8>
struct Split {
    static constexpr int kThreads = k8 ? 512 : 384;
    static constexpr int kLaunch = k8 ? 128 : 168;
    static constexpr int kLow = k8 ? 56 : 72;
    static constexpr int kHigh = k8 ? 200 : 216;
    static_assert((kThreads - 256) * kLow + 256 * kHigh <= kThreads * kLaunch, "register split exceeds the launch");
};
constexpr int kBox = kBN * 128;     // one 128-row x 64-column bf16 box (16 KB)
constexpr uint32_t kTmemCols = 512; // S_0, S_1, O_0, O_1 of 128 columns
constexpr float kRescaleThreshold = 8.0f;  // log2 units: O is rescaled only when the maximum grows by more

// kPairs: the launch has pairs of query tiles; without, a third stage takes the place of the second Q tile.
template <int D, bool kPairs, bool k8 = false>
struct PrefixCfg {
    static constexpr int kBoxes = D / 64;
    static constexpr int kTileBytes = kBoxes * kBox;                 // one Q, K or V tile
    static constexpr int kQTiles = kPairs ? 2 : 1;
    static constexpr int kStages = D == 128 ? (kPairs || k8 ? 2 : 3) : 4;
    static constexpr int kOwnTile = k8 ? 128 : 64;                   // cache rows per tile of the even-split decode
    static constexpr int kRing = D == 128 && kPairs ? 2 : 4;         // 8-bit K or V tiles on their way to be converted ...
    static constexpr int kRingBytes = kBN * D + kBN;                 // ... and their rows' exponents
    static constexpr int kRowFloats = D + 4;                         // of a result row in shared memory (bank spread)
    static constexpr int kSmemBytes = (kQTiles + 2 * kStages) * kTileBytes + 256 + (k8 ? kRing * kRingBytes : 0) + 1024;
    static_assert((1 + 4 * kStages + 6) * 8 + 4 <= 256, "barrier area too small");
    static_assert(kSmemBytes <= 232448, "more shared memory than a CTA has");
    static_assert(2 * kBM * (kRowFloats + 2) * 4 <= (kQTiles + 2 * kStages) * kTileBytes, "results do not fit");
};

struct PrefixArgs {
    float* part_o;       // [parts][Hkv][B][n_rep][D]
    float* part_lse;     // [parts][Hkv][B][n_rep]
    int B, Hkv, n_rep, seqs;   // seqs: sequences per query tile
    int prefix, n_tiles;       // K/V tiles of the prefix
    int pairs, single;         // blocks of two query tiles; whether one more block follows with the tile left
    int num_sms;
    float scale_log2;
    KvLayout lay;
};

// How the prefix is cut: stretches and K/V tiles in each, for a pair's block and for the single tile's.
struct PrefixCut {
    int splits, per, splits_single, per_single;
};

// Blocks get stretches by their cost per K/V tile, 3 for a pair and 2 for a single tile, so that the CTAs of `sms` SMs
// per kv head end together; of an 8-bit cache, where converting the tile is most of a single one's cost, alike (64
// sequences of 40 heads behind 16000 rows: 81 us, by 3 to 2 101).  More SMs never give fewer stretches.
template <bool k8>
__host__ __device__ inline PrefixCut cut_prefix(int n_tiles, int sms, int pairs, int single) {
    PrefixCut c = {};
    int want_single = 0;
    if (single) {
        want_single = k8 ? sms / (pairs + 1) : 2 * sms / (3 * pairs + 2);
        if (want_single < 1) want_single = 1;
        c.per_single = (n_tiles + want_single - 1) / want_single;
        c.splits_single = (n_tiles + c.per_single - 1) / c.per_single;
    }
    if (pairs) {
        int want = (sms - want_single) / pairs;
        if (want < 1) want = 1;
        c.per = (n_tiles + want - 1) / want;
        c.splits = (n_tiles + c.per - 1) / c.per;
    }
    return c;
}

// SMs per kv head for the prefix, so that it ends with the decode of the sequences' own rows on the other SMs: with P
// and S the SM-microseconds of the two, F the fixed time of a prefix CTA and N SMs, X SMs take F + P / X, and all is
// done after (P + S + F X) / N.  Fitted (D = 128): 2.2 us a tile for a pair, 1.4 for a single tile (0.9 beside pairs; 8-bit 2.2
// and 1.4), 4 us for the CTA; 0.55 us for a 64-row tile of the other kernel and 1.8 us of an SM for each of its CTAs.  D = 64 moves half and
// takes 0.4 of it.  Over 75 shapes timed at every X (2 to 128 sequences, prefixes of 512 to 24000 rows, 64 to 2000 own)
// this X is 1.2 % off the best one on average and 13 % at most; too few SMs cost most (64 sequences of 40 heads behind
// 32700 rows: 138 us with 9, 114 with 10, 115 with 11).
template <bool k8>
__device__ __forceinline__ int prefix_sms(const PrefixArgs& a, float own_tiles, float dim_scale) {
    const float N = (float)a.num_sms, F = 4.f;
    const float single = k8 ? (a.pairs ? 1.4f : 2.2f) : (a.pairs ? 0.9f : 1.4f);
    const float P = (float)a.Hkv * a.n_tiles * (2.2f * a.pairs + single * a.single) * dim_scale;
    const float S = 0.55f * own_tiles * dim_scale + 1.8f * fminf(own_tiles, 2.f * N);
    const float b = P + S - N * F;
    const float X = (sqrtf(b * b + 4.f * F * N * P) - b) / (2.f * F);
    return max(1, min(a.num_sms / a.Hkv, (int)(X / a.Hkv + 0.5f)));
}

__device__ __forceinline__ uint32_t col_s(int i) { return (uint32_t)(i * kBN); }
__device__ __forceinline__ uint32_t col_o(int i) { return (uint32_t)(2 * kBN + i * 128); }

// The barriers of a CTA, in shared memory behind the tiles.
template <int ST>
struct Bars {
    uint64_t *q_full, *k_full, *k_empty, *v_full, *v_empty;   // [1], then [ST] each
    uint64_t *s_full, *p_full, *o_done;                       // [2] per softmax group
    __device__ __forceinline__ explicit Bars(uint64_t* p)
        : q_full(p), k_full(p + 1), k_empty(k_full + ST), v_full(k_empty + ST), v_empty(v_full + ST),
          s_full(v_empty + ST), p_full(s_full + 2), o_done(p_full + 2) {}
};

// The converting warps of an 8-bit cache: thread t takes the 16-byte chunk t % CH of the rows CH (t / CH) .. + CH - 1
// (CH chunks a row) of every K and V tile, fetched into a ring of its own (cp.async), works out the exact bf16 values
// and stores them where TMA would have put them.  The exponents of a group's rows are fetched by its first lane.  Rows
// behind the prefix become zeros.  What it costs is latency: one warp a scheduler, so the next row is loaded before the
// present one is stored (62 -> 55 us for 4 sequences behind 32700 rows) and the tile where the prefix ends has a form of
// its own (55 -> 53).  Bit operations and a bf16 multiplication in place of the conversions took 70.
template <int D, bool kPairs>
__device__ __forceinline__ void convert_tiles(const PrefixArgs& a, const Kv8View& kv, uint8_t* sKV, uint8_t* ring,
                                              uint64_t* bars, int holder, int g, int first, int n) {
    using C = PrefixCfg<D, kPairs, true>;
    constexpr int ST = C::kStages, R = C::kRing, CH = D / 16;
    const Bars<ST> bar(bars);
    const int t = threadIdx.x & 127, lane = t & 31;
    const int c = t % CH, r0 = t / CH * CH;
    int blk = 0, row = 0;      // of tile base + lane
    int base = -32;
    auto fetch = [&](int h) {  // half tile h: K or V of tile h / 2
        if (h < 2 * n) {
            const int j = h >> 1;
            if (j >= base + 32) {
                base += 32;
                blk = row = 0;
                if (base + lane < n) kv_locate(a.lay, holder, (int64_t)(first + base + lane) * kBN, blk, row);   // a bad
            }                                                                                  // entry reads block 0
            const int at = __shfl_sync(0xffffffffu, blk, j - base), top = __shfl_sync(0xffffffffu, row, j - base) + r0;
            const uint32_t slot = smem_u32(ring + (h % R) * C::kRingBytes);
            const uint8_t* src = (h & 1 ? kv.v_pool : kv.k_pool) + at * kv.p_sb + g * kv.p_sh + top * kv.p_st + 16 * c;
#pragma unroll
            for (int i = 0; i < CH; ++i)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(slot + (r0 + i) * D + 16 * c),
                             "l"(src + i * kv.p_st)
                             : "memory");
            if (c == 0) {
                const uint8_t* exp = (h & 1 ? kv.v_exp : kv.k_exp) + at * kv.e_sb + g * kv.e_sh + top;
                asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(slot + kBN * D + r0), "l"(exp), "n"(CH)
                             : "memory");
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int h = 0; h < R - 1; ++h) fetch(h);
    for (int h = 0; h < 2 * n; ++h) {
        fetch(h + R - 1);
        const int j = h >> 1, stage = j % ST;
        const int lim = h & 1 ? a.prefix - (first + j) * kBN : kBN;   // V rows behind the prefix count as zero
        asm volatile("cp.async.wait_group %0;" ::"n"(R - 1) : "memory");
        const bool ok = mbar_wait(h & 1 ? &bar.v_empty[stage] : &bar.k_empty[stage], ((j / ST) & 1) ^ 1);
        if (!__all_sync(0xffffffffu, ok)) break;
        __syncwarp();   // the exponents that the group's first lane fetched are there
        const uint8_t* slot = ring + (h % R) * C::kRingBytes;
        uint8_t* dst = sKV + (stage * 2 + (h & 1)) * C::kTileBytes + (c >> 2) * kBox;
        uint32_t ex[CH / 4];
#pragma unroll
        for (int i = 0; i < CH / 4; ++i) ex[i] = *reinterpret_cast<const uint32_t*>(slot + kBN * D + r0 + 4 * i);
        auto load = [&](int i) { return *reinterpret_cast<const uint4*>(slot + (r0 + i) * D + 16 * c); };
        auto convert = [&](auto ends) {
            constexpr bool kEnds = decltype(ends)::value;   // the prefix ends in this tile
            uint4 w = load(0);
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                const uint4 next = load(i + 1 < CH ? i + 1 : i);   // before the stores, which it might alias for all
                const int r = r0 + i;                              // the compiler knows
                const float sc = exp_byte_scale((ex[i / 4] >> (8 * (i % 4))) & 0xFFu);
                const uint32_t in[4] = {w.x, w.y, w.z, w.w};
                uint32_t o[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t h2 = e4m3x2_to_f16x2((uint16_t)(in[e >> 1] >> (16 * (e & 1))));
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h2));
                    float x, y;
                    mul2(x, y, f.x, f.y, sc, sc);
                    o[e] = pack_bf16x2(x, y);   // exact: 4 significant bits times a power of two
                    if (kEnds && r >= lim) o[e] = 0u;
                }
                const int k = (c & 3) * 2;
                *reinterpret_cast<uint4*>(dst + r * 128 + ((k ^ (r & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
                *reinterpret_cast<uint4*>(dst + r * 128 + (((k + 1) ^ (r & 7)) << 4)) = make_uint4(o[4], o[5], o[6], o[7]);
                w = next;
            }
        };
        if (lim < kBN) convert(std::true_type{});
        else convert(std::false_type{});
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(h & 1 ? &bar.v_full[stage] : &bar.k_full[stage]);
        __syncwarp();   // all have read the exponents before the slot is fetched into again
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

// The tensor pipe's thread: for every step and group O += P V, then the group's next S = Q K^T, so that one group's
// softmax runs under the other's products.  Step k of group i works on tile k (kPair) or 2 k + i.
template <int D, bool kPairs, bool kPair, bool k8>
__device__ __forceinline__ void issue_products(uint8_t* sQ, uint8_t* sKV, uint64_t* bars, uint32_t tmem, int n) {
    using C = PrefixCfg<D, kPairs, k8>;
    constexpr int ST = C::kStages;
    const Bars<ST> bar(bars);
    constexpr uint32_t idesc_s = idesc_bf16_f32(kBM, kBN, false);
    constexpr uint32_t idesc_o = idesc_bf16_f32(kBM, D, true);
    constexpr uint32_t desc_hi = smem_desc_hi_sw128(1024);
    const int steps[2] = {kPair ? n : (n + 1) / 2, kPair ? n : n / 2};
    auto tile_of = [&](int i, int k) { return kPair ? k : 2 * k + i; };
    auto issue_s = [&](int i, int j) {
        const uint32_t qd = smem_desc_lo(smem_u32(sQ + (kPair ? i : 0) * C::kTileBytes), 16);
        const uint32_t kd = smem_desc_lo(smem_u32(sKV + (j % ST) * 2 * C::kTileBytes), 16);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            const uint32_t off = (uint32_t)(((ks >> 2) * kBox + (ks & 3) * 32) >> 4);
            tc_mma_ss_w(tmem + col_s(i), qd + off, kd + off, desc_hi, idesc_s, ks > 0 ? 1u : 0u);
        }
        tc_commit(&bar.s_full[i]);
    };
    // K tile j has been read by every product that needs it: free it if it will be refilled
    auto free_k = [&](int j) { if (j + ST < n) tc_commit(&bar.k_empty[j % ST]); };
    bool alive = mbar_wait(bar.q_full, 0);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (!alive || steps[i] == 0) continue;
        const int j = tile_of(i, 0);
        if ((i == 0 || !kPair) && !mbar_wait(&bar.k_full[j % ST], (j / ST) & 1)) { alive = false; continue; }
        tc_fence_after();
        issue_s(i, j);
        if (!kPair || i == 1) free_k(j);
    }
    for (int k = 0; k < steps[0] && alive; ++k) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (!alive || k >= steps[i]) continue;
            const int j = tile_of(i, k);
            if (!mbar_wait(&bar.p_full[i], k & 1)) { alive = false; continue; }
            if ((!kPair || i == 0) && !mbar_wait(&bar.v_full[j % ST], (j / ST) & 1)) { alive = false; continue; }
            tc_fence_after();
            const uint32_t vd = smem_desc_lo(smem_u32(sKV + (j % ST) * 2 * C::kTileBytes + C::kTileBytes), kBox);
#pragma unroll
            for (int ks = 0; ks < kBN / 16; ++ks)
                tc_mma_ts_w(tmem + col_o(i), tmem + col_s(i) + ks * 8, vd + (uint32_t)((ks * 16 * 128) >> 4), desc_hi,
                            idesc_o, (k > 0 || ks > 0) ? 1u : 0u);
            const bool last_use = !kPair || i == 1;
            if (last_use && j + ST < n) tc_commit(&bar.v_empty[j % ST]);
            if (k + 1 < steps[i]) {
                const int jn = tile_of(i, k + 1);
                if ((!kPair || i == 0) && !mbar_wait(&bar.k_full[jn % ST], (jn / ST) & 1)) { alive = false; continue; }
                tc_fence_after();
                issue_s(i, jn);   // overwrites P_i(k) only after the product above read it
                if (last_use) free_k(jn);
            } else {
                tc_commit(&bar.o_done[i]);
            }
        }
    }
}

template <int D, bool kPairs, bool k8>
__global__ void __launch_bounds__(Split<k8>::kThreads, 1)
    prefix_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmVend, PrefixArgs a,
                  StreamArgs st, Kv8View kv) {
    using C = PrefixCfg<D, kPairs, k8>;
    constexpr int kOwnTile = C::kOwnTile;
    constexpr int ST = C::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sQ = smem;
    uint8_t* sKV = sQ + C::kQTiles * C::kTileBytes;      // [ST][K | V]
    uint64_t* bars = reinterpret_cast<uint64_t*>(sKV + ST * 2 * C::kTileBytes);
    const Bars<ST> bar(bars);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar.o_done + 2);
    uint8_t* ring = reinterpret_cast<uint8_t*>(bars) + 256;   // k8

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    pdl_wait();
    // what ran before the call is complete: say so to the decode of the sequences' own rows, which runs beside this grid
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) publish_ticket(st);
    // ---- the plan, the same in every CTA: from the tiles that the other kernel will find ----
    __shared__ PrefixCut s_cut;
    __shared__ int s_holder;
    if (warp == 2) {
        // the first sequence that has the prefix: its table row is the one to read (others may be empty)
        int holder = -1;
        for (int base = 0; base < a.B && holder < 0; base += 32) {
            const bool has = base + lane < a.B && !seq_tiles<kOwnTile>(st, base + lane).short_len;
            const unsigned m = __ballot_sync(0xffffffffu, has);
            if (m != 0u) holder = base + __ffs(m) - 1;
        }
        const int own = total_tiles<kOwnTile>(st, lane);
        if (lane == 0) {
            s_holder = holder;
            s_cut = cut_prefix<k8>(a.n_tiles, prefix_sms<k8>(a, (float)own, D == 128 ? 1.f : 0.4f), a.pairs, a.single);
            if (blockIdx.x == 0 && blockIdx.y == 0) {
                st.plan[kPlanPair] = s_cut.splits;
                st.plan[kPlanSingle] = s_cut.splits_single;
            }
        }
    }
    __syncthreads();
    const int holder = s_holder;
    if (holder < 0) return;                                               // nobody has it
    const PrefixCut cut = s_cut;
    const int g = blockIdx.x;
    const int y = blockIdx.y;
    if (y >= a.pairs * cut.splits + cut.splits_single) return;            // fewer stretches than the most there may be
    const int mb = y < a.pairs * cut.splits ? y / cut.splits : a.pairs;   // a.pairs: the single tile's block
    const bool pair = kPairs && mb < a.pairs;
    const int split = y - mb * cut.splits;
    const int per = pair ? cut.per : cut.per_single;
    const int first = split * per;                       // K/V tiles first .. first + n - 1
    const int n = min(per, a.n_tiles - first);
    // Step k of softmax group i works on tile k (pair) or 2 k + i (alternating); group i has steps[i] steps.
    const int steps[2] = {pair ? n : (n + 1) / 2, pair ? n : n / 2};

    if (threadIdx.x == 0) {
        mbar_init(bar.q_full, 1);
        for (int s = 0; s < ST; ++s) {
            mbar_init(&bar.k_full[s], k8 ? 128 : 1);
            mbar_init(&bar.k_empty[s], 1);
            mbar_init(&bar.v_full[s], k8 ? 128 : 1);
            mbar_init(&bar.v_empty[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar.s_full[i], 1);
            mbar_init(&bar.p_full[i], 128);
            mbar_init(&bar.o_done[i], 1);
        }
        mbar_fence_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_trigger();   // the decode of the sequences' own rows may fill SMs as these CTAs leave them

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Split<k8>::kLow));
        if (warp == 0) {
            // ------------------------------- TMA producer -------------------------------
            if (lane == 0) {
                tma_prefetch_desc(&tmQ);
                if constexpr (!k8) {
                    tma_prefetch_desc(&tmK);
                    tma_prefetch_desc(&tmV);
                }
                const int q_tiles = pair ? 2 : 1;
                const uint32_t q_box = 128u * (uint32_t)(a.n_rep * a.seqs);   // bytes of one 64-column box
                mbar_arrive_expect_tx(bar.q_full, (uint32_t)q_tiles * C::kBoxes * q_box);
                for (int i = 0; i < q_tiles; ++i)
                    for (int bx = 0; bx < C::kBoxes; ++bx)
                        tma_load_4d(sQ + i * C::kTileBytes + bx * kBox, &tmQ, bar.q_full, bx * 64, g * a.n_rep,
                                    (2 * mb + i) * a.seqs, 0);
                for (int j = 0; !k8 && j < n; ++j) {
                    const int stage = j % ST;
                    const uint32_t phase = ((j / ST) & 1) ^ 1;
                    uint8_t* sk = sKV + stage * 2 * C::kTileBytes;
                    uint8_t* sv = sk + C::kTileBytes;
                    int blk, row;
                    kv_locate(a.lay, holder, (int64_t)(first + j) * kBN, blk, row);   // a bad entry reads block 0
                    const CUtensorMap* mv = first + j == a.n_tiles - 1 ? &tmVend : &tmV;
                    if (!mbar_wait(&bar.k_empty[stage], phase)) break;
                    mbar_arrive_expect_tx(&bar.k_full[stage], C::kTileBytes);
#pragma unroll
                    for (int bx = 0; bx < C::kBoxes; ++bx)
                        tma_load_4d(sk + bx * kBox, &tmK, &bar.k_full[stage], bx * 64, row, g, blk);
                    if (!mbar_wait(&bar.v_empty[stage], phase)) break;
                    mbar_arrive_expect_tx(&bar.v_full[stage], C::kTileBytes);
#pragma unroll
                    for (int bx = 0; bx < C::kBoxes; ++bx)
                        tma_load_4d(sv + bx * kBox, mv, &bar.v_full[stage], bx * 64, row, g, blk);
                }
            }
        } else if (warp == 1 && lane == 0) {
            if constexpr (kPairs) {
                if (pair) issue_products<D, kPairs, true, k8>(sQ, sKV, bars, tmem, n);
                else issue_products<D, kPairs, false, k8>(sQ, sKV, bars, tmem, n);
            } else {
                issue_products<D, kPairs, false, k8>(sQ, sKV, bars, tmem, n);
            }
        }
    } else if (k8 && warp >= 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Split<k8>::kLow));
        if constexpr (k8) convert_tiles<D, kPairs>(a, kv, sKV, ring, bars, holder, g, first, n);
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Split<k8>::kHigh));
        // --------------------------------- softmax ---------------------------------
        const int grp = (warp - 4) >> 2;
        const int quad = warp & 3;               // TMEM lane quadrant of this warp
        const int row = quad * 32 + lane;
        const int qt = 2 * mb + (pair ? grp : 0);
        const int b = qt * a.seqs + row / a.n_rep;
        const bool valid = row < a.seqs * a.n_rep && b < a.B;
        const bool work = __any_sync(0xffffffffu, valid);   // a warp without a valid row only keeps the barriers going
        const uint32_t t_lane = tmem + ((uint32_t)(quad * 32) << 16);
        const uint32_t t_s = t_lane + col_s(grp);
        const uint32_t t_o = t_lane + col_o(grp);
        constexpr int kAcc = 8;
        float m_run = -INFINITY, l_run = 0.f;
        bool alive = true;
        const int ns = grp == 0 ? steps[0] : steps[1];
        for (int k = 0; k < ns; ++k) {
            if (!mbar_wait(&bar.s_full[grp], k & 1)) { alive = false; break; }
            tc_fence_after();
            if (work) {
                const int j = first + (pair ? k : 2 * k + grp);
                float sv[kBN];
#pragma unroll
                for (int c = 0; c < kBN / 32; ++c)
                    tmem_ld32(t_s + c * 32, *reinterpret_cast<float(*)[32]>(&sv[c * 32]));
                tmem_wait_ld();
                const int lim = a.prefix - j * kBN;     // columns before this one are prefix rows
                if (lim < kBN) {
#pragma unroll
                    for (int c = 0; c < kBN; ++c) sv[c] = c < lim ? sv[c] : -INFINITY;
                }
                float mx[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) mx[i] = fmaxf(sv[2 * i], sv[2 * i + 1]);
#pragma unroll
                for (int c = 8; c < kBN; c += 8)
#pragma unroll
                    for (int i = 0; i < 4; ++i) mx[i] = fmax3(mx[i], sv[c + 2 * i], sv[c + 2 * i + 1]);
                mx[0] = fmax3(mx[0], mx[1], fmaxf(mx[2], mx[3]));
                const float mt = mx[0] * a.scale_log2;
                const float m_new = fmaxf(m_run, mt);
                const bool grow = (m_new - m_run) > kRescaleThreshold;   // true on the first tile
                float m_use = grow ? m_new : m_run;
                if (m_use == -INFINITY) m_use = 0.f;
                const float alpha = grow ? ex2_approx(m_run - m_use) : 1.f;
                if (k > 0 && __any_sync(0xffffffffu, grow)) {
                    // the product of step k - 1 is complete (S of step k completed after it)
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) {
                        float o[32];
                        tmem_ld32(t_o + c * 32, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] *= alpha;
                        tmem_st32(t_o + c * 32, o);
                    }
                }
                const float neg_m = -m_use;
                float sum[kAcc];
#pragma unroll
                for (int i = 0; i < kAcc; ++i) sum[i] = 0.f;
#pragma unroll
                for (int c = 0; c < kBN / 32; ++c) {
                    uint32_t pk[16];
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        float x0, x1;
                        fma2(x0, x1, sv[c * 32 + e], sv[c * 32 + e + 1], a.scale_log2, a.scale_log2, neg_m, neg_m);
                        const float p0 = ex2_approx(x0);
                        const float p1 = ex2_approx(x1);
                        add2(sum[(e >> 1) % 4 * 2], sum[(e >> 1) % 4 * 2 + 1], p0, p1);
                        pk[e >> 1] = pack_bf16x2(p0, p1);
                    }
                    tmem_st16(t_s + c * 16, pk);
                }
                tmem_wait_st();
                add2(sum[0], sum[1], sum[2], sum[3]);
                add2(sum[4], sum[5], sum[6], sum[7]);
                add2(sum[0], sum[1], sum[4], sum[5]);
                l_run = l_run * alpha + (sum[0] + sum[1]);
                m_run = m_new == -INFINITY ? -INFINITY : m_use;   // a tile of -inf scores sets no maximum
            }
            tc_fence_before();
            mbar_arrive(&bar.p_full[grp]);
        }
        alive = ns > 0 && alive && mbar_wait(&bar.o_done[grp], 0);
        // Once both groups' products are complete, the tiles' memory is free for the result rows: scaled to their final
        // weight when they are written there, so that joining two groups' rows is an addition.
        float* s_rows = reinterpret_cast<float*>(smem);                       // [2][128][kRowFloats]
        float* s_stat = s_rows + 2 * kBM * C::kRowFloats;                     // [2][128][2]: maximum and sum
        float* my_stat = s_stat + (grp * kBM + row) * 2;
        const int64_t base = (((int64_t)split * a.Hkv + g) * a.B + (int64_t)qt * a.seqs) * a.n_rep;   // row 0's part
        const int rows = min(a.seqs, a.B - qt * a.seqs) * a.n_rep;            // valid rows of this query tile
        if (!alive) l_run = 0.f;
        asm volatile("bar.sync 1, 256;" ::: "memory");   // before it the other group's products may still read the tiles
        if (!pair) {
            my_stat[0] = l_run != 0.f ? m_run : -INFINITY;
            my_stat[1] = l_run;
            asm volatile("bar.sync 1, 256;" ::: "memory");
        }
        if (work) {
            float f = l_run != 0.f ? 1.f / l_run : 0.f, lse = l_run != 0.f ? m_run + log2f(l_run) : -INFINITY;
            if (!pair) {
                const float2 other = *reinterpret_cast<const float2*>(s_stat + ((grp ^ 1) * kBM + row) * 2);
                const float M = fmaxf(my_stat[0], other.x);
                const float mine = l_run != 0.f ? ex2_approx(m_run - M) : 0.f;
                const float L = l_run * mine + (other.y != 0.f ? other.y * ex2_approx(other.x - M) : 0.f);
                f = mine != 0.f ? mine / L : 0.f;
                lse = L != 0.f ? M + log2f(L) : -INFINITY;
            }
            if (valid && (pair || grp == 0)) a.part_lse[base + row] = lse;
            float* dst = s_rows + (grp * kBM + row) * C::kRowFloats;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                float o[32];
                if (alive) {   // a group without a step has no O
                    tmem_ld32(t_o + c * 32, o);
                    tmem_wait_ld();
                }
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    const bool any = f != 0.f;
                    *reinterpret_cast<float4*>(dst + c * 32 + i) =
                        any ? make_float4(o[i] * f, o[i + 1] * f, o[i + 2] * f, o[i + 3] * f) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
            }
        }
        constexpr int kLanes = D / 4;                 // lanes that move one row, 16 bytes each
        constexpr int kRows = 32 / kLanes;            // rows a warp moves at a time
        const int lr = lane / kLanes, d = lane % kLanes * 4;
        float* part = a.part_o + base * D + d;
        if (pair) {
            __syncwarp();                             // a warp writes out the rows that it holds
            const float* src = s_rows + grp * kBM * C::kRowFloats + d;
#pragma unroll 8
            for (int i = 0; i < 32; i += kRows) {
                const int r = quad * 32 + i + lr;
                if (r < rows)
                    *reinterpret_cast<float4*>(part + (int64_t)r * D) =
                        *reinterpret_cast<const float4*>(src + r * C::kRowFloats);
            }
        } else {
            asm volatile("bar.sync 1, 256;" ::: "memory");
            const float* src = s_rows + d;
#pragma unroll 8
            for (int i = 0; i < kBM; i += 8 * kRows) {
                const int r = i + (warp - 4) * kRows + lr;
                if (r < rows) {
                    const float4 x = *reinterpret_cast<const float4*>(src + r * C::kRowFloats);
                    const float4 y = *reinterpret_cast<const float4*>(src + (kBM + r) * C::kRowFloats);
                    *reinterpret_cast<float4*>(part + (int64_t)r * D) = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

// Query tiles of `seqs` sequences, taken in pairs, and the most stretches they may be cut into.
struct PrefixPlan {
    int seqs, pairs, single;
    PrefixCut most;
};

template <bool k8>
PrefixPlan plan_prefix(int B, int Hkv, int n_rep, int prefix, int num_sms) {
    PrefixPlan p = {};
    p.seqs = kBM / n_rep;
    const int q_tiles = (B + p.seqs - 1) / p.seqs;
    p.pairs = q_tiles / 2;
    p.single = q_tiles % 2;
    p.most = cut_prefix<k8>((prefix + kBN - 1) / kBN, std::max(1, num_sms / Hkv), p.pairs, p.single);
    return p;
}

constexpr int kMaxSms = 160;

size_t shared_part_rows(int B, int H, int Hkv, int prefix) {
    // parts of the prefix: a block has no more stretches than SMs per kv head on the largest GPU, and than tiles
    const int n_rep = H / Hkv;
    const size_t parts = prefix > 0 ? std::min(std::max(1, kMaxSms / Hkv), (prefix + kBN - 1) / kBN) : 0;
    return stream_part_rows(n_rep, B, Hkv, true) + parts * Hkv * B * n_rep;
}

// A number that no other call of this process has, and that bytes left in a workspace do not hold by chance: a counter
// through a bijection of 64 bits (the finaliser of splitmix64, Steele, Lea and Flood 2014).
unsigned long long next_ticket() {
    static std::atomic<unsigned long long> calls{
        (unsigned long long)std::chrono::steady_clock::now().time_since_epoch().count() << 20};
    unsigned long long z = calls.fetch_add(1, std::memory_order_relaxed) * 0x9E3779B97F4A7C15ull;
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    z ^= z >> 31;
    return z != 0ull ? z : next_ticket();   // 0 is what a call leaves behind
}

struct PrefixMaps {
    CUtensorMap q, k, v, v_end;   // of an 8-bit cache q only
};

template <int D, bool kPairs, bool k8>
int launch_prefix_d(const PrefixArgs& a, const StreamArgs& sa, const PrefixPlan& p, const PrefixMaps& m, const Kv8View& kv,
                    cudaStream_t s) {
    auto kern = prefix_kernel<D, kPairs, k8>;
    // setmaxnreg is only safe if the compiled kernel launches with the registers the split was sized for
    static int regs_ok = -1;
    if (regs_ok < 0) {
        cudaFuncAttributes attr;
        if (int st = check_cuda(cudaFuncGetAttributes(&attr, (const void*)kern), "prefix_kernel attributes")) return st;
        regs_ok = attr.numRegs >= Split<k8>::kLaunch ? MLLM_OK : MLLM_ERR_UNSUPPORTED;
    }
    if (regs_ok != MLLM_OK) return fail(regs_ok, "prefix_kernel: compiled with fewer registers than its split needs");
    const int smem = PrefixCfg<D, kPairs, k8>::kSmemBytes;
    if (int st = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem),
                            "prefix_kernel smem attribute"))
        return st;
    return check_cuda(launch_pdl(kern, dim3(a.Hkv, p.pairs * p.most.splits + p.most.splits_single),
                                 dim3(Split<k8>::kThreads), smem, s, m.q, m.k, m.v, m.v_end, a, sa, kv),
                      "prefix_kernel launch");
}


// The decode over a bf16 cache (kv16) or an 8-bit one (kv8).
template <bool k8>
int decode_shared(const char* who, const void* q, const mllm_paged_kv* kv16, const mllm_paged_kv8* kv8, const int32_t* kv_lens,
                  int prefix_len, int batch, int num_heads, int num_kv_heads, int head_dim, int max_kv_len,
                  float softmax_scale, void* out, void* workspace, size_t workspace_bytes, cudaStream_t s) {
    const std::string w(who);
    if (batch < 0 || num_heads <= 0 || num_kv_heads <= 0 || max_kv_len <= 0)
        return fail(MLLM_ERR_INVALID_ARGUMENT, w + ": bad sizes");
    if (prefix_len < 0 || prefix_len > max_kv_len)
        return fail(MLLM_ERR_INVALID_ARGUMENT, w + ": prefix_len must be in [0, max_kv_len]");
    if (num_heads % num_kv_heads != 0)
        return fail(MLLM_ERR_INVALID_ARGUMENT, "Attention: num_heads must be divisible by num_kv_heads.");
    if (head_dim != 64 && head_dim != 128) return fail(MLLM_ERR_UNSUPPORTED, w + ": head_dim must be 64 or 128");
    const int n_rep = num_heads / num_kv_heads;
    if (n_rep > kMaxGroup) return fail(MLLM_ERR_UNSUPPORTED, w + ": GQA group larger than 8");
    if (batch > 65535 || (int64_t)batch * num_heads > 0x3fffffff)
        return fail(MLLM_ERR_UNSUPPORTED, w + ": more than 65535 sequences or 2^30 query rows");
    if (max_kv_len > 0x7fffff00) return fail(MLLM_ERR_UNSUPPORTED, w + ": max_kv_len above 2^31 - 256");
    if (!(softmax_scale > 0.f) || !std::isfinite(softmax_scale))
        return fail(MLLM_ERR_INVALID_ARGUMENT, w + ": softmax_scale must be positive");
    StreamArgs a = {};
    Kv8View view = {};
    if (int st = k8 ? paged_layout8(kv8, max_kv_len, head_dim, who, &a.lay, &view)
                    : paged_layout(kv16, max_kv_len, head_dim, who, &a.lay))
        return st;
    if (batch == 0) return ok();
    if (!q || !out || !kv_lens) return fail(MLLM_ERR_INVALID_ARGUMENT, w + ": null pointer");
    if (!aligned(q, 16) || !aligned(out, 4)) return fail(MLLM_ERR_INVALID_ARGUMENT, w + ": q/out misaligned");
    const size_t need = mllm_decode_attention_shared_workspace_size(batch, num_heads, num_kv_heads, head_dim, prefix_len);
    if (!workspace || !aligned(workspace, 256) || workspace_bytes < need)
        return fail(MLLM_ERR_WORKSPACE, w + ": workspace missing, misaligned or smaller than "
                                            "mllm_decode_attention_shared_workspace_size()");
    int num_sms = 0;
    if (int st = require_sm100(&num_sms)) return st;
    num_sms = std::min(num_sms, kMaxSms);
    const int64_t D = head_dim;
    a.q = (const __nv_bfloat16*)q;
    a.kv_lens = kv_lens;
    a.out = (__nv_bfloat16*)out;
    a.B = batch;
    a.H = num_heads;
    a.Hkv = num_kv_heads;
    a.n_rep = n_rep;
    a.max_len = max_kv_len;
    a.scale_log2 = (float)((double)softmax_scale * 1.4426950408889634);
    a.first_row = prefix_len;
    stream_place(a, workspace, head_dim, shared_part_rows(batch, num_heads, num_kv_heads, prefix_len));
    a.prefix_base = (int64_t)stream_part_rows(n_rep, batch, num_kv_heads, true);
    // bf16 K or V in boxes of box_rows rows; the rows of a block, or the first of them
    auto kv_map = [&](CUtensorMap* map, void* pool, int rows, int box_rows) {
        return encode_kv_map(map, pool, D, rows, num_kv_heads, kv16->num_blocks, kv16->row_stride, kv16->head_stride,
                             kv16->block_stride, 64, box_rows);
    };
    if (prefix_len > 0) {
        const PrefixPlan p = plan_prefix<k8>(batch, num_kv_heads, n_rep, prefix_len, num_sms);
        PrefixMaps m;
        // Q [B, H, D]: heads as the map's rows, sequences as its third dimension
        if (int st = encode_kv_map(&m.q, q, D, num_heads, batch, 1, D, num_heads * D, (int64_t)batch * num_heads * D, 64,
                                   n_rep, p.seqs))
            return st;
        if constexpr (k8) {
            m.k = m.v = m.v_end = m.q;   // not looked at
        } else {
            const int tail = prefix_len % kv16->block_size;   // rows of the prefix in its last block (0: all)
            if (int st = kv_map(&m.k, kv16->k_pool, kv16->block_size, kBN)) return st;
            if (int st = kv_map(&m.v, kv16->v_pool, kv16->block_size, kBN)) return st;
            if (int st = kv_map(&m.v_end, kv16->v_pool, tail ? tail : kv16->block_size, kBN)) return st;
        }
        PrefixArgs pa = {};
        pa.part_o = a.part_o + a.prefix_base * D;
        pa.part_lse = a.part_lse + a.prefix_base;
        pa.B = batch;
        pa.Hkv = num_kv_heads;
        pa.n_rep = n_rep;
        pa.seqs = p.seqs;
        pa.prefix = prefix_len;
        pa.n_tiles = (prefix_len + kBN - 1) / kBN;
        pa.pairs = p.pairs;
        pa.single = p.single;
        pa.num_sms = num_sms;
        pa.scale_log2 = a.scale_log2;
        pa.lay = a.lay;
        a.pair_seqs = 2 * p.pairs * p.seqs;
        a.shared = 1;
        a.ticket = next_ticket();
        int st;
        if (head_dim == 128)
            st = p.pairs ? launch_prefix_d<128, true, k8>(pa, a, p, m, view, s)
                         : launch_prefix_d<128, false, k8>(pa, a, p, m, view, s);
        else
            st = p.pairs ? launch_prefix_d<64, true, k8>(pa, a, p, m, view, s)
                         : launch_prefix_d<64, false, k8>(pa, a, p, m, view, s);
        if (st) return st;
    }
    if constexpr (k8) {
        if (int st = launch_stream_kv8(a, head_dim, kv8, view, num_sms, s)) return st;
    } else {
        CUtensorMap tmK, tmV;
        if (int st = kv_map(&tmK, kv16->k_pool, kv16->block_size, 64)) return st;
        if (int st = kv_map(&tmV, kv16->v_pool, kv16->block_size, 64)) return st;
        if (int st = launch_stream_bf16(a, head_dim, tmK, tmV, num_sms, s)) return st;
    }
    return ok();
}

}  // namespace

MLLM_DEFINE_STATUS_READER(shared_prefix)

}  // namespace mllm_b200

using namespace mllm_b200;

extern "C" size_t mllm_decode_attention_shared_workspace_size(int batch, int num_heads, int num_kv_heads, int head_dim,
                                                              int prefix_len) {
    if (batch <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads || head_dim <= 0 ||
        prefix_len < 0 || num_heads / num_kv_heads > kMaxGroup)
        return 0;
    return stream_workspace_bytes(head_dim, shared_part_rows(batch, num_heads, num_kv_heads, prefix_len), batch, num_kv_heads);
}

extern "C" int mllm_decode_attention_shared_paged_bf16(const void* q, const mllm_paged_kv* kv, const int32_t* kv_lens,
                                                       int prefix_len, int batch, int num_heads, int num_kv_heads,
                                                       int head_dim, int max_kv_len, float softmax_scale, void* out,
                                                       void* workspace, size_t workspace_bytes, mllm_stream_t stream) {
    MLLM_NVTX_RANGE("mllm_decode_attention_shared_paged_bf16");
    return decode_shared<false>("decode_attention_shared", q, kv, nullptr, kv_lens, prefix_len, batch, num_heads,
                                num_kv_heads, head_dim, max_kv_len, softmax_scale, out, workspace, workspace_bytes,
                                (cudaStream_t)stream);
}

extern "C" int mllm_decode_attention_shared_paged_kv8(const void* q, const mllm_paged_kv8* kv, const int32_t* kv_lens,
                                                      int prefix_len, int batch, int num_heads, int num_kv_heads,
                                                      int head_dim, int max_kv_len, float softmax_scale, void* out,
                                                      void* workspace, size_t workspace_bytes, mllm_stream_t stream) {
    MLLM_NVTX_RANGE("mllm_decode_attention_shared_paged_kv8");
    return decode_shared<true>("decode_attention_shared_kv8", q, nullptr, kv, kv_lens, prefix_len, batch, num_heads,
                               num_kv_heads, head_dim, max_kv_len, softmax_scale, out, workspace, workspace_bytes,
                               (cudaStream_t)stream);
}
