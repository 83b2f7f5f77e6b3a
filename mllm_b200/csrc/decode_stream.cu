// Decode attention with an even split of the cached rows over the GPU (one query per sequence), for
//   the 8-bit paged cache (kv8.cuh), and
//   the rows of a bf16 paged cache behind a prefix that the batch shares (shared_prefix.cu does the prefix).
//
// Work split.  The tiles of all (sequence, kv head) pairs, pair after pair, form one line of tiles; CTA i of G
// takes tiles i*per .. (i+1)*per - 1 of it, per = ceil(tiles / G).  Every CTA streams the same number of bytes
// whatever the lengths are, the plan is computed on the device from the lengths (a captured graph follows them),
// and there is no counter to keep between calls.  A CTA's range cuts at most its first and its last pair, so the
// partial results need two slots a CTA, whatever the lengths; a pair that lies in one CTA is written directly.
// stream_combine_kernel joins the cut pairs in CTA order (deterministic).
//
// Per tile (8-bit: 128 rows, bf16: 64; both 32 KB of K and V at D = 128) with the cached rows as the M side:
//   S^T = K Q^T      mma.sync m16n8k16, A = 16 cached rows (ldmatrix), B = the group's <= 8 query heads: no half of
//                    the MMA is padding, as it is with the heads on the M side
//   softmax          online in the exp2 domain; a thread holds two heads, the reduction runs over its 8 row lanes
//   O^T += V^T P^T   A = V^T by ldmatrix.trans, B = P^T: the C fragment of S^T turned by movmatrix
// An 8-bit row becomes halves in registers (one cvt per two values, exact).  ldmatrix moves 16-bit units, so a
// thread gets four neighbouring columns of K instead of two pairs eight apart; Q's fragments are loaded in the same
// permuted order, which leaves the contraction unchanged.  For V^T the transposed units hold two columns of two
// rows; one byte permute sorts them, and output columns 2i and 2i + 1 land in the two row halves of the MMA.
// q is scaled per head by a power of two into the range of a half (exact for elements within 2^-27 of the head's
// largest; smaller ones lose bits that lie 2^-40 below it) and the scale is taken out of S in fp32.
// Row scales: S gets 2^ek before the softmax.  2^ev multiplies P, so P^T = exp2(s - m + ev - mo + 15) with mo the running
// maximum of s - m + ev: the largest weight times scale is 2^15, the top of a half's range (65504), and none overflows it,
// however the rows' scales differ; the merge takes the 2^15 out.  With the largest at 1, what lies 2^-25 below it would
// become zero here but not in the sum l: with one dominant row, 2^18 others behind it in a warp lost 0.6 % of the output.
// Now that takes 2^-40.  The sum l uses exp2(s - m) with its own maximum in fp32.  P is rounded to a half (2^-11), to
// bf16 for a bf16 cache, since A and B of an MMA have one type; both sums stay fp32.
//
// Bound: HBM (2 (D + 1) bytes a row and kv head; 4 D for bf16).  Rows past the end of a sequence, and rows of the
// prefix in the first tile behind it, are masked to -inf in S and zeroed in V (any bits may lie there); TMA boxes wholly
// past the end are not loaded.
#include <algorithm>
#include <cmath>

#include "decode_stream.cuh"
#include "kv8.cuh"

namespace mllm_b200 {
namespace {

constexpr int kBoxRows = 64;
constexpr int kConsumerWarps = 4;
constexpr int kThreads = (kConsumerWarps + 1) * 32;
constexpr int kPad = 4;            // floats between the merge rows of two heads (bank spread)
constexpr float kTopP = 15.f;      // log2 of the largest weight times scale of an 8-bit cache's rows as a half

template <int D, bool k8>
struct Cfg {
    static constexpr int kTile = k8 ? 128 : 64;                 // rows per stage
    static constexpr int kWarpRows = kTile / kConsumerWarps;    // 32 or 16
    static constexpr int kRowBytes = k8 ? D : 2 * D;
    static constexpr int kBoxBytesRow = kRowBytes < 128 ? kRowBytes : 128;
    static constexpr int kColBoxes = kRowBytes / kBoxBytesRow;
    static constexpr int kRowBoxes = kTile / kBoxRows;
    static constexpr int kBoxBytes = kBoxRows * kBoxBytesRow;
    static constexpr int kTileBytes = kTile * kRowBytes;        // K or V
    static constexpr int kStageBytes = 2 * kTileBytes;
    static constexpr int kStages = kStageBytes >= 32768 ? 3 : 6;
    static constexpr int kExpBytes = k8 ? 2 * kTile : 0;        // K and V exponents of a stage
    static constexpr int kRedFloats = kConsumerWarps * kMaxGroup * (D + kPad);   // the warps' rows, in a stage
    static constexpr int kSmemBytes =
        kStages * (kStageBytes + kExpBytes) + 3 * kConsumerWarps * kMaxGroup * 4 + 2 * kStages * 8 + 1024;
    static_assert(kRedFloats * 4 <= kStageBytes, "a stage holds the warps' rows");
    static_assert(2 * (kSmemBytes + 1024) <= 233472, "two CTAs per SM no longer fit");
};

// 16-byte chunk c of row r of a box: the swizzle TMA applied (128-byte rows, or 64-byte rows).
template <int ROWB>
__device__ __forceinline__ uint32_t swz_chunk(uint32_t r, uint32_t c) {
    return ROWB == 128 ? r * 128u + ((c ^ (r & 7u)) << 4) : r * 64u + ((c ^ ((r >> 1) & 3u)) << 4);
}

__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Transposes an 8 x 8 matrix of 16-bit values held one row per four lanes.
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Bulk copy of a few contiguous bytes (16-byte aligned, a multiple of 16) into shared memory.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_u32(bar))
        : "memory");
}

// A barrier of the consumer warps that says whether any thread came with `flag`.
__device__ __forceinline__ bool consumers_any(bool flag) {
    uint32_t any;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, %2, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(any)
        : "r"((uint32_t)flag), "n"(kConsumerWarps * 32)
        : "memory");
    return any != 0u;
}

// The slots of whole pairs (joined with a prefix) follow two for every CTA there may be.
__device__ __forceinline__ int64_t whole_slots(const StreamArgs& a) { return 2 * (int64_t)kSharedWaves * a.ctas; }

// A pair's stretch of this CTA's tiles.
struct Walk {
    int b, g;
    int left;              // tiles of the CTA still to come, this stretch included
    int pos;               // first tile of this stretch on the line of tiles
    int t0, t1;            // tiles of the pair: this stretch
    SeqTiles s;            // the pair's rows and tiles
    __device__ __forceinline__ bool whole() const { return t0 == 0 && t1 == s.tiles; }
};

template <int TILE>
__device__ __forceinline__ void walk_open(const StreamArgs& a, Walk& w) {
    w.t1 = min(w.s.tiles, w.t0 + w.left);
}

// Moves to the next pair with tiles; false when the CTA's tiles are done.
template <int TILE>
__device__ __forceinline__ bool walk_next(const StreamArgs& a, Walk& w) {
    w.left -= w.t1 - w.t0;
    w.pos += w.t1 - w.t0;
    if (w.left <= 0) return false;
    if (++w.g == a.Hkv) {
        w.g = 0;
        do {
            if (++w.b >= a.B) return false;
            w.s = seq_tiles<TILE>(a, w.b);
        } while (w.s.tiles == 0);
    }
    w.t0 = 0;
    walk_open<TILE>(a, w);
    return true;
}

template <int D, bool k8>
__global__ void __launch_bounds__(kThreads, 2)
    stream_decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                         StreamArgs a, Kv8View kv) {
    using C = Cfg<D, k8>;
    constexpr int NS = C::kStages;
    constexpr int TILE = C::kTile;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* s_exp = smem + NS * C::kStageBytes;                       // [NS][K exps | V exps]
    float* red_m = reinterpret_cast<float*>(s_exp + NS * C::kExpBytes);   // [4][8]
    float* red_l = red_m + kConsumerWarps * kMaxGroup;
    float* red_mo = red_l + kConsumerWarps * kMaxGroup;
    uint64_t* full = reinterpret_cast<uint64_t*>(red_mo + kConsumerWarps * kMaxGroup);
    uint64_t* empty = full + NS;
    __shared__ int s_plan[6];   // tiles of this CTA, its first tile, that tile's sequence and place in it, tiles per pair,
                               // whether every pair has a CTA

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < NS; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], kConsumerWarps);
        }
        mbar_fence_init();
    }
    // Behind a prefix kernel (shared) nothing here depends on that kernel's results, but lengths, tables, queries and rows
    // come from what ran before it.  It has waited for that, and published its ticket, before it let this grid in: a
    // thread that reads the ticket back (an acquire) is ordered behind that wait and goes on beside the prefix kernel; one
    // that does not waits for the prefix kernel itself.  The loads behind it start later for that: 59 us in place of
    // 55 for 128 sequences behind 8192 rows, 25.1 in place of 24.6 for 32.
    if (!a.shared || !ticket_published(a)) pdl_wait();
    pdl_trigger();
    const int pairs = a.B * a.Hkv;
    if (a.direct) {
        if (threadIdx.x == 0) s_plan[5] = 1;
    } else if (warp == 0) {
        int longest;
        const int total = total_tiles<TILE>(a, lane, &longest);
        const bool direct = direct_pairs(pairs, longest, a.ctas, a.shared);
        const int per = tiles_per_cta(a, total);
        const int p0 = min(total, (int)blockIdx.x * per);
        const int n = direct ? 0 : min(per, total - p0);
        int before = 0;   // tiles of the sequences before this batch of 32
        if (n > 0) {
            for (int base = 0; base < a.B; base += 32) {
                const int mine = base + lane < a.B ? seq_tiles<TILE>(a, base + lane).tiles * a.Hkv : 0;
                int incl = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int up = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += up;
                }
                const unsigned past = __ballot_sync(0xffffffffu, before + incl > p0);
                if (past != 0) {
                    if (lane == __ffs(past) - 1) {
                        const int off = p0 - (before + incl - mine);
                        const int tiles = mine / a.Hkv;
                        s_plan[2] = base + lane;
                        s_plan[3] = off;          // tile within the sequence's kv heads
                        s_plan[4] = tiles;
                    }
                    break;
                }
                before += __shfl_sync(0xffffffffu, incl, 31);
            }
        }
        if (lane == 0) {
            s_plan[0] = n;
            s_plan[1] = p0;
            s_plan[5] = direct ? 1 : 0;
            if (blockIdx.x == 0) a.plan[kPlanPer] = direct ? 0 : per;   // 0: nothing to join
        }
    }
    __syncthreads();
    Walk w;
    if (s_plan[5]) {
        w.left = w.pos = w.t0 = 0;
        if ((int)blockIdx.x < pairs) {
            w.b = blockIdx.x / a.Hkv;
            w.g = blockIdx.x - w.b * a.Hkv;
            w.s = seq_tiles<TILE>(a, w.b);
            w.left = w.s.tiles;
            walk_open<TILE>(a, w);
            if (w.left == 0) {   // an empty sequence
                __nv_bfloat16* out = a.out + ((int64_t)w.b * a.H + (int64_t)w.g * a.n_rep) * D;
                for (int i = threadIdx.x; i < a.n_rep * D; i += kThreads) out[i] = __float2bfloat16_rn(0.f);
            }
        }
    } else {
        w.left = s_plan[0];
        w.pos = s_plan[1];
        if (w.left > 0) {
            w.b = s_plan[2];
            w.g = s_plan[3] / s_plan[4];
            w.t0 = s_plan[3] - w.g * s_plan[4];
            w.s = seq_tiles<TILE>(a, w.b);
            walk_open<TILE>(a, w);
        }
    }

    if (warp == kConsumerWarps) {
        // ------------------------------ producer ------------------------------
        if (lane == 0 && w.left > 0) {
            tma_prefetch_desc(&tmK);
            tma_prefetch_desc(&tmV);
            if (a.shared) asm volatile("fence.proxy.async.global;" ::: "memory");   // the rows too come behind the ticket
            int stage = 0;
            uint32_t phase = 0;
            bool alive = true;
            do {
                for (int t = w.t0; t < w.t1 && alive; ++t) {
                    const int row0 = (w.s.first_tile + t) * TILE;
                    const int boxes = C::kRowBoxes == 1 ? 1 : min(C::kRowBoxes, (w.s.len - row0 + kBoxRows - 1) / kBoxRows);
                    int blk, row;
                    kv_locate(a.lay, w.b, row0, blk, row);   // a bad table entry reads block 0 (and is recorded)
                    if (!mbar_wait(&empty[stage], phase ^ 1)) { alive = false; break; }
                    uint8_t* kdst = smem + stage * C::kStageBytes;
                    uint8_t* vdst = kdst + C::kTileBytes;
                    mbar_arrive_expect_tx(&full[stage],
                                          (uint32_t)boxes * 2u * (C::kColBoxes * C::kBoxBytes + (k8 ? kBoxRows : 0)));
                    for (int rb = 0; rb < boxes; ++rb) {
#pragma unroll
                        for (int cb = 0; cb < C::kColBoxes; ++cb) {
                            const int off = (rb * C::kColBoxes + cb) * C::kBoxBytes;
                            const int col = cb * (k8 ? 128 : 64);
                            tma_load_4d(kdst + off, &tmK, &full[stage], col, row + rb * kBoxRows, w.g, blk);
                            tma_load_4d(vdst + off, &tmV, &full[stage], col, row + rb * kBoxRows, w.g, blk);
                        }
                    }
                    if constexpr (k8) {
                        uint8_t* edst = s_exp + stage * C::kExpBytes;
                        const int64_t eoff = blk * kv.e_sb + w.g * kv.e_sh + row;
                        bulk_load(edst, kv.k_exp + eoff, boxes * kBoxRows, &full[stage]);
                        bulk_load(edst + TILE, kv.v_exp + eoff, boxes * kBoxRows, &full[stage]);
                    }
                    if (++stage == NS) { stage = 0; phase ^= 1; }
                }
            } while (alive && walk_next<TILE>(a, w));
        }
    } else if (w.left > 0) {
        // -------------------------------- consumers --------------------------------
        const int grp = lane >> 2;   // row lane (and head of the Q fragment)
        const int tig = lane & 3;    // heads 2 tig, 2 tig + 1
        constexpr int CH = C::kRowBytes / 16;            // 16-byte chunks of a row
        constexpr int KS = D / 16;                       // k-steps of S^T, and m-blocks of O^T
        constexpr int NB = C::kWarpRows / 16;            // 16-row blocks of this warp
        const int mi = lane >> 3, ri = lane & 7;
        int stage = 0;
        uint32_t phase = 0;
        bool alive = true;
        // Raw q of a pair as the B operand needs it: column n = head grp, along head_dim four neighbours (8-bit) or two
        // pairs eight apart per k-step.  The next pair's is loaded while the present one is worked on.
        uint2 raw[KS];
        auto load_q = [&](const Walk& at) {
            const bool ok = grp < a.n_rep;
            const __nv_bfloat16* qrow = a.q + ((int64_t)at.b * a.H + (int64_t)at.g * a.n_rep + (ok ? grp : 0)) * D;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                if constexpr (k8) {
                    raw[ks] = *reinterpret_cast<const uint2*>(qrow + ks * 16 + tig * 4);
                } else {
                    raw[ks].x = *reinterpret_cast<const uint32_t*>(qrow + ks * 16 + tig * 2);
                    raw[ks].y = *reinterpret_cast<const uint32_t*>(qrow + ks * 16 + tig * 2 + 8);
                }
                if (!ok) raw[ks] = make_uint2(0u, 0u);
            }
        };
        load_q(w);
        bool more;
        Walk next = w;
        do {
            uint32_t qb[KS][2];
            float sc0, sc1;          // log2-domain scales of heads 2 tig and 2 tig + 1
            if constexpr (k8) {
                float x[KS][4];
                float amax = 0.f;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const float2 lo = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[ks].x));
                    const float2 hi = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[ks].y));
                    x[ks][0] = lo.x;
                    x[ks][1] = lo.y;
                    x[ks][2] = hi.x;
                    x[ks][3] = hi.y;
#pragma unroll
                    for (int e = 0; e < 4; ++e) amax = fmaxf(amax, fabsf(x[ks][e]));
                }
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                const int eq = max((int)(__float_as_uint(amax) >> 23) - 127 - 13, kExpMin);
                const float inv = pow2i(-eq);
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    qb[ks][0] = pack_f16x2(x[ks][0] * inv, x[ks][1] * inv);
                    qb[ks][1] = pack_f16x2(x[ks][2] * inv, x[ks][3] * inv);
                }
                const float qs = pow2i(eq) * a.scale_log2;
                sc0 = __shfl_sync(0xffffffffu, qs, 8 * tig);
                sc1 = __shfl_sync(0xffffffffu, qs, 8 * tig + 4);
            } else {
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    qb[ks][0] = raw[ks].x;
                    qb[ks][1] = raw[ks].y;
                }
                sc0 = sc1 = a.scale_log2;
            }
            more = walk_next<TILE>(a, next);
            if (more) load_q(next);
            float o[KS][4];
#pragma unroll
            for (int i = 0; i < KS; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
            float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
            float mo[2] = {-INFINITY, -INFINITY};   // maximum of the weights times scales, against m

            for (int t = w.t0; t < w.t1; ++t) {
                if (!mbar_wait(&full[stage], phase)) { alive = false; break; }
                uint8_t* kst = smem + stage * C::kStageBytes;
                uint8_t* vst = kst + C::kTileBytes;
                const uint32_t kbase = smem_u32(kst), vbase = smem_u32(vst);
                const int row0 = warp * C::kWarpRows;                 // this warp's rows within the tile
                const int tile_row = (w.s.first_tile + t) * TILE;     // cache row of the tile's row 0
                const int valid = w.s.len - tile_row;                 // rows of the tile before the end
                const int lo_row = a.first_row - tile_row;            // rows before this one belong to the prefix
                auto chunk_addr = [&](uint32_t base, int row, int c) -> uint32_t {
                    constexpr int CPB = C::kBoxBytesRow / 16;
                    const int box = (row >> 6) * C::kColBoxes + c / CPB;
                    return base + box * C::kBoxBytes + swz_chunk<C::kBoxBytesRow>(row & 63, c % CPB);
                };

                // ---- S^T = K Q^T ----
                float sa[NB][4];
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    sa[nb][0] = sa[nb][1] = sa[nb][2] = sa[nb][3] = 0.f;
                    const int row = row0 + nb * 16 + 8 * (mi & 1) + ri;
#pragma unroll
                    for (int c = 0; c < CH; c += 2) {
                        uint32_t r0, r1, r2, r3;
                        ldsm_x4(chunk_addr(kbase, row, c + (mi >> 1)), r0, r1, r2, r3);
                        if constexpr (k8) {
                            mma_f16_16816(sa[nb], e4m3x2_to_f16x2((uint16_t)r0), e4m3x2_to_f16x2((uint16_t)r1),
                                          e4m3x2_to_f16x2((uint16_t)(r0 >> 16)), e4m3x2_to_f16x2((uint16_t)(r1 >> 16)),
                                          qb[c][0], qb[c][1]);
                            mma_f16_16816(sa[nb], e4m3x2_to_f16x2((uint16_t)r2), e4m3x2_to_f16x2((uint16_t)r3),
                                          e4m3x2_to_f16x2((uint16_t)(r2 >> 16)), e4m3x2_to_f16x2((uint16_t)(r3 >> 16)),
                                          qb[c + 1][0], qb[c + 1][1]);
                        } else {
                            mma_bf16_16816(sa[nb], r0, r1, r2, r3, qb[c / 2][0], qb[c / 2][1]);
                        }
                    }
                }

                // ---- online softmax: element (nb, h, e) is row row0 + 16 nb + 8 h + grp, head 2 tig + e ----
                float ev[NB][2];
                float mt[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int r = row0 + nb * 16 + 8 * h + grp;
                        const bool in = r < valid && r >= lo_row;
                        float ks = 1.f;
                        ev[nb][h] = 0.f;
                        if constexpr (k8) {
                            const uint8_t* ex = s_exp + stage * C::kExpBytes;
                            ks = exp_byte_scale(ex[r]);
                            ev[nb][h] = (float)((int)ex[TILE + r] - 127);
                        }
                        const float v0 = in ? sa[nb][2 * h] * sc0 * ks : -INFINITY;
                        const float v1 = in ? sa[nb][2 * h + 1] * sc1 * ks : -INFINITY;
                        sa[nb][2 * h] = v0;
                        sa[nb][2 * h + 1] = v1;
                        mt[0] = fmaxf(mt[0], v0);
                        mt[1] = fmaxf(mt[1], v1);
                    }
                }
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) mt[e] = fmaxf(mt[e], __shfl_xor_sync(0xffffffffu, mt[e], off));
                }
                float oscale[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float mn = fmaxf(m[e], mt[e]);
                    const float mu = mn == -INFINITY ? 0.f : mn;
                    const float shift = m[e] - mu;
                    oscale[e] = ex2_approx(shift);
                    l[e] *= oscale[e];
                    mo[e] += shift;
                    m[e] = mn;
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        sa[nb][e] -= mu;
                        sa[nb][2 + e] -= mu;
                    }
                }
                float mou[2];
                if constexpr (k8) {   // of s - m + ev, not of s + ev: that would round ev away beside a score of 2^24
                    float mot[2] = {mo[0], mo[1]};
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int e = 0; e < 2; ++e) mot[e] = fmaxf(mot[e], sa[nb][2 * h + e] + ev[nb][h]);
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1)
#pragma unroll
                        for (int e = 0; e < 2; ++e) mot[e] = fmaxf(mot[e], __shfl_xor_sync(0xffffffffu, mot[e], off));
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        mou[e] = mot[e] == -INFINITY ? 0.f : mot[e];
                        oscale[e] = ex2_approx(mo[e] - mou[e]);
                        mou[e] -= kTopP;
                        mo[e] = mot[e];
                    }
                }
                uint32_t pb[NB][2];
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float p0 = ex2_approx(sa[nb][2 * h]);
                        const float p1 = ex2_approx(sa[nb][2 * h + 1]);
                        l[0] += p0;
                        l[1] += p1;
                        uint32_t packed;
                        if constexpr (k8) {
                            packed = pack_f16x2(ex2_approx(sa[nb][2 * h] + ev[nb][h] - mou[0]),
                                                ex2_approx(sa[nb][2 * h + 1] + ev[nb][h] - mou[1]));
                        } else {
                            packed = pack_bf16x2(p0, p1);
                        }
                        pb[nb][h] = movmatrix_trans(packed);
                    }
                }
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    o[i][0] *= oscale[0];
                    o[i][1] *= oscale[1];
                    o[i][2] *= oscale[0];
                    o[i][3] *= oscale[1];
                }

                // ---- rows past the end, or of the prefix: zero this warp's V rows (any bit pattern may lie there) ----
                if (valid < row0 + C::kWarpRows || lo_row > row0) {
                    for (int i = lane; i < C::kWarpRows * CH; i += 32) {
                        const int r = row0 + i / CH, c = i % CH;
                        if (r >= valid || r < lo_row)
                            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(chunk_addr(vbase, r, c)), "r"(0)
                                         : "memory");
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }

                // ---- O^T += V^T P^T ----
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    const int row = row0 + nb * 16 + 8 * (mi & 1) + ri;
#pragma unroll
                    for (int c = 0; c < CH; c += 2) {
                        uint32_t r0, r1, r2, r3;
                        ldsm_x4_trans(chunk_addr(vbase, row, c + (mi >> 1)), r0, r1, r2, r3);
                        if constexpr (k8) {
                            r0 = __byte_perm(r0, 0u, 0x3120);
                            r1 = __byte_perm(r1, 0u, 0x3120);
                            r2 = __byte_perm(r2, 0u, 0x3120);
                            r3 = __byte_perm(r3, 0u, 0x3120);
                            mma_f16_16816(o[c], e4m3x2_to_f16x2((uint16_t)r0), e4m3x2_to_f16x2((uint16_t)(r0 >> 16)),
                                          e4m3x2_to_f16x2((uint16_t)r1), e4m3x2_to_f16x2((uint16_t)(r1 >> 16)),
                                          pb[nb][0], pb[nb][1]);
                            mma_f16_16816(o[c + 1], e4m3x2_to_f16x2((uint16_t)r2), e4m3x2_to_f16x2((uint16_t)(r2 >> 16)),
                                          e4m3x2_to_f16x2((uint16_t)r3), e4m3x2_to_f16x2((uint16_t)(r3 >> 16)),
                                          pb[nb][0], pb[nb][1]);
                        } else {
                            mma_bf16_16816(o[c / 2], r0, r2, r1, r3, pb[nb][0], pb[nb][1]);
                        }
                    }
                }
                if (t + 1 == w.t1) break;            // the stretch's last stage is kept for the merge
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty[stage]);
                if (++stage == NS) { stage = 0; phase ^= 1; }
            }

            // ---- merge the four warps, in the memory of the stretch's last stage (the next tiles are on their way) ----
            float* red_o = reinterpret_cast<float*>(smem + stage * C::kStageBytes);   // [4][8][D + kPad]
            // all have read that stage, and the last stretch's statistics; if one gave up a wait, all leave together
            if (consumers_any(!alive)) break;
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) {
                l[0] += __shfl_xor_sync(0xffffffffu, l[0], off);
                l[1] += __shfl_xor_sync(0xffffffffu, l[1], off);
            }
            if (grp == 0) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    red_m[warp * kMaxGroup + 2 * tig + e] = m[e];
                    red_l[warp * kMaxGroup + 2 * tig + e] = l[e];
                    red_mo[warp * kMaxGroup + 2 * tig + e] = k8 ? mo[e] : 0.f;
                }
            }
            // column of o[i][2h + .]: 8-bit rows 16 i + 2 grp + h, bf16 rows 16 i + 8 h + grp
            auto o_col = [&](int i, int h) -> int { return k8 ? 16 * i + 2 * grp + h : 16 * i + 8 * h + grp; };
            float* dst = red_o + warp * kMaxGroup * (D + kPad);
#pragma unroll
            for (int i = 0; i < KS; ++i) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    dst[(2 * tig + e) * (D + kPad) + o_col(i, 0)] = o[i][e];
                    dst[(2 * tig + e) * (D + kPad) + o_col(i, 1)] = o[i][2 + e];
                }
            }
            asm volatile("bar.sync 1, %0;" ::"n"(kConsumerWarps * 32) : "memory");
            // A thread joins four columns of a head: the final row, or the stretch's own attention row (normalised) and
            // log2 of its weight as a part.  A whole pair's part (to be joined with the prefix) has a slot of its own; a
            // cut pair's takes the CTA's first slot if the CTA begins in it, else the second.
            const bool final_row = w.whole() && !a.shared;
            const int64_t slot = w.whole() ? whole_slots(a) + (int64_t)w.b * a.Hkv + w.g
                                           : 2 * (int64_t)blockIdx.x + (w.pos == s_plan[1] ? 0 : 1);
            for (int i = threadIdx.x; i < a.n_rep * (D / 4); i += kConsumerWarps * 32) {
                const int h = i / (D / 4), d = 4 * (i % (D / 4));
                float M = red_m[h];
#pragma unroll
                for (int v = 1; v < kConsumerWarps; ++v) M = fmaxf(M, red_m[v * kMaxGroup + h]);
                const float Mu = M == -INFINITY ? 0.f : M;
                float mov[kConsumerWarps], MO = -INFINITY;   // the warps' mo against M
#pragma unroll
                for (int v = 0; v < kConsumerWarps; ++v) {
                    mov[v] = red_mo[v * kMaxGroup + h] + (red_m[v * kMaxGroup + h] - Mu);
                    MO = fmaxf(MO, mov[v]);
                }
                const float MOu = MO == -INFINITY ? 0.f : MO;
                float L = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int v = 0; v < kConsumerWarps; ++v) {
                    L += red_l[v * kMaxGroup + h] * ex2_approx(red_m[v * kMaxGroup + h] - Mu);
                    const float ow = ex2_approx(mov[v] - MOu);
                    const float4 r = *reinterpret_cast<const float4*>(red_o + (v * kMaxGroup + h) * (D + kPad) + d);
                    x[0] = fmaf(r.x, ow, x[0]);
                    x[1] = fmaf(r.y, ow, x[1]);
                    x[2] = fmaf(r.z, ow, x[2]);
                    x[3] = fmaf(r.w, ow, x[3]);
                }
                const float f = L != 0.f ? ex2_approx(MOu) / L : 0.f;
                constexpr float kTop = k8 ? 1.f / (1 << (int)kTopP) : 1.f;   // before f, which may be near the smallest numbers
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = x[e] * kTop * f;
                if (final_row) {
                    uint32_t* orow = reinterpret_cast<uint32_t*>(a.out + ((int64_t)w.b * a.H + w.g * a.n_rep + h) * D + d);
                    orow[0] = pack_bf16x2(x[0], x[1]);
                    orow[1] = pack_bf16x2(x[2], x[3]);
                } else {
                    *reinterpret_cast<float4*>(a.part_o + (slot * a.n_rep + h) * D + d) = make_float4(x[0], x[1], x[2], x[3]);
                    if (d == 0) a.part_lse[slot * a.n_rep + h] = L != 0.f ? Mu + log2f(L) : -INFINITY;
                }
            }
            if (!s_plan[5] && w.t0 == 0 && threadIdx.x == 0) a.plan[kPlanHead + w.b * a.Hkv + w.g] = w.pos;   // where the pair begins
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // before TMA writes the stage again
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[stage]);
            if (++stage == NS) { stage = 0; phase ^= 1; }
            w = next;
        } while (more);
    }
    // One CTA waits, so that this grid ends after the prefix kernel's; were it all of them, those that are done would
    // hold their SMs until then.
    if (a.shared && blockIdx.x == gridDim.x - 1) pdl_wait();
}

// Joins the parts of every (sequence, query head): the stretches of the cut pairs and, with a shared prefix, the
// prefix's parts.  A part is a normalised row and log2 of its weight: out = sum_i 2^(e_i - M) row_i / sum_i 2^(e_i - M),
// parts in a fixed order.  A warp takes one query head, so nothing waits at a barrier: the time of this kernel is that
// of its chain of dependent loads (the pair's place, the weights, the rows), and its launch.
constexpr int kCombineWarps = 4;

template <int D, int TILE>
__global__ void __launch_bounds__(kCombineWarps * 32) stream_combine_kernel(StreamArgs a) {
    constexpr int E = D / 32;        // columns per lane
    constexpr int U = 8;             // rows in flight
    const int lane = threadIdx.x & 31;
    const int bh = blockIdx.x * kCombineWarps + (threadIdx.x >> 5);
    if (bh >= a.B * a.H) return;
    const int b = bh / a.H, h = bh - b * a.H, g = h / a.n_rep, r = h - g * a.n_rep;
    pdl_wait();
    if (a.shared && blockIdx.x == 0 && threadIdx.x == 0) *a.ready = 0ull;
    const SeqTiles s = seq_tiles<TILE>(a, b);
    const int per = a.plan[kPlanPer], p0 = a.plan[kPlanHead + b * a.Hkv + g];   // p0 means nothing without tiles
    const int pre = a.shared ? a.plan[b < a.pair_seqs ? kPlanPair : kPlanSingle] : 0;
    if (per == 0) return;                 // every pair had a CTA of its own
    const int n_pre = s.short_len ? 0 : pre;
    int c0, own;
    if (!own_parts(p0, s.tiles, per, most_ctas(a.ctas, a.shared), &c0, &own)) record_error(kErrTimeout);
    if (own == 1 && n_pre == 0) return;   // written directly
    const int n = own + n_pre;            // 0: nothing to attend to
    auto part = [&](int i) -> int64_t {   // index of part i's row in part_o and part_lse
        if (i >= own) return a.prefix_base + (((int64_t)(i - own) * a.Hkv + g) * a.B + b) * a.n_rep + r;
        const int c = c0 + i;
        const int64_t slot = own == 1 ? whole_slots(a) + (int64_t)b * a.Hkv + g
                                      : 2 * (int64_t)c + (c * per >= p0 ? 0 : 1);
        return slot * a.n_rep + r;
    };
    float acc[E], sum = 0.f, M = -INFINITY;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    for (int i0 = 0; i0 < n; i0 += 32) {
        const int m = min(32, n - i0);
        const int64_t mine = part(min(i0 + lane, n - 1));
        const float w = lane < m ? a.part_lse[mine] : -INFINITY;
        auto load = [&](int i, float (&v)[E]) {
            const float* src = a.part_o + __shfl_sync(0xffffffffu, mine, i & 31) * D + lane * E;
            if constexpr (E == 4) {
                const float4 x = *reinterpret_cast<const float4*>(src);
                v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
            } else {
                const float2 x = *reinterpret_cast<const float2*>(src);
                v[0] = x.x, v[1] = x.y;
            }
        };
        float v[U][E];
#pragma unroll
        for (int u = 0; u < U; ++u) load(min(u, m - 1), v[u]);   // on their way while the weights are
        float top = w;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        top = fmaxf(top, M);
        const float Mu = top == -INFINITY ? 0.f : top;
        const float scale = ex2_approx(M - Mu);
        M = top;
        sum *= scale;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] *= scale;
        const float wgt = ex2_approx(w - Mu);
        for (int j = 0; j < m; j += U) {
            if (j > 0) {
#pragma unroll
                for (int u = 0; u < U; ++u) load(min(j + u, m - 1), v[u]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float f = __shfl_sync(0xffffffffu, wgt, (j + u) & 31);
                if (j + u < m) {
                    sum += f;
#pragma unroll
                    for (int e = 0; e < E; ++e) acc[e] += f * v[u][e];
                }
            }
        }
    }
    const bool any = sum > 0.f || sum != sum;
    __nv_bfloat16* out = a.out + (int64_t)bh * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; e += 2)
        *reinterpret_cast<uint32_t*>(out + e) = pack_bf16x2(any ? acc[e] / sum : 0.f, any ? acc[e + 1] / sum : 0.f);
}

constexpr int kMaxCtas = 2 * 160;

}  // namespace

size_t stream_part_rows(int n_rep, int batch, int num_kv_heads, bool shared) {
    return (2 * (size_t)kMaxCtas * (shared ? kSharedWaves : 1) + (shared ? (size_t)batch * num_kv_heads : 0)) * n_rep;
}

constexpr size_t kTicketBytes = 16;   // keeps the parts' alignment

size_t stream_workspace_bytes(int D, size_t part_rows, int batch, int num_kv_heads) {
    return (kTicketBytes + part_rows * (size_t)(D + 1) * 4 + (kPlanHead + (size_t)batch * num_kv_heads) * 4 + 255) & ~size_t(255);
}

void stream_place(StreamArgs& a, void* workspace, int D, size_t part_rows) {
    a.ready = static_cast<unsigned long long*>(workspace);
    a.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + kTicketBytes);
    a.part_lse = a.part_o + part_rows * D;
    a.plan = reinterpret_cast<int*>(a.part_lse + part_rows);
}

namespace {

template <int D, bool k8>
int launch_stream_d(StreamArgs& a, const Kv8View& kv, const CUtensorMap& tmK, const CUtensorMap& tmV, int num_sms,
                    cudaStream_t s) {
    using C = Cfg<D, k8>;
    // no more CTAs than tiles there can be
    const int64_t most = (int64_t)a.B * a.Hkv * ((a.max_len + C::kTile - 1) / C::kTile - a.first_row / C::kTile);
    if (most > 0x7fffffffLL - 65536) return fail(MLLM_ERR_UNSUPPORTED, "decode_attention: batch too large for one call");
    a.ctas = std::min(2 * num_sms, kMaxCtas);
    const int grid = std::max(stream_ctas(most, a.ctas, a.shared),
                              direct_pairs((int64_t)a.B * a.Hkv, 0, a.ctas, a.shared) ? a.B * a.Hkv : 1);
    auto kern = stream_decode_kernel<D, k8>;
    if (int st = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes),
                            "stream_decode smem attribute"))
        return st;
    a.direct = direct_pairs((int64_t)a.B * a.Hkv, (a.max_len + C::kTile - 1) / C::kTile, a.ctas, a.shared) ? 1 : 0;
    if (int st = check_cuda(launch_pdl(kern, dim3(grid), dim3(kThreads), C::kSmemBytes, s, tmK, tmV, a, kv),
                            "stream_decode_kernel launch"))
        return st;
    if (a.direct) return MLLM_OK;
    return check_cuda(launch_pdl(stream_combine_kernel<D, C::kTile>,
                                 dim3((unsigned)(((int64_t)a.B * a.H + kCombineWarps - 1) / kCombineWarps)),
                                 dim3(kCombineWarps * 32), 0, s, a),
                      "stream_combine_kernel launch");
}

}  // namespace

int launch_stream_bf16(StreamArgs& a, int head_dim, const CUtensorMap& tmK, const CUtensorMap& tmV, int num_sms,
                       cudaStream_t s) {
    return head_dim == 128 ? launch_stream_d<128, false>(a, Kv8View{}, tmK, tmV, num_sms, s)
                           : launch_stream_d<64, false>(a, Kv8View{}, tmK, tmV, num_sms, s);
}

int launch_stream_kv8(StreamArgs& a, int head_dim, const mllm_paged_kv8* kv, const Kv8View& view, int num_sms, cudaStream_t s) {
    CUtensorMap tmK, tmV;
    if (int st = encode_kv8_map(&tmK, kv->k_pool, head_dim, kv->block_size, a.Hkv, kv->num_blocks, kv->row_stride,
                                kv->head_stride, kv->block_stride, kBoxRows))
        return st;
    if (int st = encode_kv8_map(&tmV, kv->v_pool, head_dim, kv->block_size, a.Hkv, kv->num_blocks, kv->row_stride,
                                kv->head_stride, kv->block_stride, kBoxRows))
        return st;
    return head_dim == 128 ? launch_stream_d<128, true>(a, view, tmK, tmV, num_sms, s)
                           : launch_stream_d<64, true>(a, view, tmK, tmV, num_sms, s);
}

MLLM_DEFINE_STATUS_READER(decode_stream)

}  // namespace mllm_b200

using namespace mllm_b200;

extern "C" size_t mllm_decode_attention_kv8_workspace_size(int batch, int num_heads, int num_kv_heads, int head_dim) {
    if (batch <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads || head_dim <= 0) return 0;
    const size_t rows = stream_part_rows(num_heads / num_kv_heads, batch, num_kv_heads, false);
    return stream_workspace_bytes(head_dim, rows, batch, num_kv_heads);
}

extern "C" int mllm_decode_attention_paged_kv8(const void* q, const mllm_paged_kv8* kv, const int32_t* kv_lens, int batch,
                                               int num_heads, int num_kv_heads, int head_dim, int max_kv_len,
                                               float softmax_scale, void* out, void* workspace, size_t workspace_bytes,
                                               mllm_stream_t stream) {
    MLLM_NVTX_RANGE("mllm_decode_attention_paged_kv8");
    if (batch < 0 || num_heads <= 0 || num_kv_heads <= 0 || max_kv_len <= 0)
        return fail(MLLM_ERR_INVALID_ARGUMENT, "decode_attention_kv8: bad sizes");
    if (num_heads % num_kv_heads != 0)
        return fail(MLLM_ERR_INVALID_ARGUMENT, "Attention: num_heads must be divisible by num_kv_heads.");
    if (head_dim != 64 && head_dim != 128)
        return fail(MLLM_ERR_UNSUPPORTED, "decode_attention_kv8: head_dim must be 64 or 128");
    const int n_rep = num_heads / num_kv_heads;
    if (n_rep > kMaxGroup) return fail(MLLM_ERR_UNSUPPORTED, "decode_attention_kv8: GQA group larger than 8");
    if (batch > 65535 || (int64_t)batch * num_heads > 0x3fffffff)
        return fail(MLLM_ERR_UNSUPPORTED, "decode_attention_kv8: more than 65535 sequences or 2^30 query rows");
    if (max_kv_len > 0x7fffff00)
        return fail(MLLM_ERR_UNSUPPORTED, "decode_attention_kv8: max_kv_len above 2^31 - 256");
    if (!(softmax_scale > 0.f) || !std::isfinite(softmax_scale))
        return fail(MLLM_ERR_INVALID_ARGUMENT, "decode_attention_kv8: softmax_scale must be positive");
    StreamArgs a = {};
    Kv8View view;
    if (int st = paged_layout8(kv, max_kv_len, head_dim, "decode_attention_kv8", &a.lay, &view)) return st;
    if (batch == 0) return ok();
    if (!q || !out || !kv_lens) return fail(MLLM_ERR_INVALID_ARGUMENT, "decode_attention_kv8: null pointer");
    if (!aligned(q, 8) || !aligned(out, 4))
        return fail(MLLM_ERR_INVALID_ARGUMENT, "decode_attention_kv8: q/out misaligned");
    if (!workspace || !aligned(workspace, 256) ||
        workspace_bytes < mllm_decode_attention_kv8_workspace_size(batch, num_heads, num_kv_heads, head_dim))
        return fail(MLLM_ERR_WORKSPACE, "decode_attention_kv8: workspace missing, misaligned or smaller than "
                                        "mllm_decode_attention_kv8_workspace_size()");
    int num_sms = 0;
    if (int st = require_sm100(&num_sms)) return st;
    a.q = (const __nv_bfloat16*)q;
    a.kv_lens = kv_lens;
    a.out = (__nv_bfloat16*)out;
    a.B = batch;
    a.H = num_heads;
    a.Hkv = num_kv_heads;
    a.n_rep = n_rep;
    a.max_len = max_kv_len;
    a.scale_log2 = (float)((double)softmax_scale * 1.4426950408889634);
    stream_place(a, workspace, head_dim, stream_part_rows(n_rep, batch, num_kv_heads, false));
    if (int st = launch_stream_kv8(a, head_dim, kv, view, num_sms, (cudaStream_t)stream)) return st;
    return ok();
}
