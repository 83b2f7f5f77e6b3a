// Rows into and out of the 8-bit paged KV cache (kv8.cuh has the format).
//
//   kv8_epilogue_kernel   QKV epilogue with a quantising append: per-head RMSNorm (optional) and RoPE of
//                         q and k in fp32, q rounded once to bf16, k and v rows rounded once to e4m3 and
//                         written with their exponents to the cache rows of their sequences
//   kv8_read_kernel       cached rows back as bf16 (exact), for the prefill kernel
//
// Against qkv_epilogue.cu, which rounds to bf16 after the norm as the reference does: here the value
// stays fp32 until its one rounding, because the stored 8 bits cannot reproduce the reference's bits
// anyway and one rounding is nearer to the formula.  Both kernels are bound by HBM bytes at prefill
// sizes and by latency at decode sizes.
#include <algorithm>
#include <type_traits>

#include "kv8.cuh"
#include "rope_math.cuh"

namespace mllm_b200 {
namespace {

struct Epilogue8Args {
    const __nv_bfloat16* q;
    const __nv_bfloat16* k;
    const __nv_bfloat16* v;
    int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;
    int T, H, Hkv, n_seqs;
    const int64_t* positions;    // [T], or the tables
    float log_theta;
    const float* rope_cos;       // [T, D]
    const float* rope_sin;
    const __nv_bfloat16* q_gamma;
    const __nv_bfloat16* k_gamma;
    float eps;
    __nv_bfloat16* q_out;
    int64_t o_st, o_sh;
    const int32_t* cu_seqlens;   // [n_seqs + 1]
    const int32_t* start;        // [n_seqs] cache rows before the call
    KvLayout lay;
    Kv8View kv;
};

// A warp takes one token (or, when tokens are few, a part of its rows), a group of D / 16 lanes a head row at a
// time: lane j of it holds the columns 8j .. 8j+7 and D/2 + 8j .. D/2 + 8j+7, so both halves of a RoPE pair are in
// one thread, a row moves as 16-byte loads, and norm sums and maxima are three (two) xor-shuffles for a whole warp
// of rows.  What the rows of a token share (its sequence, cache row, angles) is worked out once per warp and serves
// all its rows, and the norm weights are folded into the angles' coefficients; with one warp per token instead of
// two this overhead, as large as the work on six rows, halves.  The next rows are loaded before the present ones are
// worked on.
constexpr int kEpiWarps = 4;       // tokens per CTA
constexpr int kEpiThreads = kEpiWarps * 32;
constexpr int kEpiCtas = 4;        // per SM: 128 registers a thread
constexpr int kRowsInFlight = 2;   // q rows a group loads together

struct Row8 {
    uint4 lo, hi;
};

__device__ __forceinline__ void unpack8(uint4 w, float (&x)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(u[i] << 16);
        x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
}

// One 16-byte load where the address allows it, else element by element (a projection's rows may start
// at any element).
__device__ __forceinline__ uint4 load8(const __nv_bfloat16* p, bool wide) {
    if (wide) return *reinterpret_cast<const uint4*>(p);
    const uint16_t* u = reinterpret_cast<const uint16_t*>(p);
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = (uint32_t)u[2 * i] | ((uint32_t)u[2 * i + 1] << 16);
    return make_uint4(r[0], r[1], r[2], r[3]);
}

// Coefficients of y_lo = x_lo a + x_hi b, y_hi = x_hi c + x_lo d: the rotation, with the norm weights in it.
struct Rotation {
    float a[8], b[8], c[8], d[8];
};

template <int D>
__device__ __forceinline__ void fold(Rotation& r, const float* cos_, const float* sin_, const __nv_bfloat16* gamma, int j,
                                     bool wide) {
    float gl[8], gh[8];
    if (gamma != nullptr) {
        unpack8(load8(gamma + 8 * j, wide), gl);
        unpack8(load8(gamma + D / 2 + 8 * j, wide), gh);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) gl[e] = gh[e] = 1.f;
    }
#pragma unroll
    for (int e = 0; e < 8; e += 4) {   // a group's lanes read neighbouring 16-byte pieces
        const float4 cl = *reinterpret_cast<const float4*>(cos_ + 8 * j + e);
        const float4 sl = *reinterpret_cast<const float4*>(sin_ + 8 * j + e);
        const float4 ch = *reinterpret_cast<const float4*>(cos_ + D / 2 + 8 * j + e);
        const float4 sh = *reinterpret_cast<const float4*>(sin_ + D / 2 + 8 * j + e);
        mul2(r.a[e], r.a[e + 1], cl.x, cl.y, gl[e], gl[e + 1]);
        mul2(r.a[e + 2], r.a[e + 3], cl.z, cl.w, gl[e + 2], gl[e + 3]);
        mul2(r.b[e], r.b[e + 1], -sl.x, -sl.y, gh[e], gh[e + 1]);
        mul2(r.b[e + 2], r.b[e + 3], -sl.z, -sl.w, gh[e + 2], gh[e + 3]);
        mul2(r.c[e], r.c[e + 1], ch.x, ch.y, gh[e], gh[e + 1]);
        mul2(r.c[e + 2], r.c[e + 3], ch.z, ch.w, gh[e + 2], gh[e + 3]);
        mul2(r.d[e], r.d[e + 1], sh.x, sh.y, gl[e], gl[e + 1]);
        mul2(r.d[e + 2], r.d[e + 3], sh.z, sh.w, gl[e + 2], gl[e + 3]);
    }
}

// RMSNorm (where asked) and rotation of one row; the group's lanes hold its columns.
template <int LPR>
__device__ __forceinline__ void norm_rotate(const Row8& row, const Rotation& r, bool norm, float eps, unsigned gmask,
                                            float (&lo)[8], float (&hi)[8]) {
    float x[8], y[8];
    unpack8(row.lo, x);
    unpack8(row.hi, y);
    float rr = 1.f;
    if (norm) {
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            fma2(s0, s1, x[e], x[e + 1], x[e], x[e + 1], s0, s1);
            fma2(s0, s1, y[e], y[e + 1], y[e], y[e + 1], s0, s1);
        }
        float ss = s0 + s1;
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(gmask, ss, o);
        rr = rsqrtf(ss * (1.f / (16 * LPR)) + eps);
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            mul2(x[e], x[e + 1], x[e], x[e + 1], rr, rr);
            mul2(y[e], y[e + 1], y[e], y[e + 1], rr, rr);
        }
    }
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        float u0, u1;
        mul2(u0, u1, y[e], y[e + 1], r.b[e], r.b[e + 1]);
        fma2(lo[e], lo[e + 1], x[e], x[e + 1], r.a[e], r.a[e + 1], u0, u1);
        mul2(u0, u1, x[e], x[e + 1], r.d[e], r.d[e + 1]);
        fma2(hi[e], hi[e + 1], y[e], y[e + 1], r.c[e], r.c[e + 1], u0, u1);
    }
}

// Quantises a row and writes it with its exponent.
template <int D, int LPR>
__device__ __forceinline__ void store_row8(float (&lo)[8], float (&hi)[8], unsigned gmask, int j, bool at, uint8_t* dst,
                                           uint8_t* exp) {
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmax3_abs_nan(lo[e], hi[e], top);
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) top = fmax3_abs_nan(top, __shfl_xor_sync(gmask, top, o), 0.f);
    // The row (the group's lanes agree) has elements that are not finite, or that would be rounded to 256 * 2^kExpMax,
    // which is no bf16 number.
    const bool odd = !(top < 248.f * 0x1p120f);
    if (odd) {
        // the former are stored as NaN (the conversion would saturate an infinity), the others as if they were not there;
        // the latter as the largest that is one
        top = 0.f;
        auto hold = [&](float& x) {
            if (fabsf(x) < INFINITY) x = fminf(fmaxf(x, -kRowMax), kRowMax), top = fmaxf(top, fabsf(x));
            else x = NAN;
        };
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            hold(lo[e]);
            hold(hi[e]);
        }
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(gmask, top, o));
    }
    const int e2 = row_exponent(top);
    const float inv = pow2i(-e2);
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        mul2(lo[e], lo[e + 1], lo[e], lo[e + 1], inv, inv);
        mul2(hi[e], hi[e + 1], hi[e], hi[e + 1], inv, inv);
    }
    if (!at) return;
    *reinterpret_cast<uint2*>(dst + 8 * j) =
        make_uint2(pack_e4m3x4(lo[0], lo[1], lo[2], lo[3]), pack_e4m3x4(lo[4], lo[5], lo[6], lo[7]));
    *reinterpret_cast<uint2*>(dst + D / 2 + 8 * j) =
        make_uint2(pack_e4m3x4(hi[0], hi[1], hi[2], hi[3]), pack_e4m3x4(hi[4], hi[5], hi[6], hi[7]));
    if (j == 0) *exp = (uint8_t)(e2 + 127);
}

// Where a token's K and V rows go.  The warp's lanes call it together.
struct TokenSlot {
    int seq = 0, first = 0, end = 0;   // the sequence that owns the token, and its tokens (end: look again from there on)
    int start = 0;                     // its cache rows before the call
    bool owned = false;
};

// Fills `s` for token t: its sequence is the number of sequences that end at or before it (32 ends per ballot).
__device__ __forceinline__ void find_sequence(const Epilogue8Args& a, int t, int lane, TokenSlot& s) {
    s.seq = 0;
    for (int base = 0; base < a.n_seqs; base += 32) {
        const int i = base + lane;
        const unsigned ended = __ballot_sync(0xffffffffu, i < a.n_seqs && a.cu_seqlens[i + 1] <= t);
        s.seq += __popc(ended);
        if (ended != 0xffffffffu) break;
    }
    const bool in = s.seq < a.n_seqs;
    s.first = in ? a.cu_seqlens[s.seq] : 0x7fffffff;
    s.owned = s.first <= t;
    s.end = s.owned ? a.cu_seqlens[s.seq + 1] : s.first;   // where no sequence's tokens end: with the next one's first
    s.start = s.owned ? a.start[s.seq] : 0;
}

template <int D, bool kWide, bool kTable>
__global__ void __launch_bounds__(kEpiThreads, kEpiCtas) kv8_epilogue_kernel(Epilogue8Args a) {
    constexpr int LPR = D / 16;                     // lanes per row
    constexpr int GROUPS = 32 / LPR;                // rows a warp works on at a time
    __shared__ __align__(16) float s_angle[kEpiWarps][2][D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = blockIdx.x * kEpiWarps + warp;
    if (t >= a.T) return;
    const int j = lane % LPR;
    const int grp = lane / LPR + blockIdx.y * GROUPS;
    const int step = GROUPS * gridDim.y;
    pdl_wait();
    pdl_trigger();

    const __nv_bfloat16* q = a.q + (int64_t)t * a.q_st + 8 * j;
    const __nv_bfloat16* k = a.k + (int64_t)t * a.k_st + 8 * j;
    const __nv_bfloat16* v = a.v + (int64_t)t * a.v_st + 8 * j;
    const Row8 none = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
    auto load_row = [&](const __nv_bfloat16* base, int64_t sh, int r, int n) -> Row8 {
        if (r >= n) return none;
        const __nv_bfloat16* src = base + r * sh;
        return {load8(src, kWide), load8(src + D / 2, kWide)};
    };
    // the group's first rows of each kind are on their way while the token's shared values are worked out
    Row8 krow = load_row(k, a.k_sh, grp, a.Hkv), vrow = load_row(v, a.v_sh, grp, a.Hkv), rows[kRowsInFlight];
#pragma unroll
    for (int i = 0; i < kRowsInFlight; ++i) rows[i] = load_row(q, a.q_sh, grp + i * step, a.H);

    TokenSlot ts;
    find_sequence(a, t, lane, ts);
    if (!ts.owned) return;                          // no sequence's token: nothing of it is written
    int blk = 0, crow = 0;
    bool at = false;
    if (ts.start < 0) {
        if (lane == 0 && blockIdx.y == 0) record_error(kErrBadLength);
    } else {
        at = kv_locate(a.lay, ts.seq, (int64_t)ts.start + (t - ts.first), blk, crow);
    }

    // the token's angles
    float* s_cos = s_angle[warp][0];
    float* s_sin = s_angle[warp][1];
    if constexpr (kTable) {
#pragma unroll
        for (int d = lane; d < D; d += 32) {
            s_cos[d] = a.rope_cos[(int64_t)t * D + d];
            s_sin[d] = a.rope_sin[(int64_t)t * D + d];
        }
    } else {
        const int64_t pos = a.positions[t];
#pragma unroll
        for (int d = lane; d < D / 2; d += 32) {
            float c, s;
            rope_angle_cos_sin(pos, d, D, a.log_theta, c, s);
            s_cos[d] = s_cos[d + D / 2] = c;
            s_sin[d] = s_sin[d + D / 2] = s;
        }
    }
    __syncwarp();
    // A group's lanes take the same branches; another group's in the warp may not, so the shuffles name the
    // group's lanes only.
    const unsigned gmask = ((1u << LPR) - 1u) << (lane - j);
    const bool norm = a.q_gamma != nullptr;
    Rotation rot;
    float lo[8], hi[8];

    // ---- k, then v ----
    fold<D>(rot, s_cos, s_sin, a.k_gamma, j, kWide);
    {
        uint8_t* pool = a.kv.k_pool + blk * a.kv.p_sb + crow * a.kv.p_st;
        uint8_t* exps = a.kv.k_exp + blk * a.kv.e_sb + crow;
        for (int g = grp; g < a.Hkv; g += step) {
            const Row8 next = load_row(k, a.k_sh, g + step, a.Hkv);
            norm_rotate<LPR>(krow, rot, norm, a.eps, gmask, lo, hi);
            store_row8<D, LPR>(lo, hi, gmask, j, at, pool + g * a.kv.p_sh, exps + g * a.kv.e_sh);
            krow = next;
        }
        pool = a.kv.v_pool + blk * a.kv.p_sb + crow * a.kv.p_st;
        exps = a.kv.v_exp + blk * a.kv.e_sb + crow;
        for (int g = grp; g < a.Hkv; g += step) {
            const Row8 next = load_row(v, a.v_sh, g + step, a.Hkv);
            unpack8(vrow.lo, lo);
            unpack8(vrow.hi, hi);
            store_row8<D, LPR>(lo, hi, gmask, j, at, pool + g * a.kv.p_sh, exps + g * a.kv.e_sh);
            vrow = next;
        }
    }
    // ---- q ----
    fold<D>(rot, s_cos, s_sin, a.q_gamma, j, kWide);
    __nv_bfloat16* out = a.q_out + (int64_t)t * a.o_st + 8 * j;
    for (int h0 = grp; h0 < a.H; h0 += step * kRowsInFlight) {
        Row8 next[kRowsInFlight];
#pragma unroll
        for (int i = 0; i < kRowsInFlight; ++i) next[i] = load_row(q, a.q_sh, h0 + (kRowsInFlight + i) * step, a.H);
#pragma unroll
        for (int i = 0; i < kRowsInFlight; ++i) {
            const int h = h0 + i * step;
            if (h >= a.H) break;
            norm_rotate<LPR>(rows[i], rot, norm, a.eps, gmask, lo, hi);
            __nv_bfloat16* dst = out + h * a.o_sh;
            *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16x2(lo[0], lo[1]), pack_bf16x2(lo[2], lo[3]),
                                                        pack_bf16x2(lo[4], lo[5]), pack_bf16x2(lo[6], lo[7]));
            *reinterpret_cast<uint4*>(dst + D / 2) = make_uint4(pack_bf16x2(hi[0], hi[1]), pack_bf16x2(hi[2], hi[3]),
                                                                pack_bf16x2(hi[4], hi[5]), pack_bf16x2(hi[6], hi[7]));
        }
#pragma unroll
        for (int i = 0; i < kRowsInFlight; ++i) rows[i] = next[i];
    }
}

// The same for many tokens.  The kernel above is bound by the loads that its registers can hold in flight (72 us for
// 16017 tokens of 32 + 2 x 8 heads of 128, 380 MB).  Here every lane fetches its 32 bytes of a row into a ring of its
// own in shared memory (cp.async; a lane reads back only what it fetched, so the rows need no barrier), kRing batches
// of rows ahead, across tokens: 64 us, 5.9 TB/s, where a copy of that size makes 6.0.  Warps take tokens in turn, so
// that all SMs work on neighbouring rows of HBM (consecutive tokens per warp: 68 to 71 us), and look the sequence up
// only when it changes.
constexpr int kRing = 4;           // batches of 32 / LPR rows in flight per warp
constexpr int kAngles = 4;         // angle rows: a token has at least three batches, so the loads run up to two tokens ahead
constexpr int kStreamCtas = 4;     // CTAs per SM

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

template <int D, bool kTable>
__global__ void __launch_bounds__(kEpiThreads, kStreamCtas) kv8_epilogue_stream_kernel(Epilogue8Args a) {
    constexpr int LPR = D / 16;
    constexpr int GROUPS = 32 / LPR;
    __shared__ __align__(16) uint4 s_ring[kEpiWarps][kRing][2][32];
    __shared__ __align__(16) float s_angle[kEpiWarps][kAngles][2][D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int j = lane % LPR, grp = lane / LPR;
    const int w = blockIdx.x * kEpiWarps + warp, warps = gridDim.x * kEpiWarps;
    pdl_wait();
    pdl_trigger();
    if (w >= a.T) return;
    const int nk = (a.Hkv + GROUPS - 1) / GROUPS, nq = (a.H + GROUPS - 1) / GROUPS;

    // ---- the fetching side: the group's row fr of kind fk (k, v, q) of token ft, at fp, into slot fs ----
    int ft = w, fi = 0;                    // the token, and which of this warp's it is
    int fk = 0, fr = grp, fn = a.Hkv, fs = 0;
    const __nv_bfloat16* fp = a.k + (int64_t)w * a.k_st + grp * a.k_sh + 8 * j;
    int64_t fstep = GROUPS * a.k_sh;
    int left = nk;                         // batches of the kind still to fetch
    const uint32_t ring = smem_u32(&s_ring[warp][0][0][lane]);
    auto fetch = [&]() {
        if (ft < a.T) {
            if (fr < fn) {
                cp_async16(ring + fs * 1024, fp);
                cp_async16(ring + fs * 1024 + 512, fp + D / 2);
            }
            if (kTable && fk == 0 && left == nk) {
                float (*ang)[D] = s_angle[warp][fi % kAngles];
                for (int d = 4 * lane; d < D; d += 128) {
                    cp_async16(smem_u32(&ang[0][d]), a.rope_cos + (int64_t)ft * D + d);
                    cp_async16(smem_u32(&ang[1][d]), a.rope_sin + (int64_t)ft * D + d);
                }
            }
            fp += fstep;
            fr += GROUPS;
            if (--left == 0) {             // on to the next kind, or the next token
                fr = grp;
                if (fk == 0) {
                    fk = 1;
                    left = nk;
                    fp = a.v + (int64_t)ft * a.v_st + grp * a.v_sh + 8 * j;
                    fstep = GROUPS * a.v_sh;
                } else if (fk == 1) {
                    fk = 2;
                    left = nq;
                    fn = a.H;
                    fp = a.q + (int64_t)ft * a.q_st + grp * a.q_sh + 8 * j;
                    fstep = GROUPS * a.q_sh;
                } else {
                    ft += warps;
                    ++fi;
                    fk = 0;
                    left = nk;
                    fn = a.Hkv;
                    fp = a.k + (int64_t)ft * a.k_st + grp * a.k_sh + 8 * j;
                    fstep = GROUPS * a.k_sh;
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (++fs == kRing) fs = 0;
    };
#pragma unroll
    for (int i = 0; i < kRing - 1; ++i) fetch();

    int cs = 0;
    // The next batch's rows: kRing - 1 groups are in flight, so the oldest is complete when at most kRing - 2 are not.
    auto take = [&]() -> Row8 {
        asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 2) : "memory");
        const Row8 r = {s_ring[warp][cs][0][lane], s_ring[warp][cs][1][lane]};
        if (++cs == kRing) cs = 0;
        return r;
    };
    const unsigned gmask = ((1u << LPR) - 1u) << (lane - j);
    const bool norm = a.q_gamma != nullptr;
    Rotation rot;
    float lo[8], hi[8];
    TokenSlot ts;
    for (int t = w, it = 0; t < a.T; t += warps, ++it) {
        if (t >= ts.end) find_sequence(a, t, lane, ts);
        int blk = 0, crow = 0;
        bool at = false;
        if (ts.owned) {
            if (ts.start < 0) {
                if (lane == 0) record_error(kErrBadLength);
            } else {
                at = kv_locate(a.lay, ts.seq, (int64_t)ts.start + (t - ts.first), blk, crow);
            }
        }
        float* s_cos = s_angle[warp][it % kAngles][0];
        float* s_sin = s_angle[warp][it % kAngles][1];
        if constexpr (kTable) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 2) : "memory");   // the token's first batch, and its angles
        } else {
            const int64_t pos = a.positions[t];
#pragma unroll
            for (int d = lane; d < D / 2; d += 32) {
                float c, s;
                rope_angle_cos_sin(pos, d, D, a.log_theta, c, s);
                s_cos[d] = s_cos[d + D / 2] = c;
                s_sin[d] = s_sin[d + D / 2] = s;
            }
        }
        __syncwarp();      // every lane's angles
        fold<D>(rot, s_cos, s_sin, a.k_gamma, j, true);
        uint8_t* pool = a.kv.k_pool + blk * a.kv.p_sb + crow * a.kv.p_st;
        uint8_t* exps = a.kv.k_exp + blk * a.kv.e_sb + crow;
        for (int g = grp; g < nk * GROUPS; g += GROUPS) {
            const Row8 row = take();
            fetch();
            norm_rotate<LPR>(row, rot, norm, a.eps, gmask, lo, hi);
            store_row8<D, LPR>(lo, hi, gmask, j, at && g < a.Hkv, pool + g * a.kv.p_sh, exps + g * a.kv.e_sh);
        }
        pool = a.kv.v_pool + blk * a.kv.p_sb + crow * a.kv.p_st;
        exps = a.kv.v_exp + blk * a.kv.e_sb + crow;
        for (int g = grp; g < nk * GROUPS; g += GROUPS) {
            const Row8 row = take();
            fetch();
            unpack8(row.lo, lo);
            unpack8(row.hi, hi);
            store_row8<D, LPR>(lo, hi, gmask, j, at && g < a.Hkv, pool + g * a.kv.p_sh, exps + g * a.kv.e_sh);
        }
        fold<D>(rot, s_cos, s_sin, a.q_gamma, j, true);
        __nv_bfloat16* out = a.q_out + (int64_t)t * a.o_st + 8 * j;
        for (int h = grp; h < nq * GROUPS; h += GROUPS) {
            const Row8 row = take();
            fetch();
            norm_rotate<LPR>(row, rot, norm, a.eps, gmask, lo, hi);
            if (h < a.H && ts.owned) {
                __nv_bfloat16* dst = out + h * a.o_sh;
                *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16x2(lo[0], lo[1]), pack_bf16x2(lo[2], lo[3]),
                                                            pack_bf16x2(lo[4], lo[5]), pack_bf16x2(lo[6], lo[7]));
                *reinterpret_cast<uint4*>(dst + D / 2) = make_uint4(pack_bf16x2(hi[0], hi[1]), pack_bf16x2(hi[2], hi[3]),
                                                                    pack_bf16x2(hi[4], hi[5]), pack_bf16x2(hi[6], hi[7]));
            }
        }
    }
}

struct Read8Args {
    const int32_t* first;        // [n], or NULL: row 0
    const int32_t* lens;         // [n]
    int n, Hkv, rows;
    __nv_bfloat16* k_out;        // [n, Hkv, rows, D] with strides
    __nv_bfloat16* v_out;
    int64_t o_sb, o_sh, o_st;
    KvLayout lay;
    Kv8View kv;
};

// 8 columns of a row per thread (an 8-byte load, a 16-byte store, so that a warp's stores are contiguous), D / 8
// threads a row; a thread takes its columns of K and V of a few rows, so that one look into the block table serves
// both, and has all their loads in flight.  blockIdx.y is the (sequence, kv head).
constexpr int kReadThreads = 256;
constexpr int kReadRowsPerThread = 2;

template <int D>
__global__ void __launch_bounds__(kReadThreads, 6) kv8_read_kernel(Read8Args a) {
    constexpr int TPR = D / 8;
    constexpr int RPB = kReadThreads / TPR;
    pdl_wait();
    pdl_trigger();
    const int b = blockIdx.y / a.Hkv, g = blockIdx.y - b * a.Hkv;
    const int c = threadIdx.x % TPR;
    const int r0 = blockIdx.x * (kReadRowsPerThread * RPB) + threadIdx.x / TPR;
    int first = a.first ? a.first[b] : 0, len = a.lens[b];
    if (first < 0 || len < 0) {
        if (threadIdx.x == 0) record_error(kErrBadLength);
        first = len = 0;
    }
    uint2 w[kReadRowsPerThread][2];
    float sc[kReadRowsPerThread][2];
#pragma unroll
    for (int i = 0; i < kReadRowsPerThread; ++i) {
        const int r = r0 + i * RPB;
        w[i][0] = w[i][1] = make_uint2(0u, 0u);
        sc[i][0] = sc[i][1] = 0.f;
        if (r < a.rows && r < len - first) {
            int blk, row;
            if (kv_locate(a.lay, b, (int64_t)first + r, blk, row)) {
                const int64_t at = blk * a.kv.p_sb + g * a.kv.p_sh + row * a.kv.p_st + 8 * c;
                const int64_t ea = blk * a.kv.e_sb + g * a.kv.e_sh + row;
                w[i][0] = __ldcs(reinterpret_cast<const uint2*>(a.kv.k_pool + at));
                w[i][1] = __ldcs(reinterpret_cast<const uint2*>(a.kv.v_pool + at));
                sc[i][0] = exp_byte_scale(a.kv.k_exp[ea]);
                sc[i][1] = exp_byte_scale(a.kv.v_exp[ea]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < kReadRowsPerThread; ++i) {
        const int r = r0 + i * RPB;
        if (r >= a.rows) break;
        const int64_t at = (int64_t)b * a.o_sb + (int64_t)g * a.o_sh + (int64_t)r * a.o_st + 8 * c;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            const uint32_t in[2] = {w[i][kv].x, w[i][kv].y};
            uint32_t o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t h = e4m3x2_to_f16x2((uint16_t)(in[e >> 1] >> (16 * (e & 1))));
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
                // exact: 4 significant bits times a power of two
                o[e] = pack_bf16x2(f.x * sc[i][kv], f.y * sc[i][kv]);
            }
            *reinterpret_cast<uint4*>((kv ? a.v_out : a.k_out) + at) = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
}

}  // namespace

MLLM_DEFINE_STATUS_READER(kv8_rows)

}  // namespace mllm_b200

using namespace mllm_b200;

extern "C" int mllm_qkv_epilogue_varlen_paged_kv8(
    const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_st, int64_t k_sh, const void* v, int64_t v_st,
    int64_t v_sh, int total_tokens, int num_heads, int num_kv_heads, int head_dim, const int64_t* positions,
    double rope_theta, const float* rope_cos, const float* rope_sin, const void* q_norm_weight,
    const void* k_norm_weight, double rms_norm_eps, void* q_out, int64_t q_out_st, int64_t q_out_sh,
    const mllm_paged_kv8* kv, const int32_t* cu_seqlens, int batch, const int32_t* cache_start, mllm_stream_t stream) {
    MLLM_NVTX_RANGE("mllm_qkv_epilogue_varlen_paged_kv8");
    if (total_tokens < 0 || batch < 0 || num_heads <= 0 || num_kv_heads <= 0 || total_tokens > 0x3fffffff)
        return fail(MLLM_ERR_INVALID_ARGUMENT, "qkv_epilogue_kv8: bad sizes");
    if (num_heads % num_kv_heads != 0)
        return fail(MLLM_ERR_INVALID_ARGUMENT, "Attention: num_heads must be divisible by num_kv_heads.");
    if (head_dim != 64 && head_dim != 128)
        return fail(MLLM_ERR_UNSUPPORTED, "qkv_epilogue_kv8: head_dim must be 64 or 128");
    if ((q_norm_weight == nullptr) != (k_norm_weight == nullptr))
        return fail(MLLM_ERR_INVALID_ARGUMENT, "qkv_epilogue_kv8: give both q/k norm weights or neither");
    if ((rope_cos == nullptr) != (rope_sin == nullptr))
        return fail(MLLM_ERR_INVALID_ARGUMENT, "qkv_epilogue_kv8: give both rope tables or neither");
    if (rope_cos == nullptr && positions == nullptr)
        return fail(MLLM_ERR_INVALID_ARGUMENT, "qkv_epilogue_kv8: positions or rope tables required");
    if (rope_cos == nullptr && !(rope_theta > 0.0))
        return fail(MLLM_ERR_INVALID_ARGUMENT, "qkv_epilogue_kv8: rope_theta must be positive");
    Epilogue8Args a = {};
    if (int st = paged_layout8(kv, 0, head_dim, "qkv_epilogue_kv8", &a.lay, &a.kv)) return st;
    if (total_tokens == 0 || batch == 0) return ok();
    if (!q || !k || !v || !q_out || !cu_seqlens || !cache_start)
        return fail(MLLM_ERR_INVALID_ARGUMENT, "qkv_epilogue_kv8: null pointer");
    if (!aligned(q, 2) || !aligned(k, 2) || !aligned(v, 2))
        return fail(MLLM_ERR_INVALID_ARGUMENT, "qkv_epilogue_kv8: q/k/v misaligned");
    if (!aligned(q_out, 16) || q_out_st % 8 || q_out_sh % 8)
        return fail(MLLM_ERR_INVALID_ARGUMENT, "qkv_epilogue_kv8: q_out and its strides must be multiples of 16 bytes");
    int num_sms = 0;
    if (int st = require_sm100(&num_sms)) return st;
    a.q = (const __nv_bfloat16*)q;
    a.k = (const __nv_bfloat16*)k;
    a.v = (const __nv_bfloat16*)v;
    a.q_st = q_st; a.q_sh = q_sh;
    a.k_st = k_st; a.k_sh = k_sh;
    a.v_st = v_st; a.v_sh = v_sh;
    a.T = total_tokens;
    a.H = num_heads;
    a.Hkv = num_kv_heads;
    a.n_seqs = batch;
    a.positions = positions;
    a.log_theta = rope_cos ? 0.f : rope_log_theta(rope_theta);
    a.rope_cos = rope_cos;
    a.rope_sin = rope_sin;
    a.q_gamma = (const __nv_bfloat16*)q_norm_weight;
    a.k_gamma = (const __nv_bfloat16*)k_norm_weight;
    a.eps = (float)rms_norm_eps;
    a.q_out = (__nv_bfloat16*)q_out;
    a.o_st = q_out_st; a.o_sh = q_out_sh;
    a.cu_seqlens = cu_seqlens;
    a.start = cache_start;
    // 16-byte loads need every row to start on 16 bytes
    bool wide = aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(q_norm_weight, 16) && aligned(k_norm_weight, 16);
    for (int64_t s : {q_st, q_sh, k_st, k_sh, v_st, v_sh}) wide = wide && s % 8 == 0;
    // few tokens: a token's rows over several warps, up to one row per group of lanes
    const int groups = 32 / (head_dim / 16);
    const int most = (std::max(num_heads, num_kv_heads) + groups - 1) / groups;
    const int parts = std::max(1, std::min(most, 8 * num_sms / total_tokens));
    const dim3 grid((total_tokens + kEpiWarps - 1) / kEpiWarps, parts);
    const int warps = kStreamCtas * kEpiWarps * num_sms;
    const bool stream_rows = wide && aligned(rope_cos, 16) && aligned(rope_sin, 16) && total_tokens >= warps;
    auto launch = [&](void (*kern)(Epilogue8Args)) {
        return launch_pdl(kern, grid, dim3(kEpiThreads), 0, (cudaStream_t)stream, a);
    };
    auto pick = [&](auto table) {
        constexpr bool kTable = decltype(table)::value;
        if (stream_rows) {
            const dim3 g(kStreamCtas * num_sms);
            return head_dim == 128 ? launch_pdl(kv8_epilogue_stream_kernel<128, kTable>, g, dim3(kEpiThreads), 0,
                                                (cudaStream_t)stream, a)
                                   : launch_pdl(kv8_epilogue_stream_kernel<64, kTable>, g, dim3(kEpiThreads), 0,
                                                (cudaStream_t)stream, a);
        }
        if (head_dim == 128)
            return wide ? launch(kv8_epilogue_kernel<128, true, kTable>) : launch(kv8_epilogue_kernel<128, false, kTable>);
        return wide ? launch(kv8_epilogue_kernel<64, true, kTable>) : launch(kv8_epilogue_kernel<64, false, kTable>);
    };
    const cudaError_t e = rope_cos ? pick(std::true_type{}) : pick(std::false_type{});
    if (int st = check_cuda(e, "kv8_epilogue_kernel launch")) return st;
    return ok();
}

extern "C" int mllm_kv8_read_bf16(const mllm_paged_kv8* kv, const int32_t* first_rows, const int32_t* kv_lens, int batch,
                                  int num_kv_heads, int head_dim, int rows, void* k_out, void* v_out, int64_t out_sb,
                                  int64_t out_sh, int64_t out_st, mllm_stream_t stream) {
    MLLM_NVTX_RANGE("mllm_kv8_read_bf16");
    if (batch < 0 || num_kv_heads <= 0 || rows < 0) return fail(MLLM_ERR_INVALID_ARGUMENT, "kv8_read: bad sizes");
    if (head_dim != 64 && head_dim != 128) return fail(MLLM_ERR_UNSUPPORTED, "kv8_read: head_dim must be 64 or 128");
    Read8Args a = {};
    if (int st = paged_layout8(kv, 0, head_dim, "kv8_read", &a.lay, &a.kv)) return st;
    if ((int64_t)batch * num_kv_heads > 65535)
        return fail(MLLM_ERR_UNSUPPORTED, "kv8_read: more than 65535 (sequence, kv head) pairs");
    if (batch == 0 || rows == 0) return ok();
    if (!kv_lens || !k_out || !v_out) return fail(MLLM_ERR_INVALID_ARGUMENT, "kv8_read: null pointer");
    if (!aligned(k_out, 16) || !aligned(v_out, 16) || out_sb % 8 || out_sh % 8 || out_st % 8 || out_st < head_dim)
        return fail(MLLM_ERR_INVALID_ARGUMENT, "kv8_read: outputs and their strides must be multiples of 16 bytes");
    if (int st = require_sm100()) return st;
    a.first = first_rows;
    a.lens = kv_lens;
    a.n = batch;
    a.Hkv = num_kv_heads;
    a.rows = rows;
    a.k_out = (__nv_bfloat16*)k_out;
    a.v_out = (__nv_bfloat16*)v_out;
    a.o_sb = out_sb; a.o_sh = out_sh; a.o_st = out_st;
    const int rpb = kReadThreads / (head_dim / 8) * kReadRowsPerThread;
    const dim3 grid((rows + rpb - 1) / rpb, batch * num_kv_heads);
    cudaError_t e = head_dim == 128
        ? launch_pdl(kv8_read_kernel<128>, grid, dim3(kReadThreads), 0, (cudaStream_t)stream, a)
        : launch_pdl(kv8_read_kernel<64>, grid, dim3(kReadThreads), 0, (cudaStream_t)stream, a);
    if (int st = check_cuda(e, "kv8_read_kernel launch")) return st;
    return ok();
}
