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

// A group of D / 8 lanes owns one head row; lane j of it holds the columns 4j .. 4j+3 and
// D/2 + 4j .. D/2 + 4j+3, so both halves of a RoPE pair are in one thread, a row moves as 8-byte loads,
// and norm sums and maxima are xor-shuffles inside the group.
constexpr int kEpiThreads = 256;
constexpr int kRowsInFlight = 3;   // rows a group loads before it works on the first

struct Row8 {
    uint2 lo, hi;
};

__device__ __forceinline__ void unpack4(uint2 w, float (&x)[4]) {
    const __nv_bfloat162 a = *reinterpret_cast<const __nv_bfloat162*>(&w.x);
    const __nv_bfloat162 b = *reinterpret_cast<const __nv_bfloat162*>(&w.y);
    x[0] = __bfloat162float(a.x);
    x[1] = __bfloat162float(a.y);
    x[2] = __bfloat162float(b.x);
    x[3] = __bfloat162float(b.y);
}

// One 8-byte load where the address allows it, else element by element (a projection's rows may start
// at any element).
__device__ __forceinline__ uint2 load4(const __nv_bfloat16* p, bool wide) {
    if (wide) return *reinterpret_cast<const uint2*>(p);
    const uint16_t* u = reinterpret_cast<const uint16_t*>(p);
    return make_uint2((uint32_t)u[0] | ((uint32_t)u[1] << 16), (uint32_t)u[2] | ((uint32_t)u[3] << 16));
}

template <int D>
__global__ void __launch_bounds__(kEpiThreads) kv8_epilogue_kernel(Epilogue8Args a, bool wide) {
    constexpr int LPR = D / 8;                      // lanes per row
    constexpr int GROUPS = kEpiThreads / LPR;
    const int t = blockIdx.x;
    const int lane = threadIdx.x & 31;
    const int j = threadIdx.x % LPR;
    const int grp = threadIdx.x / LPR + blockIdx.y * GROUPS;
    const int step = GROUPS * gridDim.y;
    const int total = a.H + 2 * a.Hkv;
    pdl_wait();
    pdl_trigger();

    auto row_src = [&](int r) -> const __nv_bfloat16* {
        if (r < a.H) return a.q + (int64_t)t * a.q_st + (int64_t)r * a.q_sh;
        if (r < a.H + a.Hkv) return a.k + (int64_t)t * a.k_st + (int64_t)(r - a.H) * a.k_sh;
        return a.v + (int64_t)t * a.v_st + (int64_t)(r - a.H - a.Hkv) * a.v_sh;
    };
    Row8 rows[kRowsInFlight];
    auto load_rows = [&](int r0) {
#pragma unroll
        for (int i = 0; i < kRowsInFlight; ++i) {
            const int r = r0 + i * step;
            if (r < total) {
                const __nv_bfloat16* src = row_src(r);
                rows[i].lo = load4(src + 4 * j, wide);
                rows[i].hi = load4(src + D / 2 + 4 * j, wide);
            } else {
                rows[i].lo = rows[i].hi = make_uint2(0u, 0u);
            }
        }
    };
    load_rows(grp);

    // the token's sequence: the number of sequences that end at or before it (32 ends per ballot)
    int seq = 0;
    for (int base = 0; base < a.n_seqs; base += 32) {
        const int i = base + lane;
        const unsigned ended = __ballot_sync(0xffffffffu, i < a.n_seqs && a.cu_seqlens[i + 1] <= t);
        seq += __popc(ended);
        if (ended != 0xffffffffu) break;
    }
    const bool owned = seq < a.n_seqs && a.cu_seqlens[seq] <= t;
    if (!owned) return;                             // no sequence's token: nothing of it is written
    const int64_t slot = (int64_t)a.start[seq] + (t - a.cu_seqlens[seq]);
    int blk = 0, crow = 0;
    bool at = false;
    if (a.start[seq] < 0) {
        if (threadIdx.x == 0 && blockIdx.y == 0) record_error(kErrBadLength);
    } else {
        at = kv_locate(a.lay, seq, slot, blk, crow);
    }

    float c_lo[4], s_lo[4], c_hi[4], s_hi[4];
    if (a.rope_cos != nullptr) {
        const float* c = a.rope_cos + (int64_t)t * D;
        const float* s = a.rope_sin + (int64_t)t * D;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            c_lo[i] = c[4 * j + i];
            s_lo[i] = s[4 * j + i];
            c_hi[i] = c[D / 2 + 4 * j + i];
            s_hi[i] = s[D / 2 + 4 * j + i];
        }
    } else {
        const int64_t pos = a.positions[t];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            rope_angle_cos_sin(pos, 4 * j + i, D, a.log_theta, c_lo[i], s_lo[i]);
            c_hi[i] = c_lo[i];
            s_hi[i] = s_lo[i];
        }
    }

    // A group's lanes leave the loop together; lanes of another group in the warp may go on, so the
    // shuffles name the group's lanes only.
    const unsigned gmask = (LPR == 32 ? 0xffffffffu : ((1u << LPR) - 1u)) << (lane - j);
    for (int r0 = grp; r0 < total; r0 += step * kRowsInFlight) {
        if (r0 != grp) load_rows(r0);
#pragma unroll
        for (int i = 0; i < kRowsInFlight; ++i) {
            const int r = r0 + i * step;
            if (r >= total) break;
            const bool is_v = r >= a.H + a.Hkv;
            const bool is_q = r < a.H;
            float lo[4], hi[4];
            unpack4(rows[i].lo, lo);
            unpack4(rows[i].hi, hi);
            if (!is_v) {
                const __nv_bfloat16* gamma = is_q ? a.q_gamma : a.k_gamma;
                if (gamma != nullptr) {
                    float ss = 0.f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) ss = fmaf(lo[e], lo[e], fmaf(hi[e], hi[e], ss));
#pragma unroll
                    for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(gmask, ss, o);
                    const float rr = 1.f / sqrtf(ss * (1.f / D) + a.eps);
                    float gl[4], gh[4];
                    unpack4(load4(gamma + 4 * j, wide), gl);
                    unpack4(load4(gamma + D / 2 + 4 * j, wide), gh);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        lo[e] *= rr * gl[e];
                        hi[e] *= rr * gh[e];
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = lo[e], y = hi[e];
                    lo[e] = x * c_lo[e] - y * s_lo[e];
                    hi[e] = y * c_hi[e] + x * s_hi[e];
                }
            }
            if (is_q) {
                __nv_bfloat16* dst = a.q_out + (int64_t)t * a.o_st + (int64_t)r * a.o_sh;
                *reinterpret_cast<uint2*>(dst + 4 * j) = make_uint2(pack_bf16x2(lo[0], lo[1]), pack_bf16x2(lo[2], lo[3]));
                *reinterpret_cast<uint2*>(dst + D / 2 + 4 * j) =
                    make_uint2(pack_bf16x2(hi[0], hi[1]), pack_bf16x2(hi[2], hi[3]));
                continue;
            }
            float amax = 0.f;   // over finite elements
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = fabsf(lo[e]), y = fabsf(hi[e]);
                amax = fmaxf(amax, fmaxf(x < INFINITY ? x : 0.f, y < INFINITY ? y : 0.f));
            }
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(gmask, amax, o));
            const int e2 = row_exponent(amax);
            const float inv = pow2i(-e2);
            float ql[4], qh[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                ql[e] = fabsf(lo[e]) < INFINITY ? lo[e] * inv : NAN;
                qh[e] = fabsf(hi[e]) < INFINITY ? hi[e] * inv : NAN;
            }
            if (!at) continue;
            const int g = is_v ? r - a.H - a.Hkv : r - a.H;
            uint8_t* dst = (is_v ? a.kv.v_pool : a.kv.k_pool) + blk * a.kv.p_sb + g * a.kv.p_sh + crow * a.kv.p_st;
            *reinterpret_cast<uint32_t*>(dst + 4 * j) = pack_e4m3x4(ql[0], ql[1], ql[2], ql[3]);
            *reinterpret_cast<uint32_t*>(dst + D / 2 + 4 * j) = pack_e4m3x4(qh[0], qh[1], qh[2], qh[3]);
            if (j == 0)
                ((is_v ? a.kv.v_exp : a.kv.k_exp) + blk * a.kv.e_sb + g * a.kv.e_sh)[crow] = (uint8_t)(e2 + 127);
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

// 16 bytes of a row per thread: D / 16 threads a row, 256 threads over 256 / (D / 16) rows of one
// (sequence, kv head); blockIdx.z is K or V.
constexpr int kReadThreads = 256;
constexpr int kReadRowsPerThread = 2;

template <int D>
__global__ void __launch_bounds__(kReadThreads) kv8_read_kernel(Read8Args a) {
    constexpr int TPR = D / 16;
    constexpr int RPB = kReadThreads / TPR;
    pdl_wait();
    pdl_trigger();
    const int b = blockIdx.y / a.Hkv, g = blockIdx.y - b * a.Hkv;
    const bool is_v = blockIdx.z != 0;
    const uint8_t* pool = is_v ? a.kv.v_pool : a.kv.k_pool;
    const uint8_t* exps = is_v ? a.kv.v_exp : a.kv.k_exp;
    __nv_bfloat16* out = (is_v ? a.v_out : a.k_out) + (int64_t)b * a.o_sb + (int64_t)g * a.o_sh;
    const int c = threadIdx.x % TPR;
    const int64_t first = a.first ? a.first[b] : 0;
    const int64_t len = a.lens[b];
    if ((first < 0 || len < 0) && threadIdx.x == 0) record_error(kErrBadLength);
    uint4 w[kReadRowsPerThread];
    float sc[kReadRowsPerThread];
#pragma unroll
    for (int i = 0; i < kReadRowsPerThread; ++i) {
        const int r = (blockIdx.x * kReadRowsPerThread + i) * RPB + threadIdx.x / TPR;
        w[i] = make_uint4(0u, 0u, 0u, 0u);
        sc[i] = 0.f;
        if (r < a.rows && first >= 0 && first + r < len) {
            int blk, row;
            if (kv_locate(a.lay, b, first + r, blk, row)) {
                w[i] = *reinterpret_cast<const uint4*>(pool + blk * a.kv.p_sb + g * a.kv.p_sh + row * a.kv.p_st + 16 * c);
                sc[i] = exp_byte_scale((exps + blk * a.kv.e_sb + g * a.kv.e_sh)[row]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < kReadRowsPerThread; ++i) {
        const int r = (blockIdx.x * kReadRowsPerThread + i) * RPB + threadIdx.x / TPR;
        if (r >= a.rows) continue;
        const uint32_t in[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
        uint32_t o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t h = e4m3x2_to_f16x2((uint16_t)(in[e >> 1] >> (16 * (e & 1))));
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
            o[e] = pack_bf16x2(f.x * sc[i], f.y * sc[i]);   // exact: 4 significant bits times a power of two
        }
        uint4* dst = reinterpret_cast<uint4*>(out + (int64_t)r * a.o_st + 16 * c);
        dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
        dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
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
    if (!aligned(q_out, 8) || q_out_st % 4 || q_out_sh % 4)
        return fail(MLLM_ERR_INVALID_ARGUMENT, "qkv_epilogue_kv8: q_out and its strides must be multiples of 8 bytes");
    if (int st = require_sm100()) return st;
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
    // 8-byte loads need every row to start on 8 bytes
    bool wide = aligned(q, 8) && aligned(k, 8) && aligned(v, 8) && aligned(q_norm_weight, 8) && aligned(k_norm_weight, 8);
    for (int64_t s : {q_st, q_sh, k_st, k_sh, v_st, v_sh}) wide = wide && s % 4 == 0;
    const dim3 grid(total_tokens);
    cudaError_t e = head_dim == 128
        ? launch_pdl(kv8_epilogue_kernel<128>, grid, dim3(kEpiThreads), 0, (cudaStream_t)stream, a, wide)
        : launch_pdl(kv8_epilogue_kernel<64>, grid, dim3(kEpiThreads), 0, (cudaStream_t)stream, a, wide);
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
    const int rpb = kReadThreads / (head_dim / 16) * kReadRowsPerThread;
    const dim3 grid((rows + rpb - 1) / rpb, batch * num_kv_heads, 2);
    cudaError_t e = head_dim == 128
        ? launch_pdl(kv8_read_kernel<128>, grid, dim3(kReadThreads), 0, (cudaStream_t)stream, a)
        : launch_pdl(kv8_read_kernel<64>, grid, dim3(kReadThreads), 0, (cudaStream_t)stream, a);
    if (int st = check_cuda(e, "kv8_read_kernel launch")) return st;
    return ok();
}
