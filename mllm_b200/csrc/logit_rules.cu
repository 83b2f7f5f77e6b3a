// Rules on logits before a token is picked: repetition, presence and frequency penalties, biases and a mask of
// allowed tokens, each row with its own.
//
//   seen  = the token occurs in the row's history;  c = how often among its generated part
//   x     = logit;  if seen: x / r (x >= 0) or x * r (x < 0);  x -= c f;  if c > 0: x -= p;  x += sum of its biases
//   out   = allowed ? x : -inf                           in fp32, rounded once to the logits' type
//
// One CTA takes a stretch of one row's vocabulary.  It reads the row's whole history (8 bytes a token, small against
// the row and in L2 after the first CTA) and counts the tokens of its stretch in shared memory, so nothing has to be
// cleared or kept in global memory and any number of calls may run at once; a bit marks the tokens that have a bias.
// Then it streams the stretch with 16-byte loads: bits are copied where neither a counter nor the mask says otherwise,
// and the few tokens with a counter are worked out where they lie, each lane looping over its own (a branch per token,
// taken by a warp whenever one of its lanes does, took 22.9 us for 64 bf16 rows instead of 14.2).  Streaming first and
// redoing the touched tokens in a second pass over the history took 25 us for 64 fp32 rows instead of 19: its loads
// depend on one another and nothing else is left to do meanwhile.  Everything is taken in a fixed order: counts are whole numbers, and a token's biases are
// summed in list order by the thread that owns the token.
//
// Bound: HBM, the row read and written once, behind the counting: 64 rows of 151936 fp32 logits with up to 5000 tokens of
// history, 40 biases and a mask take 16.5 us, 80 MB at 4.8 TB/s, and with 100 tokens of history 13.7.  128 rows take
// 40 us, 161 MB at 4.0 TB/s.  The logits are read as data that is not needed again, so that L2 keeps what is written: with
// plain loads 64 rows that L2 does not hold took 19.6 us, 16.1 where it does either way.
#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "host_util.h"

namespace mllm_b200 {
namespace {

constexpr int kThreads = 512;
constexpr int kMinStretch = 1024;
constexpr int kMaxStretch = 26 * 1024;   // 104 KB of counters: two CTAs fit on an SM
constexpr int kMinCtas = 2;
constexpr int kHeld = 2;                 // history tokens a thread loads together
constexpr int kMaxBias = 1024;
constexpr unsigned kSeen = 0x80000000u;  // counter bits: the token is in the prompt part of the history ...
constexpr unsigned kBiased = 0x40000000u; // ... it has a bias; the rest counts it in the generated part

struct RuleArgs {
    const void* logits;
    void* out;
    int64_t l_stride, o_stride;
    int vocab, stretch;
    const int64_t* hist;
    int64_t hist_stride;
    int hist_cols;
    const int32_t* hist_lens;
    const int32_t* out_start;
    const float* rep;
    const float* pres;
    const float* freq;
    const int64_t* bias_ids;
    const float* bias_vals;
    int64_t bias_stride;
    int bias_cols;
    const int32_t* bias_lens;
    const uint32_t* allowed;      // bit v % 32 of word v / 32
    int64_t allowed_stride;
};

__device__ __forceinline__ float load_f32(const float* p) { return *p; }
__device__ __forceinline__ float load_f32(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store_f32(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_f32(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ int checked_len(const int32_t* lens, int row, int cols) {
    const int n = lens[row];
    if (n < 0 || n > cols) {
        record_error(kErrBadLength);
        return n < 0 ? 0 : cols;
    }
    return n;
}

template <typename T, bool kWide>
__global__ void __launch_bounds__(kThreads, kMinCtas) logit_rules_kernel(RuleArgs a) {
    extern __shared__ __align__(16) unsigned s_count[];   // [stretch], only with a history or biases
    __shared__ int s_id[kMaxBias];
    __shared__ float s_val[kMaxBias];
    const int row = blockIdx.y;
    const int v0 = blockIdx.x * a.stretch;
    const int n = min(a.stretch, a.vocab - v0);
    const int t = threadIdx.x;
    const bool counted = a.hist != nullptr || a.bias_ids != nullptr;
    if (counted)
        for (int i = t; i < (n + 3) / 4; i += kThreads) reinterpret_cast<uint4*>(s_count)[i] = make_uint4(0u, 0u, 0u, 0u);
    pdl_wait();
    pdl_trigger();
    const T* x = static_cast<const T*>(a.logits) + (int64_t)row * a.l_stride + v0;
    T* y = static_cast<T*>(a.out) + (int64_t)row * a.o_stride + v0;
    const uint32_t* allow = a.allowed ? a.allowed + (int64_t)row * a.allowed_stride + v0 / 32 : nullptr;

    // The first loads of everything go out together: the history's do not wait for its length (its columns exist).
    const int64_t* hist = a.hist ? a.hist + (int64_t)row * a.hist_stride : nullptr;
    const int cols = hist ? a.hist_cols : 0;
    int64_t tok[kHeld];
#pragma unroll
    for (int u = 0; u < kHeld; ++u) tok[u] = t + u * kThreads < cols ? hist[t + u * kThreads] : -1;
    const int64_t bias_row = (int64_t)row * a.bias_stride;
    const int bias_cols = a.bias_ids ? a.bias_cols : 0;
    int64_t bias_id = t < bias_cols ? a.bias_ids[bias_row + t] : -1;
    float bias_val = t < bias_cols ? a.bias_vals[bias_row + t] : 0.f;
    constexpr int E = 16 / (int)sizeof(T);           // 4 or 8 tokens per 16 bytes
    constexpr int U = 2;                             // 16-byte loads in flight, while as many are worked on
    const int nv = kWide ? n / E : 0;
    uint4 w[U], next_w[U];
    auto load = [&](int i0) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + u * kThreads < nv) next_w[u] = __ldcs(reinterpret_cast<const uint4*>(x) + i0 + u * kThreads);
    };
    load(t);
    const int n_hist = hist ? checked_len(a.hist_lens, row, a.hist_cols) : 0;
    const int n_bias = a.bias_ids ? checked_len(a.bias_lens, row, a.bias_cols) : 0;
    const int made = hist && a.out_start ? a.out_start[row] : 0;
    const float r = a.rep ? a.rep[row] : 1.f, p = a.pres ? a.pres[row] : 0.f, f = a.freq ? a.freq[row] : 0.f;

    if (counted) {
        __syncthreads();     // the counters are clear
        auto place = [&](int64_t id) -> int {   // of a token in the stretch, or -1
            const int64_t at = id - v0;
            return at >= 0 && at < n ? (int)at : -1;
        };
        auto count = [&](int i, int64_t id) {
            const int at = i < n_hist ? place(id) : -1;
            if (at < 0) return;
            if (i >= made) atomicAdd(&s_count[at], 1u);
            else atomicOr(&s_count[at], kSeen);
        };
        for (int i0 = t; i0 < n_hist; i0 += kHeld * kThreads) {
            int64_t next[kHeld];   // on their way while the present ones are counted
#pragma unroll
            for (int u = 0; u < kHeld; ++u) {
                const int i = i0 + (kHeld + u) * kThreads;
                next[u] = i < n_hist ? hist[i] : -1;
            }
#pragma unroll
            for (int u = 0; u < kHeld; ++u) count(i0 + u * kThreads, tok[u]);
#pragma unroll
            for (int u = 0; u < kHeld; ++u) tok[u] = next[u];
        }
        for (int i = t; i < n_bias; i += kThreads) {
            if (i != t) {
                bias_id = a.bias_ids[bias_row + i];
                bias_val = a.bias_vals[bias_row + i];
            }
            const int at = place(bias_id);
            s_id[i] = at;
            s_val[i] = bias_val;
            if (at >= 0) atomicOr(&s_count[at], kBiased);
        }
        __syncthreads();
    }

    // A touched token's logit; c is its counter.
    auto ruled = [&](float v, unsigned c, int i) {
        const unsigned made_c = c & ~(kSeen | kBiased);
        if ((c & kSeen) || made_c) v = v < 0.f ? v * r : __fdiv_rn(v, r);
        if (made_c) v = v - (float)made_c * f - p;
        if (c & kBiased) {
            float b = 0.f;
            for (int j = 0; j < n_bias; ++j)
                if (s_id[j] == i) b += s_val[j];
            v += b;
        }
        return v;
    };
    if constexpr (kWide) {
        constexpr uint32_t kAll = (1u << E) - 1u;
        for (int i0 = t; i0 < nv; i0 += U * kThreads) {
#pragma unroll
            for (int u = 0; u < U; ++u) w[u] = next_w[u];
            load(i0 + U * kThreads);
            uint32_t m[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + u * kThreads;
                m[u] = i < nv && allow ? (allow[i * E >> 5] >> (i * E & 31)) & kAll : kAll;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + u * kThreads;
                if (i >= nv) break;
                uint32_t* c = reinterpret_cast<uint32_t*>(&w[u]);
                if (counted) {
                    uint32_t hit = 0u;
#pragma unroll
                    for (int e = 0; e < E; e += 4) {
                        const uint4 k = *reinterpret_cast<const uint4*>(s_count + i * E + e);
                        hit |= ((k.x ? 1u : 0u) | (k.y ? 2u : 0u) | (k.z ? 4u : 0u) | (k.w ? 8u : 0u)) << e;
                    }
                    hit &= m[u];
                    while (hit != 0u) {   // a lane's own few: a branch per token would run for all of a warp's
                        const int e = __ffs(hit) - 1;
                        hit &= hit - 1u;
                        constexpr int P = E / 4;   // tokens in 32 bits
                        const int q = e / P, sh = P == 2 ? 16 * (e & 1) : 0;
                        const uint32_t bits = q < 2 ? (q == 0 ? c[0] : c[1]) : (q == 2 ? c[2] : c[3]);
                        T v;
                        if constexpr (P == 1) v = __uint_as_float(bits);
                        else v = __ushort_as_bfloat16((unsigned short)(bits >> sh));
                        store_f32(&v, ruled(load_f32(&v), s_count[i * E + e], i * E + e));
                        uint32_t now;
                        if constexpr (P == 1) now = __float_as_uint(v);
                        else now = (bits & ~(0xFFFFu << sh)) | ((uint32_t)__bfloat16_as_ushort(v) << sh);
#pragma unroll
                        for (int d = 0; d < 4; ++d) c[d] = d == q ? now : c[d];
                    }
                }
                if (m[u] != kAll) {
                    if constexpr (sizeof(T) == 4) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) c[e] = (m[u] >> e) & 1u ? c[e] : 0xFF800000u;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t lo = (m[u] >> (2 * e)) & 1u ? c[e] & 0xFFFFu : 0xFF80u;
                            const uint32_t hi = (m[u] >> (2 * e + 1)) & 1u ? c[e] & 0xFFFF0000u : 0xFF800000u;
                            c[e] = lo | hi;
                        }
                    }
                }
                reinterpret_cast<uint4*>(y)[i] = w[u];
            }
        }
    }
    for (int i = nv * E + t; i < n; i += kThreads) {   // the last few, or all where 16-byte loads are not possible
        const bool ok = allow == nullptr || ((allow[i >> 5] >> (i & 31)) & 1u);
        const unsigned c = counted ? s_count[i] : 0u;
        const T v = x[i];
        if (!ok) store_f32(y + i, -INFINITY);
        else if (c == 0u) y[i] = v;
        else store_f32(y + i, ruled(load_f32(&v), c, i));
    }
}

// Whether any row of `len` bytes of one tensor meets one of the other's (rows sa and sb bytes apart): both in ascending
// order.
bool rows_meet(uintptr_t a, uintptr_t sa, uintptr_t b, uintptr_t sb, int rows, uintptr_t len) {
    for (int i = 0, j = 0; i < rows && j < rows;) {
        const uintptr_t pa = a + i * sa, pb = b + j * sb;
        if (pa + len <= pb) ++i;
        else if (pb + len <= pa) ++j;
        else return true;
    }
    return false;
}

}  // namespace

MLLM_DEFINE_STATUS_READER(logit_rules)

}  // namespace mllm_b200

using namespace mllm_b200;

extern "C" int mllm_logit_rules(const void* logits, int logits_bf16, int64_t row_stride, int batch, int vocab,
                                const int64_t* history, int64_t history_stride, int history_cols,
                                const int32_t* history_lens, const int32_t* output_start, const float* repetition,
                                const float* presence, const float* frequency, const int64_t* bias_ids,
                                const float* bias_values, int64_t bias_stride, int bias_cols, const int32_t* bias_lens,
                                const uint32_t* allowed, int64_t allowed_stride, void* out, int64_t out_stride,
                                mllm_stream_t stream) {
    MLLM_NVTX_RANGE("mllm_logit_rules");
    if (vocab <= 0) return fail(MLLM_ERR_INVALID_ARGUMENT, "logit_rules: empty logits");
    if (batch < 0 || row_stride < vocab || out_stride < vocab)
        return fail(MLLM_ERR_INVALID_ARGUMENT, "logit_rules: bad sizes");
    if (batch > 65535) return fail(MLLM_ERR_UNSUPPORTED, "logit_rules: more than 65535 rows");
    if ((history == nullptr) != (history_lens == nullptr))
        return fail(MLLM_ERR_INVALID_ARGUMENT, "logit_rules: give both history and history_lens or neither");
    if (history && (history_cols < 0 || history_stride < history_cols))
        return fail(MLLM_ERR_INVALID_ARGUMENT, "logit_rules: bad history_cols or history_stride");
    if (!history && (repetition || presence || frequency || output_start))
        return fail(MLLM_ERR_INVALID_ARGUMENT, "logit_rules: penalties need a history");
    if ((bias_ids == nullptr) != (bias_values == nullptr) || (bias_ids == nullptr) != (bias_lens == nullptr))
        return fail(MLLM_ERR_INVALID_ARGUMENT, "logit_rules: give all of bias_ids, bias_values and bias_lens or none");
    if (bias_ids && (bias_cols < 0 || bias_stride < bias_cols))
        return fail(MLLM_ERR_INVALID_ARGUMENT, "logit_rules: bad bias_cols or bias_stride");
    if (history && history_cols > (int)~(kSeen | kBiased))
        return fail(MLLM_ERR_UNSUPPORTED, "logit_rules: more than 2^30 - 1 columns of history");
    if (bias_ids && bias_cols > kMaxBias)
        return fail(MLLM_ERR_UNSUPPORTED, "logit_rules: more than 1024 biases a row");
    if (allowed && allowed_stride < (vocab + 31) / 32)
        return fail(MLLM_ERR_INVALID_ARGUMENT, "logit_rules: allowed_stride below ceil(vocab / 32)");
    if (batch == 0) return ok();
    if (!logits || !out) return fail(MLLM_ERR_INVALID_ARGUMENT, "logit_rules: null pointer");
    const int es = logits_bf16 ? 2 : 4;
    if (!aligned(logits, es) || !aligned(out, es) || !aligned(allowed, 4) ||
        !aligned(history, 8) || !aligned(history_lens, 4) || !aligned(output_start, 4) || !aligned(repetition, 4) ||
        !aligned(presence, 4) || !aligned(frequency, 4) || !aligned(bias_ids, 8) || !aligned(bias_values, 4) ||
        !aligned(bias_lens, 4))
        return fail(MLLM_ERR_INVALID_ARGUMENT, "logit_rules: misaligned pointer");
    const bool in_place = logits == out && (batch == 1 || row_stride == out_stride);
    if (!in_place && rows_meet((uintptr_t)logits, (uintptr_t)row_stride * es, (uintptr_t)out, (uintptr_t)out_stride * es, batch,
                               (uintptr_t)vocab * es))
        return fail(MLLM_ERR_INVALID_ARGUMENT, "logit_rules: out overlaps the logits without being the same rows");
    int num_sms = 0;
    if (int st = require_sm100(&num_sms)) return st;
    RuleArgs a = {};
    a.logits = logits;
    a.out = out;
    a.l_stride = row_stride;
    a.o_stride = out_stride;
    a.vocab = vocab;
    a.hist = history_cols > 0 ? history : nullptr;
    a.hist_stride = history_stride;
    a.hist_cols = history_cols;
    a.hist_lens = history_lens;
    a.out_start = output_start;
    a.rep = repetition;
    a.pres = presence;
    a.freq = frequency;
    a.bias_ids = bias_cols > 0 ? bias_ids : nullptr;
    a.bias_vals = bias_values;
    a.bias_stride = bias_stride;
    a.bias_cols = bias_cols;
    a.bias_lens = bias_lens;
    a.allowed = allowed;
    a.allowed_stride = allowed_stride;
    // A row is cut so that all CTAs of the batch fill whole waves of the resident ones, as few waves as the limit on a
    // stretch allows: every CTA reads its row's whole history, so few long stretches beat many short ones (4 fp32 rows
    // take 5.3 us in one wave and 7.4 in two, 32 rows 9.7 and 12.1).
    const int64_t slots = (int64_t)kMinCtas * num_sms;
    const int64_t least = ((int64_t)vocab + kMaxStretch - 1) / kMaxStretch;
    const int64_t waves = (least * batch + slots - 1) / slots;
    const int64_t per_row = slots * waves / batch;
    const int stretch = std::max(kMinStretch, (int)(((int64_t)vocab + per_row - 1) / per_row + 255) / 256 * 256);
    a.stretch = stretch;
    const dim3 grid((vocab + stretch - 1) / stretch, batch);
    const int smem = a.hist || a.bias_ids ? stretch * 4 : 0;
    const bool wide = aligned(logits, 16) && aligned(out, 16) && row_stride * es % 16 == 0 && out_stride * es % 16 == 0;
    auto launch = [&](void (*kern)(RuleArgs)) -> int {
        if (int st = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxStretch * 4),
                                "logit_rules smem attribute"))
            return st;
        return check_cuda(launch_pdl(kern, grid, dim3(kThreads), smem, (cudaStream_t)stream, a), "logit_rules_kernel launch");
    };
    int st;
    if (logits_bf16)
        st = wide ? launch(logit_rules_kernel<__nv_bfloat16, true>) : launch(logit_rules_kernel<__nv_bfloat16, false>);
    else
        st = wide ? launch(logit_rules_kernel<float, true>) : launch(logit_rules_kernel<float, false>);
    if (st) return st;
    return ok();
}
