// Rules on logits before a token is picked: repetition, presence and frequency penalties, biases and a mask of
// allowed tokens, each row with its own.
//
//   seen  = the token occurs in the row's history;  c = how often among its generated part
//   x     = logit;  if seen: x / r (x >= 0) or x * r (x < 0);  x -= c f;  if c > 0: x -= p;  x += sum of its biases
//   out   = allowed ? x : -inf                           in fp32, rounded once to the logits' type
//
// One CTA takes a stretch of one row's vocabulary.  Counting: the CTA reads the row's whole history (8 bytes a
// token, small against the row and in L2 after the first CTA) and counts the tokens of its stretch in shared
// memory, so nothing has to be cleared or kept in global memory and any number of calls may run at once.  The
// stretch is streamed with 16-byte loads, copying bits or writing -inf; no counter is looked at there, because
// only the few tokens with a bias or a count change.  Those are then redone, each by the thread that owns its
// first list entry (biases) or that takes its count (history), so every token is written once more at most and
// the result does not depend on the order of the threads.
//
// Bound: HBM, the row read and written once.  The stretch is chosen so that the CTAs fill the GPU a few times
// over at large batches and once at a batch of one, and its counters leave room for two CTAs per SM.
#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "host_util.h"

namespace mllm_b200 {
namespace {

constexpr int kThreads = 512;
constexpr int kMinStretch = 1024;
constexpr int kMaxStretch = 24 * 1024;   // 96 KB of counters
constexpr int kMaxBias = 1024;
constexpr unsigned kSeen = 0x80000000u;  // counter bit of a prompt token; the rest counts generated ones

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
__global__ void __launch_bounds__(kThreads) logit_rules_kernel(RuleArgs a) {
    extern __shared__ unsigned s_count[];      // [stretch], only with a history
    __shared__ int s_id[kMaxBias];
    __shared__ float s_val[kMaxBias];
    const int row = blockIdx.y;
    const int v0 = blockIdx.x * a.stretch;
    const int n = min(a.stretch, a.vocab - v0);
    const int t = threadIdx.x;
    if (a.hist != nullptr)
        for (int i = t; i < n; i += kThreads) s_count[i] = 0u;
    pdl_wait();
    pdl_trigger();
    const T* x = static_cast<const T*>(a.logits) + (int64_t)row * a.l_stride + v0;
    T* y = static_cast<T*>(a.out) + (int64_t)row * a.o_stride + v0;
    const uint32_t* allow = a.allowed ? a.allowed + (int64_t)row * a.allowed_stride + v0 / 32 : nullptr;
    auto is_allowed = [&](int i) { return allow == nullptr || ((allow[i >> 5] >> (i & 31)) & 1u); };

    const int64_t* hist = a.hist ? a.hist + (int64_t)row * a.hist_stride : nullptr;
    const int n_hist = hist ? checked_len(a.hist_lens, row, a.hist_cols) : 0;
    const int n_bias = a.bias_ids ? checked_len(a.bias_lens, row, a.bias_cols) : 0;
    __syncthreads();
    if (n_hist > 0) {
        const int made = a.out_start ? a.out_start[row] : 0;
        for (int i = t; i < n_hist; i += kThreads) {
            const int64_t at = hist[i] - v0;
            if (at < 0 || at >= n) continue;
            if (i >= made) atomicAdd(&s_count[at], 1u);
            else atomicOr(&s_count[at], kSeen);
        }
    }
    for (int i = t; i < n_bias; i += kThreads) {
        const int64_t at = a.bias_ids[(int64_t)row * a.bias_stride + i] - v0;
        s_id[i] = at >= 0 && at < n ? (int)at : -1;
        s_val[i] = a.bias_vals[(int64_t)row * a.bias_stride + i];
    }

    // ---- the stretch, bits copied or -inf ----
    if constexpr (kWide) {
        constexpr int E = 16 / (int)sizeof(T);       // 4 or 8 tokens per 16 bytes
        constexpr uint32_t kAll = (1u << E) - 1u;
        constexpr int U = 4;                         // loads in flight
        const int nv = n / E;
        for (int i0 = t; i0 < nv; i0 += U * kThreads) {
            uint4 w[U];
            uint32_t m[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + u * kThreads;
                if (i < nv) {
                    w[u] = __ldcs(reinterpret_cast<const uint4*>(x) + i);
                    m[u] = allow ? (allow[i * E >> 5] >> (i * E & 31)) & kAll : kAll;
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + u * kThreads;
                if (i >= nv) break;
                if (m[u] != kAll) {
                    uint32_t* c = reinterpret_cast<uint32_t*>(&w[u]);
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
        for (int i = nv * E + t; i < n; i += kThreads) {
            const T v = x[i];
            if (is_allowed(i)) y[i] = v;
            else store_f32(y + i, -INFINITY);
        }
    } else {
        for (int i = t; i < n; i += kThreads) {
            const T v = x[i];
            if (is_allowed(i)) y[i] = v;
            else store_f32(y + i, -INFINITY);
        }
    }
    if (n_hist == 0 && n_bias == 0) return;
    __syncthreads();     // counts and biases complete, and the stretch written (y is read back below)

    const float r = a.rep ? a.rep[row] : 1.f, p = a.pres ? a.pres[row] : 0.f, f = a.freq ? a.freq[row] : 0.f;
    auto redo = [&](int i, unsigned count, float bias) {
        if (!is_allowed(i)) return;
        float v = load_f32(y + i);      // the logit itself: the copy above did not change it
        if (count != 0u) {
            v = v < 0.f ? v * r : __fdiv_rn(v, r);
            const unsigned c = count & ~kSeen;
            if (c != 0u) v = v - (float)c * f - p;
        }
        store_f32(y + i, v + bias);
    };
    for (int i = t; i < n_bias; i += kThreads) {
        const int id = s_id[i];
        if (id < 0) continue;
        bool first = true;
        for (int j = 0; j < i && first; ++j) first = s_id[j] != id;
        if (!first) continue;
        float b = 0.f;                  // a token listed more than once gets the sum, in list order
        for (int j = i; j < n_bias; ++j)
            if (s_id[j] == id) b += s_val[j];
        unsigned count = 0u;
        if (hist) {
            count = s_count[id];
            s_count[id] = 0u;
        }
        redo(id, count, b);
    }
    if (n_hist == 0) return;
    __syncthreads();
    for (int i = t; i < n_hist; i += kThreads) {
        const int64_t at = hist[i] - v0;
        if (at < 0 || at >= n) continue;
        const unsigned count = atomicExch(&s_count[at], 0u);
        if (count != 0u) redo((int)at, count, 0.f);
    }
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
    if (bias_ids && bias_cols > kMaxBias)
        return fail(MLLM_ERR_UNSUPPORTED, "logit_rules: more than 1024 biases a row");
    if (allowed && allowed_stride < (vocab + 31) / 32)
        return fail(MLLM_ERR_INVALID_ARGUMENT, "logit_rules: allowed_stride below ceil(vocab / 32)");
    if (batch == 0) return ok();
    if (!logits || !out) return fail(MLLM_ERR_INVALID_ARGUMENT, "logit_rules: null pointer");
    const int es = logits_bf16 ? 2 : 4;
    if (!aligned(logits, es) || !aligned(out, es) || !aligned(allowed, 4))
        return fail(MLLM_ERR_INVALID_ARGUMENT, "logit_rules: misaligned pointer");
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
    // stretches per row: about three CTAs per SM over the batch, within the limits on a stretch
    const int want = std::max(1, 3 * num_sms / batch);
    int stretch = (vocab + want - 1) / want;
    stretch = std::min(kMaxStretch, std::max(kMinStretch, (stretch + 255) / 256 * 256));
    a.stretch = stretch;
    const dim3 grid((vocab + stretch - 1) / stretch, batch);
    const int smem = a.hist ? stretch * 4 : 0;
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
