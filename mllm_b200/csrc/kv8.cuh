// The 8-bit KV cache (mllm_paged_kv8): a K or V row of one token and kv head is D e4m3 values and one
// exponent byte e + 127, standing for value * 2^e.
//
// Why a power of two per row.  e4m3 is itself a floating-point format: scaling a row by anything but a
// power of two changes which values are representable, not how finely, so a full scale factor buys no
// precision (it would only use the last 1/8 of the top binade better).  A power of two costs one byte
// per row instead of four, makes value * 2^e exact in bf16 (4 significant bits), and lets attention fold
// the scale into the softmax exponent.
//
// e is the smallest integer in [kExpMin, kExpMax] with max|row| <= 448 * 2^e, the maximum taken over the
// row's finite elements.  Below 2^kExpMin * 2^-9 elements become zero; the bound keeps 2^e and 2^-e normal
// fp32 numbers and value * 2^e a normal bf16 number; for the latter, elements above kRowMax are stored as that.  A
// non-finite element is stored as NaN (the format has no infinity, and saturating one would hide it).
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <string>

#include "common.cuh"
#include "host_util.h"
#include "kv_layout.cuh"

namespace mllm_b200 {

constexpr int kExpMin = -100;
constexpr int kExpMax = 120;
constexpr float kRowMax = 240.f * 0x1p120f;   // 256 * 2^120 is beyond bf16's largest number

// 2^e for -126 <= e <= 127.
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// A cached row's scale from its exponent byte (byte 0, a row never written, gives 0).
__device__ __forceinline__ float exp_byte_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// The exponent of a row whose largest finite magnitude is amax: amax = m 2^x with 1 <= m < 2, and
// m 2^x <= 1.75 * 2^8 * 2^e.
__device__ __forceinline__ int row_exponent(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int x = (int)(u >> 23) - 127;                       // subnormals land far below kExpMin
    const int e = x - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return min(max(e, kExpMin), kExpMax);
}

// Four fp32 values (already multiplied by 2^-e) as e4m3 bytes, nearest even, lowest index lowest byte.
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return (uint32_t)lo | ((uint32_t)hi << 16);
}

// Two e4m3 bytes (the low or high half of a word) as two halves, exactly.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint16_t v) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
    return r;
}

// Device view of a paged 8-bit cache: pools in bytes, block table as in KvLayout.
struct Kv8View {
    uint8_t* k_pool;
    uint8_t* v_pool;
    uint8_t* k_exp;
    uint8_t* v_exp;
    int64_t p_sb, p_sh, p_st;   // pool strides per block, head, row
    int64_t e_sb, e_sh;         // exponent strides per block, head (rows are adjacent)
};

// Host side: checks a descriptor for a call that addresses `rows` rows per sequence of `head_dim`
// columns and fills the device layouts.
inline int paged_layout8(const mllm_paged_kv8* kv, int64_t rows, int head_dim, const char* who, KvLayout* lay,
                         Kv8View* view) {
    const std::string w(who);
    if (kv == nullptr) return fail(MLLM_ERR_INVALID_ARGUMENT, w + ": paged cache descriptor is NULL");
    if (!kv->k_pool || !kv->v_pool || !kv->k_exp || !kv->v_exp || !kv->block_table)
        return fail(MLLM_ERR_INVALID_ARGUMENT, w + ": paged cache pools, exponents and block table must be given");
    if (kv->block_size <= 0 || kv->block_size % 128 != 0)
        return fail(MLLM_ERR_INVALID_ARGUMENT, w + ": block_size must be a positive multiple of 128");
    if (kv->num_blocks <= 0 || kv->max_blocks_per_seq <= 0 || kv->table_stride < kv->max_blocks_per_seq)
        return fail(MLLM_ERR_INVALID_ARGUMENT, w + ": bad num_blocks, max_blocks_per_seq or table_stride");
    if (kv->row_stride < head_dim || kv->head_stride < head_dim || kv->block_stride < head_dim ||
        kv->row_stride % 16 || kv->head_stride % 16 || kv->block_stride % 16)
        return fail(MLLM_ERR_INVALID_ARGUMENT, w + ": pool strides must be multiples of 16 bytes, at least head_dim");
    if (kv->exp_head_stride < 16 || kv->exp_block_stride < 16 || kv->exp_head_stride % 16 || kv->exp_block_stride % 16)
        return fail(MLLM_ERR_INVALID_ARGUMENT, w + ": exponent strides must be positive multiples of 16 bytes");
    if (!aligned(kv->k_pool, 16) || !aligned(kv->v_pool, 16) || !aligned(kv->k_exp, 16) || !aligned(kv->v_exp, 16))
        return fail(MLLM_ERR_INVALID_ARGUMENT, w + ": pools and exponents must be 16-byte aligned");
    if (rows > (int64_t)kv->max_blocks_per_seq * kv->block_size)
        return fail(MLLM_ERR_INVALID_ARGUMENT, w + ": rows exceed max_blocks_per_seq * block_size");
    lay->table = kv->block_table;
    lay->table_stride = kv->table_stride;
    lay->block_size = kv->block_size;
    lay->num_blocks = kv->num_blocks;
    lay->max_blocks = kv->max_blocks_per_seq;
    view->k_pool = static_cast<uint8_t*>(kv->k_pool);
    view->v_pool = static_cast<uint8_t*>(kv->v_pool);
    view->k_exp = static_cast<uint8_t*>(kv->k_exp);
    view->v_exp = static_cast<uint8_t*>(kv->v_exp);
    view->p_sb = kv->block_stride;
    view->p_sh = kv->head_stride;
    view->p_st = kv->row_stride;
    view->e_sb = kv->exp_block_stride;
    view->e_sh = kv->exp_head_stride;
    return MLLM_OK;
}

}  // namespace mllm_b200
