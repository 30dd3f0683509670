// The 8-bit paged cache: e4m3 elements and one e8m0 scale a row (one token, one KV head).
#pragma once

#include <cuda_fp8.h>

#include "batch.cuh"

namespace b200 {

// The scale 2^e as a number, from its byte e + 127; 255: NaN.
B200_DEVICE float e8m0_value(uint32_t b) {
    return __uint_as_float(b == 255u ? 0x7FC00000u : (b ? b << 23 : 0x00400000u));
}
// e + 127 for the least whole e >= -127 with top <= 448 2^e = 1.75 2^(e + 8), from top's bits: an added
// 2^21 - 1 carries into the exponent where the fraction is above .75.
B200_DEVICE uint32_t e8m0_of(uint32_t top_bits) {
    const int b = static_cast<int>((top_bits + 0x1FFFFFu) >> 23) - 8;
    return static_cast<uint32_t>(max(b, 0));
}
// 2^-e
B200_DEVICE float e8m0_inverse(uint32_t b) { return __uint_as_float((254u - b) << 23); }  // b <= 247

// The four e4m3 numbers of a word as F16 (exact): bytes 0 and 1, and 2 and 3.
B200_DEVICE void e4m3x4_to_f16(uint32_t w, uint32_t &lo, uint32_t &hi) {
    asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
}

inline int check_pool_q8(const b200_kv_pool_q8 *p) {
    if (!p || !p->k || !p->v || !p->k_scale || !p->v_scale || p->n_blocks <= 0 || p->block_tokens <= 0 ||
        p->n_head_kv <= 0 || p->head_dim <= 0)
        return B200_ERR_INVALID_ARGUMENT;
    if (p->n_blocks > INT32_MAX || p->block_tokens > INT32_MAX || p->n_head_kv > (1 << 24) / p->head_dim ||
        (p->head_dim != 64 && p->head_dim != 128) || !rows_aligned16(p->k, p->block_stride, p->tok_stride, 1) ||
        !rows_aligned16(p->v, p->head_stride, 0, 1))
        return B200_ERR_NOT_SUPPORTED;
    return B200_OK;
}

}  // namespace b200
