// Arguments of the packed causal attention kernels (b200_flash_attn_packed).
#pragma once

#include "batch.cuh"

namespace b200 {

struct PackedArgs {
    const void *q = nullptr, *k = nullptr, *v = nullptr;
    void *out = nullptr;
    int64_t q_tok = 0, q_head = 0, k_tok = 0, k_head = 0, v_tok = 0, v_head = 0, o_tok = 0, o_head = 0;  // elements
    const int32_t *cu_q = nullptr, *cu_k = nullptr;
    int64_t total_q = 0, total_k = 0;
    int n_seqs = 0, Hq = 0, Hkv = 0, G = 0, D = 0;
    float sl2 = 0.f;  // scale * log2 e
    int32_t dtype = 0;
    void *ws = nullptr;
    int32_t *status = nullptr;
};

// The tensor-core kernel; cudaErrorNotSupported (nothing launched) where it does not apply.
size_t packed_tc_workspace(int64_t n_seqs, int64_t total_q, int64_t total_k, int64_t D, int64_t Hq, int64_t Hkv,
                           int32_t dtype);
cudaError_t packed_tc_launch(const PackedArgs &a, cudaStream_t stream);

}  // namespace b200
