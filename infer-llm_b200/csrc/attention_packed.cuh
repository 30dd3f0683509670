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

// Where a sequence's offsets are out of range: reports it, and clears the query rows that no other
// sequence covers, so that an output made for the call holds nothing else. Run by one warp of the
// grid's last CTA, which found its own tile (or none) in the same offsets.
B200_DEVICE void clear_uncovered(const PackedArgs &a) {
    const int lane = threadIdx.x & 31;
    int64_t q0, k0;
    int nq, nk;
    const auto runs = [&](int s) {  // (an empty sequence's keys do not matter)
        const bool ok_q = packed_range(a.cu_q, s, a.total_q, q0, nq), ok_k = packed_range(a.cu_k, s, a.total_k, k0, nk);
        return ok_q && (ok_k || nq == 0);
    };
    bool bad = false;
    for (int s = lane; s < a.n_seqs; s += 32) bad |= !runs(s);
    if (!__any_sync(0xffffffffu, bad)) return;
    if (lane == 0) set_status(a.status, B200_DEV_BAD_POSITION);
    const int64_t e = a.dtype == B200_DTYPE_F32 ? 4 : 2;
    const int chunks = a.D * static_cast<int>(e) / 16;  // of a head
    for (int t = 0; t < a.total_q;) {  // from one covered run of rows to the next
        int end = 0, next = static_cast<int>(a.total_q);
        for (int s = lane; s < a.n_seqs; s += 32) {
            if (!runs(s) || nq == 0) continue;
            if (t < q0) next = min(next, static_cast<int>(q0));
            else if (t < q0 + nq) end = max(end, static_cast<int>(q0 + nq));
        }
        end = __reduce_max_sync(0xffffffffu, end);
        next = __reduce_min_sync(0xffffffffu, next);
        for (; t < next && end == 0; ++t) {
            char *row = static_cast<char *>(a.out) + t * a.o_tok * e;
            for (int c = lane; c < a.Hq * chunks; c += 32)
                *reinterpret_cast<uint4 *>(row + (c / chunks) * a.o_head * e + c % chunks * 16) = make_uint4(0, 0, 0, 0);
        }
        t = max(t, end);
    }
}

// The tensor-core kernel; cudaErrorNotSupported (nothing launched) where it does not apply.
size_t packed_tc_workspace(int64_t n_seqs, int64_t total_q, int64_t total_k, int64_t D, int64_t Hq, int64_t Hkv,
                           int32_t dtype);
cudaError_t packed_tc_launch(const PackedArgs &a, cudaStream_t stream);

}  // namespace b200
