// Arguments of the batched one-token attention over paged caches (b200_flash_attn_paged_batch), and its launch for sequences that
// share prefixes.
#pragma once

#include "paged_line.cuh"
#include "shared_prefix.cuh"

namespace b200 {

struct PbArgs {
    const void *q = nullptr;
    void *out = nullptr;
    int64_t q_seq = 0, q_head = 0, o_seq = 0, o_head = 0;  // elements
    const char *k = nullptr, *v = nullptr;
    int64_t block_stride = 0, tok_stride = 0, head_stride = 0;  // bytes
    int64_t n_blocks = 0;
    const int32_t *table = nullptr, *lens = nullptr;
    int64_t table_stride = 0;
    int64_t max_keys = 0;  // positions a table row covers (fits 31 bits)
    uint32_t bt = 1;
    int n_seqs = 0, G = 0, VH = 0, HG = 0;  // query heads a KV head; (KV head, head group) pairs; groups a KV head
    float sl2 = 0.f;                        // scale * log2 e
    float *ws = nullptr;
    float *whole = nullptr;  // with prefixes: a record a pair, of those that one CTA took whole
    int32_t *status = nullptr;
};

// Whether sequences with so many keys, prefixes included, take one launch of clusters.
bool paged_batch_one_launch(int64_t n_seqs, int64_t max_keys, int64_t G, int64_t Hkv, int32_t dtype);
// The sequences' own keys, joined with what the prefixes' kernel left (launched before on the stream; it lets this grid start early).
// `a.ws` and `a.whole` as the sizes of paged_batch_prefix_bytes.
size_t paged_batch_prefix_bytes(int64_t n_seqs, int64_t max_keys, int64_t D, int64_t G, int64_t Hkv, int32_t dtype);
cudaError_t paged_batch_prefix_launch(PbArgs a, const PrefixArgs &px, int64_t Hkv, int64_t D, int32_t dtype, void *workspace, cudaStream_t st);

}  // namespace b200
