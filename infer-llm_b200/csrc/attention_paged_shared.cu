// b200_flash_attn_paged_shared: one query token for each of many sequences that share prefixes, against a paged K/V cache.
//
// out_b = softmax over the keys of the prefix of b's group and b's own keys, of the one pool.
#include "attention_rows.cuh"
#include "paged_line.cuh"

namespace b200 {
namespace {

struct SharedArgs {
    const void *q = nullptr;
    void *out = nullptr;
    int64_t q_seq = 0, q_head = 0, o_seq = 0, o_head = 0;  // elements
    const char *k = nullptr, *v = nullptr;
    int64_t block_stride = 0, tok_stride = 0, head_stride = 0;  // elements
    int64_t n_blocks = 0;
    const int32_t *table = nullptr, *lens = nullptr, *prefix_table = nullptr, *prefix_lens = nullptr, *cu = nullptr;
    int64_t table_stride = 0, prefix_stride = 0;
    int64_t max_keys = 0, max_prefix = 0;  // positions a table row covers (fits 31 bits)
    uint32_t bt = 1;
    int n_seqs = 0, n_groups = 0, G = 0, Hkv = 0;
    float sl2 = 0.f;  // scale * log2 e
    int32_t *status = nullptr;
};

template <typename T, int D>
__global__ void __launch_bounds__(32 * kArWarps) shared_rows_kernel(const __grid_constant__ SharedArgs a) {
    constexpr int E = D / 32;
    const int b = static_cast<int>(blockIdx.x / static_cast<unsigned>(a.Hkv)), h = blockIdx.x % static_cast<unsigned>(a.Hkv);
    const int64_t len = __ldg(a.lens + b), keys = min64(max64(len, 0), a.max_keys);
    const int group = a.n_groups ? warp_find_row(a.cu, a.n_groups, b) : -1;
    const bool in = group >= 0 && __ldg(a.cu + group) >= 0 && __ldg(a.cu + group + 1) <= a.n_seqs;
    const int64_t plen = in ? __ldg(a.prefix_lens + group) : 0, prefix = min64(max64(plen, 0), a.max_prefix);
    if ((len != keys || plen != prefix) && threadIdx.x == 0 && h == 0) set_status(a.status, B200_DEV_BAD_POSITION);
    if (blockIdx.x == 0)
        for (int g = threadIdx.x; g < a.n_groups; g += blockDim.x) {
            int64_t f;
            int n;
            if (!packed_range(a.cu, g, a.n_seqs, f, n)) set_status(a.status, B200_DEV_BAD_POSITION);
        }
    bool bad = false;
    const auto block_of = [&](const int32_t *table, uint32_t slot) { return static_cast<int64_t>(__ldg(table + slot)); };
    const int32_t *ptable = a.prefix_table + (in ? group : 0) * a.prefix_stride;
    for (int64_t s = threadIdx.x; s * a.bt < prefix; s += blockDim.x) {
        const int64_t blk = block_of(ptable, static_cast<uint32_t>(s));
        bad |= blk < 0 || blk >= a.n_blocks;
    }
    bad = __syncthreads_or(bad);
    if (bad && threadIdx.x == 0) set_status(a.status, B200_DEV_BAD_POSITION);
    const T *q = static_cast<const T *>(a.q) + b * a.q_seq + static_cast<int64_t>(h) * a.G * a.q_head;
    T *out = static_cast<T *>(a.out) + b * a.o_seq + static_cast<int64_t>(h) * a.G * a.o_head;
    attend_rows<D>(
        a.G, bad ? 0 : prefix + keys, a.sl2,
        [&](int64_t j, int lane, float (&k)[E], float (&v)[E]) {
            const bool own = j >= prefix;
            const uint32_t pos = static_cast<uint32_t>(own ? j - prefix : j), slot = pos / a.bt;
            const int64_t blk = block_of(own ? a.table + b * a.table_stride : ptable, slot);
            if (blk < 0 || blk >= a.n_blocks) {
                set_status(a.status, B200_DEV_BAD_POSITION);
                return false;
            }
            const int64_t at = blk * a.block_stride + (pos - slot * a.bt) * a.tok_stride + h * a.head_stride + lane * E;
            for (int e = 0; e < E; ++e) {
                k[e] = to_f32<T>(reinterpret_cast<const T *>(a.k)[at + e]);
                v[e] = to_f32<T>(reinterpret_cast<const T *>(a.v)[at + e]);
            }
            return true;
        },
        [&](int g, int d) { return to_f32<T>(q[g * a.q_head + d]); },
        [&](int g, int d, float x) { out[g * a.o_head + d] = from_f32<T>(x); });
}

template <typename T>
cudaError_t shared_by_dim(const SharedArgs &a, int64_t D, cudaStream_t st) {
    const int64_t pairs = static_cast<int64_t>(a.n_seqs) * a.Hkv;
    if (pairs > INT32_MAX) return cudaErrorNotSupported;
    if (D == 128) shared_rows_kernel<T, 128><<<static_cast<unsigned>(pairs), 32 * kArWarps, 0, st>>>(a);
    else shared_rows_kernel<T, 64><<<static_cast<unsigned>(pairs), 32 * kArWarps, 0, st>>>(a);
    return cudaGetLastError();
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

size_t b200_flash_attn_paged_shared_workspace_bytes(int64_t n_seqs, int64_t max_keys, int64_t n_groups, int64_t max_prefix,
                                                    int64_t D, int64_t Hq, int64_t Hkv, int32_t dtype) {
    return 0;
}

int b200_flash_attn_paged_shared(const void *q, int64_t q_seq_stride, int64_t q_head_stride, void *out,
                                 int64_t out_seq_stride, int64_t out_head_stride, const b200_kv_pool *pool,
                                 const int32_t *prefix_table, int64_t prefix_stride, int64_t prefix_blocks,
                                 const int32_t *prefix_lens, const int32_t *cu_seqs, int64_t n_groups,
                                 const int32_t *block_table, int64_t table_stride, int64_t max_blocks,
                                 const int32_t *seq_lens, int64_t n_seqs, int64_t Hq, float scale, void *workspace,
                                 size_t workspace_bytes, int32_t *dev_status, void *stream) {
    if (n_seqs < 0 || n_groups < 0 || Hq <= 0) return B200_ERR_INVALID_ARGUMENT;
    const int rc = check_pool(pool);
    if (rc != B200_OK) return rc;
    const int64_t D = pool->head_dim, Hkv = pool->n_head_kv;
    if (Hq % Hkv) return B200_ERR_INVALID_ARGUMENT;
    if (n_seqs == 0) return B200_OK;
    if (!q || !out || !block_table || !seq_lens || max_blocks <= 0 || table_stride < max_blocks ||
        (n_groups > 0 && (!prefix_table || !prefix_lens || !cu_seqs || prefix_blocks <= 0 || prefix_stride < prefix_blocks)))
        return B200_ERR_INVALID_ARGUMENT;
    const int e = dtype_bytes(pool->dtype);
    if ((D != 64 && D != 128) || n_seqs > kMostRows || n_groups > kMostRows || Hq > 65536 ||
        !rows_aligned16(q, q_seq_stride, q_head_stride, e) || !rows_aligned16(out, out_seq_stride, out_head_stride, e))
        return B200_ERR_NOT_SUPPORTED;
    const auto positions = [&](int64_t blocks) {
        return blocks > kMostKeys / pool->block_tokens ? kMostKeys : blocks * pool->block_tokens;
    };
    SharedArgs a;
    a.max_keys = positions(max_blocks);
    a.max_prefix = n_groups ? positions(prefix_blocks) : 0;
    const size_t need =
        b200_flash_attn_paged_shared_workspace_bytes(n_seqs, a.max_keys, n_groups, a.max_prefix, D, Hq, Hkv, pool->dtype);
    if (need && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < need))
        return B200_ERR_INVALID_ARGUMENT;
    a.q = q;
    a.out = out;
    a.q_seq = q_seq_stride;
    a.q_head = q_head_stride;
    a.o_seq = out_seq_stride;
    a.o_head = out_head_stride;
    a.k = static_cast<const char *>(pool->k);
    a.v = static_cast<const char *>(pool->v);
    a.block_stride = pool->block_stride;
    a.tok_stride = pool->tok_stride;
    a.head_stride = pool->head_stride;
    a.n_blocks = pool->n_blocks;
    a.table = block_table;
    a.lens = seq_lens;
    a.prefix_table = prefix_table;
    a.prefix_lens = prefix_lens;
    a.cu = cu_seqs;
    a.table_stride = table_stride;
    a.prefix_stride = prefix_stride;
    a.bt = static_cast<uint32_t>(pool->block_tokens);
    a.n_seqs = static_cast<int>(n_seqs);
    a.n_groups = static_cast<int>(n_groups);
    a.G = static_cast<int>(Hq / Hkv);
    a.Hkv = static_cast<int>(Hkv);
    a.sl2 = (scale > 0.f ? scale : 1.0f / sqrtf(static_cast<float>(D))) * kLog2e;
    a.status = dev_status;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (pool->dtype) {
        case B200_DTYPE_F16: return status_of(shared_by_dim<__half>(a, D, st));
        case B200_DTYPE_BF16: return status_of(shared_by_dim<__nv_bfloat16>(a, D, st));
    }
    return status_of(shared_by_dim<float>(a, D, st));
}

}  // extern "C"
