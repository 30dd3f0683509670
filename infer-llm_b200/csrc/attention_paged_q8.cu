// b200_flash_attn_paged_batch_q8: one query token for each of many sequences against an 8-bit paged cache.
//
// out_b = sum_j softmax_j(scale 2^ek_j q_b . kq_j) 2^ev_j vq_j over the keys j < seq_lens[b].
#include "attention_rows.cuh"
#include "gemv.cuh"
#include "paged_q8.cuh"

namespace b200 {
namespace {

constexpr int64_t kMostKeys = INT32_MAX - 256;

struct P8Args {
    const void *q = nullptr;
    void *out = nullptr;
    int64_t q_seq = 0, q_head = 0, o_seq = 0, o_head = 0;  // elements
    const char *k = nullptr, *v = nullptr;
    const unsigned char *ke = nullptr, *ve = nullptr;
    int64_t block_stride = 0, tok_stride = 0, head_stride = 0;
    int64_t scale_block = 0, scale_tok = 0, scale_head = 0;
    int64_t n_blocks = 0;
    const int32_t *table = nullptr, *lens = nullptr;
    int64_t table_stride = 0;
    int64_t max_keys = 0;  // positions a table row covers (fits 31 bits)
    uint32_t bt = 1;
    int n_seqs = 0, G = 0, Hkv = 0;
    float sl2 = 0.f;  // scale * log2 e
    int32_t *status = nullptr;
};

template <typename T, int D>
__global__ void __launch_bounds__(32 * kArWarps) paged_q8_rows_kernel(const __grid_constant__ P8Args a) {
    constexpr int E = D / 32;
    const int b = static_cast<int>(blockIdx.x / static_cast<unsigned>(a.Hkv)), h = blockIdx.x % static_cast<unsigned>(a.Hkv);
    const int64_t len = __ldg(a.lens + b), keys = min64(max64(len, 0), a.max_keys);
    if (len != keys && threadIdx.x == 0 && h == 0) set_status(a.status, B200_DEV_BAD_POSITION);
    const T *q = static_cast<const T *>(a.q) + b * a.q_seq + static_cast<int64_t>(h) * a.G * a.q_head;
    T *out = static_cast<T *>(a.out) + b * a.o_seq + static_cast<int64_t>(h) * a.G * a.o_head;
    attend_rows<D>(
        a.G, keys, a.sl2,
        [&](int64_t j, int lane, float (&k)[E], float (&v)[E]) {
            const uint32_t slot = static_cast<uint32_t>(j) / a.bt;
            const int64_t blk = __ldg(a.table + b * a.table_stride + slot), t = static_cast<uint32_t>(j) - slot * a.bt;
            if (blk < 0 || blk >= a.n_blocks) {
                set_status(a.status, B200_DEV_BAD_POSITION);
                return false;
            }
            const int64_t at = blk * a.block_stride + t * a.tok_stride + h * a.head_stride + lane * E;
            const int64_t se = blk * a.scale_block + t * a.scale_tok + h * a.scale_head;
            const float fk = e8m0_value(a.ke[se]), fv = e8m0_value(a.ve[se]);
            for (int e = 0; e < E; e += 2) {
                const uint32_t x = e4m3x2_to_f16x2(*reinterpret_cast<const uint16_t *>(a.k + at + e));
                const uint32_t y = e4m3x2_to_f16x2(*reinterpret_cast<const uint16_t *>(a.v + at + e));
                const float2 xf = __half22float2(*reinterpret_cast<const __half2 *>(&x));
                const float2 yf = __half22float2(*reinterpret_cast<const __half2 *>(&y));
                k[e] = xf.x * fk, k[e + 1] = xf.y * fk, v[e] = yf.x * fv, v[e + 1] = yf.y * fv;
            }
            return true;
        },
        [&](int g, int d) { return to_f32<T>(q[g * a.q_head + d]); },
        [&](int g, int d, float x) { out[g * a.o_head + d] = from_f32<T>(x); });
}

template <typename T>
cudaError_t p8_by_dim(const P8Args &a, int64_t D, cudaStream_t st) {
    const int64_t pairs = static_cast<int64_t>(a.n_seqs) * a.Hkv;
    if (pairs > INT32_MAX) return cudaErrorNotSupported;
    if (D == 128) paged_q8_rows_kernel<T, 128><<<static_cast<unsigned>(pairs), 32 * kArWarps, 0, st>>>(a);
    else paged_q8_rows_kernel<T, 64><<<static_cast<unsigned>(pairs), 32 * kArWarps, 0, st>>>(a);
    return cudaGetLastError();
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

size_t b200_flash_attn_paged_batch_q8_workspace_bytes(int64_t n_seqs, int64_t max_keys, int64_t D, int64_t Hq, int64_t Hkv) {
    return 0;
}

int b200_flash_attn_paged_batch_q8(const void *q, int64_t q_seq_stride, int64_t q_head_stride, void *out,
                                   int64_t out_seq_stride, int64_t out_head_stride, int32_t dtype,
                                   const b200_kv_pool_q8 *pool, const int32_t *block_table, int64_t table_stride,
                                   int64_t max_blocks, const int32_t *seq_lens, int64_t n_seqs, int64_t Hq, float scale,
                                   void *workspace, size_t workspace_bytes, int32_t *dev_status, void *stream) {
    const int e = dtype_bytes(dtype);
    if (n_seqs < 0 || Hq <= 0 || !e) return B200_ERR_INVALID_ARGUMENT;
    const int rc = check_pool_q8(pool);
    if (rc != B200_OK) return rc;
    const int64_t D = pool->head_dim, Hkv = pool->n_head_kv;
    if (Hq % Hkv) return B200_ERR_INVALID_ARGUMENT;
    if (n_seqs == 0) return B200_OK;
    if (!q || !out || !block_table || !seq_lens || max_blocks <= 0 || table_stride < max_blocks)
        return B200_ERR_INVALID_ARGUMENT;
    if (n_seqs > kMostRows || Hq > 65536 || !rows_aligned16(q, q_seq_stride, q_head_stride, e) ||
        !rows_aligned16(out, out_seq_stride, out_head_stride, e))
        return B200_ERR_NOT_SUPPORTED;
    // a length and a tile past it fit 31 bits: the tail of a table of more positions is not used
    const int64_t max_keys =
        max_blocks > kMostKeys / pool->block_tokens ? kMostKeys : max_blocks * pool->block_tokens;
    const size_t need = b200_flash_attn_paged_batch_q8_workspace_bytes(n_seqs, max_keys, D, Hq, Hkv);
    if (need && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < need))
        return B200_ERR_INVALID_ARGUMENT;
    P8Args a;
    a.q = q;
    a.out = out;
    a.q_seq = q_seq_stride;
    a.q_head = q_head_stride;
    a.o_seq = out_seq_stride;
    a.o_head = out_head_stride;
    a.k = static_cast<const char *>(pool->k);
    a.v = static_cast<const char *>(pool->v);
    a.ke = static_cast<const unsigned char *>(pool->k_scale);
    a.ve = static_cast<const unsigned char *>(pool->v_scale);
    a.block_stride = pool->block_stride;
    a.tok_stride = pool->tok_stride;
    a.head_stride = pool->head_stride;
    a.scale_block = pool->scale_block_stride;
    a.scale_tok = pool->scale_tok_stride;
    a.scale_head = pool->scale_head_stride;
    a.n_blocks = pool->n_blocks;
    a.table = block_table;
    a.lens = seq_lens;
    a.table_stride = table_stride;
    a.bt = static_cast<uint32_t>(pool->block_tokens);
    a.max_keys = max_keys;
    a.n_seqs = static_cast<int>(n_seqs);
    a.G = static_cast<int>(Hq / Hkv);
    a.Hkv = static_cast<int>(Hkv);
    a.sl2 = (scale > 0.f ? scale : 1.0f / sqrtf(static_cast<float>(D))) * kLog2e;
    a.status = dev_status;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case B200_DTYPE_F16: return status_of(p8_by_dim<__half>(a, D, st));
        case B200_DTYPE_BF16: return status_of(p8_by_dim<__nv_bfloat16>(a, D, st));
    }
    return status_of(p8_by_dim<float>(a, D, st));
}

}  // extern "C"
