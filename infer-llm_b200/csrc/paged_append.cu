// b200_paged_kv_append: the K / V rows of a packed batch of new tokens into the blocks
// of their sequences. A copy: bytes bound it (each row read once and written once), and
// for one decode step's few rows the latency of one dependent chain, row -> sequence ->
// block -> store. A warp takes up to 2 KB of one row of K or V: its loads (four of 16
// bytes a lane) are issued before the lookups, so the chain and the loads overlap. Index
// arithmetic is 32-bit and one division a warp: in 64 bits it took two thirds of the issue
// slots (4096 F32 rows of 8 heads of 128, 67 MB: 16.2 us, now 14.6, 4.6 TB/s). 64 BF16 rows: 5 us
// on the device.
#include "batch.cuh"

namespace b200 {
namespace {

struct AppendArgs {
    const char *src[2];       // K, V rows
    char *dst[2];             // the pool's K, V
    int64_t src_tok[2], src_head[2];  // bytes
    int64_t block_stride, tok_stride, head_stride;  // bytes
    const int32_t *cu, *lens, *table;
    int64_t table_stride, max_blocks, n_blocks, n_tokens;
    uint32_t block_tokens;
    int32_t n_seqs, chunks, head_chunks;  // 16-byte chunks of a row / of a head
    int32_t step_heads, step_chunks;      // 32 chunks as whole heads and the rest
    int32_t *status;
    B200_DEVICE void next(int &h, int &r) const {
        h += step_heads, r += step_chunks;
        if (r >= head_chunks) ++h, r -= head_chunks;
    }
};

constexpr int kAppendThreads = 128;
constexpr int kLaneChunks = 4;

__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const AppendArgs a) {
    const int lane = threadIdx.x & 31, kv = blockIdx.z;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * (kAppendThreads / 32) + (threadIdx.x >> 5);
    if (t >= a.n_tokens) return;
    // Head h and chunk r of it, for chunk c of the row; 32 chunks on is one addition with a carry.
    const int c0 = blockIdx.y * 32 * kLaneChunks + lane;
    const int h0 = static_cast<int>(static_cast<unsigned>(c0) / static_cast<unsigned>(a.head_chunks));
    const int r0 = c0 - h0 * a.head_chunks;
    const char *src = a.src[kv] + t * a.src_tok[kv];
    uint4 x[kLaneChunks];
    int h = h0, r = r0;
#pragma unroll
    for (int i = 0; i < kLaneChunks; ++i) {
        if (c0 + 32 * i < a.chunks) x[i] = __ldg(reinterpret_cast<const uint4 *>(src + h * a.src_head[kv] + r * 16));
        a.next(h, r);
    }
    const int s = warp_find_row(a.cu, a.n_seqs, t);
    if (s < 0) {
        if (lane == 0) set_status(a.status, B200_DEV_BAD_POSITION);
        return;
    }
    const int64_t pos = static_cast<int64_t>(__ldg(a.lens + s)) - __ldg(a.cu + s + 1) + t;  // < 2^31: t is a row of s
    const int64_t slot = pos < 0 ? -1 : static_cast<int64_t>(static_cast<unsigned>(pos) / a.block_tokens);
    const int64_t blk = slot >= 0 && slot < a.max_blocks ? __ldg(a.table + s * a.table_stride + slot) : -1;
    if (blk < 0 || blk >= a.n_blocks) {
        if (lane == 0) set_status(a.status, B200_DEV_BAD_POSITION);
        return;
    }
    char *dst = a.dst[kv] + blk * a.block_stride + (pos - slot * a.block_tokens) * a.tok_stride;
    h = h0, r = r0;
#pragma unroll
    for (int i = 0; i < kLaneChunks; ++i) {
        if (c0 + 32 * i < a.chunks) *reinterpret_cast<uint4 *>(dst + h * a.head_stride + r * 16) = x[i];
        a.next(h, r);
    }
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200_paged_kv_append(const void *k, int64_t k_tok_stride, int64_t k_head_stride, const void *v,
                                    int64_t v_tok_stride, int64_t v_head_stride, const int32_t *cu_new,
                                    const int32_t *seq_lens, int64_t n_seqs, int64_t n_tokens,
                                    const b200_kv_pool *pool, const int32_t *block_table, int64_t table_stride,
                                    int64_t max_blocks, int32_t *dev_status, void *stream) {
    if (n_seqs < 0 || n_tokens < 0) return B200_ERR_INVALID_ARGUMENT;
    const int rc = check_pool(pool);
    if (rc != B200_OK) return rc;
    if (n_tokens == 0) return B200_OK;
    if (!k || !v || !cu_new || !seq_lens || !block_table || n_seqs == 0 || max_blocks <= 0 || table_stride < max_blocks)
        return B200_ERR_INVALID_ARGUMENT;
    const int e = dtype_bytes(pool->dtype);
    if (!rows_aligned16(k, k_tok_stride, k_head_stride, e) || !rows_aligned16(v, v_tok_stride, v_head_stride, e) ||
        n_seqs > kMostRows || n_tokens > kMostRows || pool->n_head_kv > (1 << 24) / pool->head_dim)
        return B200_ERR_NOT_SUPPORTED;
    AppendArgs a = {};
    a.src[0] = static_cast<const char *>(k);
    a.src[1] = static_cast<const char *>(v);
    a.dst[0] = static_cast<char *>(pool->k);
    a.dst[1] = static_cast<char *>(pool->v);
    a.src_tok[0] = k_tok_stride * e;
    a.src_tok[1] = v_tok_stride * e;
    a.src_head[0] = k_head_stride * e;
    a.src_head[1] = v_head_stride * e;
    a.block_stride = pool->block_stride * e;
    a.tok_stride = pool->tok_stride * e;
    a.head_stride = pool->head_stride * e;
    a.cu = cu_new;
    a.lens = seq_lens;
    a.table = block_table;
    a.table_stride = table_stride;
    a.max_blocks = max_blocks;
    a.n_blocks = pool->n_blocks;
    a.block_tokens = static_cast<uint32_t>(pool->block_tokens);
    a.n_tokens = n_tokens;
    a.n_seqs = static_cast<int32_t>(n_seqs);
    a.head_chunks = static_cast<int32_t>(pool->head_dim * e / 16);
    a.chunks = static_cast<int32_t>(pool->n_head_kv) * a.head_chunks;
    a.step_heads = 32 / a.head_chunks;
    a.step_chunks = 32 % a.head_chunks;
    a.status = dev_status;
    constexpr int kWarps = kAppendThreads / 32, kWarpChunks = 32 * kLaneChunks;
    const dim3 grid(static_cast<unsigned>((n_tokens + kWarps - 1) / kWarps),
                    static_cast<unsigned>((a.chunks + kWarpChunks - 1) / kWarpChunks), 2);  // y <= 2^15
    paged_append_kernel<<<grid, kAppendThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
    return status_of(cudaGetLastError());
}
