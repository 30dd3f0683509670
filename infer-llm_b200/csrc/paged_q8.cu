// b200_paged_kv_append_q8 and b200_paged_kv_read_q8: packed rows into an 8-bit paged cache, and back.
//
// A row x of D elements becomes q = e4m3(x 2^-e) and e, the least whole number with max |x| <= 448 2^e. A power of two as
// scale leaves x 2^-e exact, so an element is rounded once and the answer does not depend on how a quotient is
// rounded; within a factor of two of the range it costs e4m3, whose steps are relative, no accuracy.
// Both are passes over bytes: 4096 F32 rows of 8 heads of 128 (42 MB) into the cache 14 us a call, 3.0 TB/s; 32 k BF16 rows (198
// MB) out of it 36 us, 5.5 TB/s, 84 % of a large copy's rate. For one decode step's few rows the dependent chain row -> sequence
// -> block -> store bounds them (64 rows 3 us on the device).
#include "paged_q8.cuh"

namespace b200 {
namespace {

struct Q8Args {
    const char *src[2] = {};  // append: K, V rows
    char *dst[2] = {};        // read: K, V rows
    char *pool[2] = {}, *scale[2] = {};
    int64_t row_tok[2] = {}, row_head[2] = {};  // bytes
    int64_t block_stride = 0, tok_stride = 0, head_stride = 0;
    int64_t scale_block = 0, scale_tok = 0, scale_head = 0;
    const int32_t *cu = nullptr, *lens = nullptr, *table = nullptr;
    int64_t table_stride = 0, max_blocks = 0, n_blocks = 0, n_tokens = 0;
    uint32_t block_tokens = 1, bt_mul = 0, bt_shift = 0;  // x / block_tokens = x bt_mul / 2^bt_shift for x < 2^31
    int32_t n_seqs = 0, chunks = 0;  // 16-byte chunks of a token's rows of F32, F16 or BF16
    int32_t *status = nullptr;
};

constexpr int kQ8Threads = 128, kQ8Chunks = 4;

// Block and place in it of packed row t of sequence s, a sequence's rows being its last positions; false if the sequence's
// offsets, the position or the block are out of range.
B200_DEVICE bool q8_place(const Q8Args &a, int s, int64_t t, int64_t &block, int64_t &place) {
    const int64_t end = __ldg(a.cu + s + 1), pos = __ldg(a.lens + s) - end + t;  // < 2^31: t is a row of s
    if (__ldg(a.cu + s) < 0 || end > a.n_tokens || pos < 0) return false;
    const int64_t slot = static_cast<int64_t>(static_cast<uint64_t>(pos) * a.bt_mul >> a.bt_shift);
    if (slot >= a.max_blocks) return false;
    block = __ldg(a.table + s * a.table_stride + slot);
    place = pos - slot * a.block_tokens;
    return block >= 0 && block < a.n_blocks;
}

// A warp takes up to four 16-byte chunks a lane of one token's K or V rows; the lanes of a head reduce its largest
// magnitude. Loads are issued before the lookups.
template <typename T, int D>
__global__ void __launch_bounds__(kQ8Threads) paged_append_q8_kernel(const Q8Args a) {
    constexpr int E = 16 / sizeof(T), L = D / E;  // elements of a chunk, lanes of a head (8, 16 or 32)
    const int lane = threadIdx.x & 31, kv = blockIdx.z;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * (kQ8Threads / 32) + (threadIdx.x >> 5);
    if (t >= a.n_tokens) return;
    const int c0 = blockIdx.y * 32 * kQ8Chunks + lane, h0 = c0 / L, r = c0 % L;
    const char *src = a.src[kv] + t * a.row_tok[kv] + r * 16;
    uint4 x[kQ8Chunks];
#pragma unroll
    for (int i = 0; i < kQ8Chunks; ++i)
        x[i] = c0 + 32 * i < a.chunks
                   ? __ldg(reinterpret_cast<const uint4 *>(src + (h0 + i * (32 / L)) * a.row_head[kv]))
                   : make_uint4(0, 0, 0, 0);
    const int s = warp_find_row(a.cu, a.n_seqs, t);
    int64_t block = 0, place = 0;
    if (s < 0 || !q8_place(a, s, t, block, place)) {
        if (lane == 0) set_status(a.status, B200_DEV_BAD_POSITION);
        return;
    }
    char *dst = a.pool[kv] + block * a.block_stride + place * a.tok_stride + r * E;
    char *scale = a.scale[kv] + block * a.scale_block + place * a.scale_tok;
#pragma unroll
    for (int i = 0; i < kQ8Chunks; ++i) {
        float v[E];
        const T *e = reinterpret_cast<const T *>(&x[i]);
        uint32_t top = 0;  // magnitudes as bits: in the order of the numbers, infinities and NaN above all
#pragma unroll
        for (int j = 0; j < E; ++j) {
            v[j] = to_f32<T>(e[j]);
            top = max(top, __float_as_uint(v[j]) & 0x7FFFFFFFu);
        }
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const bool odd = top >= 0x7F800000u;
        const uint32_t b = odd ? 255u : e8m0_of(top);
        const float inv = odd ? 0.f : e8m0_inverse(b);
        uint32_t q[E / 4];
#pragma unroll
        for (int j = 0; j < E; j += 4) {
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[j] * inv, v[j + 1] * inv), __NV_SATFINITE, __NV_E4M3);
            const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[j + 2] * inv, v[j + 3] * inv), __NV_SATFINITE, __NV_E4M3);
            q[j / 4] = odd ? 0u : lo | hi << 16;
        }
        if (c0 + 32 * i >= a.chunks) continue;
        const int h = h0 + i * (32 / L);
        if constexpr (E == 4) *reinterpret_cast<uint32_t *>(dst + h * a.head_stride) = q[0];
        else *reinterpret_cast<uint2 *>(dst + h * a.head_stride) = make_uint2(q[0], q[E / 4 - 1]);
        if (r == 0) scale[h * a.scale_head] = static_cast<char>(b);
    }
}

// The same chunks the other way, K and V by one warp: its lookups serve both (198 MB 39 -> 36 us; append, whose loads come before
// them, 13.9 -> 14.4).
template <typename T, int D>
__global__ void __launch_bounds__(kQ8Threads) paged_read_q8_kernel(const Q8Args a) {
    constexpr int E = 16 / sizeof(T), L = D / E;
    const int lane = threadIdx.x & 31;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * (kQ8Threads / 32) + (threadIdx.x >> 5);
    if (t >= a.n_tokens) return;
    const int s = warp_find_row(a.cu, a.n_seqs, t);
    // outside every sequence: left as it was
    if (s < 0 && (t < __ldg(a.cu) || t >= __ldg(a.cu + a.n_seqs))) return;
    const int c0 = blockIdx.y * 32 * kQ8Chunks + lane, h0 = c0 / L, r = c0 % L;
    int64_t block = 0, place = 0;
    const bool ok = s >= 0 && q8_place(a, s, t, block, place);
    if (!ok && lane == 0) set_status(a.status, B200_DEV_BAD_POSITION);
    const int64_t data_at = block * a.block_stride + place * a.tok_stride + h0 * a.head_stride + r * E;
    const int64_t scale_at = block * a.scale_block + place * a.scale_tok + h0 * a.scale_head;
    uint32_t q[2][kQ8Chunks][E / 4], b[2][kQ8Chunks];
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
        const char *src = a.pool[kv] + data_at, *scale = a.scale[kv] + scale_at;
#pragma unroll
        for (int i = 0; i < kQ8Chunks; ++i) {
            const bool in = ok && c0 + 32 * i < a.chunks;
            const char *at = src + i * (32 / L) * a.head_stride;
            if constexpr (E == 4) {
                q[kv][i][0] = in ? __ldg(reinterpret_cast<const uint32_t *>(at)) : 0u;
            } else {
                const uint2 u = in ? __ldg(reinterpret_cast<const uint2 *>(at)) : make_uint2(0, 0);
                q[kv][i][0] = u.x, q[kv][i][E / 4 - 1] = u.y;
            }
            b[kv][i] = in ? __ldg(reinterpret_cast<const unsigned char *>(scale + i * (32 / L) * a.scale_head)) : 0u;
        }
    }
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
        char *dst = a.dst[kv] + t * a.row_tok[kv] + h0 * a.row_head[kv] + r * 16;
#pragma unroll
        for (int i = 0; i < kQ8Chunks; ++i) {
            if (c0 + 32 * i >= a.chunks) continue;
            const float f = e8m0_value(b[kv][i]);
            T x[E];
#pragma unroll
            for (int j = 0; j < E; j += 4) {
                uint32_t h[2];
                e4m3x4_to_f16(q[kv][i][j / 4], h[0], h[1]);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&h[u]));
                    x[j + 2 * u] = from_f32<T>(v.x * f);
                    x[j + 2 * u + 1] = from_f32<T>(v.y * f);
                }
            }
            *reinterpret_cast<uint4 *>(dst + i * (32 / L) * a.row_head[kv]) = *reinterpret_cast<const uint4 *>(x);
        }
    }
}

Q8Args q8_args(const b200_kv_pool_q8 *p, const int32_t *table, int64_t table_stride, int64_t max_blocks, const int32_t *cu,
               const int32_t *lens, int64_t n_seqs, int64_t n_tokens, int64_t k_tok, int64_t k_head, int64_t v_tok,
               int64_t v_head, int e, int32_t *status) {
    Q8Args a;
    a.pool[0] = static_cast<char *>(p->k);
    a.pool[1] = static_cast<char *>(p->v);
    a.scale[0] = static_cast<char *>(p->k_scale);
    a.scale[1] = static_cast<char *>(p->v_scale);
    a.row_tok[0] = k_tok * e;
    a.row_tok[1] = v_tok * e;
    a.row_head[0] = k_head * e;
    a.row_head[1] = v_head * e;
    a.block_stride = p->block_stride;
    a.tok_stride = p->tok_stride;
    a.head_stride = p->head_stride;
    a.scale_block = p->scale_block_stride;
    a.scale_tok = p->scale_tok_stride;
    a.scale_head = p->scale_head_stride;
    a.cu = cu;
    a.lens = lens;
    a.table = table;
    a.table_stride = table_stride;
    a.max_blocks = max_blocks;
    a.n_blocks = p->n_blocks;
    a.block_tokens = static_cast<uint32_t>(p->block_tokens);
    reciprocal31(a.block_tokens, a.bt_mul, a.bt_shift);
    a.n_seqs = static_cast<int32_t>(n_seqs);
    a.n_tokens = n_tokens;
    a.chunks = static_cast<int32_t>(p->n_head_kv * p->head_dim * e / 16);
    a.status = status;
    return a;
}

template <typename T>
int q8_launch(bool append, int64_t D, const Q8Args &a, cudaStream_t st) {
    constexpr int kWarps = kQ8Threads / 32, kWarpChunks = 32 * kQ8Chunks;
    const dim3 grid(static_cast<unsigned>((a.n_tokens + kWarps - 1) / kWarps),
                    static_cast<unsigned>((a.chunks + kWarpChunks - 1) / kWarpChunks), append ? 2 : 1);  // y <= 2^15
    if (append && D == 128) paged_append_q8_kernel<T, 128><<<grid, kQ8Threads, 0, st>>>(a);
    else if (append) paged_append_q8_kernel<T, 64><<<grid, kQ8Threads, 0, st>>>(a);
    else if (D == 128) paged_read_q8_kernel<T, 128><<<grid, kQ8Threads, 0, st>>>(a);
    else paged_read_q8_kernel<T, 64><<<grid, kQ8Threads, 0, st>>>(a);
    return status_of(cudaGetLastError());
}

int q8_by_type(bool append, int32_t dtype, int64_t D, const Q8Args &a, void *stream) {
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case B200_DTYPE_F16: return q8_launch<__half>(append, D, a, st);
        case B200_DTYPE_BF16: return q8_launch<__nv_bfloat16>(append, D, a, st);
    }
    return q8_launch<float>(append, D, a, st);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

int b200_paged_kv_append_q8(const void *k, int64_t k_tok_stride, int64_t k_head_stride, const void *v, int64_t v_tok_stride,
                            int64_t v_head_stride, int32_t dtype, const int32_t *cu_new, const int32_t *seq_lens,
                            int64_t n_seqs, int64_t n_tokens, const b200_kv_pool_q8 *pool, const int32_t *block_table,
                            int64_t table_stride, int64_t max_blocks, int32_t *dev_status, void *stream) {
    const int e = dtype_bytes(dtype);
    if (n_seqs < 0 || n_tokens < 0 || !e) return B200_ERR_INVALID_ARGUMENT;
    const int rc = check_pool_q8(pool);
    if (rc != B200_OK) return rc;
    if (n_tokens == 0) return B200_OK;
    if (!k || !v || !cu_new || !seq_lens || !block_table || n_seqs == 0 || max_blocks <= 0 || table_stride < max_blocks)
        return B200_ERR_INVALID_ARGUMENT;
    if (!rows_aligned16(k, k_tok_stride, k_head_stride, e) || !rows_aligned16(v, v_tok_stride, v_head_stride, e) ||
        n_seqs > kMostRows || n_tokens > kMostRows)
        return B200_ERR_NOT_SUPPORTED;
    Q8Args a = q8_args(pool, block_table, table_stride, max_blocks, cu_new, seq_lens, n_seqs, n_tokens, k_tok_stride,
                       k_head_stride, v_tok_stride, v_head_stride, e, dev_status);
    a.src[0] = static_cast<const char *>(k);
    a.src[1] = static_cast<const char *>(v);
    return q8_by_type(true, dtype, pool->head_dim, a, stream);
}

int b200_paged_kv_read_q8(const b200_kv_pool_q8 *pool, const int32_t *block_table, int64_t table_stride, int64_t max_blocks,
                          const int32_t *cu_rows, const int32_t *seq_lens, int64_t n_seqs, int64_t n_rows, void *k,
                          int64_t k_tok_stride, int64_t k_head_stride, void *v, int64_t v_tok_stride, int64_t v_head_stride,
                          int32_t dtype, int32_t *dev_status, void *stream) {
    const int e = dtype_bytes(dtype);
    if (n_seqs < 0 || n_rows < 0 || !e) return B200_ERR_INVALID_ARGUMENT;
    const int rc = check_pool_q8(pool);
    if (rc != B200_OK) return rc;
    if (n_rows == 0) return B200_OK;
    if (!k || !v || !cu_rows || !seq_lens || !block_table || n_seqs == 0 || max_blocks <= 0 || table_stride < max_blocks)
        return B200_ERR_INVALID_ARGUMENT;
    if (!rows_aligned16(k, k_tok_stride, k_head_stride, e) || !rows_aligned16(v, v_tok_stride, v_head_stride, e) ||
        n_seqs > kMostRows || n_rows > kMostRows)
        return B200_ERR_NOT_SUPPORTED;
    Q8Args a = q8_args(pool, block_table, table_stride, max_blocks, cu_rows, seq_lens, n_seqs, n_rows, k_tok_stride,
                       k_head_stride, v_tok_stride, v_head_stride, e, dev_status);
    a.dst[0] = static_cast<char *>(k);
    a.dst[1] = static_cast<char *>(v);
    return q8_by_type(false, dtype, pool->head_dim, a, stream);
}

}  // extern "C"
