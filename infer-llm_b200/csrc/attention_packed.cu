// b200_flash_attn_packed: causal GQA attention of packed sequences, and its plain kernel.
//
// out_i = sum_j softmax_j(scale q_i . k_j) v_j over the keys j <= nk - nq + i of row i's own
// sequence. packed_ffma_kernel computes it with F32 FFMA for every type: 64 rows (tokens
// times the heads that share a KV head) against 64-key tiles, running maximum and sum,
// scores and output in registers as 4 x 4 and 4 x D/16 blocks a thread. The FFMA rate
// bounds it. It serves what the tensor-core kernel does not: F32 calls with few keys, more than 128
// query heads a KV head, strides that a tensor map cannot hold.
#include "attention_packed.cuh"
#include "gemv.cuh"

namespace b200 {
namespace {

constexpr int64_t kMostRows = INT32_MAX - 1024;  // row numbers of a tile past the last one fit 31 bits
constexpr int kPkRows = 64, kPkKeys = 64, kPkThreads = 256;
constexpr int kPkPad = kPkRows + 4;

B200_DEVICE void load4(const float *p, float (&x)[4]) {
    const float4 v = __ldg(reinterpret_cast<const float4 *>(p));
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
}
template <typename T>
B200_DEVICE void load4(const T *p, float (&x)[4]) {
    const uint2 v = __ldg(reinterpret_cast<const uint2 *>(p));
    const T *e = reinterpret_cast<const T *>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = to_f32<T>(e[i]);
}

template <int D>
constexpr size_t packed_smem() {
    return (2 * static_cast<size_t>(D) * kPkPad + static_cast<size_t>(kPkKeys) * D) * 4;
}

template <typename T, int D>
__global__ void __launch_bounds__(kPkThreads, 2) packed_ffma_kernel(const PackedArgs a) {
    extern __shared__ __align__(16) float pk_smem[];
    float *qt = pk_smem;               // [D][row]
    float *kt = qt + D * kPkPad;       // [D][key]; then P [key][row]
    float *vs = kt + D * kPkPad;       // [key][D]
    const int kvh = blockIdx.x % a.Hkv;
    const PackedTile p = find_packed_tile(a.cu_q, a.cu_k, a.n_seqs, a.total_q, a.total_k, a.G, kPkRows,
                                          blockIdx.x / a.Hkv, a.status);
    if (p.seq < 0) return;
    const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
    const int rows = min(kPkRows, p.nq * a.G - p.tile * kPkRows);
    const int r0 = p.tile * kPkRows;
    const T *q = static_cast<const T *>(a.q), *k = static_cast<const T *>(a.k), *v = static_cast<const T *>(a.v);
    // four elements a load; lanes take neighbouring rows, so the transposed stores do not collide
#pragma unroll
    for (int i0 = 0; i0 < kPkRows * D / 4; i0 += kPkThreads) {
        const int i = i0 + tid, r = i % kPkRows, d = i / kPkRows * 4;
        float x[4] = {0.f, 0.f, 0.f, 0.f};
        if (r < rows) {
            const int tok = (r0 + r) / a.G, h = kvh * a.G + (r0 + r) % a.G;
            load4(q + (p.q0 + tok) * a.q_tok + h * a.q_head + d, x);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) qt[(d + e) * kPkPad + r] = x[e];
    }
    int last[4];  // last key each row sees (relative to the sequence)
#pragma unroll
    for (int i = 0; i < 4; ++i) last[i] = 4 * ty + i < rows ? p.nk - p.nq + (r0 + 4 * ty + i) / a.G : -1;
    float m[4], l[4], o[4][D / 16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int e = 0; e < D / 16; ++e) o[i][e] = 0.f;
    }
    const int end = p.nk - p.nq + (r0 + rows - 1) / a.G + 1;  // keys the tile's last row sees
    for (int k0 = 0; k0 < end; k0 += kPkKeys) {
        __syncthreads();
#pragma unroll
        for (int i0 = 0; i0 < kPkKeys * D / 4; i0 += kPkThreads) {
            const int i = i0 + tid, j = i % kPkKeys, d = i / kPkKeys * 4;
            const int64_t t = p.k0 + k0 + j;
            float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
            if (k0 + j < end) {
                load4(k + t * a.k_tok + kvh * a.k_head + d, x);
                load4(v + t * a.v_tok + kvh * a.v_head + d, y);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) kt[(d + e) * kPkPad + j] = x[e];
            *reinterpret_cast<float4 *>(vs + j * D + d) = make_float4(y[0], y[1], y[2], y[3]);
        }
        __syncthreads();
        float s[4][4] = {};
#pragma unroll 8
        for (int d = 0; d < D; ++d) {
            const float4 x = *reinterpret_cast<const float4 *>(qt + d * kPkPad + 4 * ty);
            const float4 y = *reinterpret_cast<const float4 *>(kt + d * kPkPad + 4 * tx);
            const float xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[i][j] = fmaf(xs[i], ys[j], s[i][j]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[i][j] = k0 + 4 * tx + j <= last[i] ? s[i][j] * a.sl2 : -INFINITY;
                mx = fmaxf(mx, s[i][j]);
            }
#pragma unroll
            for (int w = 1; w < 16; w <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
            const float mn = fmaxf(m[i], mx), ms = mn == -INFINITY ? 0.f : mn;
            const float al = exp2_approx(m[i] - ms);
            m[i] = mn;
            l[i] *= al;
#pragma unroll
            for (int e = 0; e < D / 16; ++e) o[i][e] *= al;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[i][j] = exp2_approx(s[i][j] - ms);
                l[i] += s[i][j];
            }
        }
        __syncthreads();  // the keys have been read
#pragma unroll
        for (int j = 0; j < 4; ++j)
            *reinterpret_cast<float4 *>(kt + (4 * tx + j) * kPkPad + 4 * ty) = make_float4(s[0][j], s[1][j], s[2][j], s[3][j]);
        __syncthreads();
        // a key that a row does not see has P = 0, and 0 times a V that is no number would
        // not be 0: such products are left out where the tile has hidden keys
        const bool all = k0 + kPkKeys - 1 <= p.nk - p.nq + r0 / a.G;
#pragma unroll 4
        for (int j = 0; j < kPkKeys; ++j) {
            const float4 x = *reinterpret_cast<const float4 *>(kt + j * kPkPad + 4 * ty);
            const float xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
                const float4 y = *reinterpret_cast<const float4 *>(vs + j * D + 64 * c + 4 * tx);
                const float ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (all || k0 + j <= last[i]) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[i][4 * c + e] = fmaf(xs[i], ys[e], o[i][4 * c + e]);
                    }
            }
        }
    }
    T *out = static_cast<T *>(a.out);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = 4 * ty + i;
#pragma unroll
        for (int w = 1; w < 16; w <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], w);
        if (r >= rows) continue;
        const float inv = l[i] != 0.f ? 1.0f / l[i] : 0.f;  // no key, or scores of -inf alone: zeros
        T *dst = out + (p.q0 + (r0 + r) / a.G) * a.o_tok + (kvh * a.G + (r0 + r) % a.G) * a.o_head;
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) dst[64 * c + 4 * tx + e] = from_f32<T>(o[i][4 * c + e] * inv);
    }
}

// F32 calls with so few keys in all take the FFMA kernel: one launch of one key tile against the
// tensor cores' two launches (16 / 8 heads of 128: 64 tokens 24.6 us against 25.6, 100 tokens 36.9
// against 27.6; the second launch also costs the caller ~3 us).
bool packed_short(int32_t dtype, int64_t total_k) { return dtype == B200_DTYPE_F32 && total_k <= kPkKeys; }

template <typename T, int D>
cudaError_t packed_ffma_launch(const PackedArgs &a, cudaStream_t st) {
    auto kern = packed_ffma_kernel<T, D>;
    cudaError_t e = once_per_device(reinterpret_cast<const void *>(kern), ATTR_SMEM, [&] {
        return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    static_cast<int>(packed_smem<D>()));
    });
    if (e != cudaSuccess) return e;
    const int64_t ctas = most_packed_tiles(a.n_seqs, a.total_q, a.G, kPkRows) * a.Hkv;
    if (ctas > INT32_MAX) return cudaErrorNotSupported;
    return b200_launch(kern, dim3(static_cast<unsigned>(ctas)), dim3(kPkThreads), packed_smem<D>(), st, false, a);
}

template <typename T>
cudaError_t packed_by_dim(const PackedArgs &a, cudaStream_t st) {
    return a.D == 128 ? packed_ffma_launch<T, 128>(a, st) : packed_ffma_launch<T, 64>(a, st);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

size_t b200_flash_attn_packed_workspace_bytes(int64_t n_seqs, int64_t total_q, int64_t total_k, int64_t D, int64_t Hq,
                                              int64_t Hkv, int32_t dtype) {
    if (n_seqs <= 0 || total_q <= 0 || total_k <= 0 || D <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv ||
        packed_short(dtype, total_k))
        return 0;
    return packed_tc_workspace(n_seqs, total_q, total_k, D, Hq, Hkv, dtype);
}

int b200_flash_attn_packed(const void *q, int64_t q_tok_stride, int64_t q_head_stride, const void *k,
                           int64_t k_tok_stride, int64_t k_head_stride, const void *v, int64_t v_tok_stride,
                           int64_t v_head_stride, void *out, int64_t out_tok_stride, int64_t out_head_stride,
                           const int32_t *cu_q, const int32_t *cu_k, int64_t n_seqs, int64_t total_q, int64_t total_k,
                           int64_t D, int64_t Hq, int64_t Hkv, float scale, int32_t dtype, void *workspace,
                           size_t workspace_bytes, int32_t *dev_status, void *stream) {
    const int e = dtype_bytes(dtype);
    if (n_seqs < 0 || total_q < 0 || total_k < 0 || D <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || !e)
        return B200_ERR_INVALID_ARGUMENT;
    if (n_seqs == 0 || total_q == 0) return B200_OK;
    if (!q || !out || !cu_q || !cu_k || (total_k > 0 && (!k || !v))) return B200_ERR_INVALID_ARGUMENT;
    if ((D != 64 && D != 128) || Hq > 65536 || n_seqs >= INT32_MAX || total_q * (Hq / Hkv) > kMostRows ||
        total_k > kMostRows || !rows_aligned16(q, q_tok_stride, q_head_stride, e) ||
        !rows_aligned16(k, k_tok_stride, k_head_stride, e) || !rows_aligned16(v, v_tok_stride, v_head_stride, e) ||
        !rows_aligned16(out, out_tok_stride, out_head_stride, e))
        return B200_ERR_NOT_SUPPORTED;
    const size_t need = b200_flash_attn_packed_workspace_bytes(n_seqs, total_q, total_k, D, Hq, Hkv, dtype);
    if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)))
        return B200_ERR_INVALID_ARGUMENT;
    PackedArgs a;
    a.q = q;
    a.k = k;
    a.v = v;
    a.out = out;
    a.q_tok = q_tok_stride;
    a.q_head = q_head_stride;
    a.k_tok = k_tok_stride;
    a.k_head = k_head_stride;
    a.v_tok = v_tok_stride;
    a.v_head = v_head_stride;
    a.o_tok = out_tok_stride;
    a.o_head = out_head_stride;
    a.cu_q = cu_q;
    a.cu_k = cu_k;
    a.total_q = total_q;
    a.total_k = total_k;
    a.n_seqs = static_cast<int>(n_seqs);
    a.Hq = static_cast<int>(Hq);
    a.Hkv = static_cast<int>(Hkv);
    a.G = static_cast<int>(Hq / Hkv);
    a.D = static_cast<int>(D);
    a.sl2 = (scale > 0.f ? scale : 1.0f / sqrtf(static_cast<float>(D))) * kLog2e;
    a.dtype = dtype;
    a.ws = workspace;
    a.status = dev_status;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!packed_short(dtype, total_k)) {
        const cudaError_t tc = packed_tc_launch(a, st);
        if (tc != cudaErrorNotSupported) return status_of(tc);
    }
    switch (dtype) {
        case B200_DTYPE_F16: return status_of(packed_by_dim<__half>(a, st));
        case B200_DTYPE_BF16: return status_of(packed_by_dim<__nv_bfloat16>(a, st));
    }
    return status_of(packed_by_dim<float>(a, st));
}

}  // extern "C"
