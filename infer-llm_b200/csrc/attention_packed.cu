// b200_flash_attn_packed: causal GQA attention of packed sequences, and its plain kernel.
//
// out_i = sum_j softmax_j(scale q_i . k_j) v_j over the keys j <= nk - nq + i of row i's own
// sequence. packed_ffma_kernel computes it with F32 FFMA for every type, 64 rows a CTA
// (attention_packed_ffma.cuh). It serves what the tensor-core kernel does not: F32 calls with few keys, more than 128
// query heads a KV head, strides that a tensor map cannot hold.
#include "attention_packed_ffma.cuh"
#include "gemv.cuh"

namespace b200 {
namespace {

template <typename T, int D>
__global__ void __launch_bounds__(kPkThreads, 2) packed_ffma_kernel(const PackedArgs a) {
    extern __shared__ __align__(16) float pk_smem[];
    const int kvh = blockIdx.x % a.Hkv;
    const PackedTile p = find_packed_tile(a.cu_q, a.cu_k, a.n_seqs, a.total_q, a.total_k, a.G, kPkRows,
                                          blockIdx.x / a.Hkv, a.status);
    if (blockIdx.x == gridDim.x - 1 && threadIdx.x < 32) clear_uncovered(a);
    if (p.seq < 0) return;
    const int r0 = p.tile * kPkRows, rows = min(kPkRows, p.nq * a.G - r0);
    T *out = static_cast<T *>(a.out);
    ffma_rows<T, D>(a, p, kvh, r0, rows, 0, p.nk, pk_smem, threadIdx.x, [] { __syncthreads(); },
                    [&](int r, int c, const float (&x)[4], float, float) {
                        T *dst = out + (p.q0 + (r0 + r) / a.G) * a.o_tok + (kvh * a.G + (r0 + r) % a.G) * a.o_head + c;
#pragma unroll
                        for (int e = 0; e < 4; ++e) dst[e] = from_f32<T>(x[e]);
                    });
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
                                    static_cast<int>(ffma_smem<D>()));
    });
    if (e != cudaSuccess) return e;
    const int64_t ctas = most_packed_tiles(a.n_seqs, a.total_q, a.G, kPkRows) * a.Hkv;
    if (ctas > INT32_MAX) return cudaErrorNotSupported;
    return b200_launch(kern, dim3(static_cast<unsigned>(ctas)), dim3(kPkThreads), ffma_smem<D>(), st, false, a);
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
    if ((D != 64 && D != 128) || Hq > 65536 || n_seqs > kMostRows || total_q > kMostRows / (Hq / Hkv) ||
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
