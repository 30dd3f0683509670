// b200_adjust_logits: penalties, biases and masks of each row's request on its logits, before a token is drawn.
//
//   x <- x / r or x r (known), x - f count - p (drawn), x + bias, -inf (masked)
//
// A pass over the logits, which HBM bounds; what has to be known of a token (how often it was drawn, whether the row knows it, its bias)
// is gathered before, in shared memory, for the chunk of the vocabulary that a CTA takes: it
// walks its row's history and counts what falls into its chunk. Counts are whole numbers, so their order does not matter.
// A row's history is walked once per chunk, from L2: a chunk of 8192 tokens (19 of a vocabulary of 151936) keeps that
// below the logits' own bytes up to 8192 F32 tokens of history; smaller chunks where there are few rows.
#include "batch.cuh"
#include "gemv.cuh"

namespace b200 {
namespace {

struct AdjustArgs {
    const void *in = nullptr;
    void *out = nullptr;
    int64_t in_row = 0, out_row = 0, n_rows = 0, n_tokens = 0, n_biases = 0, mask_row = 0;  // rows: elements (mask: words)
    int32_t vocab = 0, chunk = 0, chunks = 0;
    const int32_t *tokens = nullptr, *cu_tokens = nullptr, *prompt_lens = nullptr;
    const float *repetition = nullptr, *frequency = nullptr, *presence = nullptr;
    const int32_t *bias_ids = nullptr, *cu_bias = nullptr;
    const float *bias_values = nullptr;
    const uint32_t *mask = nullptr;
    int32_t *status = nullptr;
};

constexpr int kAdThreads = 256;
constexpr uint32_t kKnown = 1u << 31;  // a token of the history; the bits below count how often it was drawn

// The row's range of a packed list, empty (and reported) where the offsets are out of order or range.
B200_DEVICE void list_range(const int32_t *cu, int64_t row, int64_t total, int32_t *status, int64_t &from, int64_t &to) {
    from = __ldg(cu + row), to = __ldg(cu + row + 1);
    if (from >= 0 && from <= to && to <= total) return;
    if (threadIdx.x == 0) set_status(status, B200_DEV_BAD_POSITION);
    from = to = 0;
}

// A row's penalty, `off` where there is none or it makes no sense.
B200_DEVICE float penalty(const float *p, int64_t row, float off, bool positive, int32_t *status) {
    if (!p) return off;
    const float x = __ldg(p + row);
    if (fabsf(x) < INFINITY && (!positive || x > 0.f)) return x;
    if (threadIdx.x == 0) set_status(status, B200_DEV_BAD_LOGITS);
    return off;
}

template <typename T>
__global__ void __launch_bounds__(kAdThreads) adjust_logits_kernel(const __grid_constant__ AdjustArgs a) {
    constexpr int V = 16 / sizeof(T);
    extern __shared__ __align__(16) uint32_t ad_smem[];
    const int64_t row = blockIdx.x / static_cast<unsigned>(a.chunks);
    const int first = static_cast<int>(blockIdx.x % static_cast<unsigned>(a.chunks)) * a.chunk;
    const T *in = static_cast<const T *>(a.in) + row * a.in_row;
    T *out = static_cast<T *>(a.out) + row * a.out_row;
    // The chunk begins where its vectors are aligned in `in`: up to V - 1 elements before `first`
    const int skew = static_cast<int>(reinterpret_cast<uintptr_t>(in) / sizeof(T) % V);
    const int begin = first - skew, end = min(begin + a.chunk, a.vocab);  // this CTA's tokens
    // (the last chunk's end is the row's: chunks * chunk >= vocab + V)
    const bool in_place = a.in == a.out;
    const bool wide = reinterpret_cast<uintptr_t>(out) / sizeof(T) % V == static_cast<unsigned>(skew);
    uint32_t *known = ad_smem, *bias = ad_smem + (a.tokens ? a.chunk : 0);
    const int words = (a.tokens ? a.chunk : 0) + (a.bias_ids ? a.chunk : 0);
    bool any = false;  // a token of this chunk is known or biased
    float rep = 1.f, freq = 0.f, pres = 0.f;
    if (words) {
        for (int i = threadIdx.x; i < words / 4; i += kAdThreads) reinterpret_cast<uint4 *>(ad_smem)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        if (a.tokens) {
            rep = penalty(a.repetition, row, 1.f, true, a.status);
            freq = penalty(a.frequency, row, 0.f, false, a.status);
            pres = penalty(a.presence, row, 0.f, false, a.status);
            int64_t from, to;
            list_range(a.cu_tokens, row, a.n_tokens, a.status, from, to);
            const int64_t drawn = from + (a.prompt_lens ? max(0, __ldg(a.prompt_lens + row)) : 0);
            for (int64_t i = from + threadIdx.x; i < to; i += kAdThreads) {
                const int t = __ldg(a.tokens + i);
                if (t < 0 || t >= a.vocab) set_status(a.status, B200_DEV_BAD_TOKEN);
                else if (t >= begin && t < end) {
                    any = true;
                    if (i >= drawn) atomicAdd(known + (t - begin), 1u);
                    atomicOr(known + (t - begin), kKnown);
                }
            }
        }
        if (a.bias_ids) {
            int64_t from, to;
            list_range(a.cu_bias, row, a.n_biases, a.status, from, to);
            for (int64_t i = from + threadIdx.x; i < to; i += kAdThreads) {
                const int t = __ldg(a.bias_ids + i);
                if (t < 0 || t >= a.vocab) set_status(a.status, B200_DEV_BAD_TOKEN);
                else if (t >= begin && t < end) {
                    any = true;
                    atomicMax(bias + (t - begin), static_cast<uint32_t>(i + 1));  // of several the last
                }
            }
        }
        any = __syncthreads_or(any);
    }
    const auto adjusted = [&](T x, int t) {
        float y = to_f32<T>(x);
        if (a.tokens) {
            const uint32_t u = known[t - begin];
            if (u) {
                y = y > 0.f ? y / rep : y * rep;
                const uint32_t count = u & ~kKnown;
                if (count) y = y - freq * static_cast<float>(count) - pres;
            }
        }
        if (a.bias_ids) {
            const uint32_t i = bias[t - begin];
            if (i) y += __ldg(a.bias_values + (i - 1));
        }
        return from_f32<T>(y);
    };
    const uint32_t *mask = a.mask ? a.mask + row * a.mask_row : nullptr;
    const int last_word = (a.vocab - 1) >> 5;
    for (int t = begin + V * static_cast<int>(threadIdx.x); t < end; t += V * kAdThreads) {
        uint32_t allowed = ~0u;  // bit j: token t + j may be drawn
        if (mask) {
            const int at = max(t, 0), w = at >> 5;
            const uint32_t lo = __ldg(mask + w), hi = w < last_word ? __ldg(mask + w + 1) : 0u;
            allowed = __funnelshift_r(lo, hi, at & 31) << (at - t);
        }
        const bool whole = t >= 0 && t + V <= a.vocab;
        constexpr uint32_t kAll = (1u << V) - 1u;
        if (in_place && !any && (allowed & kAll) == kAll) continue;
        if (whole) {
            uint4 u = *reinterpret_cast<const uint4 *>(in + t);
            T *e = reinterpret_cast<T *>(&u);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (any) e[j] = adjusted(e[j], t + j);
                if (!(allowed >> j & 1u)) e[j] = from_f32<T>(-INFINITY);
            }
            if (wide) {
                *reinterpret_cast<uint4 *>(out + t) = u;
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) out[t + j] = e[j];
            }
        } else {
            for (int j = max(0, -t); j < V && t + j < a.vocab; ++j) {
                const T x = any ? adjusted(in[t + j], t + j) : in[t + j];
                out[t + j] = allowed >> j & 1u ? x : from_f32<T>(-INFINITY);
            }
        }
    }
}

template <typename T>
cudaError_t adjust_launch(AdjustArgs a, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    a.chunk = 8192;
    while (a.chunk > 1024 && a.n_rows * ((a.vocab + a.chunk - 1) / a.chunk) < 4 * device_sm_count()) a.chunk /= 2;
    a.chunks = (a.vocab + V - 1 + a.chunk - 1) / a.chunk;
    if (a.n_rows > INT32_MAX / a.chunks) return cudaErrorNotSupported;
    const size_t smem = static_cast<size_t>(a.chunk) * 4 * ((a.tokens ? 1 : 0) + (a.bias_ids ? 1 : 0));
    auto kern = adjust_logits_kernel<T>;
    const cudaError_t e = once_per_device(reinterpret_cast<const void *>(kern), ATTR_SMEM, [&] {
        return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 65536);
    });
    if (e != cudaSuccess) return e;
    kern<<<static_cast<unsigned>(a.n_rows * a.chunks), kAdThreads, smem, st>>>(a);
    return cudaGetLastError();
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200_adjust_logits(const void *logits, int64_t row_stride, void *out, int64_t out_row_stride, int64_t n_rows,
                                  int64_t n_vocab, int32_t dtype, const int32_t *tokens, int64_t n_tokens,
                                  const int32_t *cu_tokens, const int32_t *prompt_lens, const float *repetition,
                                  const float *frequency, const float *presence, const int32_t *bias_ids,
                                  const float *bias_values, int64_t n_biases, const int32_t *cu_bias, const uint32_t *mask,
                                  int64_t mask_stride, int32_t *dev_status, void *stream) {
    const int e = dtype_bytes(dtype);
    if (n_rows < 0 || n_vocab <= 0 || n_tokens < 0 || n_biases < 0 || !e) return B200_ERR_INVALID_ARGUMENT;
    if (n_rows == 0) return B200_OK;
    if (!logits || !out || row_stride < 0 || mask_stride < 0 || (n_rows > 1 && out_row_stride < n_vocab) ||
        (logits == out && row_stride != out_row_stride && n_rows > 1))
        return B200_ERR_INVALID_ARGUMENT;
    if ((n_tokens > 0 && !tokens) || (tokens && !cu_tokens) || (n_biases > 0 && !bias_ids) ||
        (bias_ids && (!bias_values || !cu_bias)))
        return B200_ERR_INVALID_ARGUMENT;
    if (!cu_tokens && (prompt_lens || repetition || frequency || presence)) return B200_ERR_INVALID_ARGUMENT;
    if (n_vocab > (1 << 21) || n_tokens > kMostRows || n_biases > kMostRows || reinterpret_cast<uintptr_t>(logits) % e ||
        reinterpret_cast<uintptr_t>(out) % e)
        return B200_ERR_NOT_SUPPORTED;
    AdjustArgs a;
    a.in = logits;
    a.out = out;
    a.in_row = row_stride;
    a.out_row = out_row_stride;
    a.n_rows = n_rows;
    a.n_tokens = n_tokens;
    a.n_biases = n_biases;
    a.mask_row = mask_stride;
    a.vocab = static_cast<int32_t>(n_vocab);
    a.tokens = n_tokens > 0 ? tokens : nullptr;
    a.cu_tokens = cu_tokens;
    a.prompt_lens = prompt_lens;
    a.repetition = repetition;
    a.frequency = frequency;
    a.presence = presence;
    a.bias_ids = n_biases > 0 ? bias_ids : nullptr;
    a.bias_values = bias_values;
    a.cu_bias = cu_bias;
    a.mask = mask;
    a.status = dev_status;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case B200_DTYPE_F16: return status_of(adjust_launch<__half>(a, st));
        case B200_DTYPE_BF16: return status_of(adjust_launch<__nv_bfloat16>(a, st));
    }
    return status_of(adjust_launch<float>(a, st));
}
