// b200_adjust_logits: penalties, biases and masks of each row's request on its logits, before a token is drawn.
//
//   x <- x / r or x r (known), x - f count - p (drawn), x + bias, -inf (masked)
//
// A pass over the logits, which HBM bounds, by CTAs that take a chunk of a row's vocabulary each. What a row's history and biases say
// concerns few tokens: a CTA walks them for those of its chunk, sets a bit a token, counts the bits before each word, and so has a
// slot of its own for each such token, in which it counts; the pass then writes the chunk with the masked tokens replaced, and
// last come the tokens with slots, a thread each. Half of the warps pass and half walk at the same time, since the walk's chain
// (offsets, tokens, counters) is as long as the pass. The pass goes through a ring in shared memory that bulk copies fill and
// empty; a thread takes a mask word and its 32 tokens. 256 rows of 151936 F32 with up to 4000 tokens of history, masks and biases:
// 70 us, 4.5 TB/s, 69 % of a large copy's rate; the pass alone 55 with masks, 53 without (a library copy of these bytes 51). What
// is left is the walk, and the named tokens' scattered reads and writes. Otherwise: a mask word looked up for each vector of four
// 74 us for the pass, 88 in all; the pass through registers 82 in all, whole chunks in shared memory 112, two kernels 80 to 123;
// three stages and three CTAs an SM 74, five CTAs with half the slots 71. Counts are whole numbers, so their order does not matter.
#include "batch.cuh"
#include "gemv.cuh"
#include "tcgen05.cuh"

namespace b200 {
namespace {

struct AdjustArgs {
    const void *in = nullptr;
    void *out = nullptr;
    int64_t in_row = 0, out_row = 0, n_rows = 0, n_tokens = 0, n_biases = 0, mask_row = 0;  // rows: elements (mask: words)
    int32_t vocab = 0;
    const int32_t *tokens = nullptr, *cu_tokens = nullptr, *prompt_lens = nullptr;
    const float *repetition = nullptr, *frequency = nullptr, *presence = nullptr;
    const int32_t *bias_ids = nullptr, *cu_bias = nullptr;
    const float *bias_values = nullptr;
    const uint32_t *mask = nullptr;
    int32_t *status = nullptr;
};

constexpr int kAdPass = 128, kAdWalk = 128, kAdThreads = kAdPass + kAdWalk;  // threads that pass, and that walk
constexpr int kAdCtas = 4;                                        // an SM
constexpr int kAdStages = 2, kAdStep = 32 * kAdPass;              // stages of the ring, and their tokens
constexpr int kAdChunk = 16384, kAdSlots = 2048, kAdAtOnce = 8;  // tokens and slots of a CTA at most; list entries a thread asks for at once
constexpr uint32_t kKnown = 1u << 31;  // in a slot: a token of the history; the bits below count how often it was drawn

// The row's range of a packed list, empty (and reported) where the offsets are out of order or range.
B200_DEVICE void list_range(const int32_t *cu, int64_t row, int64_t total, int32_t *status, int64_t &from, int64_t &to) {
    from = __ldg(cu + row), to = __ldg(cu + row + 1);
    if (from >= 0 && from <= to && to <= total) return;
    set_status(status, B200_DEV_BAD_POSITION);
    from = to = 0;
}

// A row's penalty, `off` where there is none or it makes no sense.
B200_DEVICE float penalty(const float *p, int64_t row, float off, bool positive, int32_t *status) {
    if (!p) return off;
    const float x = __ldg(p + row);
    if (fabsf(x) < INFINITY && (!positive || x > 0.f)) return x;
    set_status(status, B200_DEV_BAD_LOGITS);
    return off;
}

// visit(i, load(i)) for i = tid, tid + kAdWalk, ... below n, kAdAtOnce loads at once.
template <typename Load, typename Visit>
B200_DEVICE void batches(int n, int tid, Load load, Visit visit) {
    for (int i0 = tid; i0 < n; i0 += kAdAtOnce * kAdWalk) {
        decltype(load(0)) x[kAdAtOnce] = {};
#pragma unroll
        for (int j = 0; j < kAdAtOnce; ++j)
            if (i0 + j * kAdWalk < n) x[j] = load(i0 + j * kAdWalk);
#pragma unroll
        for (int j = 0; j < kAdAtOnce; ++j)
            if (i0 + j * kAdWalk < n) visit(i0 + j * kAdWalk, x[j]);
    }
}

// Which of the 32 tokens from t on may be drawn, as bits.
B200_DEVICE uint32_t allowed_bits(const uint32_t *mask, int t, int vocab) {
    if (!mask || t >= vocab) return ~0u;
    const int at = max(t, 0), w = at >> 5;
    const uint32_t lo = __ldg(mask + w), hi = (at & 31) && w < (vocab - 1) >> 5 ? __ldg(mask + w + 1) : 0u;
    return __funnelshift_r(lo, hi, at & 31) << (at - t);
}

// steps: the chunk is so many stages of the ring.
template <typename T>
__global__ void __launch_bounds__(kAdThreads, kAdCtas) adjust_logits_kernel(const __grid_constant__ AdjustArgs a, const int steps) {
    constexpr int V = 16 / sizeof(T), kStep = kAdStep, kWords = kAdChunk / 32, kPer = kWords / kAdWalk;
    static_assert(kPer == 4 && kAdChunk % kStep == 0, "four words a thread that walks, whole steps");
    __shared__ __align__(16) uint32_t named[kWords];  // bit t % 32 of word t / 32: token begin + t is named
    __shared__ __align__(8) uint16_t before[kWords];  // named tokens before the word
    __shared__ uint32_t known[kAdSlots], bias[kAdSlots];
    __shared__ uint16_t token[kAdSlots];
    __shared__ int warp_sums[kAdWalk / 32], total;
    extern __shared__ __align__(16) unsigned char ad_ring[];
    T(*ring)[kStep] = reinterpret_cast<T(*)[kStep]>(ad_ring);
    __shared__ uint64_t landed[kAdStages];
    const int64_t row = blockIdx.x;
    const T *in = static_cast<const T *>(a.in) + row * a.in_row;
    T *out = static_cast<T *>(a.out) + row * a.out_row;
    // The chunk begins where its vectors are aligned in `in`, up to V - 1 elements before a multiple of its size. (The last
    // chunk's end is the row's: chunks * steps * kStep >= vocab + V - 1.)
    const int skew = static_cast<int>(reinterpret_cast<uintptr_t>(in) / sizeof(T) % V);
    const int begin = static_cast<int>(blockIdx.y) * steps * kStep - skew;
    const uint32_t *mask = a.mask ? a.mask + row * a.mask_row : nullptr;
    const bool walks = threadIdx.x >= kAdPass;
    const int tid = walks ? threadIdx.x - kAdPass : threadIdx.x, lane = tid & 31;

    // The lists, and a slot a token that they name: the first kAdSlots, the others later. Threads that walk only.
    int64_t bias_from = 0;
    const int32_t *tokens = nullptr, *biases = nullptr;
    int n = 0, m = 0, prompt = 0;
    // (a last chunk that only another alignment needs begins behind the row: its span is nothing)
    const uint32_t least = static_cast<uint32_t>(max(begin, 0));
    const uint32_t span = static_cast<uint32_t>(max(0, min(begin + steps * kStep, a.vocab) - max(begin, 0)));
    const auto in_chunk = [&](int t) { return static_cast<uint32_t>(t) - least < span; };
    const auto count = [&](int first) {
        for (int i = tid; i < min(total - first, kAdSlots); i += kAdWalk) known[i] = bias[i] = 0;
        named_sync(1, kAdWalk);
        const auto slot_of = [&](int t) {  // kAdSlots and more: none
            if (!in_chunk(t)) return ~0u;
            const uint32_t at = static_cast<uint32_t>(t - begin), w = at >> 5;
            const uint32_t slot = before[w] + __popc(named[w] & ((1u << (at & 31)) - 1u)) - static_cast<uint32_t>(first);
            if (slot < kAdSlots) token[slot] = static_cast<uint16_t>(at);
            return slot;
        };
        batches(n, tid, [&](int i) { return __ldg(tokens + i); }, [&](int i, int t) {
            const uint32_t slot = slot_of(t);
            if (slot >= kAdSlots) return;
            atomicOr(known + slot, kKnown);
            if (i >= prompt) atomicAdd(known + slot, 1u);
        });
        batches(m, tid, [&](int i) { return __ldg(biases + i); }, [&](int i, int t) {
            const uint32_t slot = slot_of(t);
            if (slot < kAdSlots) atomicMax(bias + slot, static_cast<uint32_t>(i + 1));  // of several the last
        });
    };
    if (!walks && (mask || a.in != a.out)) {  // (in place, only a mask needs the pass)
        const bool wide = static_cast<int>(reinterpret_cast<uintptr_t>(out) / sizeof(T) % V) == skew;
        // whole vectors of the row, [vlo, vhi), go through the ring; its first and last tokens one by one
        const int vlo = skew ? V - skew : 0, vhi = vlo + max(0, a.vocab - vlo) / V * V;
        if (tid < 2 * V) {
            const int t = tid < V ? tid : vhi + tid - V;
            if (t < (tid < V ? min(vlo, a.vocab) : a.vocab) && t >= begin && t < begin + steps * kStep)
                out[t] = allowed_bits(mask, t, a.vocab) & 1u ? in[t] : from_f32<T>(-INFINITY);
        }
        // a stage's vectors
        const auto first_of = [&](int step) { return max(begin + step * kStep, vlo); };
        const auto count_of = [&](int step) { return max(0, min(begin + (step + 1) * kStep, vhi) - first_of(step)); };
        const auto stage_of = [&](int step) { return ring[step % kAdStages] + (first_of(step) - begin - step * kStep); };
        const auto fill = [&](int step) {  // by one thread
            const uint32_t bytes = static_cast<uint32_t>(count_of(step)) * static_cast<uint32_t>(sizeof(T));
            mbar_arrive_expect_tx(&landed[step % kAdStages], bytes);
            if (bytes) bulk_g2s(stage_of(step), in + first_of(step), bytes, &landed[step % kAdStages], policy_evict_first());
        };
        if (tid == 0) {
            for (int i = 0; i < kAdStages; ++i) mbar_init(&landed[i], 1);
            fence_barrier_init();
            for (int i = 0; i < min(kAdStages - 1, steps); ++i) fill(i);
        }
        named_sync(2, kAdPass);
        uint32_t allowed = allowed_bits(mask, begin + 32 * tid, a.vocab);
        for (int step = 0; step < steps; ++step) {
            const uint32_t next = step + 1 < steps ? allowed_bits(mask, begin + (step + 1) * kStep + 32 * tid, a.vocab) : ~0u;
            if (!wait_poll(&landed[step % kAdStages], (step / kAdStages) & 1, nullptr)) set_status(a.status, B200_DEV_TIMEOUT);
            if (allowed != ~0u) {
                constexpr int NV = 32 / V;
                T *mine = ring[step % kAdStages] + 32 * tid;
                const int turn = sizeof(T) == 4 ? lane : lane >> 1;  // lanes at different vectors: no two at one bank
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const int v = (j + turn) % NV;
                    const uint32_t bits = allowed >> (v * V);
                    uint4 *at = reinterpret_cast<uint4 *>(mine + v * V), y = *at;
                    T *e = reinterpret_cast<T *>(&y);
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        if (!(bits >> i & 1u)) e[i] = from_f32<T>(-INFINITY);
                    *at = y;
                }
            }
            allowed = next;
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            named_sync(2, kAdPass);  // the stage is as it is to be written
            if (!wide) {
                const T *stage = stage_of(step);
                for (int i = tid; i < count_of(step); i += kAdPass) out[first_of(step) + i] = stage[i];
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                named_sync(2, kAdPass);
            }
            if (tid == 0) {
                const uint32_t bytes = static_cast<uint32_t>(count_of(step)) * static_cast<uint32_t>(sizeof(T));
                if (wide && bytes)
                    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(out + first_of(step)),
                                 "r"(smem_addr(stage_of(step))), "r"(bytes)
                                 : "memory");
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                // the stage filled next is the one written a step ago
                asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
                if (step + kAdStages - 1 < steps) fill(step + kAdStages - 1);
            }
        }
        // the chunk is written, for whoever changes tokens of it
        if (tid == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    } else if (walks) {
        int64_t from = 0, to = 0, bias_to = 0;
        // (offsets are looked at where the lists hold nothing too)
        if (a.cu_tokens) list_range(a.cu_tokens, row, a.n_tokens, a.status, from, to);
        if (a.tokens && a.prompt_lens) prompt = max(0, __ldg(a.prompt_lens + row));
        if (a.cu_bias) list_range(a.cu_bias, row, a.n_biases, a.status, bias_from, bias_to);
        tokens = a.tokens + from, biases = a.bias_ids + bias_from;
        n = static_cast<int>(to - from), m = static_cast<int>(bias_to - bias_from);
        *reinterpret_cast<uint4 *>(named + kPer * tid) = make_uint4(0, 0, 0, 0);
        named_sync(1, kAdWalk);
        bool odd = false;  // an id that names no token (the first chunk's CTA reports it)
        const auto mark = [&](int, int t) {
            const uint32_t at = static_cast<uint32_t>(t - begin);
            if (in_chunk(t)) atomicOr(named + (at >> 5), 1u << (at & 31));
            odd |= static_cast<uint32_t>(t) >= static_cast<uint32_t>(a.vocab);
        };
        batches(n, tid, [&](int i) { return __ldg(tokens + i); }, mark);
        batches(m, tid, [&](int i) { return __ldg(biases + i); }, mark);
        if (odd && blockIdx.y == 0) set_status(a.status, B200_DEV_BAD_TOKEN);
        named_sync(1, kAdWalk);
        const uint4 w4 = *reinterpret_cast<const uint4 *>(named + kPer * tid);
        const int c0 = __popc(w4.x), c1 = c0 + __popc(w4.y), c2 = c1 + __popc(w4.z), own = c2 + __popc(w4.w);
        int up_to = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, up_to, o);
            if (lane >= o) up_to += y;
        }
        if (lane == 31) warp_sums[tid >> 5] = up_to;
        named_sync(1, kAdWalk);
        int base = up_to - own, sum = 0;
#pragma unroll
        for (int w = 0; w < kAdWalk / 32; ++w) {
            if (w < tid >> 5) base += warp_sums[w];
            sum += warp_sums[w];
        }
        *reinterpret_cast<ushort4 *>(before + kPer * tid) = make_ushort4(base, base + c0, base + c1, base + c2);
        if (tid == 0) total = sum;
        named_sync(1, kAdWalk);
        if (sum > 0) count(0);
    }
    __syncthreads();  // the slots are counted, and the pass has written their tokens
    if (total == 0 && (blockIdx.y || threadIdx.x)) return;
    // (the first chunk's CTA looks at the row's penalties where it has no token for them too)
    const float rep = penalty(a.repetition, row, 1.f, true, a.status);
    const float freq = penalty(a.frequency, row, 0.f, false, a.status);
    const float pres = penalty(a.presence, row, 0.f, false, a.status);
    if (total == 0) return;
    const float *bias_values = a.bias_ids ? a.bias_values + __ldg(a.cu_bias + row) : nullptr;
    for (int first = 0;;) {
        for (int i = threadIdx.x; i < min(total - first, kAdSlots); i += kAdThreads) {
            const int t = begin + token[i];
            const uint32_t u = known[i], drawn = u & ~kKnown, b = bias[i];
            if (mask && !(__ldg(mask + (t >> 5)) >> (t & 31) & 1u)) continue;
            float y = to_f32<T>(in[t]);  // in place: still what it was
            if (u) y = y > 0.f ? y / rep : y * rep;
            if (drawn) y = y - freq * static_cast<float>(drawn) - pres;
            if (b) y += __ldg(bias_values + (b - 1));
            out[t] = from_f32<T>(y);
        }
        first += kAdSlots;
        if (first >= total) return;
        __syncthreads();  // the slots are free again
        if (walks) count(first);
        __syncthreads();
    }
}

template <typename T>
cudaError_t adjust_launch(const AdjustArgs &a, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    int steps = kAdChunk / kAdStep;
    const auto chunks = [&] { return (a.vocab + V - 1 + steps * kAdStep - 1) / (steps * kAdStep); };
    while (steps > 1 && a.n_rows * chunks() < kAdCtas * device_sm_count()) steps /= 2;  // fewer CTAs than run at once
    if (a.n_rows > INT32_MAX) return cudaErrorNotSupported;
    auto kern = adjust_logits_kernel<T>;
    constexpr int kRing = kAdStages * kAdStep * static_cast<int>(sizeof(T));
    const cudaError_t e = once_per_device(reinterpret_cast<const void *>(kern), ATTR_SMEM, [&] {
        return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kRing);
    });
    if (e != cudaSuccess) return e;
    const dim3 grid(static_cast<unsigned>(a.n_rows), static_cast<unsigned>(chunks()));  // y <= 2^9 + 1
    return b200_launch(kern, grid, dim3(kAdThreads), kRing, st, false, a, steps);
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
