// b200_sample: temperature, top-k, top-p and min-p sampling of one token per row of
// logits from given uniform numbers.
//
// Token weights are whole numbers, w_i = floor(2^40 exp((x_i - max) / T)), so sums need no
// order and the answer does not depend on the split. The kept set of top-k and top-p is a
// head of the tokens ordered by (logit descending, index ascending), so it is described by
// a threshold: every logit above K, and the first r (by index) of those equal to K. Nothing
// is sorted: K is found by counting.
//
//  * A row belongs to one cluster of C CTAs, each with a contiguous chunk of the vocabulary
//    kept in its shared memory, so the logits are read from HBM once. The CTAs exchange
//    maxima, histograms and sums through distributed shared memory; no workspace.
//  * Threshold: one histogram (count and weight) of the chunk over bins of equal width in
//    (x - max) / T, merged over the cluster, gives the bin in which the k-th token, or the
//    token that completes the nucleus, lies. Tokens below e^-28 of the likeliest have weight
//    0 and are left out everywhere. The bin's tokens (at most kList, else the bin is split
//    again over its ordered bit patterns) are gathered and ranked by comparison.
//  * Draw: every warp sums the kept weights of its contiguous piece; a scan over the pieces
//    names the one in which the drawn sum lies, and its warp walks it.
// Bound: one read of the logits for a large batch; for a few rows the chain of about six
// cluster exchanges.
#include "batch.cuh"
#include "gemv.cuh"

namespace b200 {
namespace {

constexpr int kSmThreads = 512;
constexpr int kSmWarps = kSmThreads / 32;
constexpr int kBins = 512;   // one a thread
constexpr int kList = 512;   // tokens ranked directly, one a thread
constexpr int kMaxCluster = 8;
constexpr float kFloor = -28.0f;  // 2^40 e^-28 < 1
static_assert(kBins == kSmThreads && kList == kSmThreads, "one bin and one listed token a thread");

struct SampleArgs {
    const void *logits;
    int64_t row_stride;
    const float *u, *temperature, *top_p, *min_p;
    const int32_t *top_k;
    int32_t *out;
    int32_t *status;
    int32_t vocab, chunk, cluster;  // chunk: tokens a CTA takes
};

// Shared memory read by the other CTAs of the cluster, and this CTA's own.
struct SampleShared {
    // exchanged
    uint32_t cnt[kBins];
    unsigned long long wgt[kBins];
    uint32_t list[kList];
    unsigned long long piece_w[kSmWarps];  // kept weight above K, a warp's piece
    uint32_t piece_eq[kSmWarps];           // tokens equal to K
    float top;
    uint32_t listed, bad;
    // own
    uint32_t mcnt[kBins], lcnt[kBins];     // merged: first histogram, later ones
    unsigned long long mwgt[kBins], lwgt[kBins];
    uint32_t akey[kList];
    unsigned long long awgt[kList];
    uint32_t warp_c[kSmWarps];
    unsigned long long warp_w[kSmWarps];
    float warp_f[kSmWarps];
    uint32_t warp_b[kSmWarps];
    int32_t bin;
    uint32_t bin_c, key, ties;
    unsigned long long above_c, above_w, sum;
};

B200_DEVICE uint32_t ld_dsmem_u32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
B200_DEVICE unsigned long long ld_dsmem_u64(uint32_t addr) {
    unsigned long long v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
    return v;
}
B200_DEVICE uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

// Bit pattern of x in an order that follows the values (x is no NaN; -0 was made +0).
B200_DEVICE uint32_t order_key(float x) {
    const uint32_t u = __float_as_uint(x);
    return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
B200_DEVICE float key_value(uint32_t k) {
    return __uint_as_float((k >> 31) ? k ^ 0x80000000u : ~k);
}

struct Scale {
    float top, inv_t;
    B200_DEVICE float z(float x) const { return (x - top) * inv_t; }
    B200_DEVICE unsigned long long weight(float x) const {
        const float y = z(x);
        return y > kFloor ? __float2ull_rz(expf(y) * 1099511627776.0f) : 0ull;
    }
    B200_DEVICE int bin(float zz) const { return min(static_cast<int>(zz * (-kBins / -kFloor)), kBins - 1); }
};

template <typename T, bool HELD>
struct Chunk {
    const T *held;    // shared memory (HELD) or the row's chunk in global memory
    int n;
    B200_DEVICE float operator[](int i) const {
        if constexpr (HELD) return to_f32<T>(held[i]) + 0.0f;
        else return to_f32<T>(__ldg(held + i)) + 0.0f;
    }
};

template <typename T, bool HELD>
struct Sampler {
    const SampleArgs &a;
    SampleShared &s;
    Chunk<T, HELD> x;
    Scale sc;
    int tid, warp, lane;
    uint32_t rank, nc;

    // Merges the cluster's histograms into mc / mw (bin `tid` by each thread). The caller
    // has passed a cluster barrier since they were filled.
    B200_DEVICE void merge(uint32_t *mc, unsigned long long *mw) {
        uint32_t c = 0;
        unsigned long long w = 0;
        for (uint32_t r = 0; r < nc; ++r) {
            c += ld_dsmem_u32(dsmem_addr(&s.cnt[tid], r));
            w += ld_dsmem_u64(dsmem_addr(&s.wgt[tid], r));
        }
        mc[tid] = c;
        mw[tid] = w;
    }

    // The bin in which the running measure (count or weight) reaches `target`, given what
    // lies above the bins; s.bin = -1 if it does not. Leaves s.above_*, s.bin_c.
    B200_DEVICE void find(const uint32_t *mc, const unsigned long long *mw, unsigned long long above_c,
                          unsigned long long above_w, unsigned long long target, bool by_weight) {
        const uint32_t c = mc[tid];
        const unsigned long long w = mw[tid];
        uint32_t ic = c;
        unsigned long long iw = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t yc = __shfl_up_sync(0xffffffffu, ic, o);
            const unsigned long long yw = __shfl_up_sync(0xffffffffu, iw, o);
            if (lane >= o) ic += yc, iw += yw;
        }
        if (lane == 31) s.warp_c[warp] = ic, s.warp_w[warp] = iw;
        if (tid == 0) s.bin = -1;
        __syncthreads();
        unsigned long long pc = above_c, pw = above_w;
        for (int i = 0; i < warp; ++i) pc += s.warp_c[i], pw += s.warp_w[i];
        pc += ic - c;
        pw += iw - w;
        const unsigned long long lo = by_weight ? pw : pc, hi = by_weight ? pw + w : pc + c;
        if (lo < target && target <= hi) {
            s.bin = tid;
            s.bin_c = c;
            s.above_c = pc;
            s.above_w = pw;
        }
        __syncthreads();
    }

    B200_DEVICE void clear_histogram() {
        s.cnt[tid] = 0;
        s.wgt[tid] = 0;
        __syncthreads();
    }

    // Finds K and r for `target` (a count of tokens, or a sum of weights) from the merged
    // first histogram: s.key, s.ties, and s.sum, the weight of the head they describe.
    // Every CTA of the cluster takes the same path. False: the whole row is kept.
    B200_DEVICE bool select(unsigned long long target, bool by_weight) {
        find(s.mcnt, s.mwgt, 0, 0, target, by_weight);
        const int bin0 = s.bin;
        if (bin0 < 0) return false;
        uint32_t lo = 0, hi = order_key(sc.top);
        uint32_t n = s.bin_c;
        unsigned long long ac = s.above_c, aw = s.above_w;
        const auto member = [&](float v, uint32_t key) {
            const float z = sc.z(v);
            return z > kFloor && sc.bin(z) == bin0 && key >= lo && key <= hi;
        };
        while (n > kList && lo < hi) {  // split the bin over its bit patterns, descending
            const int shift = max(0, 32 - __clz(static_cast<int>(hi - lo)) - 9);
            cluster_sync();  // nobody reads the histogram any more
            clear_histogram();
            for (int i = tid; i < x.n; i += kSmThreads) {
                const float v = x[i];
                const uint32_t key = order_key(v);
                if (member(v, key)) {
                    atomicAdd(&s.cnt[(hi - key) >> shift], 1u);
                    atomicAdd(&s.wgt[(hi - key) >> shift], sc.weight(v));
                }
            }
            cluster_sync();
            merge(s.lcnt, s.lwgt);
            __syncthreads();
            find(s.lcnt, s.lwgt, ac, aw, target, by_weight);
            const uint32_t off = static_cast<uint32_t>(s.bin) << shift;
            hi -= off;
            const uint32_t width = (1u << shift) - 1u;
            lo = hi - lo > width ? hi - width : lo;
            n = s.bin_c;
            ac = s.above_c;
            aw = s.above_w;
            __syncthreads();
        }
        if (n > kList) {  // one bit pattern is left
            if (tid == 0) settle(lo, ac, aw, target, by_weight);
            __syncthreads();
            return true;
        }
        if (tid == 0) s.listed = 0;
        __syncthreads();
        for (int i = tid; i < x.n; i += kSmThreads) {
            const float v = x[i];
            const uint32_t key = order_key(v);
            if (member(v, key)) s.list[atomicAdd(&s.listed, 1u)] = key;
        }
        cluster_sync();
        uint32_t base = 0;
        for (uint32_t r = 0; r < nc; ++r) {
            const uint32_t m = ld_dsmem_u32(dsmem_addr(&s.listed, r));
            if (tid < static_cast<int>(m)) s.akey[base + tid] = ld_dsmem_u32(dsmem_addr(&s.list[tid], r));
            base += m;
        }
        cluster_sync();  // the lists may be written again
        if (tid < static_cast<int>(n)) s.awgt[tid] = sc.weight(key_value(s.akey[tid]));
        __syncthreads();
        if (tid < static_cast<int>(n)) {
            const uint32_t mine = s.akey[tid];
            unsigned long long c = ac, w = aw, eq = 0;
            for (uint32_t j = 0; j < n; ++j) {
                const uint32_t k = s.akey[j];
                if (k > mine) c += 1, w += s.awgt[j];
                eq += k == mine;
            }
            const unsigned long long below = by_weight ? w : c;
            if (below < target && target <= below + (by_weight ? eq * s.awgt[tid] : eq))
                settle(mine, c, w, target, by_weight);  // equal tokens write the same values
        }
        __syncthreads();
        return true;
    }

    B200_DEVICE void settle(uint32_t key, unsigned long long c, unsigned long long w, unsigned long long target,
                            bool by_weight) {
        const unsigned long long each = sc.weight(key_value(key));
        const unsigned long long r = by_weight ? (target - w + each - 1) / each : target - c;
        s.key = key;
        s.ties = static_cast<uint32_t>(r);
        s.sum = w + r * each;
    }
};

template <typename T, bool HELD>
__global__ void __launch_bounds__(kSmThreads, 2) sample_kernel(const SampleArgs a) {
    extern __shared__ __align__(16) unsigned char sm_raw[];
    SampleShared &s = *reinterpret_cast<SampleShared *>(sm_raw);
    T *held = reinterpret_cast<T *>(sm_raw + (sizeof(SampleShared) + 15) / 16 * 16);
    const uint32_t nc = a.cluster, rank = nc > 1 ? cluster_rank() : 0;
    const int64_t row = blockIdx.x / nc;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t begin = static_cast<int64_t>(rank) * a.chunk;
    const int n = static_cast<int>(max64(0, min64(a.chunk, a.vocab - begin)));
    const T *src = static_cast<const T *>(a.logits) + row * a.row_stride + begin;

    // the chunk, its maximum, and whether it has a NaN or +inf
    float mx = -INFINITY;
    bool bad = false;
    const auto take = [&](T v) {
        const float f = to_f32<T>(v);
        bad |= !(f < INFINITY);
        mx = fmaxf(mx, f);
    };
    constexpr int V = 16 / sizeof(T);
    const bool vec = (reinterpret_cast<uintptr_t>(src) & 15) == 0;
    const int n4 = vec ? n / V : 0;
    for (int i0 = tid; i0 < n4; i0 += 4 * kSmThreads) {
        uint4 r[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i0 + j * kSmThreads < n4) r[j] = __ldg(reinterpret_cast<const uint4 *>(src) + i0 + j * kSmThreads);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i0 + j * kSmThreads < n4) {
                if constexpr (HELD) reinterpret_cast<uint4 *>(held)[i0 + j * kSmThreads] = r[j];
                const T *e = reinterpret_cast<const T *>(&r[j]);
#pragma unroll
                for (int q = 0; q < V; ++q) take(e[q]);
            }
    }
    for (int i = n4 * V + tid; i < n; i += kSmThreads) {
        const T v = __ldg(src + i);
        if constexpr (HELD) held[i] = v;
        take(v);
    }
    const float temp = __ldg(a.temperature + row);
    const float u = __ldg(a.u + row);
    const int32_t top_k = a.top_k ? __ldg(a.top_k + row) : 0;
    const float top_p = a.top_p ? __ldg(a.top_p + row) : 1.0f;
    const float min_p = a.min_p ? __ldg(a.min_p + row) : 0.0f;
    bad |= temp != temp || u != u || top_p != top_p || min_p != min_p;
    mx = warp_max(mx);
    bad = __any_sync(0xffffffffu, bad);
    if (lane == 0) s.warp_f[warp] = mx, s.warp_b[warp] = bad;
    s.cnt[tid] = 0;
    s.wgt[tid] = 0;
    __syncthreads();
    if (warp == 0) {
        mx = warp_max(lane < kSmWarps ? s.warp_f[lane] : -INFINITY);
        bad = __any_sync(0xffffffffu, lane < kSmWarps && s.warp_b[lane]);
        if (lane == 0) s.top = mx, s.bad = bad;
    }
    cluster_sync();
    mx = -INFINITY;
    bad = false;
    for (uint32_t r = 0; r < nc; ++r) {
        mx = fmaxf(mx, ld_dsmem(dsmem_addr(&s.top, r)));
        bad |= ld_dsmem_u32(dsmem_addr(&s.bad, r)) != 0;
    }
    if (bad || mx == -INFINITY) {
        if (rank == 0 && tid == 0) {
            a.out[row] = -1;
            set_status(a.status, B200_DEV_BAD_LOGITS);
        }
        cluster_sync();
        return;
    }
    const float inv = 1.0f / temp;
    const bool cold = !(temp > 0.f) || inv == INFINITY;
    Sampler<T, HELD> f{a, s, {HELD ? held : src, n}, {mx + 0.0f, cold ? 1.0f : inv}, tid, warp, lane, rank, nc};

    // the kept head: keys above `key`, and the first `ties` equal to it
    uint32_t key = 0, ties = 0;
    if (cold) {
        key = order_key(mx + 0.0f);
        ties = 1;
    } else if (top_k > 0 && top_k < a.vocab || top_p < 1.0f) {
        for (int i = tid; i < n; i += kSmThreads) {
            const float v = f.x[i], z = f.sc.z(v);
            if (z > kFloor) {
                const int b = f.sc.bin(z);
                atomicAdd(&s.cnt[b], 1u);
                atomicAdd(&s.wgt[b], f.sc.weight(v));
            }
        }
        cluster_sync();
        f.merge(s.mcnt, s.mwgt);
        __syncthreads();
        unsigned long long sum = 0;
        bool cut = false;
        if (top_k > 0) cut = f.select(static_cast<unsigned long long>(top_k), false);
        if (cut) {
            key = s.key, ties = s.ties, sum = s.sum;
        } else {
            for (int i = lane; i < kBins; i += 32) sum += s.mwgt[i];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
        __syncthreads();
        if (top_p < 1.0f) {
            const double want = static_cast<double>(top_p) * static_cast<double>(sum);
            const unsigned long long target = want >= 1.0 ? static_cast<unsigned long long>(want) : 1ull;
            if (f.select(target, true)) key = s.key, ties = s.ties;
        }
    }
    const double floor_p = static_cast<double>(fminf(fmaxf(min_p, 0.0f), 1.0f)) * 1099511627776.0;
    const unsigned long long least = static_cast<unsigned long long>(floor_p);

    // kept weight of each warp's contiguous piece
    const int piece = (a.chunk / kSmWarps + 31) / 32 * 32;
    const int p0 = warp * piece, p1 = min(n, p0 + piece);
    unsigned long long pw = 0;
    uint32_t pe = 0;
    for (int i = p0 + lane; i < p1; i += 32) {
        const float v = f.x[i];
        const uint32_t k = order_key(v);
        if (k > key) {
            const unsigned long long w = f.sc.weight(v);
            if (w >= least) pw += w;
        } else if (k == key) {
            ++pe;
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        pw += __shfl_xor_sync(0xffffffffu, pw, o);
        pe += __shfl_xor_sync(0xffffffffu, pe, o);
    }
    if (lane == 0) s.piece_w[warp] = pw, s.piece_eq[warp] = pe;
    cluster_sync();
    // every warp scans all pieces of the cluster (lane: pieces lane, lane + 32, ... in order)
    unsigned long long each = ties ? f.sc.weight(key_value(key)) : 0ull;
    if (each < least) each = 0;
    const int pieces = static_cast<int>(nc) * kSmWarps;
    unsigned long long total = 0, before = 0;  // before: kept weight ahead of this warp's piece
    uint32_t eq_total = 0, eq_before = 0;
    const int mine = static_cast<int>(rank) * kSmWarps + warp;
    for (int i0 = 0; i0 < pieces; i0 += 32) {
        const int i = i0 + lane;
        unsigned long long w = 0;
        uint32_t e = 0;
        if (i < pieces) {
            w = ld_dsmem_u64(dsmem_addr(&s.piece_w[i % kSmWarps], i / kSmWarps));
            e = ld_dsmem_u32(dsmem_addr(&s.piece_eq[i % kSmWarps], i / kSmWarps));
        }
        uint32_t ie = e;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, ie, o);
            if (lane >= o) ie += y;
        }
        const uint32_t eb = eq_total + ie - e;  // equal tokens ahead of piece i
        const uint32_t kept = eb < ties ? min(e, ties - eb) : 0u;
        unsigned long long iw = w + kept * each;
        const unsigned long long own = iw;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long y = __shfl_up_sync(0xffffffffu, iw, o);
            if (lane >= o) iw += y;
        }
        if (mine >= i0 && mine < i0 + 32) {
            before = total + __shfl_sync(0xffffffffu, iw - own, mine - i0);
            eq_before = __shfl_sync(0xffffffffu, eb, mine - i0);
        }
        total += __shfl_sync(0xffffffffu, iw, 31);
        eq_total += __shfl_sync(0xffffffffu, ie, 31);
    }
    const double want = static_cast<double>(u) * static_cast<double>(total);
    unsigned long long at = want > 0.0 ? static_cast<unsigned long long>(want) : 0ull;
    if (want >= static_cast<double>(total) || at >= total) at = total - 1;
    // the warp whose piece holds the drawn sum walks it
    const uint32_t my_kept = eq_before < ties ? min(pe, ties - eq_before) : 0u;
    if (at >= before && at < before + pw + my_kept * each) {
        unsigned long long run = before;
        uint32_t eq = eq_before;
        for (int i0 = p0; i0 < p1; i0 += 32) {
            const int i = i0 + lane;
            unsigned long long w = 0;
            bool same = false;
            if (i < p1) {
                const float v = f.x[i];
                const uint32_t k = order_key(v);
                same = k == key;
                if (k > key) {
                    w = f.sc.weight(v);
                    if (w < least) w = 0;
                }
            }
            const uint32_t sm = __ballot_sync(0xffffffffu, same);
            if (same && eq + __popc(sm & ((1u << lane) - 1u)) < ties) w = each;
            eq += __popc(sm);
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned long long y = __shfl_up_sync(0xffffffffu, w, o);
                if (lane >= o) w += y;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, run + w > at);
            if (hit) {
                if (lane == 0) a.out[row] = static_cast<int32_t>(begin + i0 + __ffs(hit) - 1);
                break;
            }
            run += __shfl_sync(0xffffffffu, w, 31);
        }
    }
    cluster_sync();  // no CTA's shared memory goes away while it is read
}

constexpr size_t kOwnBytes = (sizeof(SampleShared) + 15) / 16 * 16;
constexpr size_t kMostShared = 227 * 1024;
constexpr size_t kHalfShared = 113 * 1024;  // two CTAs an SM: 228 KB less 1 KB for each

template <typename T, bool HELD>
cudaError_t sample_launch_as(const SampleArgs &a, int64_t rows, cudaStream_t st) {
    auto kern = sample_kernel<T, HELD>;
    cudaError_t e = once_per_device(reinterpret_cast<const void *>(kern), ATTR_SMEM, [&] {
        return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kMostShared));
    });
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(rows * a.cluster));
    cfg.blockDim = dim3(kSmThreads);
    cfg.dynamicSmemBytes = kOwnBytes + (HELD ? static_cast<size_t>(a.chunk) * sizeof(T) : 0);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(a.cluster);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, a);
}

template <typename T>
cudaError_t sample_launch(SampleArgs a, int64_t rows, cudaStream_t st) {
    // CTAs a row: about 2,048 tokens each while a row's CTAs are fewer than the SMs; more
    // rows take fewer, as far as two chunks still fit an SM
    const int64_t sms = device_sm_count();
    int c = 1;
    while (c < kMaxCluster && a.vocab > 2048 * c && rows * c < sms) c *= 2;
    while (c < kMaxCluster && kOwnBytes + (a.vocab + c - 1) / c * sizeof(T) > kHalfShared) c *= 2;
    a.cluster = c;
    a.chunk = static_cast<int32_t>(((a.vocab + c - 1) / c + 63) / 64 * 64);
    if (kOwnBytes + static_cast<size_t>(a.chunk) * sizeof(T) <= kMostShared) return sample_launch_as<T, true>(a, rows, st);
    return sample_launch_as<T, false>(a, rows, st);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200_sample(const void *logits, int64_t row_stride, int64_t n_rows, int64_t n_vocab, int32_t dtype,
                           const float *u, const float *temperature, const int32_t *top_k, const float *top_p,
                           const float *min_p, int32_t *out_ids, int32_t *dev_status, void *stream) {
    if (n_rows < 0 || n_vocab <= 0 || row_stride < 0 || !dtype_bytes(dtype)) return B200_ERR_INVALID_ARGUMENT;
    if (n_rows == 0) return B200_OK;
    if (!logits || !u || !temperature || !out_ids) return B200_ERR_INVALID_ARGUMENT;
    if (n_vocab > (1 << 21) || n_rows > INT32_MAX / kMaxCluster) return B200_ERR_NOT_SUPPORTED;
    SampleArgs a = {};
    a.logits = logits;
    a.row_stride = row_stride;
    a.u = u;
    a.temperature = temperature;
    a.top_p = top_p;
    a.min_p = min_p;
    a.top_k = top_k;
    a.out = out_ids;
    a.status = dev_status;
    a.vocab = static_cast<int32_t>(n_vocab);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case B200_DTYPE_F16: return status_of(sample_launch<__half>(a, n_rows, st));
        case B200_DTYPE_BF16: return status_of(sample_launch<__nv_bfloat16>(a, n_rows, st));
    }
    return status_of(sample_launch<float>(a, n_rows, st));
}
