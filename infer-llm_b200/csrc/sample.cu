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
//    kept in its shared memory, so the logits are read from HBM once; where many rows would queue for
//    that room, or one has none, the passes read the chunk from L2. The CTAs exchange maxima,
//    histograms and sums through distributed shared memory; no workspace.
//  * A histogram over bins of equal width in (x - max) / T, merged over the cluster, gives the bin
//    in which the k-th token, or the token that completes the nucleus, lies. A weight is added as
//    three words of 14 bits: 32-bit shared-memory additions run at full rate, 64-bit ones
//    are compare-and-swap loops (16 us a row). Tokens below e^-28 of the likeliest have
//    weight 0 and are left out everywhere.
//  * If the bins up to it hold at most kList tokens, as for a head of a few hundred, the first
//    CTA gathers them, sorts them and draws among them. For a short top-k the bins of the threads' own
//    largest tokens tell where to stop, and nothing else is counted.
//  * Otherwise the threshold is looked for in its bin alone: its tokens are ranked, or the bin is
//    split again over its ordered bit patterns. Then the kept weight of each warp's
//    contiguous piece is summed, and the CTA in whose chunk the drawn sum lies searches
//    that piece.
// Bound: for a few rows the chain of about four cluster exchanges (151936 F32 logits: 14 to 18 us with one row); for
// a large batch the instructions of the passes, each token's weight (an exponential and a 64-bit
// shift) taking ~44 issue slots a warp, beside those chains. 256 rows of 151936 F32: greedy 55 us (2.8
// TB/s), top-k 50 88, no filter 124, top-p 0.95 168 to 343 as the row is steep or flat, mixed filters 145 to 155.
#include "batch.cuh"
#include "gemv.cuh"

namespace b200 {
namespace {

constexpr int kSmThreads = 512;
constexpr int kSmWarps = kSmThreads / 32;
constexpr int kBins = 512;   // one a thread
constexpr int kList = 512;   // tokens ranked directly, one a thread
constexpr int kMaxCluster = 8;
constexpr int kMostChunk = 1 << 18;  // tokens a CTA takes: so many words of 14 bits sum up within 32
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
    uint32_t cnt[kBins], wgt[3][kBins];  // tokens; their weights in words of 14 bits
    uint32_t list[kList], list_at[kList];
    unsigned long long part;     // kept weight above K
    uint32_t equal;              // tokens equal to K
    float top;
    uint32_t listed, bad;
    // own
    uint32_t mcnt[kBins];             // the first histogram, merged
    unsigned long long mwgt[kBins];
    unsigned long long sorted[kList], awgt[kList];
    uint32_t aat[kList];
    uint32_t warp_c[kSmWarps], piece_eq[kSmWarps];
    unsigned long long warp_w[kSmWarps], piece_w[kSmWarps];
    float warp_f[kSmWarps];
    uint32_t warp_b[kSmWarps];
    int32_t bin;
    uint32_t bin_c, key, ties;
    unsigned long long above_c, above_w, upto_c, sum;
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
    // floor(2^40 e^z) from the bits of the exponential, which is at most 1 (a conversion to 64
    // bits runs at a fraction of the rate of the shifts)
    B200_DEVICE unsigned long long weight(float x) const {
        const float y = z(x);
        if (!(y > kFloor)) return 0ull;
        const uint32_t e = __float_as_uint(expf(y));
        return (static_cast<unsigned long long>((e & 0x7FFFFFu) | 0x800000u) << 17) >> (127u - (e >> 23));
    }
    // A value below every token whose bin is at most b (b = kBins - 1: of any bin), and one above
    // those of bin b on: wide enough for the rounding of z and of the bins' edges. One
    // comparison then rules most tokens out; the exact test takes the rest.
    B200_DEVICE float below(int b) const { return edge(b + 0.75f) - slack(); }
    B200_DEVICE float above(int b) const { return edge(b - 0.75f) + slack(); }
    B200_DEVICE float edge(float b) const { return top + kFloor / kBins / inv_t * b; }
    B200_DEVICE float slack() const { return 1e-5f * (fabsf(top) - kFloor / inv_t); }
    // the bin nearest to kBins z / kFloor (adding 2^23 leaves the whole number in the low bits)
    B200_DEVICE static int bin(float zz) {
        return min(static_cast<int>(__float_as_uint(fmaf(zz, kBins / kFloor, 8388608.0f)) & 0x3FFu), kBins - 1);
    }
};

template <typename T, bool HELD>
struct Chunk {
    const T *held;    // shared memory (HELD) or the row's chunk in global memory
    int n;
    B200_DEVICE float operator[](int i) const {
        if constexpr (HELD) return to_f32<T>(held[i]) + 0.0f;
        else return to_f32<T>(__ldg(held + i)) + 0.0f;
    }
    // fn(value, index) for the tokens [from + 4 lane, ...) below `to` of `lanes` lanes that take
    // four consecutive ones at a time; `from` is a multiple of four
    template <typename F>
    B200_DEVICE void each(int from, int to, int lane, int lanes, F fn) const {
        if constexpr (HELD) {
            const int whole = from + ((to - from) & ~3);
            for (int i = from + 4 * lane; i < whole; i += 4 * lanes) {
                alignas(16) T v[4];
                if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4 *>(v) = *reinterpret_cast<const uint4 *>(held + i);
                else *reinterpret_cast<uint2 *>(v) = *reinterpret_cast<const uint2 *>(held + i);
#pragma unroll
                for (int j = 0; j < 4; ++j) fn(to_f32<T>(v[j]) + 0.0f, i + j);
            }
            if (whole + lane < to) fn((*this)[whole + lane], whole + lane);
        } else {
            // from L2, as a rule: four loads of 16 bytes a thread in flight
            constexpr int V = 16 / sizeof(T);
            const int whole = (reinterpret_cast<uintptr_t>(held) & 15) == 0 ? from + (to - from) / V * V : from;
            for (int i = from + V * lane; i < whole; i += 4 * V * lanes) {
                uint4 r[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (i + j * V * lanes < whole) r[j] = __ldg(reinterpret_cast<const uint4 *>(held + i + j * V * lanes));
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (i + j * V * lanes < whole) {
                        const T *e = reinterpret_cast<const T *>(&r[j]);
#pragma unroll
                        for (int q = 0; q < V; ++q) fn(to_f32<T>(e[q]) + 0.0f, i + j * V * lanes + q);
                    }
            }
#pragma unroll 4
            for (int i = whole + lane; i < to; i += lanes) fn((*this)[i], i);
        }
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

    // Sum of v over the CTA, in every thread. Ends with a barrier.
    B200_DEVICE unsigned long long cta_sum(unsigned long long v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane == 0) s.warp_w[warp] = v;
        __syncthreads();
        unsigned long long t = 0;
#pragma unroll
        for (int w = 0; w < kSmWarps; ++w) t += s.warp_w[w];
        __syncthreads();
        return t;
    }
    // Sum of v over the threads before this one.
    B200_DEVICE unsigned long long cta_before(unsigned long long v) {
        unsigned long long incl = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        if (lane == 31) s.warp_w[warp] = incl;
        __syncthreads();
        unsigned long long t = incl - v;
        for (int w = 0; w < warp; ++w) t += s.warp_w[w];
        __syncthreads();
        return t;
    }
    // Bin `tid` of the cluster's histograms. The caller has passed a cluster barrier since they
    // were filled.
    B200_DEVICE uint32_t merged_count() const {
        uint32_t c = 0;
        for (uint32_t r = 0; r < nc; ++r) c += ld_dsmem_u32(dsmem_addr(&s.cnt[tid], r));
        return c;
    }
    B200_DEVICE unsigned long long merged_weight() const {
        unsigned long long w = 0;
        for (uint32_t r = 0; r < nc; ++r)
#pragma unroll
            for (int i = 0; i < 3; ++i)
                w += static_cast<unsigned long long>(ld_dsmem_u32(dsmem_addr(&s.wgt[i][tid], r))) << (14 * i);
        return w;
    }
    B200_DEVICE void clear_histogram() {
        s.cnt[tid] = 0;
#pragma unroll
        for (int i = 0; i < 3; ++i) s.wgt[i][tid] = 0;
        __syncthreads();
    }
    B200_DEVICE void count(int b) { atomicAdd(&s.cnt[b], 1u); }
    B200_DEVICE void add_weight(int b, unsigned long long w) {
        // a chunk has at most kMostChunk tokens: no word overflows
        if (w & 0x3FFFu) atomicAdd(&s.wgt[0][b], static_cast<uint32_t>(w) & 0x3FFFu);
        atomicAdd(&s.wgt[1][b], static_cast<uint32_t>(w >> 14) & 0x3FFFu);
        if (w >> 28) atomicAdd(&s.wgt[2][b], static_cast<uint32_t>(w >> 28));
    }

    // The bin at which the running count or weight of the bins (bin `tid` holds c tokens of
    // weight w), on top of what is ahead of them, reaches `target`: s.bin (-1 if it does not),
    // s.bin_c, s.above_c and s.above_w (ahead of the bin), s.upto_c (tokens up to it).
    B200_DEVICE void find(uint32_t c, unsigned long long w, unsigned long long ahead_c, unsigned long long ahead_w,
                          unsigned long long target, bool by_weight) {
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
        unsigned long long pc = ahead_c + (ic - c), pw = ahead_w + (iw - w);
        for (int i = 0; i < warp; ++i) pc += s.warp_c[i], pw += s.warp_w[i];
        const unsigned long long lo = by_weight ? pw : pc, hi = by_weight ? pw + w : pc + c;
        if (lo < target && target <= hi) {
            s.bin = tid;
            s.bin_c = c;
            s.above_c = pc;
            s.above_w = pw;
            s.upto_c = pc + c;
        }
        __syncthreads();
    }

    // Appends the tokens that `member(value)` names to this CTA's list; s.listed counts those past
    // its end too.
    template <typename F>
    B200_DEVICE void collect(F member) {
        if (tid == 0) s.listed = 0;
        __syncthreads();
        x.each(0, x.n, tid, kSmThreads, [&](float v, int i) {
            if (member(v)) {
                const uint32_t at = atomicAdd(&s.listed, 1u);
                if (at < kList) {
                    s.list[at] = order_key(v);
                    s.list_at[at] = static_cast<uint32_t>(i);
                }
            }
        });
    }
    // Token `tid` of the cluster's lists, the CTAs' lists in order: its key and index in the
    // vocabulary; returns the lists' length. The caller has passed a cluster barrier since they
    // were filled.
    B200_DEVICE uint32_t fetch_listed(uint32_t &key, uint32_t &at) {
        uint32_t m[kMaxCluster], n = 0, from = 0, r = 0, base = 0;
#pragma unroll
        for (uint32_t i = 0; i < kMaxCluster; ++i) m[i] = i < nc ? ld_dsmem_u32(dsmem_addr(&s.listed, i)) : 0u;
#pragma unroll
        for (uint32_t i = 0; i < kMaxCluster; ++i) {
            if (static_cast<uint32_t>(tid) >= n && static_cast<uint32_t>(tid) < n + m[i]) r = i, from = tid - n, base = i * a.chunk;
            n += m[i];
        }
        key = at = 0;
        if (static_cast<uint32_t>(tid) < n) {
            key = ld_dsmem_u32(dsmem_addr(&s.list[from], r));
            at = ld_dsmem_u32(dsmem_addr(&s.list_at[from], r)) + base;
        }
        return n;
    }

    // Appends the tokens of bins 0 to `last`, and returns the lists' length. Ends with a cluster barrier.
    B200_DEVICE uint32_t collect_bins(int last) {
        const float low = sc.below(last);
        collect([&](float v) {
            if (v < low) return false;
            const float z = sc.z(v);
            return z > kFloor && Scale::bin(z) <= last;
        });
        cluster_sync();
        uint32_t n = 0;
        for (uint32_t r = 0; r < nc; ++r) n += ld_dsmem_u32(dsmem_addr(&s.listed, r));
        return n;
    }

    // Sorts the first n threads' values, descending; the others' are 0 (bitonic; exchanges
    // within a warp by shuffles, across warps through s.sorted).
    B200_DEVICE unsigned long long sort_descending(unsigned long long v, uint32_t n) {
        const int size = n <= 32 ? 32 : 1 << (32 - __clz(static_cast<int>(n - 1)));
#pragma unroll 1
        for (int k = 2; k <= size; k <<= 1) {
#pragma unroll 1
            for (int j = k >> 1; j > 0; j >>= 1) {
                unsigned long long o = 0;
                if (j >= 32) {
                    __syncthreads();
                    s.sorted[tid] = v;
                    __syncthreads();
                    o = s.sorted[tid ^ j];
                } else if (tid < size) {
                    o = __shfl_xor_sync(0xffffffffu, v, j);
                }
                const bool larger = ((tid & j) == 0) == ((tid & k) == 0);  // this thread keeps the larger one
                if (tid < size) v = (v > o) == larger ? v : o;
            }
        }
        return v;
    }

    // Finds K and r (s.key, s.ties) for the head of `target` tokens, or of weight `target`,
    // and s.sum, the head's weight, from the merged first histogram (`weights`: which has the
    // weights too). False: the whole row is kept. Every CTA takes the same path.
    B200_DEVICE bool select(unsigned long long target, bool by_weight, bool weights) {
        find(s.mcnt[tid], s.mwgt[tid], 0, 0, target, by_weight);
        const int bin0 = s.bin;
        if (bin0 < 0) return false;
        uint32_t lo = 0, hi = order_key(sc.top), n = s.bin_c;
        unsigned long long ac = s.above_c, aw = s.above_w;
        // the bin's values lie in an interval a little wider than its edges
        const float x_lo = sc.below(bin0), x_hi = sc.above(bin0);
        const auto member = [&](float v) {
            if (v < x_lo || v > x_hi) return false;
            const float z = sc.z(v);
            const uint32_t key = order_key(v);
            return z > kFloor && sc.bin(z) == bin0 && key >= lo && key <= hi;
        };
        if (x_hi < sc.top) hi = order_key(x_hi);
        if (x_lo > -INFINITY && x_lo < sc.top) lo = order_key(x_lo);
        while (n > kList && lo < hi) {  // split the bin over its bit patterns, descending
            const int shift = max(0, 32 - __clz(static_cast<int>(hi - lo)) - 9);
            cluster_sync();  // nobody reads the histogram any more
            clear_histogram();
            x.each(0, x.n, tid, kSmThreads, [&](float v, int) {
                if (member(v)) {
                    const int b = static_cast<int>((hi - order_key(v)) >> shift);
                    count(b);
                    if (weights) add_weight(b, sc.weight(v));
                }
            });
            cluster_sync();
            find(merged_count(), weights ? merged_weight() : 0ull, ac, aw, target, by_weight);
            hi -= static_cast<uint32_t>(s.bin) << shift;
            const uint32_t width = (1u << shift) - 1u;
            lo = hi - lo > width ? hi - width : lo;
            n = s.bin_c;
            ac = s.above_c;
            aw = s.above_w;
            __syncthreads();
        }
        uint32_t key = lo, at;
        unsigned long long each = sc.weight(key_value(lo));
        if (n > kList) {  // one bit pattern is left
            const unsigned long long r = by_weight ? (target - aw + each - 1) / each : target - ac;
            if (tid == 0) s.key = lo, s.ties = static_cast<uint32_t>(r), s.sum = aw + r * each;
            __syncthreads();
            return true;
        }
        collect(member);
        cluster_sync();
        fetch_listed(key, at);
        cluster_sync();  // the lists may be written again
        // in order, the token at which the measure reaches the target
        const bool have = tid < static_cast<int>(n);
        const unsigned long long v =
            sort_descending(have ? static_cast<unsigned long long>(key) << 32 | (0xFFFFFFFFu - at) : 0ull, n);
        key = static_cast<uint32_t>(v >> 32);
        each = have ? sc.weight(key_value(key)) : 0ull;
        const unsigned long long before = aw + cta_before(each);
        s.sorted[tid] = v;
        __syncthreads();
        if (have && (by_weight ? before < target && target <= before + each : ac + tid + 1 == target)) {
            int first = tid;  // of the run of equal tokens
            while (first > 0 && static_cast<uint32_t>(s.sorted[first - 1] >> 32) == key) --first;
            s.key = key;
            s.ties = static_cast<uint32_t>(tid - first) + 1;
            s.sum = before + each;
        }
        __syncthreads();
        return true;
    }

    B200_DEVICE unsigned long long share_of(float p, unsigned long long sum) const {
        const double want = static_cast<double>(p) * static_cast<double>(sum);
        return want >= 1.0 ? static_cast<unsigned long long>(want) : 1ull;
    }
    B200_DEVICE static unsigned long long drawn(float u, unsigned long long total) {
        const double want = static_cast<double>(u) * static_cast<double>(total);
        unsigned long long at = want > 0.0 ? static_cast<unsigned long long>(want) : 0ull;
        return want >= static_cast<double>(total) || at >= total ? total - 1 : at;
    }

    // The whole draw among the listed tokens, which hold the kept head (first CTA).
    B200_DEVICE void draw_listed(int32_t top_k, float top_p, unsigned long long row_sum, unsigned long long least, float u,
                                 int32_t *out) {
        uint32_t key, at;
        const uint32_t n = fetch_listed(key, at);
        const unsigned long long v = sort_descending(
            static_cast<uint32_t>(tid) < n ? static_cast<unsigned long long>(key) << 32 | (0xFFFFFFFFu - at) : 0ull, n);
        const uint32_t head = top_k > 0 ? min(n, static_cast<uint32_t>(top_k)) : n;
        bool keep = static_cast<uint32_t>(tid) < head;
        at = 0xFFFFFFFFu - static_cast<uint32_t>(v);
        const unsigned long long w = keep ? sc.weight(key_value(static_cast<uint32_t>(v >> 32))) : 0ull;
        if (top_p < 1.0f) {
            const unsigned long long sum = top_k > 0 ? cta_sum(w) : row_sum;
            const unsigned long long before = cta_before(w);
            keep = keep && (tid == 0 || before < share_of(top_p, sum));
        }
        keep = keep && w >= least;
        // the kept tokens by index: each sums the kept weight at smaller indices
        s.aat[tid] = keep ? at : 0xFFFFFFFFu;
        s.awgt[tid] = keep ? w : 0ull;
        const unsigned long long total = cta_sum(keep ? w : 0ull);
        const unsigned long long goal = drawn(u, total);
        if (__any_sync(0xffffffffu, keep)) {
            unsigned long long ahead = 0;
#pragma unroll 4
            for (uint32_t j = 0; j < head; ++j)
                if (s.aat[j] < at) ahead += s.awgt[j];
            if (keep && ahead <= goal && goal < ahead + w) *out = static_cast<int32_t>(at);
        }
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
    const float temp = __ldg(a.temperature + row);
    const float u = __ldg(a.u + row);
    const int32_t top_k = a.top_k ? __ldg(a.top_k + row) : 0;
    const float top_p = a.top_p ? __ldg(a.top_p + row) : 1.0f;
    const float min_p = a.min_p ? __ldg(a.min_p + row) : 0.0f;
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
    bad |= temp != temp || u != u || top_p != top_p || min_p != min_p;
    const float own = mx;
    mx = warp_max(mx);
    bad = __any_sync(0xffffffffu, bad);
    if (lane == 0) s.warp_f[warp] = mx, s.warp_b[warp] = bad;
    s.cnt[tid] = 0;
#pragma unroll
    for (int i = 0; i < 3; ++i) s.wgt[i][tid] = 0;
    __syncthreads();
    if (warp == 0) {
        mx = warp_max(lane < kSmWarps ? s.warp_f[lane] : -INFINITY);
        bad = __any_sync(0xffffffffu, lane < kSmWarps && s.warp_b[lane]);
        if (lane == 0) s.top = mx, s.bad = bad;
    }
    cluster_sync();
    mx = -INFINITY;
    bad = false;
    uint32_t first = 0;  // the first chunk with the maximum
    for (uint32_t r = 0; r < nc; ++r) {
        const float top = ld_dsmem(dsmem_addr(&s.top, r));
        if (top > mx) mx = top, first = r;
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
    Sampler<T, HELD> f{a, s, {HELD ? held : src, n}, {mx + 0.0f, inv}, tid, warp, lane, rank, nc};
    if (!(temp > 0.f) || inv == INFINITY) {
        // the first token with the maximum, without sums (256 held rows of 151936 F32: 74 us, by sums 107)
        if (rank == first) {
            int best = INT_MAX;
            f.x.each(0, n, tid, kSmThreads, [&](float v, int i) {
                if (v == mx) best = min(best, i);
            });
            best = __reduce_min_sync(0xffffffffu, best);
            if (lane == 0) s.warp_c[warp] = static_cast<uint32_t>(best);
            __syncthreads();
            if (warp == 0) {
                const uint32_t at = __reduce_min_sync(0xffffffffu, s.warp_c[lane % kSmWarps]);
                if (lane == 0) a.out[row] = static_cast<int32_t>(begin + at);
            }
        }
        cluster_sync();  // no CTA's shared memory goes away while it is read
        return;
    }
    const bool by_k = top_k > 0 && top_k < a.vocab, by_p = top_p < 1.0f;
    const double floor_p = static_cast<double>(fminf(fmaxf(min_p, 0.0f), 1.0f)) * 1099511627776.0;
    const unsigned long long least = static_cast<unsigned long long>(floor_p);

    // the kept head: keys above `key`, and the first `ties` equal to it
    uint32_t key = 0, ties = 0;
    if (by_k || by_p) {
        if (by_k && top_k <= kList / 2) {
            // Of the threads' largest tokens, top_k lie in bins 0 to s.bin, so the head does. Those bins hold few
            // more, as a rule, and no pass has to count all tokens.
            const float z = f.sc.z(own);
            if (z > kFloor) f.count(f.sc.bin(z));
            cluster_sync();
            f.find(f.merged_count(), 0, 0, 0, static_cast<unsigned long long>(top_k), false);
            const int last = s.bin;
            if (last >= 0 && f.collect_bins(last) <= kList) {
                if (rank == 0) f.draw_listed(top_k, top_p, 0, least, u, a.out + row);
                cluster_sync();  // no CTA's shared memory goes away while it is read
                return;
            }
            cluster_sync();  // nobody reads the histogram any more
            f.clear_histogram();
        }
        const float low = f.sc.below(kBins - 1);
        f.x.each(0, n, tid, kSmThreads, [&](float v, int) {
            if (v < low) return;
            const float z = f.sc.z(v);
            if (z > kFloor) {
                const int b = f.sc.bin(z);
                f.count(b);
                if (by_p) f.add_weight(b, f.sc.weight(v));
            }
        });
        cluster_sync();
        s.mcnt[tid] = f.merged_count();
        s.mwgt[tid] = by_p ? f.merged_weight() : 0ull;
        unsigned long long sum = by_p && !by_k ? f.cta_sum(s.mwgt[tid]) : 0ull;  // of the row
        // the last bin that the head reaches into
        if (by_k) f.find(s.mcnt[tid], s.mwgt[tid], 0, 0, static_cast<unsigned long long>(top_k), false);
        else f.find(s.mcnt[tid], s.mwgt[tid], 0, 0, f.share_of(top_p, sum), true);
        const int last = s.bin;
        if (last >= 0 && s.upto_c <= kList) {
            f.collect_bins(last);
            if (rank == 0) f.draw_listed(by_k ? top_k : 0, top_p, sum, least, u, a.out + row);
            cluster_sync();  // no CTA's shared memory goes away while it is read
            return;
        }
        __syncthreads();
        bool cut = false;
        if (by_k) cut = f.select(static_cast<unsigned long long>(top_k), false, by_p);
        if (cut) key = s.key, ties = s.ties, sum = s.sum;
        __syncthreads();
        if (by_p) {
            if (by_k && !cut) sum = f.cta_sum(s.mwgt[tid]);
            if (f.select(f.share_of(top_p, sum), true, true)) key = s.key, ties = s.ties;
        }
    }

    // kept weight of each warp's contiguous piece
    const int piece = (a.chunk / kSmWarps + 127) / 128 * 128;
    {
        const int p0 = min(n, warp * piece), p1 = min(n, p0 + piece);
        unsigned long long pw = 0;
        uint32_t pe = 0;
        // (key 0 keeps the whole row; min-p leaves out what lies below its own bin)
        const float k_value = key ? key_value(key) : -INFINITY;
        // `least` whole units, not min_p: the two differ by up to a factor of two where min_p is a few units
        const float low = f.sc.below(
            least > 0 ? min(kBins - 1, static_cast<int>(logf(static_cast<float>(least) * 0x1p-40f) * (kBins / kFloor)) + 2) : kBins - 1);
        f.x.each(p0, p1, lane, 32, [&](float v, int) {
            if (v < k_value || v < low) return;
            if (v > k_value) {
                const unsigned long long w = f.sc.weight(v);
                if (w >= least) pw += w;
            } else {
                ++pe;
            }
        });
        pe = __reduce_add_sync(0xffffffffu, pe);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) pw += __shfl_xor_sync(0xffffffffu, pw, o);
        if (lane == 0) s.piece_w[warp] = pw, s.piece_eq[warp] = pe;
        __syncthreads();
        if (tid == 0) {
            unsigned long long cw = 0;
            uint32_t ce = 0;
            for (int i = 0; i < kSmWarps; ++i) cw += s.piece_w[i], ce += s.piece_eq[i];
            s.part = cw;
            s.equal = ce;
        }
    }
    cluster_sync();
    unsigned long long each = ties ? f.sc.weight(key_value(key)) : 0ull;
    if (each < least) each = 0;
    unsigned long long total = 0, before = 0;  // kept weight of the row; ahead of this chunk
    uint32_t eq = 0, eq_before = 0;
    for (uint32_t r = 0; r < nc; ++r) {
        const uint32_t e = ld_dsmem_u32(dsmem_addr(&s.equal, r));
        if (r == rank) before = total, eq_before = eq;
        total += ld_dsmem_u64(dsmem_addr(&s.part, r)) + (eq < ties ? min(e, ties - eq) : 0u) * each;
        eq += e;
    }
    const unsigned long long goal = f.drawn(u, total);
    // the CTA in whose chunk the drawn sum lies: the piece, then the token
    if (goal >= before) {
        int p = -1;
        unsigned long long at = before;
        uint32_t ep = eq_before;
        for (int i = 0; i < kSmWarps; ++i) {
            const unsigned long long w = s.piece_w[i] + (ep < ties ? min(s.piece_eq[i], ties - ep) : 0u) * each;
            if (goal < at + w) {
                p = i;
                break;
            }
            at += w;
            ep += s.piece_eq[i];
        }
        if (p >= 0) {  // the whole CTA: `per` consecutive tokens a thread
            const int per = (piece + kSmThreads - 1) / kSmThreads;
            const int i0 = min(n, min((p + 1) * piece, p * piece + tid * per));
            const int i1 = min(n, min((p + 1) * piece, i0 + per));
            unsigned long long w = 0, e = 0;
            for (int i = i0; i < i1; ++i) {
                const float v = f.x[i];
                const uint32_t k = order_key(v);
                if (k > key) {
                    const unsigned long long x = f.sc.weight(v);
                    if (x >= least) w += x;
                }
                e += k == key;
            }
            const unsigned long long eb = ep + f.cta_before(e);  // equal tokens ahead of this thread
            unsigned long long kept = eb < ties ? (ties - eb < e ? ties - eb : e) : 0ull;
            w += kept * each;
            unsigned long long run = at + f.cta_before(w);
            if (run <= goal && goal < run + w) {
                for (int i = i0; i < i1; ++i) {
                    const float v = f.x[i];
                    const uint32_t k = order_key(v);
                    unsigned long long x = 0;
                    if (k > key) {
                        x = f.sc.weight(v);
                        if (x < least) x = 0;
                    } else if (k == key && kept > 0) {
                        x = each;
                        --kept;
                    }
                    if (goal < run + x) {
                        a.out[row] = static_cast<int32_t>(begin + i);
                        break;
                    }
                    run += x;
                }
            }
        }
    }
    cluster_sync();  // no CTA's shared memory goes away while it is read
}

constexpr size_t kOwnBytes = (sizeof(SampleShared) + 15) / 16 * 16;
constexpr size_t kMostShared = 227 * 1024;
constexpr size_t kHalfShared = 113 * 1024;  // two CTAs an SM: 228 KB less 1 KB for each
static_assert(kMostShared / 2 < kMostChunk / 2, "rows that fit eight CTAs' shared memory fit four chunks");

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
    // rows take fewer, as far as two chunks still fit an SM. F32, 1 / 2 / 4 / 8 CTAs a row: one row of
    // 32003 24.5 / 19.5 / 16.4 / 16.4 us; 64 rows 31 / 24 / 22 / 35, 256 rows 55 / 47 / 64 / 113; one row of
    // 151936 104 / 59 / 25 / 22 (before top-k stopped at the threads' own largest tokens; 14 to 18 now).
    const int64_t sms = device_sm_count();
    int c = 1;
    while (c < kMaxCluster && a.vocab > 2048 * c && rows * c < sms) c *= 2;
    while (c < kMaxCluster && kOwnBytes + (a.vocab + c - 1) / c * sizeof(T) > kHalfShared) c *= 2;
    const auto bytes = [&] { return kOwnBytes + (a.vocab + c - 1) / c * sizeof(T) + 64 * sizeof(T); };
    bool held = bytes() <= kMostShared;
    // Rows of which an SM holds an eighth or two are few at a time, and each waits on its own exchanges. With
    // more than three rounds of them the passes read the rows again from L2 instead, by fewer CTAs a
    // row. F32, held in clusters of 8 against 2 or 4 from L2: 64 rows of 151936 74 us against 77 (held), 128
    // rows 115 against 99, 256 rows 205 against 164 (4), 600 rows 441 against 290 (2) and 307 (4).
    if (held && c == kMaxCluster && rows * c > 3 * sms * (bytes() <= kHalfShared ? 2 : 1)) {
        held = false;
        c = rows * 2 >= 5 * sms && a.vocab <= 2 * kMostChunk ? 2 : 4;
    }
    a.cluster = c;
    a.chunk = static_cast<int32_t>(((a.vocab + c - 1) / c + 63) / 64 * 64);
    return held ? sample_launch_as<T, true>(a, rows, st) : sample_launch_as<T, false>(a, rows, st);
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
    if (n_vocab > kMaxCluster * kMostChunk || n_rows > INT32_MAX / kMaxCluster) return B200_ERR_NOT_SUPPORTED;
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
