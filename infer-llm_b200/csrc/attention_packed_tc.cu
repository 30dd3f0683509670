// Packed causal attention on the 5th-generation tensor cores, for F16, BF16 and F32.
//
// A slot is a 128-row accumulator: scores S (128 x 128 keys) and output O (128 x D) in tensor
// memory, and one softmax warpgroup with a thread per row. Two slots run on an SM, two of one CTA or
// one of each of two CTAs. A step i belongs to slot i % SL:
//   S = Q . K^T           (M 128, N 128 keys, K D; both operands in shared memory)
//   P = 2^(S sl2 - m)     (softmax warps; 16-bit P written over S in tensor memory)
//   O += P . V            (M 128, N D, K 128 keys; A = P from tensor memory)
// While one slot's softmax runs, the tensor cores work for the other. The slots are
//   NT = 2, SL = 2: two query tiles over the same key tiles (K and V are read once for both);
//   NT = 1, SL = 2: one query tile, even key tiles in slot 0 and odd ones in slot 1, joined at the
//           end (half as long a chain for calls with few query tiles);
//   NT = 1, SL = 1: one query tile in one slot, two CTAs an SM (short contexts: one CTA's start and
//           end run beside the other's steps).
// With fewer query tiles than SMs and long contexts the key tiles are also cut into `parts`, a CTA
// each (NT = 1); packed_join_kernel weighs the parts' rows by their sums.
// A query tile's rows are tokens times the G heads of a KV head (row = token * G + head), as
// many whole tokens as fit 128 rows, so the heads that share keys share every tile.
// Warp roles: warp 0 TMA, warp 1 tensor cores, warps 2-3 V check, then four softmax warps a slot, and
// for F32 warps 12-15 the output's sum. They share out the CTA's registers (80 + 2 x 120 + 192 = 4 x 128
// for F32, 88 + 2 x 208 = 3 x 168 with two slots, 56 + 200 = 2 x 128 with one).
//   * The running maximum moves only when it grows by more than 2^8, so rescaling O is rare
//     (the result is unchanged: every p is bounded by 2^8). Statistics are F32. 16-bit types: P is
//     one number of the element type, the sum is taken before that rounding. It is what the second
//     product takes at one product's cost; two terms of P would add half to the tensor work. The errors against
//     64 bits grow by it from 1.5e-3 to 2.0e-3 of the output (8192 BF16 tokens) and from 2.1e-4 to 2.6e-4 (F16).
//   * Hidden keys of a tile (past a row's last key, of the next sequence, or past the end)
//     have P = 0, but 0 times a V that is no number is not 0. The V check looks for such
//     rows in the tiles that hide keys, clears them in shared memory, and notes them; 16-bit rows that
//     do see one of them add its term in the epilogue.
//   * F32 (NT = 1) runs as three F16 products. With a tile's values scaled by a power of two to a
//     largest magnitude in [2^14, 2^15), x = hi + lo of two F16 numbers holds 22 bits
//     of x (and an absolute 2^-39 of the tile's largest), and x y = hi hi + hi lo + lo hi
//     up to 2^-22. packed_split_kernel writes K and V so, as hi and lo planes with one
//     exponent per 128-key tile and KV head; Q rows are split by the softmax threads
//     (an exponent per row), P by construction (p <= 1, times 2^14). V, whose columns each make an output of their
//     own, has its lo times 2^11: it is as large as hi then, not among F16's subnormals, and
//     2^-50 of the tile's largest is held. P hi times it comes first, and the next product takes the sum times 2^-11
//     (2048 tokens 82 us, with plain lo 81; K so too 85).
//     One exponent does only for rows and columns of like magnitude: a tile of K or V in which a row's or a
//     column's largest is below 2^-16 of the tile's, or which holds Inf or NaN, is marked, and a CTA that met one does
//     its rows over with F32 FFMA (attention_packed_ffma.cuh; 2048 tokens with one such key 868 us). So
//     neither hidden keys nor other columns cost a row its bits. The tensor cores
//     round their sums toward zero: over a long row that bias reached 1e-5 at 8192 keys. So each
//     step's O starts from zero (lo products first), and a fourth warpgroup adds the steps
//     up in F32 registers, each with its own row maximum and V exponent. An FFMA kernel has no
//     such rounding but a 20th of the rate; TF32 products would keep 11 bits.
// Bound: at long contexts the chain scores -> softmax -> P -> product of a slot, against which the other
// slot's runs: 8192 BF16 tokens, 32 / 8 heads of 128, 505 to 522 us by GPU, 1.05 to 1.09 PFLOP/s (64 to 66 % of a
// large library matrix product's rate); the tensor cores are busy 54 to 60 % of the time. 2048 F32 tokens, 16 / 8
// heads of 128, 81 to 82 us (209 to 212 TFLOP/s of the call's, 630 of the three products), the split kernel 7 us of it. Short
// calls: a CTA's start and end, ~6 us (look-up 1, first copies 1.4, last product 0.8 to 1.7, output 2), beside ~0.9
// us a step: 10 prompts of 1 to 1333 BF16 tokens, 16 / 8 heads of 128, 35 us. Two slots take all 512
// columns of tensor memory and most of an SM's registers.
// Every mbarrier wait is bounded; one that runs out records B200_DEV_TIMEOUT, and the CTA
// waits (bounded) for its copies and products and frees its tensor memory.
#include "attention_packed_ffma.cuh"
#include "gemv.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

#include <type_traits>

namespace b200 {
namespace {

constexpr int kPtRows = 128, kPtKeys = 128;
template <typename T, int SL>
constexpr int kPtThreads = 128 + 128 * SL + (__is_same(T, float) ? 128 : 0);
constexpr int kMaskedTiles = 4;  // key tiles in which some row of a CTA hides keys (at most 256 tokens)
constexpr float kPtRescale = 8.0f;
constexpr int kPolyStep = 4;  // 8192 BF16 keys: none 522 us, every 4th pair 504 to 513, every 2nd slower than none

// NT: query tiles a CTA; SL: slots; PL: planes of an operand tile (2: hi and lo of F32)
template <int D, int NT, int SL, int PL>
struct PtGeometry {
    static_assert(PL == 1 || NT == 1, "F32 tiles leave room for one query tile");
    static constexpr uint32_t kBox = kPtKeys * 128;           // 64 elements of 128 rows
    static constexpr uint32_t kTile = (D / 64) * kBox;        // a plane of a 128-row tile of Q, K or V
    // one slot: two CTAs an SM
    static constexpr int kStages = SL == 1 ? 256 / D : (D == 128 ? (NT * PL == 2 ? 5 : 6) : 8);
    static constexpr uint32_t kOffRing = NT * PL * kTile;
    static constexpr uint32_t kOffBar = kOffRing + kStages * kTile;  // 44 words, then the CTA's PackedTile
    static constexpr uint32_t kOffStat = kOffBar + 384;       // F32: (m, l) of each slot's step
    static constexpr uint32_t kOffBad = kOffStat + (PL == 2 ? 2 * kPtRows * 8 : 0);  // [kMaskedTiles][4] words, "any", "wide"
    static constexpr size_t kSmem = kOffBad + 128;
    static_assert(kSmem <= (SL == 1 ? 113 : 227) * 1024, "shared memory of an SM");
    static_assert(PL == 1 || ffma_smem<D>() <= kOffBar, "rows done over by FFMA");
};

// K and V tiles of a key-tile sequence, numbered in the order of their first use.
// PAIRS: K and V of a tile follow one another; else K runs a tile ahead.
template <bool PAIRS>
B200_DEVICE int plane_k(int t) { return PAIRS ? 2 * t : (t == 0 ? 0 : 2 * t - 1); }
template <bool PAIRS>
B200_DEVICE int plane_v(int t, int n) { return PAIRS ? 2 * t + 1 : t + min(t + 2, n); }

// Tile `at` of the query tiles of all sequences (M tokens each) in the order of their key tiles, most
// first, so that the last CTAs to start are the shortest (10 prompts of 1 to 1333 BF16 tokens: 39 us against 46 in
// the sequences' order). A whole warp: a lane a sequence (at most 32), and bisection over the number of key
// tiles, which takes ~1 us more than find_packed_tile.
B200_DEVICE PackedTile find_heaviest_tile(const PackedArgs &a, int M, int64_t at, int32_t *status) {
    const int lane = threadIdx.x & 31;
    int64_t q0 = 0, k0 = 0;
    int nq = 0, nk = 0;
    bool ok = true;
    if (lane < a.n_seqs) {
        const bool ok_q = packed_range(a.cu_q, lane, a.total_q, q0, nq), ok_k = packed_range(a.cu_k, lane, a.total_k, k0, nk);
        ok = ok_q && (ok_k || nq == 0);
        if (!ok) set_status(status, B200_DEV_BAD_POSITION);
    }
    // x / M for x < 2^31 by a product that is at most one too large
    const unsigned scale = 0xFFFFFFFFu / static_cast<unsigned>(M) + 1u;
    const auto over_m = [&](unsigned x) {
        const unsigned y = M == 1 ? x : __umulhi(x, scale);
        return static_cast<int>(y - (y * M > x ? 1u : 0u));
    };
    const int tiles = over_m(static_cast<unsigned>(nq) + static_cast<unsigned>(M) - 1u);
    // the lane's tiles with at least c key tiles (the last token of tile i sees min(nq, (i + 1) M) + nk - nq keys)
    const auto with = [&](int c) {
        const int64_t x = static_cast<int64_t>(c - 1) * kPtKeys - (nk - nq);  // tokens that see fewer
        if (c <= 0) return tiles;
        return nq == 0 || nq <= x ? 0 : tiles - min(tiles - 1, over_m(static_cast<unsigned>(max64(0, x))));
    };
    PackedTile p;
    int lo = 0, hi = __reduce_max_sync(0xffffffffu, (nk + kPtKeys - 1) / kPtKeys) + 1;  // key tiles of tile `at`: in [lo, hi)
    if (static_cast<int64_t>(__reduce_add_sync(0xffffffffu, static_cast<unsigned>(tiles))) <= at) return p;
    while (hi - lo > 1) {
        const int c = (lo + hi) >> 1;
        if (static_cast<int64_t>(__reduce_add_sync(0xffffffffu, static_cast<unsigned>(with(c)))) > at) lo = c;
        else hi = c;
    }
    const int more = with(hi), same = with(lo) - more;
    int incl = same;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    const int rank = static_cast<int>(at) - static_cast<int>(__reduce_add_sync(0xffffffffu, static_cast<unsigned>(more)));
    const int l = __ffs(static_cast<int>(__ballot_sync(0xffffffffu, incl > rank))) - 1;
    p.seq = __shfl_sync(0xffffffffu, ok ? lane : -1, l);
    p.tile = __shfl_sync(0xffffffffu, tiles - more - same + (rank - (incl - same)), l);
    p.nq = __shfl_sync(0xffffffffu, nq, l);
    p.nk = __shfl_sync(0xffffffffu, nk, l);
    p.q0 = __shfl_sync(0xffffffffu, q0, l);
    p.k0 = __shfl_sync(0xffffffffu, k0, l);
    return p;
}

// Matrix descriptors of 128-byte-swizzled tiles differ only in their low word (address and
// leading byte offset): 64-byte rows of 8-row atoms 1024 bytes apart, version 1. Forming
// the words for an instruction by 64-bit arithmetic costs the issuing thread ~130 cycles,
// twice the product's own 64; a 32-bit add of a constant does not.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
B200_DEVICE uint32_t desc_low(uint32_t saddr, uint32_t lbo) { return ((saddr & 0x3FFFFu) >> 4) | ((lbo >> 4) << 16); }
// The whole warp runs these, converged, and one elected lane issues: with the operands the same
// in every lane, addresses stay in uniform registers. From one lane's branch each instruction
// moves its own there first (8192 BF16 keys: 588 us against 510).
B200_DEVICE uint32_t elect_lane() {
    uint32_t e;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(e));
    return e;
}
B200_DEVICE void mma_ss(uint32_t e, uint32_t d, uint32_t a_low, uint32_t b_low, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n .reg .pred p, e;\n .reg .b64 da, db;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 e, %6, 0;\n mov.b64 da, {%1, %5};\n"
        " mov.b64 db, {%2, %5};\n @e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}" ::"r"(d),
        "r"(a_low), "r"(b_low), "r"(idesc), "r"(static_cast<uint32_t>(accumulate)), "r"(kDescHigh), "r"(e)
        : "memory");
}
B200_DEVICE void mma_ts(uint32_t e, uint32_t d, uint32_t a, uint32_t b_low, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n .reg .pred p, e;\n .reg .b64 db;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 e, %6, 0;\n mov.b64 db, {%2, %5};\n"
        " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n}" ::"r"(d),
        "r"(a), "r"(b_low), "r"(idesc), "r"(static_cast<uint32_t>(accumulate)), "r"(kDescHigh), "r"(e)
        : "memory");
}
// The same onto D times 2^-kLoShift.
constexpr int kLoShift = 11;
B200_DEVICE void mma_ts_onto_lo(uint32_t e, uint32_t d, uint32_t a, uint32_t b_low, uint32_t idesc) {
    asm volatile(
        "{\n .reg .pred p, e;\n .reg .b64 db;\n setp.eq.b32 p, 0, 0;\n setp.ne.b32 e, %5, 0;\n mov.b64 db, {%2, %4};\n"
        " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p, %6;\n}" ::"r"(d),
        "r"(a), "r"(b_low), "r"(idesc), "r"(kDescHigh), "r"(e), "n"(kLoShift)
        : "memory");
}
B200_DEVICE void commit_if(uint32_t e, uint64_t *bar) {
    asm volatile(
        "{\n .reg .pred e;\n setp.ne.b32 e, %1, 0;\n"
        " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(smem_addr(bar)),
        "r"(e)
        : "memory");
}

// Two F32 operations in one instruction.
B200_DEVICE uint64_t pair_of(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
B200_DEVICE float2 of_pair(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
B200_DEVICE uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
B200_DEVICE uint64_t add_pair(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// 2^x of two values in FP32 arithmetic, for x <= 8: 2^round(x) by the exponent field times a
// least-maximum polynomial of the rest in [-1/2, 1/2]. x below -125 gives 2^-125, and so does a NaN: it
// serves tiles that hide no keys (x = -inf) and rows whose scores' maximum is finite. Degree 3 is within 7.5e-5 (BF16 rounds P to
// 2^-9), degree 4 within 2.6e-6 (F16 to 2^-12).
template <bool BF16>
B200_DEVICE float2 exp2_poly_pair(float2 x) {
    constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23: adding it rounds to whole numbers
    const auto both = [](float v) { return pair_of(v, v); };
    const uint64_t c = pair_of(fmaxf(x.x, -125.0f), fmaxf(x.y, -125.0f));
    const uint64_t t = add_pair(c, both(kMagic));
    const uint64_t f = fma_pair(add_pair(t, both(-kMagic)), both(-1.0f), c);
    uint64_t p;
    if constexpr (BF16) {
        p = fma_pair(f, both(0.0551716648f), both(0.242611125f));
        p = fma_pair(p, f, both(0.693260968f));
        p = fma_pair(p, f, both(0.999928057f));
    } else {
        p = fma_pair(f, both(0.00957010128f), both(0.0559178591f));
        p = fma_pair(p, f, both(0.240247443f));
        p = fma_pair(p, f, both(0.693121791f));
        p = fma_pair(p, f, both(0.999999285f));
    }
    const float2 tf = of_pair(t), pf = of_pair(p);
    return make_float2(__uint_as_float(__float_as_uint(pf.x) + (__float_as_uint(tf.x) << 23)),
                       __uint_as_float(__float_as_uint(pf.y) + (__float_as_uint(tf.y) << 23)));
}
B200_DEVICE uint64_t mul_pair(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
B200_DEVICE float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// NaN if one of them is
B200_DEVICE float max2_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
B200_DEVICE float max3_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

template <typename T>
B200_DEVICE uint32_t pack_pair(float x, float y) {
    if constexpr (__is_same(T, __half)) {
        const __half2 h = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}

// F32 operands split for the tensor cores: planes of F16 rows [2][total_k][Hkv][D], and per
// (key tile, KV head) the exponents of K and of V. And the parts of a query tile's keys.
struct SplitView {
    const int32_t *exps = nullptr;
    int64_t total_k = 0;
    int parts = 1;            // of each query tile's keys
    float *part_o = nullptr;  // [CTA][128][D], with parts > 1
    float2 *part_ml = nullptr;
    bool by_weight = false;   // query tiles in the order of their key tiles
};
constexpr int kTop = 14;  // largest magnitudes in [2^14, 2^15); P <= 1 times 2^14
// Rows and columns within 2^16 of their tile's largest: their elements hold 22 bits, or an absolute 2^-23 (K)
// or 2^-33 (V) of the row's and the column's largest.
constexpr int kSpread = 16;
// A word of `exps`: the exponent, and whether the tile takes FFMA.
B200_DEVICE int exps_word(int e, bool wide) { return 2 * e + static_cast<int>(wide); }
B200_DEVICE int exps_exponent(int word) { return word >> 1; }
B200_DEVICE bool exps_wide(int word) { return word & 1; }
constexpr int kMostScale = 100;  // exponents of Q and K that add up past it: their product takes FFMA

// A tile's place in `exps`: increasing along the packed keys for any lengths, since
// floor(x) + ceil(y) <= floor(x + y) + 1.
B200_DEVICE int64_t split_index(int64_t k0, int seq, int t) { return k0 / kPtKeys + seq + t; }

B200_DEVICE float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(max(-126, min(127, e)) + 127) << 23); }

// floor(log2 x) of the largest finite magnitude (as its bits), at least -100
B200_DEVICE int top_exponent(uint32_t bits) { return max(-100, static_cast<int>(bits >> 23) - 127); }
B200_DEVICE uint32_t finite_magnitude(float x) {
    const uint32_t u = __float_as_uint(x) & 0x7FFFFFFFu;
    return u < 0x7F800000u ? u : 0u;
}
constexpr float kLoScale = static_cast<float>(1 << kLoShift);  // of V
// hi + lo / lo_scale = x (22 bits); a value that is no number stays one, in hi
B200_DEVICE void split_f16(float x, float lo_scale, __half &hi, __half &lo) {
    hi = __float2half_rn(x);
    lo = finite_magnitude(x) || x == 0.f ? __float2half_rn((x - __half2float(hi)) * lo_scale) : __half(0.f);
}
B200_DEVICE void split_f16x2(uint64_t v, uint32_t &hi, uint32_t &lo) {
    const float2 x = of_pair(v);
    const __half2 h = __floats2half2_rn(x.x, x.y);
    const float2 f = __half22float2(h);
    const float2 d = of_pair(add_pair(v, pair_of(-f.x, -f.y)));
    const __half2 r = __floats2half2_rn(d.x, d.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&r);
}

constexpr int kSplitThreads = 256;

// One CTA: the K or V rows of one key tile and KV head, as hi and lo planes with the tile's
// exponent, and whether its rows and columns spread too far for one. A pass over the bytes: HBM bounds it (2048 keys, 8 heads of 128: 17 MB in, 17 MB out, 7 us
// with its launch; the attention kernel's start overlaps it).
template <int D>
__global__ void __launch_bounds__(kSplitThreads) packed_split_kernel(const PackedArgs a, __half *planes, int32_t *exps) {
    constexpr int V4 = D / 4, PER = kPtKeys * V4 / kSplitThreads;  // float4 a row, a thread
    constexpr int W = kSplitThreads / 32;
    __shared__ uint32_t warp_top[W], warp_low[W], warp_any[W], col_top[W][D], col_low[D / 32];
    grid_launch_dependents();
    const int kvh = (blockIdx.x >> 1) % a.Hkv, is_v = blockIdx.x & 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const PackedTile p = find_packed_tile(a.cu_k, a.cu_k, a.n_seqs, a.total_k, a.total_k, 1, kPtKeys,
                                          (blockIdx.x >> 1) / a.Hkv, nullptr);
    if (p.seq < 0) return;
    const float *src = static_cast<const float *>(is_v ? a.v : a.k) + kvh * (is_v ? a.v_head : a.k_head);
    const int64_t tok = is_v ? a.v_tok : a.k_tok;
    const int rows = min(kPtKeys, p.nk - p.tile * kPtKeys);
    const int64_t first = p.k0 + static_cast<int64_t>(p.tile) * kPtKeys;
    // magnitudes: the largest finite one (`top`), of each row and column, the least of those that
    // are not zero (`low`), and of any kind (`any`)
    const auto nonzero = [](uint32_t m) { return m ? m : 0xFFFFFFFFu; };
    float4 x[PER];
    uint32_t low = 0xFFFFFFFFu, any = 0, top = 0, col[4] = {};
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = threadIdx.x + i * kSplitThreads, r = e / V4, c = e % V4;
        x[i] = r < rows ? __ldg(reinterpret_cast<const float4 *>(src + (first + r) * tok) + c) : make_float4(0.f, 0.f, 0.f, 0.f);
        const float v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
        uint32_t row = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t m = finite_magnitude(v[j]);
            any = max(any, __float_as_uint(v[j]) & 0x7FFFFFFFu);
            row = max(row, m);
            col[j] = max(col[j], m);
        }
        if constexpr (V4 == 32) {
            row = __reduce_max_sync(0xffffffffu, row);
        } else {  // two rows a warp
#pragma unroll
            for (int o = V4 / 2; o > 0; o >>= 1) row = max(row, __shfl_xor_sync(0xffffffffu, row, o));
        }
        low = min(low, nonzero(row));
        top = max(top, row);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (V4 == 16) col[j] = max(col[j], __shfl_xor_sync(0xffffffffu, col[j], 16));
        if (lane < V4) col_top[warp][4 * lane + j] = col[j];
    }
    if constexpr (V4 == 16) {
        low = min(low, __shfl_xor_sync(0xffffffffu, low, 16));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 16));
    }
    any = __reduce_max_sync(0xffffffffu, any);
    if (lane == 0) warp_top[warp] = top, warp_low[warp] = low, warp_any[warp] = any;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) top = max(top, warp_top[w]);
    const int e = top ? top_exponent(top) : kTop;  // (a tile of zeros: any)
    const float s = pow2(kTop - e), lo_scale = is_v ? kLoScale : 1.0f;
    if (threadIdx.x < D) {
        uint32_t c = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) c = max(c, col_top[w][threadIdx.x]);
        c = __reduce_min_sync(0xffffffffu, nonzero(c));
        if (lane == 0) col_low[warp] = c;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 0; w < W; ++w) low = min(low, warp_low[w]), any = max(any, warp_any[w]);
        for (int w = 0; w < D / 32; ++w) low = min(low, col_low[w]);
        const bool wide = any >= 0x7F800000u || static_cast<int>(min(low, 0x7F800000u) >> 23) - 127 < e - kSpread;
        exps[(split_index(p.k0, p.seq, p.tile) * a.Hkv + kvh) * 2 + is_v] = exps_word(e - kTop, wide);
    }
    const int64_t plane = a.total_k * a.Hkv * D;
    __half *dst = planes + (is_v ? 2 * plane : 0) + kvh * D;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int el = threadIdx.x + i * kSplitThreads, r = el / V4, c = el % V4;
        if (r >= rows) continue;
        __half h[4], l[4];
        split_f16(x[i].x * s, lo_scale, h[0], l[0]);
        split_f16(x[i].y * s, lo_scale, h[1], l[1]);
        split_f16(x[i].z * s, lo_scale, h[2], l[2]);
        split_f16(x[i].w * s, lo_scale, h[3], l[3]);
        __half *d = dst + (first + r) * a.Hkv * D + 4 * c;
        *reinterpret_cast<uint2 *>(d) = *reinterpret_cast<const uint2 *>(h);
        *reinterpret_cast<uint2 *>(d + plane) = *reinterpret_cast<const uint2 *>(l);
    }
}

template <typename T, int D, int NT, int SL>
__global__ void __launch_bounds__(kPtThreads<T, SL>, SL == 1 ? 2 : 1)
    packed_tc_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                     const __grid_constant__ CUtensorMap tv, const PackedArgs a, const SplitView sp) {
    constexpr bool SPLIT = __is_same(T, float);
    constexpr int PL = SPLIT ? 2 : 1;
    using Ge = PtGeometry<D, NT, SL, PL>;
    static_assert(SL == 2 || (NT == 1 && !SPLIT), "one slot holds one query tile");
    constexpr bool kPairs = NT == 2 || SL == 1, kJoin = NT == 1 && SL == 2;  // kJoin: the slots halve the key tiles
    constexpr int kColumns = 256 * SL;  // of tensor memory
    constexpr bool kBf16 = __is_same(T, __nv_bfloat16);
    constexpr uint32_t kIdS = idesc_f16(kPtRows, kPtKeys, kBf16, false, false);
    constexpr uint32_t kIdO = idesc_f16(kPtRows, D, kBf16, false, true);
    constexpr int S = Ge::kStages;
    extern __shared__ __align__(1024) unsigned char pt_smem[];  // as the swizzled tiles want
    unsigned char *base = pt_smem;
    const uint32_t sbase = smem_addr(base);
    uint64_t *bars = reinterpret_cast<uint64_t *>(base + Ge::kOffBar);
    uint64_t *full = bars;            // [S] a plane of a K or V tile landed
    uint64_t *empty = bars + S;       // [S] plane read by its last product
    uint64_t *q_full = bars + 2 * S;
    uint64_t *s_full = q_full + 1;    // [2] scores of the slot's step complete (and all earlier products)
    uint64_t *p_part = s_full + 2;    // [2] O rescaled and the first 96 keys' P written (F32: all of P)
    uint64_t *p_full = p_part + 2;    // [2] all of P written
    uint64_t *o_final = p_full + 2;   // [2] the slot's last product complete (F32: each step's)
    uint64_t *v_ok = o_final + 2;     // [kMaskedTiles] the masked tile's V checked
    uint64_t *v_ask = v_ok + kMaskedTiles;  // [kMaskedTiles] its V landed: to be checked
    uint64_t *o_empty = v_ask + kMaskedTiles;  // [2] F32: the step's O has been added up
    uint64_t *st_full = o_empty + 2;           // [2] F32: the step's (m, l) written
    uint64_t *idle = st_full + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(idle + 1);
    uint32_t *bad = reinterpret_cast<uint32_t *>(base + Ge::kOffBad);

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(q_full, SPLIT ? 256 : 1);
        for (int s = 0; s < 2; ++s) {
            mbar_init(&s_full[s], 1);
            mbar_init(&p_part[s], 128);
            mbar_init(&p_full[s], 128);
            mbar_init(&o_final[s], 1);
            mbar_init(&o_empty[s], 128);
            mbar_init(&st_full[s], 128);
        }
        for (int s = 0; s < kMaskedTiles; ++s) {
            mbar_init(&v_ok[s], 64);
            mbar_init(&v_ask[s], 1);
        }
        mbar_init(idle, 1);
        fence_barrier_init();
        for (const CUtensorMap *m : {&tq, &tk, &tv})
            asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
    }
    if (threadIdx.x < 4 * kMaskedTiles + 2) bad[threadIdx.x] = 0;
    uint32_t &any_wide = bad[4 * kMaskedTiles + 1];  // F32: a key tile was not held by two F16 numbers
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"(kColumns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        if (blockIdx.x == gridDim.x - 1) clear_uncovered(a);
    }

    const int G = a.G, BQ = kPtRows / G, MT = NT * BQ;  // tokens of a query tile, of the CTA
    const int kvh = blockIdx.x / sp.parts % a.Hkv, part = blockIdx.x % sp.parts;
    // (one warp looks, while others prepare barriers and tensor memory)
    PackedTile *found = reinterpret_cast<PackedTile *>(bars + 44);
    if (warp == 3) {
        const int64_t at = blockIdx.x / (sp.parts * a.Hkv);
        const PackedTile f = sp.by_weight ? find_heaviest_tile(a, MT, at, a.status)
                                          : find_packed_tile(a.cu_q, a.cu_k, a.n_seqs, a.total_q, a.total_k, 1, MT, at, a.status);
        if (lane == 0) *found = f;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    PackedTile p;
    p.seq = __shfl_sync(0xffffffffu, found->seq, 0);
    p.tile = __shfl_sync(0xffffffffu, found->tile, 0);
    p.nq = __shfl_sync(0xffffffffu, found->nq, 0);
    p.nk = __shfl_sync(0xffffffffu, found->nk, 0);
    p.q0 = __shfl_sync(0xffffffffu, found->q0, 0);
    p.k0 = __shfl_sync(0xffffffffu, found->k0, 0);
    const bool some = p.seq >= 0;                      // not past the last tile
    const int t0 = p.tile * MT;                        // first token
    const int shift = p.nk - p.nq;                     // token t sees keys 0 .. t + shift
    const int seen = min(p.nq, t0 + MT) + shift;       // keys the last token sees (may be <= 0)
    const int tiles = some && seen > 0 ? (seen + kPtKeys - 1) / kPtKeys : 0;  // key tiles, of which this CTA's:
    const int ta = tiles * part / sp.parts, nt = tiles * (part + 1) / sp.parts - ta;
    const int steps = NT * nt;
    // the CTA's tiles from this one on hide keys from some row
    const int first_masked = max(0, (t0 + shift + 1) / kPtKeys - ta);
    const int64_t k0 = p.k0 + static_cast<int64_t>(ta) * kPtKeys;  // its first key

    const auto col_s = [&](int slot) { return tmem + static_cast<uint32_t>(slot * kPtKeys); };
    const auto col_o = [&](int slot) { return tmem + 128u * SL + static_cast<uint32_t>(slot * 128); };
    const auto wait = [&](uint64_t *bar, uint32_t parity) {
        if (wait_poll(bar, parity, nullptr)) return true;
        set_status(a.status, B200_DEV_TIMEOUT);
        return false;
    };

    // softmax and output threads: a row of the slot's query tile, a lane of tensor memory
    const int slot = (warp - 4) >> 2, qq = warp & 3;
    const int r = 32 * qq + lane;
    const uint32_t lanes = static_cast<uint32_t>(32 * qq) << 16;
    const int tok = t0 + (NT == 2 ? slot * BQ : 0) + r / G;
    const bool live = some && r < BQ * G && tok < p.nq;
    const int last = live ? tok + shift - ta * kPtKeys : -1;  // last of the CTA's keys that the row sees
    const T *q_row = static_cast<const T *>(a.q) + (p.q0 + tok) * a.q_tok + (kvh * G + r % G) * a.q_head;
    // Rows of a query tile (first token t) from shared memory to the output: a thread writes its
    // row's 16-byte chunk c to row r, chunk c ^ (r % 8) of `stage`, and the group's threads
    // then copy whole rows (a row written by its own thread reaches 32 lines an instruction).
    constexpr int kRowChunks = D * static_cast<int>(sizeof(T)) / 16;
    const auto store_rows = [&](const unsigned char *stage, int t, int id, int threads) {
        const int step = threads / kRowChunks, dt = step / G, dg = step % G, c = id % kRowChunks;
        int row = id / kRowChunks, g = row % G;
        t += row / G;
#pragma unroll 4
        for (; row < BQ * G && t < p.nq; row += step) {
            T *to_row = static_cast<T *>(a.out) + (p.q0 + t) * a.o_tok + (kvh * G + g) * a.o_head;
            reinterpret_cast<uint4 *>(to_row)[c] =
                *reinterpret_cast<const uint4 *>(stage + (row * kRowChunks + (c ^ (row & 7))) * 16);
            t += dt;
            g += dg;
            if (g >= G) g -= G, ++t;
        }
    };
    const auto staged = [&](unsigned char *stage, int c) {
        return reinterpret_cast<uint4 *>(stage + (r * kRowChunks + (c ^ (r & 7))) * 16);
    };
    // this CTA's part of the row: its normalised output, and (m, l) to weigh it by
    const int64_t part_row = static_cast<int64_t>(blockIdx.x) * kPtRows + r;
    // x (columns [c, c + 32) of the row's output) plus the terms of the cleared V rows it sees
    const auto add_cleared = [&](float (&x)[32], int c, float m_row, float inv) {
        for (int w = 0; w < 4 * kMaskedTiles; ++w) {
            for (uint32_t mask = bad[w]; mask; mask &= mask - 1) {
                const int key = first_masked * kPtKeys + 32 * w + __ffs(static_cast<int>(mask)) - 1;
                if (key > last) continue;
                const T *kr = static_cast<const T *>(a.k) + (k0 + key) * a.k_tok + kvh * a.k_head;
                const T *vr = static_cast<const T *>(a.v) + (k0 + key) * a.v_tok + kvh * a.v_head;
                float s = 0.f;
                for (int d = 0; d < D; ++d) s = fmaf(to_f32<T>(q_row[d]), to_f32<T>(kr[d]), s);
                const float pr = exp2_approx(fmaf(s, a.sl2, -m_row)) * inv;
#pragma unroll
                for (int j = 0; j < 32; ++j) x[j] = fmaf(pr, to_f32<T>(vr[c + j]), x[j]);
            }
        }
    };

    if (warp < 4) {
        if constexpr (SPLIT) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        else if constexpr (SL == 1) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        else asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == 0 && lane == 0 && nt > 0) {
            // ---- TMA
            const uint64_t pol = policy_evict_last();  // K / V are read again by the other query tiles
            if (!SPLIT) {
                mbar_arrive_expect_tx(q_full, NT * (D / 64) * static_cast<uint32_t>(BQ * G) * 128u);
                for (int x = 0; x < NT; ++x)
                    for (int b = 0; b < D / 64; ++b)
                        tma_load_3d(sbase + x * Ge::kTile + b * Ge::kBox, &tq, 64 * b, kvh * G,
                                    static_cast<int32_t>(p.q0) + t0 + x * BQ, smem_addr(q_full), pol);
            }
            if (SPLIT) grid_wait();  // the split planes (Q is split here meanwhile)
            int issued = 0;
            const auto tile = [&](const CUtensorMap *map, int t) {
                for (int h = PL - 1; h >= 0; --h) {  // lo, then hi
                    const int st = issued % S;
                    if (issued >= S && !wait(&empty[st], ((issued / S) - 1) & 1)) return false;
                    mbar_arrive_expect_tx(&full[st], Ge::kTile);
#pragma unroll
                    for (int b = 0; b < D / 64; ++b)
                        tma_load_3d(sbase + Ge::kOffRing + st * Ge::kTile + b * Ge::kBox, map, 64 * b, kvh,
                                    static_cast<int32_t>(k0 + h * sp.total_k) + t * kPtKeys, smem_addr(&full[st]), pol);
                    ++issued;
                }
                return true;
            };
            bool ok = true;
            if (!kPairs) {
                ok = tile(&tk, 0) && (nt < 2 || tile(&tk, 1));
                for (int t = 0; t < nt && ok; ++t) ok = tile(&tv, t) && (t + 2 >= nt || tile(&tk, t + 2));
            } else {
                for (int t = 0; t < nt && ok; ++t) ok = tile(&tk, t) && tile(&tv, t);
            }
            // copies still landing in this CTA's shared memory
            if (!SPLIT) wait_poll(q_full, 0, nullptr);
            for (int i = max(0, issued - S); i < issued; ++i) wait_poll(&full[i % S], (i / S) & 1, nullptr);
        } else if (warp == 1 && nt > 0) {
            // ---- tensor cores
            const uint32_t e = elect_lane();
            // Every lane polls, and the warp is converged again before the next instructions: the
            // lanes share the uniform registers that these take their operands from.
            const auto all = [&](uint64_t *bar, uint32_t parity) {
                const bool ok = __all_sync(0xffffffffu, wait(bar, parity)) != 0;
                __syncwarp();
                return ok;
            };
            const auto at = [&](int pl) { return sbase + Ge::kOffRing + (pl % S) * Ge::kTile; };
            const auto landed = [&](int pl) { return all(&full[pl % S], (pl / S) & 1); };
            // S (+)= a plane of Q . a plane of K
            const auto scores = [&](int slot, uint32_t q, int pl, bool add) {
                const uint32_t d = col_s(slot), qa = desc_low(q, 16), ka = desc_low(at(pl), 16);
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {  // 16 columns: 32 bytes inside a 128-byte row
                    const uint32_t off = ((kk >> 2) * Ge::kBox + 32 * (kk & 3)) >> 4;
                    mma_ss(e, d, qa + off, ka + off, kIdS, add || kk > 0);
                }
            };
            // O (+)= P . a plane of V. P lies over the scores: 16 keys in 8 columns; F32: each 32
            // columns hold hi, then lo of their 32 keys
            const auto values = [&](int slot, bool lo, int pl, int from, int to, bool add, bool onto_lo) {
                const uint32_t d = col_o(slot), pa = col_s(slot) + (lo ? 16 : 0), va = desc_low(at(pl), Ge::kBox);
#pragma unroll
                for (int kk = from; kk < to; ++kk) {  // 16 keys: two 1024-byte atoms
                    const uint32_t pk = pa + (SPLIT ? 32 * (kk >> 1) + 8 * (kk & 1) : 8 * kk), vk = va + kk * (2048 >> 4);
                    if (onto_lo && kk == 0) mma_ts_onto_lo(e, d, pk, vk, kIdO);
                    else mma_ts(e, d, pk, vk, kIdO, add || kk > 0);
                }
            };
            constexpr int KK = kPtKeys / 16, KH = 3 * KK / 4;  // products of a V tile; of P's first part
            const auto issue_s = [&](int i) {
                const int slot = i % SL, pl = PL * plane_k<kPairs>(NT == 2 ? i >> 1 : i);
                const uint32_t q = sbase + (NT == 2 ? slot : 0) * Ge::kTile;
                if (!landed(pl)) return false;
                tc_fence_after();
                scores(slot, q, pl, false);
                if (SPLIT) {  // the small products first: the sum loses least
                    commit_if(e, &empty[pl % S]);
                    if (!landed(pl + 1)) return false;
                    tc_fence_after();
                    scores(slot, q + Ge::kTile, pl + 1, true);
                    scores(slot, q, pl + 1, true);
                }
                commit_if(e, &s_full[slot]);
                if (NT == 1 || slot == 1) commit_if(e, &empty[(pl + PL - 1) % S]);
                return true;
            };
            bool ok = all(q_full, 0);
            for (int i = 0; i < min(SL, steps) && ok; ++i) ok = issue_s(i);
            for (int i = 0; i < steps && ok; ++i) {
                const int slot = i % SL, t = NT == 2 ? i >> 1 : i, pl = PL * plane_v<kPairs>(t, nt);
                const bool check = t >= first_masked && (NT == 1 || slot == 0);
                ok = landed(pl) && (!SPLIT || !check || landed(pl + 1));
                if (!ok) break;
                if (check) {  // done while the softmax runs
                    if (e) mbar_arrive(&v_ask[t - first_masked]);
                    __syncwarp();
                }
                ok = all(&p_part[slot], (i / SL) & 1) && (!check || all(&v_ok[t - first_masked], 0)) &&
                     (!SPLIT || i < 2 || all(&o_empty[slot], ((i >> 1) - 1) & 1));
                if (!ok) break;
                tc_fence_after();
                if (SPLIT) {
                    values(slot, false, pl, 0, KK, false, false);
                    commit_if(e, &empty[pl % S]);
                    ok = landed(pl + 1);
                    if (!ok) break;
                    tc_fence_after();
                    values(slot, true, pl + 1, 0, KK, true, true);
                    values(slot, false, pl + 1, 0, KK, true, false);
                } else {
                    values(slot, false, pl, 0, KH, i >= SL, false);
                    ok = all(&p_full[slot], (i / SL) & 1);
                    if (!ok) break;
                    tc_fence_after();
                    values(slot, false, pl, KH, KK, true, false);
                }
                if (NT == 1 || slot == 1) commit_if(e, &empty[(pl + PL - 1) % S]);
                if (SPLIT || i + SL >= steps) commit_if(e, &o_final[slot]);
                if (i + SL < steps) ok = issue_s(i + SL);
            }
            // no product may still use tensor memory or the ring when the CTA exits
            commit_if(e, idle);
            wait_poll(idle, 0, nullptr);
        } else if (warp >= 2) {
            // ---- V check: rows of the masked tiles that hold Inf or NaN, cleared and noted
            constexpr uint32_t kExp = kBf16 ? 0x7F80u : 0x7C00u;
            for (int t = first_masked; t < nt; ++t) {
                const int pl = PL * plane_v<kPairs>(t, nt);
                // the tensor-core warp has seen this phase of `full` and holds it until the
                // check is done, so its parity is not ambiguous here
                if (!__all_sync(0xffffffffu, wait(&v_ask[t - first_masked], 0) && wait(&full[pl % S], (pl / S) & 1) &&
                                                 (!SPLIT || wait(&full[(pl + 1) % S], ((pl + 1) / S) & 1))))
                    break;
                unsigned char *v = base + Ge::kOffRing + (pl % S) * Ge::kTile;
                unsigned char *v2 = base + Ge::kOffRing + ((pl + PL - 1) % S) * Ge::kTile;  // F32: both planes
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int row = 64 * half + (warp - 2) * 32 + lane;
                    bool odd = false;
#pragma unroll 4
                    for (int c = 0; c < PL * D / 8; ++c) {
                        const uint4 u = *reinterpret_cast<const uint4 *>(
                            (c < D / 8 ? v : v2) + ((c % (D / 8)) >> 3) * Ge::kBox + row * 128 + (((c & 7) ^ (row & 7)) << 4));
                        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            odd |= (w[j] & kExp) == kExp || ((w[j] >> 16) & kExp) == kExp;
                    }
                    const uint32_t mask = __ballot_sync(0xffffffffu, odd);
                    if (mask) {
                        for (int c = 0; odd && c < D / 8; ++c) {
                            const uint32_t off = (c >> 3) * Ge::kBox + row * 128 + (c & 7) * 16;
                            *reinterpret_cast<uint4 *>(v + off) = make_uint4(0, 0, 0, 0);
                            *reinterpret_cast<uint4 *>(v2 + off) = make_uint4(0, 0, 0, 0);
                        }
                        if (lane == 0) {
                            bad[(t - first_masked) * 4 + row / 32] = mask;
                            bad[4 * kMaskedTiles] = 1;
                        }
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(&v_ok[t - first_masked]);
            }
        }
    } else if (SPLIT && warp >= 12) {
        // ---- F32: the output's sum
        if constexpr (SPLIT) {
            asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
            float2 *stat = reinterpret_cast<float2 *>(base + Ge::kOffStat);  // [slot][row]
            const int32_t *exps = sp.exps + (split_index(p.k0, p.seq, ta) * a.Hkv + kvh) * 2;
            const int64_t ex_step = static_cast<int64_t>(a.Hkv) * 2;
            // the steps' O added up. Step i holds sum p v = O 2^(m + ev); l counts in 2^m
            float acc[D], L = 0.f, M = -INFINITY, R = -INFINITY;
#pragma unroll
            for (int d = 0; d < D; ++d) acc[d] = 0.f;
            // The exponents. (They are read by plain loads: a load through the read-only path may be moved
            // ahead of the wait, to where the split kernel is still at work.)
            grid_wait();
            int word = steps > 0 ? __ldcg(exps + 1) : 0;
            bool ok = true, wide = false;
#pragma unroll 1
            for (int i = 0; i < steps; ++i) {
                const int sl = i & 1;
                ok = __all_sync(0xffffffffu, wait(&st_full[sl], (i >> 1) & 1) && wait(&o_final[sl], (i >> 1) & 1));
                if (!ok) break;
                tc_fence_after();
                const float2 st = stat[sl * kPtRows + r];
                const float e = st.x + static_cast<float>(exps_exponent(word));
                wide |= exps_wide(word);
                if (i + 1 < steps) word = __ldcg(exps + (i + 1) * ex_step + 1);
                if (st.x > M) {
                    L *= exp2_approx(M - st.x);
                    M = st.x;
                }
                const float f_l = st.x == -INFINITY ? 0.f : exp2_approx(st.x - M);
                L = fmaf(f_l, st.y, L);
                const float Rn = fmaxf(R, e);
                const float f_old = R == -INFINITY ? 0.f : exp2_approx(R - Rn);
                const float f_new = e == -INFINITY ? 0.f : exp2_approx(e - Rn);
                if (__any_sync(0xffffffffu, Rn > R)) {
#pragma unroll
                    for (int d = 0; d < D; ++d) acc[d] *= f_old;
                }
                R = Rn;
#pragma unroll
                for (int c = 0; c < D / 16; ++c) {
                    float o[16];
                    tc_ld16(col_o(sl) + lanes + 16 * c, o);
#pragma unroll
                    for (int j = 0; j < 16; ++j) acc[16 * c + j] = fmaf(o[j], f_new, acc[16 * c + j]);
                }
                tc_fence_before();
                mbar_arrive(&o_empty[sl]);
            }
            const float inv = L != 0.f ? 1.0f / L : 0.f;  // a row that sees no key: zeros
            // P and l both carry 2^kTop; two factors, neither of which overflows
            const float half = R == -INFINITY ? 0.f : 0.5f * (R - M);
            const float undo = exp2_approx(half);
            if (steps == 0) ok = __all_sync(0xffffffffu, wait(q_full, 0));  // Q's planes are written by now
            if (wide) any_wide = 1;
            named_sync(4, 384);
            ok = ok && !any_wide;  // else the softmax threads do the rows over
            if (ok && sp.parts > 1 && live) sp.part_ml[part_row] = make_float2(M, L);
            if (ok) {
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    float x[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j) x[j] = acc[32 * c + j] * inv * undo * undo;
                    if (sp.parts == 1) {  // over Q: every product with it is complete
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            *reinterpret_cast<float4 *>(staged(base, 8 * c + j)) =
                                make_float4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
                    } else if (live) {
#pragma unroll
                        for (int j = 0; j < 32; j += 4)
                            *reinterpret_cast<float4 *>(sp.part_o + part_row * D + 32 * c + j) =
                                make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
                    }
                }
            }
            named_sync(2, 128);
            if (sp.parts == 1 && ok && some) store_rows(base, t0, r, 128);
        }
    } else if constexpr (SPLIT) {
        // ---- F32 softmax
        asm volatile("setmaxnreg.dec.sync.aligned.u32 120;");
        float2 *stat = reinterpret_cast<float2 *>(base + Ge::kOffStat);  // [slot][row]
        const int32_t *exps = sp.exps + (split_index(p.k0, p.seq, ta) * a.Hkv + kvh) * 2;
        const int64_t ex_step = static_cast<int64_t>(a.Hkv) * 2;
        // the row of Q as hi and lo planes: this warpgroup writes half of its columns
        const float4 *q4 = reinterpret_cast<const float4 *>(q_row) + slot * (D / 8);
        float4 x[D / 8];
#pragma unroll
        for (int c = 0; c < D / 8; ++c) x[c] = live ? __ldg(q4 + c) : make_float4(0.f, 0.f, 0.f, 0.f);
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < D / 8; ++c)
            top = max(max(top, max(finite_magnitude(x[c].x), finite_magnitude(x[c].y))),
                      max(finite_magnitude(x[c].z), finite_magnitude(x[c].w)));
        uint32_t *tops = reinterpret_cast<uint32_t *>(stat);  // free until the first scores
        tops[slot * kPtRows + r] = top;
        named_sync(3, 256);
        top = max(top, tops[(slot ^ 1) * kPtRows + r]);
        const int eq = top ? top_exponent(top) - kTop : 0;
        const float s = pow2(-eq);
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {  // 16-byte chunks of eight halves
            const uint64_t s2 = pair_of(s, s), e[4] = {pair_of(x[2 * c].x, x[2 * c].y), pair_of(x[2 * c].z, x[2 * c].w),
                                                       pair_of(x[2 * c + 1].x, x[2 * c + 1].y),
                                                       pair_of(x[2 * c + 1].z, x[2 * c + 1].w)};
            uint32_t h[4], lo[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) split_f16x2(mul_pair(e[j], s2), h[j], lo[j]);
            const int chunk = slot * (D / 16) + c;
            unsigned char *at = base + (chunk >> 3) * Ge::kBox + r * 128 + (((chunk & 7) ^ (r & 7)) << 4);
            *reinterpret_cast<uint4 *>(at) = make_uint4(h[0], h[1], h[2], h[3]);
            *reinterpret_cast<uint4 *>(at + Ge::kTile) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(q_full);
        grid_wait();  // the exponents
        const uint32_t ts = col_s(slot) + lanes;
        int word = slot < steps ? __ldcg(exps + slot * ex_step) : 0;
        bool wide = false;
#pragma unroll 1
        for (int i = slot; i < steps; i += 2) {
            const int ex = exps_exponent(word) + eq;
            wide |= exps_wide(word) || ex > kMostScale;
            const float sl2 = a.sl2 * pow2(ex >> 1) * pow2(ex - (ex >> 1));  // (one factor ends at 2^-126)
            if (i + 2 < steps) word = __ldcg(exps + (i + 2) * ex_step);
            if (!__all_sync(0xffffffffu, wait(&s_full[slot], (i >> 1) & 1))) break;
            tc_fence_after();
            const int vis = last + 1 - i * kPtKeys;  // keys of the tile the row sees
            const bool whole = __all_sync(0xffffffffu, vis >= kPtKeys);
            // hidden keys: scores of -inf, written back so that the second reading sees them too
            float mx[8];
#pragma unroll
            for (int c = 0; c < 4; c += 2) {
                uint32_t sv[2][32];
                tc_ld32_nowait(ts + 32 * c, sv[0]);
                tc_ld32_nowait(ts + 32 * c + 32, sv[1]);
                tc_wait_ld();
                tc_reg_fence(sv[0]);
                tc_reg_fence(sv[1]);
                if (!whole) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (32 * (c + h) + j >= vis) sv[h][j] = 0xFF800000u;
                        tc_st32(ts + 32 * (c + h), sv[h]);
                    }
                    tc_wait_st();
                }
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        const float u = __uint_as_float(sv[h][j]), v = __uint_as_float(sv[h][j + 1]);
                        float &best = mx[(j >> 1) & 7];
                        best = c == 0 && h == 0 && j < 16 ? fmaxf(u, v) : max3(best, u, v);
                    }
            }
            const float m = max3(max3(mx[0], mx[1], mx[2]), max3(mx[3], mx[4], mx[5]), fmaxf(mx[6], mx[7])) * sl2;
            const float shift_p = static_cast<float>(kTop) - (m == -INFINITY ? 0.f : m);
            const uint64_t scale2 = pair_of(sl2, sl2), shift2 = pair_of(shift_p, shift_p);
            uint64_t sum2[4] = {};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t sv[32], pv[32];
                tc_ld32_nowait(ts + 32 * c, sv);
                tc_wait_ld();
                tc_reg_fence(sv);
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float2 y =
                        of_pair(fma_pair(pair_of(__uint_as_float(sv[2 * j]), __uint_as_float(sv[2 * j + 1])), scale2, shift2));
                    const uint64_t e2 = pair_of(exp2_approx(y.x), exp2_approx(y.y));
                    sum2[j & 3] = add_pair(sum2[j & 3], e2);
                    split_f16x2(e2, pv[j], pv[16 + j]);
                }
                tc_st32(ts + 32 * c, pv);
            }
            const float2 sum = of_pair(add_pair(add_pair(sum2[0], sum2[1]), add_pair(sum2[2], sum2[3])));
            // the slot's last step has been added up (long since, as a rule), so its (m, l) too
            if (i >= 2 && !__all_sync(0xffffffffu, wait(&o_empty[slot], ((i >> 1) - 1) & 1))) break;
            stat[slot * kPtRows + r] = make_float2(m, sum.x + sum.y);
            mbar_arrive(&st_full[slot]);
            tc_wait_st();
            tc_fence_before();
            mbar_arrive(&p_part[slot]);
        }
        if (wide) any_wide = 1;
        named_sync(4, 384);  // every product is complete
        if (any_wide) {
            const int rows = min(BQ, p.nq - t0) * G, from = ta * kPtKeys, to = (ta + nt) * kPtKeys;
            for (int r0 = 0; r0 < rows; r0 += kPkRows) {
                named_sync(5, kPkThreads);  // the last rows' shared memory is free
                ffma_rows<float, D>(
                    a, p, kvh, t0 * G + r0, min(kPkRows, rows - r0), from, to, reinterpret_cast<float *>(base), threadIdx.x - 128,
                    [] { named_sync(5, kPkThreads); },
                    [&](int row, int c, const float (&x)[4], float m, float l) {
                        row += r0;
                        if (sp.parts == 1) {
                            float *to_row = static_cast<float *>(a.out) + (p.q0 + t0 + row / G) * a.o_tok + (kvh * G + row % G) * a.o_head;
                            *reinterpret_cast<float4 *>(to_row + c) = make_float4(x[0], x[1], x[2], x[3]);
                        } else {
                            const int64_t at = static_cast<int64_t>(blockIdx.x) * kPtRows + row;
                            *reinterpret_cast<float4 *>(sp.part_o + at * D + c) = make_float4(x[0], x[1], x[2], x[3]);
                            if (c == 0) sp.part_ml[at] = make_float2(m, l * pow2(kTop));  // as the other parts' sums
                        }
                    });
            }
        }
    } else {
        // ---- softmax
        if constexpr (SL == 1) asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
        else asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const uint32_t ts = col_s(slot) + lanes, to = col_o(slot) + lanes;
        float m = -INFINITY, l = 0.f;
        bool ok = true;
#pragma unroll 1
        for (int i = slot; i < steps; i += SL) {
            ok = __all_sync(0xffffffffu, wait(&s_full[slot], (i / SL) & 1));
            if (!ok) break;
            tc_fence_after();
            uint32_t sv[4][32];
#pragma unroll
            for (int c = 0; c < 4; ++c) tc_ld32_nowait(ts + 32 * c, sv[c]);
            tc_wait_ld();
#pragma unroll
            for (int c = 0; c < 4; ++c) tc_reg_fence(sv[c]);
            const int vis = last + 1 - (NT == 2 ? i >> 1 : i) * kPtKeys;  // keys of the tile the row sees
            const bool whole = __all_sync(0xffffffffu, vis >= kPtKeys);
            if (!whole) {
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (32 * c + j >= vis) sv[c][j] = 0xFF800000u;
            }
            float mx[8];  // (a NaN stays: such a row's weights must not go by the polynomial)
#pragma unroll
            for (int j = 0; j < 8; ++j) mx[j] = max2_nan(__uint_as_float(sv[0][2 * j]), __uint_as_float(sv[0][2 * j + 1]));
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int j = c == 0 ? 16 : 0; j < 32; j += 2)
                    mx[(j >> 1) & 7] = max3_nan(mx[(j >> 1) & 7], __uint_as_float(sv[c][j]), __uint_as_float(sv[c][j + 1]));
            const float top = max3_nan(max3_nan(mx[0], mx[1], mx[2]), max3_nan(mx[3], mx[4], mx[5]), max2_nan(mx[6], mx[7])) * a.sl2;
            float alpha = 1.f;
            bool grow = false;
            if (m == -INFINITY) {
                m = top;  // nothing summed so far: O and l are zero, or not yet written
            } else if (top > m + kPtRescale) {
                alpha = exp2_approx(m - top);
                m = top;
                grow = true;
            }
            // with a NaN or +inf among its scores a row has no weights, with -inf alone they are 0: not for the polynomial
            const bool odd = whole && !(fabsf(top) < INFINITY);
            bool by_poly = whole;
            if (__any_sync(0xffffffffu, grow || odd)) {
                by_poly = whole && !__any_sync(0xffffffffu, odd);
                // every earlier product of this slot completed before its scores did
                l *= alpha;
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t o[32];
                    tc_ld32_nowait(to + 32 * c, o);
                    tc_wait_ld();
                    tc_reg_fence(o);
#pragma unroll
                    for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
                    tc_st32(to + 32 * c, o);
                }
            }
            const float ms = m == -INFINITY ? 0.f : m;
            const uint64_t scale2 = pair_of(a.sl2, a.sl2), minus2 = pair_of(-ms, -ms);
            uint64_t sum[4] = {pair_of(l, 0.f), 0, 0, 0};
            // every kPolyStep-th pair by polynomial: the special-function unit takes 8 cycles a warp
            // instruction and does not overlap much with the rest of one warp's work
            const auto weigh = [&](auto poly) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t pv[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const uint64_t s2 = pair_of(__uint_as_float(sv[c][2 * j]), __uint_as_float(sv[c][2 * j + 1]));
                        const float2 x = of_pair(fma_pair(s2, scale2, minus2));
                        const float2 y = decltype(poly)::value && j % kPolyStep == kPolyStep - 1
                                             ? exp2_poly_pair<kBf16>(x)
                                             : make_float2(exp2_approx(x.x), exp2_approx(x.y));
                        sum[j & 3] = add_pair(sum[j & 3], pair_of(y.x, y.y));
                        pv[j] = pack_pair<T>(y.x, y.y);
                    }
                    tc_st16(ts + 16 * c, pv);
                    if (c == 2) {  // the tensor cores may start on the first 96 keys
                        tc_wait_st();
                        tc_fence_before();
                        mbar_arrive(&p_part[slot]);
                    }
                }
            };
            if (by_poly) weigh(std::true_type{});
            else weigh(std::false_type{});
            const float2 two = of_pair(add_pair(add_pair(sum[0], sum[1]), add_pair(sum[2], sum[3])));
            l = two.x + two.y;
            tc_wait_st();
            tc_fence_before();
            mbar_arrive(&p_full[slot]);
        }
        const bool mine = steps > slot;  // the slot had a step
        if (ok && mine) ok = __all_sync(0xffffffffu, wait(&o_final[slot], 0));
        tc_fence_after();
        // the row's output: O / l, plus what the cleared V rows would have added
        float m_row = m, l_row = l, f_own = 1.f, f_other = 0.f;
        constexpr int NC = kJoin ? D / 64 : D / 32;  // 32-column pieces this thread writes
        const int c0 = kJoin ? slot * NC : 0;
        if constexpr (kJoin) {
            // the slots' halves of the key tiles, joined: each warpgroup hands the other half of
            // its columns over through the ring (no copy or product uses it any more)
            float2 *stat = reinterpret_cast<float2 *>(base);  // over Q: every product with it is complete
            float *xch = reinterpret_cast<float *>(base + Ge::kOffRing) + slot * (D / 2) * kPtRows;
            named_sync(1, 256);  // both slots' products are complete
            stat[slot * kPtRows + r] = make_float2(m, mine ? l : 0.f);
            if (ok && mine) {
#pragma unroll 1
                for (int c = 0; c < NC; ++c) {
                    uint32_t o[32];
                    tc_ld32_nowait(to + 32 * ((slot ^ 1) * NC + c), o);
                    tc_wait_ld();
                    tc_reg_fence(o);
#pragma unroll
                    for (int j = 0; j < 32; ++j) xch[(32 * c + j) * kPtRows + r] = __uint_as_float(o[j]);
                }
            }
            named_sync(1, 256);
            const float2 other = stat[(slot ^ 1) * kPtRows + r];
            m_row = fmaxf(m, other.x);
            const float mm = m_row == -INFINITY ? 0.f : m_row;
            f_own = mine ? exp2_approx(m - mm) : 0.f;
            f_other = exp2_approx(other.x - mm);
            l_row = (mine ? l * f_own : 0.f) + other.y * f_other;
        }
        const float inv = l_row != 0.f ? 1.0f / l_row : 0.f;  // a row that sees no key: zeros
        // over the slot's query tile; kJoin: in the ring behind what the slots exchanged
        unsigned char *stage = base + (kJoin ? Ge::kOffRing + D * kPtRows * 4 : slot * Ge::kTile);
        if (ok) {
            const bool any_bad = bad[4 * kMaskedTiles] != 0;
            const float *got = reinterpret_cast<const float *>(base + Ge::kOffRing) + (slot ^ 1) * (D / 2) * kPtRows;
            const bool other_has = kJoin && steps > (slot ^ 1);
#pragma unroll 1
            for (int c = 0; c < NC; ++c) {
                uint32_t o[32];
                if (mine) {
                    tc_ld32_nowait(to + 32 * (c0 + c), o);
                    tc_wait_ld();
                    tc_reg_fence(o);
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) o[j] = 0;
                }
                float x[32];
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    x[j] = __uint_as_float(o[j]);
                    if (kJoin) x[j] = x[j] * f_own + (other_has ? got[(32 * c + j) * kPtRows + r] * f_other : 0.f);
                    x[j] *= inv;
                }
                if (any_bad && live) add_cleared(x, 32 * (c0 + c), m_row, inv);
                if (sp.parts == 1) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        *staged(stage, 4 * (c0 + c) + j) =
                            make_uint4(pack_pair<T>(x[8 * j], x[8 * j + 1]), pack_pair<T>(x[8 * j + 2], x[8 * j + 3]),
                                       pack_pair<T>(x[8 * j + 4], x[8 * j + 5]), pack_pair<T>(x[8 * j + 6], x[8 * j + 7]));
                } else if (live) {
#pragma unroll
                    for (int j = 0; j < 32; j += 4)
                        *reinterpret_cast<float4 *>(sp.part_o + part_row * D + 32 * (c0 + c) + j) =
                            make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
                }
            }
        }
        if (sp.parts > 1) {
            if (live && slot == 0) sp.part_ml[part_row] = make_float2(m_row, l_row);
        } else if constexpr (!kJoin) {
            named_sync(2 + slot, 128);
            if (ok && some) store_rows(stage, t0 + slot * BQ, r, 128);
        } else {
            named_sync(1, 256);
            if (ok && some) store_rows(stage, t0, 128 * slot + r, 256);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 2) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kColumns) : "memory");
    }
}

// rows x heads x D as {D, heads, rows} with boxes of 64 elements (128 bytes, swizzled)
bool row_map(CUtensorMap *m, bool bf16, const void *base, int64_t D, int64_t heads, int64_t rows, int64_t head, int64_t tok,
             int box_heads, int box_rows) {
    const uint64_t dims[3] = {static_cast<uint64_t>(D), static_cast<uint64_t>(heads), static_cast<uint64_t>(rows)};
    const uint64_t strides[2] = {static_cast<uint64_t>(head) * 2, static_cast<uint64_t>(tok) * 2};
    const uint32_t box[3] = {64, static_cast<uint32_t>(box_heads), static_cast<uint32_t>(box_rows)};
    return tma_encode(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, base, 3, dims, strides,
                      box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// The parts of each row joined, o = sum l_i 2^(m_i - M) o_i / sum l_i 2^(m_i - M): kPtJoinCtas CTAs per
// (query tile, KV head), a warp per row. A launch and one dependent read bound it (~4 us).
constexpr int kPtJoinThreads = 256, kPtJoinCtas = 8;
template <typename T, int D>
__global__ void __launch_bounds__(kPtJoinThreads) packed_join_kernel(const PackedArgs a, const SplitView sp) {
    constexpr int E = D / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, BQ = kPtRows / a.G;
    const PackedTile p =
        find_packed_tile(a.cu_q, a.cu_k, a.n_seqs, a.total_q, a.total_k, 1, BQ, blockIdx.x / (a.Hkv * kPtJoinCtas), nullptr);
    const int at = blockIdx.x / kPtJoinCtas, kvh = at % a.Hkv;
    grid_wait();
    if (p.seq < 0) return;
    const int rows = min(BQ, p.nq - p.tile * BQ) * a.G;
    const int64_t first = static_cast<int64_t>(at) * sp.parts * kPtRows;
    for (int r = blockIdx.x % kPtJoinCtas + kPtJoinCtas * warp; r < rows; r += kPtJoinCtas * kPtJoinThreads / 32) {
        const float2 ml = lane < sp.parts ? __ldcg(sp.part_ml + first + lane * kPtRows + r) : make_float2(-INFINITY, 0.f);
        const float M = warp_max(ml.x);
        const float w = ml.y == 0.f ? 0.f : ml.y * exp2_approx(ml.x - (M == -INFINITY ? 0.f : M));
        const float sum = warp_sum(w);
        float o[E] = {};
        for (int i = 0; i < sp.parts; ++i) {
            const float f = __shfl_sync(0xffffffffu, w, i);
            if (f == 0.f) continue;  // a part without keys for this row holds nothing
            const float *src = sp.part_o + (first + i * kPtRows + r) * D + E * lane;
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = fmaf(f, __ldcg(src + e), o[e]);
        }
        const float inv = sum != 0.f ? 1.0f / sum : 0.f;
        T *dst = static_cast<T *>(a.out) + (p.q0 + p.tile * BQ + r / a.G) * a.o_tok + (kvh * a.G + r % a.G) * a.o_head;
#pragma unroll
        for (int e = 0; e < E; ++e) dst[E * lane + e] = from_f32<T>(o[e] * inv);
    }
}

// How a call is cut: query tiles a CTA, parts of the keys, CTAs at most.
struct PtPlan {
    int nt, slots, parts;
    int64_t ctas;
};
PtPlan pt_plan(int64_t n_seqs, int64_t total_q, int64_t total_k, int64_t G, int64_t Hkv, int32_t dtype) {
    const int64_t sms = device_sm_count(), BQ = kPtRows / G;
    PtPlan p = {1, 2, 1, 0};
    // 16-bit types, us for one tile in two slots / one tile in one slot / two tiles:
    //  * long contexts: two tiles once such CTAs fill the SMs, else one in two slots (16 / 8 heads of
    //    128: 2048 tokens 36 / 40 / 41, 4096 tokens 91 / 82 / 73, 8192 tokens 259 / 257 / 228);
    //  * shorter ones: one slot and two CTAs an SM once the tiles outnumber the SMs: a CTA's start and end, ~6
    //    us, then run beside another's work (10 prompts of 1 to 1333 tokens 53 / 39 / 45, 32 of 64 27 / 18 / 27,
    //    16 of 300 53 / 37 / 41, 4 of 1024 53 / 39 / 39; but one of 2048 among short ones 35 / 39 / 41).
    if (dtype != B200_DTYPE_F32) {
        if (total_k / max64(1, n_seqs) >= 8 * kPtKeys) p.nt = total_q / (2 * BQ) * Hkv >= sms ? 2 : 1;
        else if (most_packed_tiles(n_seqs, total_q, 1, BQ) * Hkv > sms) p.slots = 1;
    }
    const int64_t tiles = most_packed_tiles(n_seqs, total_q, 1, p.nt * BQ) * Hkv;
    if (p.nt == 1 && tiles > 0) {
        // As many parts as the SMs allow, each of so many key tiles of a mean sequence at least that the
        // shorter chain pays for the join, a launch of ~4 us. A 16-bit tile takes ~1 us, an F32 one ~3 (one
        // part against the parts taken here: one BF16 token, 1601 keys, 8 / 4 heads 24.6 us against 21.5,
        // 8001 keys 71 against 26; but 200 tokens, 1500 keys 23.5 against 25.6 in two, so they stay whole.
        // F32, 16 / 8 heads: 128 tokens, 1128 keys 52 against 50; 512 tokens 36, in two 40).
        const int64_t keys = total_k / max64(1, n_seqs) / ((dtype == B200_DTYPE_F32 ? 4 : 6) * kPtKeys);
        p.parts = static_cast<int>(max64(1, min64(8, min64(sms / tiles, keys))));
    }
    p.ctas = tiles * p.parts;
    return p;
}

size_t split_bytes(int64_t n_seqs, int64_t total_k, int64_t D, int64_t Hkv, int32_t dtype) {
    if (dtype != B200_DTYPE_F32) return 0;
    // hi and lo planes of K and V, and the tiles' exponents
    const size_t n = static_cast<size_t>(total_k * Hkv * D * 8 + (total_k / kPtKeys + n_seqs + 1) * Hkv * 8);
    return (n + 255) / 256 * 256;
}

template <typename T, int D, int NT, int SL>
cudaError_t pt_launch(const PackedArgs &a, const PtPlan &plan, cudaStream_t st) {
    constexpr bool bf16 = __is_same(T, __nv_bfloat16), split = __is_same(T, float);
    using Ge = PtGeometry<D, NT, SL, split ? 2 : 1>;
    auto kern = packed_tc_kernel<T, D, NT, SL>;
    cudaError_t e = once_per_device(reinterpret_cast<const void *>(kern), ATTR_SMEM, [&] {
        return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Ge::kSmem));
    });
    if (e != cudaSuccess) return e;
    const int BQ = kPtRows / a.G;
    if (plan.ctas > INT32_MAX / kPtJoinCtas) return cudaErrorNotSupported;
    CUtensorMap mq = {}, mk, mv;
    SplitView sp;
    sp.parts = plan.parts;
    // an order matters to CTAs that wait for others; parts (and the join's order) come with fewer CTAs
    sp.by_weight = a.n_seqs > 1 && a.n_seqs <= 32 && plan.parts == 1 && plan.ctas > device_sm_count();
    if (plan.parts > 1) {
        char *parts = static_cast<char *>(a.ws) + split_bytes(a.n_seqs, a.total_k, D, a.Hkv, a.dtype);
        sp.part_ml = reinterpret_cast<float2 *>(parts);
        sp.part_o = reinterpret_cast<float *>(sp.part_ml + plan.ctas * kPtRows);
    }
    if constexpr (split) {
        const int64_t plane = a.total_k * a.Hkv * D;
        __half *planes = static_cast<__half *>(a.ws);
        int32_t *exps = reinterpret_cast<int32_t *>(planes + 4 * plane);
        sp.exps = exps;
        sp.total_k = a.total_k;
        const int64_t tiles = most_packed_tiles(a.n_seqs, a.total_k, 1, kPtKeys) * a.Hkv * 2;
        if (tiles > INT32_MAX || 2 * a.total_k > INT32_MAX - 1024 ||
            !row_map(&mk, false, planes, D, a.Hkv, 2 * a.total_k, D, a.Hkv * D, 1, kPtKeys) ||
            !row_map(&mv, false, planes + 2 * plane, D, a.Hkv, 2 * a.total_k, D, a.Hkv * D, 1, kPtKeys))
            return cudaErrorNotSupported;
        mq = mk;  // not used
        e = b200_launch(packed_split_kernel<D>, dim3(static_cast<unsigned>(tiles)), dim3(kSplitThreads), 0, st, false, a,
                        planes, exps);
        if (e != cudaSuccess) return e;
    } else {
        if (!row_map(&mq, bf16, a.q, D, a.Hq, a.total_q, a.q_head, a.q_tok, a.G, BQ) ||
            !row_map(&mk, bf16, a.k, D, a.Hkv, a.total_k, a.k_head, a.k_tok, 1, kPtKeys) ||
            !row_map(&mv, bf16, a.v, D, a.Hkv, a.total_k, a.v_head, a.v_tok, 1, kPtKeys))
            return cudaErrorNotSupported;
    }
    e = b200_launch(kern, dim3(static_cast<unsigned>(plan.ctas)), dim3(kPtThreads<T, SL>), Ge::kSmem, st, split, mq, mk, mv, a,
                    sp);
    if (e != cudaSuccess || plan.parts == 1) return e;
    return b200_launch(packed_join_kernel<T, D>, dim3(static_cast<unsigned>(plan.ctas / plan.parts * kPtJoinCtas)),
                       dim3(kPtJoinThreads), 0, st, true, a, sp);
}

template <typename T, int D>
cudaError_t pt_by_tiles(const PackedArgs &a, const PtPlan &plan, cudaStream_t st) {
    if constexpr (!__is_same(T, float))
        if (plan.nt == 2) return pt_launch<T, D, 2, 2>(a, plan, st);
    if constexpr (!__is_same(T, float))
        if (plan.slots == 1) return pt_launch<T, D, 1, 1>(a, plan, st);
    return pt_launch<T, D, 1, 2>(a, plan, st);
}

template <typename T>
cudaError_t pt_by_dim(const PackedArgs &a, const PtPlan &plan, cudaStream_t st) {
    return a.D == 128 ? pt_by_tiles<T, 128>(a, plan, st) : pt_by_tiles<T, 64>(a, plan, st);
}

}  // namespace

size_t packed_tc_workspace(int64_t n_seqs, int64_t total_q, int64_t total_k, int64_t D, int64_t Hq, int64_t Hkv,
                           int32_t dtype) {
    if (Hq / Hkv > kPtRows) return 0;
    const PtPlan plan = pt_plan(n_seqs, total_q, total_k, Hq / Hkv, Hkv, dtype);
    return split_bytes(n_seqs, total_k, D, Hkv, dtype) +
           (plan.parts > 1 ? static_cast<size_t>(plan.ctas) * kPtRows * (D * 4 + 8) : 0);
}

cudaError_t packed_tc_launch(const PackedArgs &a, cudaStream_t st) {
    if (a.total_k == 0 || a.G > kPtRows) return cudaErrorNotSupported;
    const PtPlan plan = pt_plan(a.n_seqs, a.total_q, a.total_k, a.G, a.Hkv, a.dtype);
    switch (a.dtype) {
        case B200_DTYPE_F16: return pt_by_dim<__half>(a, plan, st);
        case B200_DTYPE_BF16: return pt_by_dim<__nv_bfloat16>(a, plan, st);
    }
    return pt_by_dim<float>(a, plan, st);
}

}  // namespace b200
