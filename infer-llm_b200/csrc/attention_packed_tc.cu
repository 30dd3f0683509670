// Packed causal attention on the 5th-generation tensor cores for F16 and BF16.
//
// A CTA owns two slots, each a 128-row accumulator: scores S (128 x 128 keys) and output O
// (128 x D) in tensor memory, and one softmax warpgroup with a thread per row. A step i
// belongs to slot i % 2:
//   S = Q . K^T           (M 128, N 128 keys, K D; both operands in shared memory)
//   P = 2^(S sl2 - m)     (softmax warps; 16-bit P written over S in tensor memory)
//   O += P . V            (M 128, N D, K 128 keys; A = P from tensor memory)
// While one slot's softmax runs, the tensor cores work for the other. The slots are
//   NT = 2: two query tiles over the same key tiles (K and V are read once for both);
//   NT = 1: one query tile, even key tiles in slot 0 and odd ones in slot 1, joined at the
//           end (half as long a chain for calls with few query tiles).
// A query tile's rows are tokens times the G heads of a KV head (row = token * G + head), as
// many whole tokens as fit 128 rows, so the heads that share keys share every tile.
// Warp roles: warp 0 TMA, warp 1 tensor cores, warps 2-3 V check, warps 4-11 softmax.
//   * The running maximum moves only when it grows by more than 2^8, so rescaling O is rare
//     (the result is unchanged: every p is bounded by 2^8). Statistics are F32; P is
//     rounded to the element type, the sum is taken before that.
//   * Hidden keys of a tile (past a row's last key, of the next sequence, or past the end)
//     have P = 0, but 0 times a V that is no number is not 0. The V check looks for such
//     rows in the tiles that hide keys, clears them in shared memory, and notes them; rows that do
//     see one of them add its term in the epilogue.
// Every mbarrier wait is bounded; one that runs out records B200_DEV_TIMEOUT, and the CTA
// waits (bounded) for its copies and products and frees its tensor memory.
#include "attention_packed.cuh"
#include "gemv.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace b200 {
namespace {

constexpr int kPtRows = 128, kPtKeys = 128;
constexpr int kPtThreads = 384;
constexpr int kMaskedTiles = 4;  // key tiles in which some row of a CTA hides keys (at most 256 tokens)
constexpr float kPtRescale = 8.0f;

template <int D, int NT>
struct PtGeometry {
    static constexpr uint32_t kBox = kPtKeys * 128;           // 64 elements of 128 rows
    static constexpr uint32_t kTile = (D / 64) * kBox;        // a 128-row tile of Q, K or V
    static constexpr int kStages = D == 128 ? (NT == 2 ? 5 : 6) : 8;
    static constexpr uint32_t kOffRing = NT * kTile;
    static constexpr uint32_t kOffBar = kOffRing + kStages * kTile;
    static constexpr uint32_t kOffBad = kOffBar + 320;        // [kMaskedTiles][4] words, then "any"
    static constexpr size_t kSmem = 1024 + kOffBad + 128;
};

// The planes (K or V tiles) of a key-tile sequence in the order of their first use.
template <int NT>
B200_DEVICE int plane_k(int t) { return NT == 2 ? 2 * t : (t == 0 ? 0 : 2 * t - 1); }
template <int NT>
B200_DEVICE int plane_v(int t, int n) { return NT == 2 ? 2 * t + 1 : t + min(t + 2, n); }

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

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kPtThreads, 1)
    packed_tc_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                     const __grid_constant__ CUtensorMap tv, const PackedArgs a) {
    using Ge = PtGeometry<D, NT>;
    constexpr bool kBf16 = !__is_same(T, __half);
    constexpr uint32_t kIdS = idesc_f16(kPtRows, kPtKeys, kBf16, false, false);
    constexpr uint32_t kIdO = idesc_f16(kPtRows, D, kBf16, false, true);
    constexpr int S = Ge::kStages;
    extern __shared__ unsigned char pt_raw[];
    const uint32_t raw = smem_addr(pt_raw);
    const uint32_t sbase = (raw + 1023u) & ~1023u;
    unsigned char *base = pt_raw + (sbase - raw);
    uint64_t *bars = reinterpret_cast<uint64_t *>(base + Ge::kOffBar);
    uint64_t *full = bars;            // [S] plane landed
    uint64_t *empty = bars + S;       // [S] plane read by its last product
    uint64_t *q_full = bars + 2 * S;
    uint64_t *s_full = q_full + 1;    // [2] scores of the slot's step complete (and all earlier products)
    uint64_t *p_full = s_full + 2;    // [2] P written, O rescaled
    uint64_t *o_final = p_full + 2;   // [2] the slot's last product complete
    uint64_t *v_ok = o_final + 2;     // [kMaskedTiles] the masked tile's V checked
    uint64_t *v_ask = v_ok + kMaskedTiles;  // [kMaskedTiles] its V landed: to be checked
    uint64_t *idle = v_ask + kMaskedTiles;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(idle + 1);
    uint32_t *bad = reinterpret_cast<uint32_t *>(base + Ge::kOffBad);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = a.G, BQ = kPtRows / G, MT = NT * BQ;  // tokens of a query tile, of the CTA
    const int kvh = blockIdx.x % a.Hkv;
    const PackedTile p =
        find_packed_tile(a.cu_q, a.cu_k, a.n_seqs, a.total_q, a.total_k, 1, MT, blockIdx.x / a.Hkv, a.status);
    if (p.seq < 0) return;
    const int t0 = p.tile * MT;                        // first token
    const int shift = p.nk - p.nq;                     // token t sees keys 0 .. t + shift
    const int seen = min(p.nq, t0 + MT) + shift;       // keys the last token sees (may be <= 0)
    const int nt = seen > 0 ? (seen + kPtKeys - 1) / kPtKeys : 0;  // key tiles
    const int steps = NT * nt;
    const int first_masked = max(0, (t0 + shift + 1) / kPtKeys);  // tiles from here on hide keys from some row

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(q_full, 1);
        for (int s = 0; s < 2; ++s) {
            mbar_init(&s_full[s], 1);
            mbar_init(&p_full[s], 128);
            mbar_init(&o_final[s], 1);
        }
        for (int s = 0; s < kMaskedTiles; ++s) {
            mbar_init(&v_ok[s], 64);
            mbar_init(&v_ask[s], 1);
        }
        mbar_init(idle, 1);
        fence_barrier_init();
    }
    if (threadIdx.x < 4 * kMaskedTiles + 1) bad[threadIdx.x] = 0;
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const auto col_s = [&](int slot) { return tmem + static_cast<uint32_t>(slot * kPtKeys); };
    const auto col_o = [&](int slot) { return tmem + 256u + static_cast<uint32_t>(slot * 128); };
    const auto wait = [&](uint64_t *bar, uint32_t parity) {
        if (wait_poll(bar, parity, nullptr)) return true;
        set_status(a.status, B200_DEV_TIMEOUT);
        return false;
    };

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == 0 && lane == 0 && nt > 0) {
            // ---- TMA
            const uint64_t pol = policy_evict_last();  // K / V are read again by the other query tiles
            mbar_arrive_expect_tx(q_full, NT * (D / 64) * static_cast<uint32_t>(BQ * G) * 128u);
            for (int x = 0; x < NT; ++x)
                for (int b = 0; b < D / 64; ++b)
                    tma_load_3d(sbase + x * Ge::kTile + b * Ge::kBox, &tq, 64 * b, kvh * G,
                                static_cast<int32_t>(p.q0) + t0 + x * BQ, smem_addr(q_full), pol);
            int issued = 0;
            const auto plane = [&](const CUtensorMap *map, int t) {
                const int st = issued % S;
                if (issued >= S && !wait(&empty[st], ((issued / S) - 1) & 1)) return false;
                mbar_arrive_expect_tx(&full[st], Ge::kTile);
#pragma unroll
                for (int b = 0; b < D / 64; ++b)
                    tma_load_3d(sbase + Ge::kOffRing + st * Ge::kTile + b * Ge::kBox, map, 64 * b, kvh,
                                static_cast<int32_t>(p.k0) + t * kPtKeys, smem_addr(&full[st]), pol);
                ++issued;
                return true;
            };
            bool ok = true;
            if (NT == 1) {
                ok = plane(&tk, 0) && (nt < 2 || plane(&tk, 1));
                for (int t = 0; t < nt && ok; ++t) ok = plane(&tv, t) && (t + 2 >= nt || plane(&tk, t + 2));
            } else {
                for (int t = 0; t < nt && ok; ++t) ok = plane(&tk, t) && plane(&tv, t);
            }
            // copies still landing in this CTA's shared memory
            wait_poll(q_full, 0, nullptr);
            for (int i = max(0, issued - S); i < issued; ++i) wait_poll(&full[i % S], (i / S) & 1, nullptr);
        } else if (warp == 1 && lane == 0 && nt > 0) {
            // ---- tensor cores
            const auto at = [&](int pl) { return sbase + Ge::kOffRing + (pl % S) * Ge::kTile; };
            const auto issue_s = [&](int i) {
                const int slot = i & 1, t = NT == 2 ? i >> 1 : i, pl = plane_k<NT>(t);
                if (!wait(&full[pl % S], (pl / S) & 1)) return false;
                tc_fence_after();
                const uint32_t q = sbase + (NT == 2 ? slot : 0) * Ge::kTile, k = at(pl);
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk)
                    tc_mma_f16(col_s(slot), desc_k_sw128(q + (kk >> 2) * Ge::kBox) + 2 * (kk & 3),
                               desc_k_sw128(k + (kk >> 2) * Ge::kBox) + 2 * (kk & 3), kIdS, kk > 0 ? 1u : 0u);
                tc_commit(smem_addr(&s_full[slot]));
                if (NT == 1 || slot == 1) tc_commit(smem_addr(&empty[pl % S]));
                return true;
            };
            bool ok = wait(q_full, 0);
            for (int i = 0; i < min(2, steps) && ok; ++i) ok = issue_s(i);
            for (int i = 0; i < steps && ok; ++i) {
                const int slot = i & 1, t = NT == 2 ? i >> 1 : i, pl = plane_v<NT>(t, nt);
                const bool check = t >= first_masked && (NT == 1 || slot == 0);
                ok = wait(&full[pl % S], (pl / S) & 1);
                if (!ok) break;
                if (check) mbar_arrive(&v_ask[t - first_masked]);  // done while the softmax runs
                ok = wait(&p_full[slot], (i >> 1) & 1) && (!check || wait(&v_ok[t - first_masked], 0));
                if (!ok) break;
                tc_fence_after();
                const uint32_t v = at(pl);
#pragma unroll
                for (int kk = 0; kk < kPtKeys / 16; ++kk)
                    tc_mma_f16_ts(col_o(slot), col_s(slot) + 8 * kk, desc_mn_sw128(v + kk * 2048, Ge::kBox), kIdO,
                                  (i >= 2 || kk > 0) ? 1u : 0u);
                if (NT == 1 || slot == 1) tc_commit(smem_addr(&empty[pl % S]));
                if (i + 2 >= steps) tc_commit(smem_addr(&o_final[slot]));
                if (i + 2 < steps) ok = issue_s(i + 2);
            }
            // no product may still use tensor memory or the ring when the CTA exits
            tc_commit(smem_addr(idle));
            wait_poll(idle, 0, nullptr);
        } else if (warp >= 2) {
            // ---- V check: rows of the masked tiles that hold Inf or NaN, cleared and noted
            constexpr uint32_t kExp = kBf16 ? 0x7F80u : 0x7C00u;
            for (int t = first_masked; t < nt; ++t) {
                const int pl = plane_v<NT>(t, nt);
                // the tensor-core warp has seen this phase of `full` and holds it until the
                // check is done, so its parity is not ambiguous here
                if (!__all_sync(0xffffffffu, wait(&v_ask[t - first_masked], 0) && wait(&full[pl % S], (pl / S) & 1))) break;
                unsigned char *v = base + Ge::kOffRing + (pl % S) * Ge::kTile;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int row = 64 * half + (warp - 2) * 32 + lane;
                    bool odd = false;
#pragma unroll
                    for (int c = 0; c < D / 8; ++c) {
                        const uint4 u = *reinterpret_cast<const uint4 *>(v + (c >> 3) * Ge::kBox + row * 128 +
                                                                         (((c & 7) ^ (row & 7)) << 4));
                        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            odd |= (w[j] & kExp) == kExp || ((w[j] >> 16) & kExp) == kExp;
                    }
                    const uint32_t mask = __ballot_sync(0xffffffffu, odd);
                    if (mask) {
                        if (odd)
                            for (int c = 0; c < D / 8; ++c)
                                *reinterpret_cast<uint4 *>(v + (c >> 3) * Ge::kBox + row * 128 + (c & 7) * 16) =
                                    make_uint4(0, 0, 0, 0);
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
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        // ---- softmax: thread = row of the slot's query tile = tensor-memory lane
        const int slot = (warp - 4) >> 2, qq = warp & 3;
        const int r = 32 * qq + lane;
        const uint32_t lanes = static_cast<uint32_t>(32 * qq) << 16;
        const uint32_t ts = col_s(slot) + lanes, to = col_o(slot) + lanes;
        const int tok = t0 + (NT == 2 ? slot * BQ : 0) + r / G;
        const bool live = r < BQ * G && tok < p.nq;
        const int last = live ? tok + shift : -1;  // last key the row sees
        float m = -INFINITY, l = 0.f;
        bool ok = true;
#pragma unroll 1
        for (int i = slot; i < steps; i += 2) {
            const int k0 = (NT == 2 ? i >> 1 : i) * kPtKeys;
            ok = __all_sync(0xffffffffu, wait(&s_full[slot], (i >> 1) & 1));
            if (!ok) break;
            tc_fence_after();
            uint32_t sv[4][32];
#pragma unroll
            for (int c = 0; c < 4; ++c) tc_ld32_nowait(ts + 32 * c, sv[c]);
            tc_wait_ld();
#pragma unroll
            for (int c = 0; c < 4; ++c) tc_reg_fence(sv[c]);
            const int vis = last + 1 - k0;  // keys of the tile the row sees
            if (!__all_sync(0xffffffffu, vis >= kPtKeys)) {
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (32 * c + j >= vis) sv[c][j] = 0xFF800000u;
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int j = 0; j < 32; ++j) mx[j & 3] = fmaxf(mx[j & 3], __uint_as_float(sv[c][j]));
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.sl2;
            float alpha = 1.f;
            bool grow = false;
            if (m == -INFINITY) {
                m = top;  // nothing summed so far: O and l are zero, or not yet written
            } else if (top > m + kPtRescale) {
                alpha = exp2_approx(m - top);
                m = top;
                grow = true;
            }
            if (__any_sync(0xffffffffu, grow)) {
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
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t pv[32];
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    const float x = exp2_approx(fmaf(__uint_as_float(sv[2 * c + (j >> 4)][2 * (j & 15)]), a.sl2, -ms));
                    const float y = exp2_approx(fmaf(__uint_as_float(sv[2 * c + (j >> 4)][2 * (j & 15) + 1]), a.sl2, -ms));
                    sum[j & 1] += x;
                    sum[2 + (j & 1)] += y;
                    pv[j] = pack_pair<T>(x, y);
                }
                tc_st32(ts + 32 * c, pv);
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            tc_wait_st();
            tc_fence_before();
            mbar_arrive(&p_full[slot]);
        }
        const bool mine = steps > slot;  // the slot had a step
        if (ok && mine) ok = __all_sync(0xffffffffu, wait(&o_final[slot], 0));
        tc_fence_after();
        // the row's output: O / l, plus what the cleared V rows would have added
        float m_row = m, l_row = l, f_own = 1.f, f_other = 0.f;
        constexpr int NC = NT == 2 ? D / 32 : D / 64;  // 32-column pieces this thread writes
        const int c0 = NT == 2 ? 0 : slot * NC;
        if constexpr (NT == 1) {
            // the slots' halves of the key tiles, joined: each warpgroup hands the other half of
            // its columns over through the ring (no copy or product uses it any more)
            float2 *stat = reinterpret_cast<float2 *>(base);  // over Q: every product with it is complete
            float *xch = reinterpret_cast<float *>(base + Ge::kOffRing) + slot * (D / 2) * kPtRows;
            asm volatile("bar.sync 1, 256;" ::: "memory");  // both slots' products are complete
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
            asm volatile("bar.sync 1, 256;" ::: "memory");
            const float2 other = stat[(slot ^ 1) * kPtRows + r];
            m_row = fmaxf(m, other.x);
            const float mm = m_row == -INFINITY ? 0.f : m_row;
            f_own = mine ? exp2_approx(m - mm) : 0.f;
            f_other = exp2_approx(other.x - mm);
            l_row = (mine ? l * f_own : 0.f) + other.y * f_other;
        }
        const float inv = l_row != 0.f ? 1.0f / l_row : 0.f;  // a row that sees no key: zeros
        if (ok) {
            T *dst = static_cast<T *>(a.out) + (p.q0 + tok) * a.o_tok + (kvh * G + r % G) * a.o_head;
            const bool any_bad = bad[4 * kMaskedTiles] != 0;
            const float *got = reinterpret_cast<const float *>(base + Ge::kOffRing) + (slot ^ 1) * (D / 2) * kPtRows;
            const bool other_has = NT == 1 && steps > (slot ^ 1);
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
                    if (NT == 1) x[j] = x[j] * f_own + (other_has ? got[(32 * c + j) * kPtRows + r] * f_other : 0.f);
                }
                if (any_bad && live) {
                    const T *q = static_cast<const T *>(a.q) + (p.q0 + tok) * a.q_tok + (kvh * G + r % G) * a.q_head;
                    for (int w = 0; w < 4 * kMaskedTiles; ++w) {
                        for (uint32_t mask = bad[w]; mask; mask &= mask - 1) {
                            const int key = first_masked * kPtKeys + 32 * w + __ffs(static_cast<int>(mask)) - 1;
                            if (key > last) continue;
                            const T *kr = static_cast<const T *>(a.k) + (p.k0 + key) * a.k_tok + kvh * a.k_head;
                            const T *vr = static_cast<const T *>(a.v) + (p.k0 + key) * a.v_tok + kvh * a.v_head;
                            float s = 0.f;
                            for (int d = 0; d < D; ++d) s = fmaf(to_f32<T>(q[d]), to_f32<T>(kr[d]), s);
                            const float pr = exp2_approx(fmaf(s, a.sl2, -m_row));
#pragma unroll
                            for (int j = 0; j < 32; ++j) x[j] = fmaf(pr, to_f32<T>(vr[32 * (c0 + c) + j]), x[j]);
                        }
                    }
                }
                if (live) {
#pragma unroll
                    for (int j = 0; j < 32; j += 8)
                        *reinterpret_cast<uint4 *>(dst + 32 * (c0 + c) + j) =
                            make_uint4(pack_pair<T>(x[j] * inv, x[j + 1] * inv), pack_pair<T>(x[j + 2] * inv, x[j + 3] * inv),
                                       pack_pair<T>(x[j + 4] * inv, x[j + 5] * inv), pack_pair<T>(x[j + 6] * inv, x[j + 7] * inv));
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 2) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
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

template <typename T, int D, int NT>
cudaError_t pt_launch(const PackedArgs &a, cudaStream_t st) {
    constexpr bool bf16 = !__is_same(T, __half);
    auto kern = packed_tc_kernel<T, D, NT>;
    cudaError_t e = once_per_device(reinterpret_cast<const void *>(kern), ATTR_SMEM, [&] {
        return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    static_cast<int>(PtGeometry<D, NT>::kSmem));
    });
    if (e != cudaSuccess) return e;
    const int BQ = kPtRows / a.G;
    CUtensorMap mq, mk, mv;
    if (!row_map(&mq, bf16, a.q, D, a.Hq, a.total_q, a.q_head, a.q_tok, a.G, BQ) ||
        !row_map(&mk, bf16, a.k, D, a.Hkv, a.total_k, a.k_head, a.k_tok, 1, kPtKeys) ||
        !row_map(&mv, bf16, a.v, D, a.Hkv, a.total_k, a.v_head, a.v_tok, 1, kPtKeys))
        return cudaErrorNotSupported;
    const int64_t ctas = most_packed_tiles(a.n_seqs, a.total_q, 1, NT * BQ) * a.Hkv;
    if (ctas > INT32_MAX) return cudaErrorNotSupported;
    return b200_launch(kern, dim3(static_cast<unsigned>(ctas)), dim3(kPtThreads), PtGeometry<D, NT>::kSmem, st, false, mq,
                       mk, mv, a);
}

template <typename T, int D>
cudaError_t pt_by_tiles(const PackedArgs &a, cudaStream_t st) {
    // two query tiles a CTA once such CTAs fill the SMs
    const int64_t pairs = a.total_q * a.G / (2 * kPtRows) * a.Hkv;
    return pairs >= device_sm_count() ? pt_launch<T, D, 2>(a, st) : pt_launch<T, D, 1>(a, st);
}

template <typename T>
cudaError_t pt_by_dim(const PackedArgs &a, cudaStream_t st) {
    return a.D == 128 ? pt_by_tiles<T, 128>(a, st) : pt_by_tiles<T, 64>(a, st);
}

}  // namespace

cudaError_t packed_tc_launch(const PackedArgs &a, cudaStream_t st) {
    if (a.total_k == 0 || a.G > kPtRows) return cudaErrorNotSupported;
    switch (a.dtype) {
        case B200_DTYPE_F16: return pt_by_dim<__half>(a, st);
        case B200_DTYPE_BF16: return pt_by_dim<__nv_bfloat16>(a, st);
    }
    return cudaErrorNotSupported;
}

}  // namespace b200
