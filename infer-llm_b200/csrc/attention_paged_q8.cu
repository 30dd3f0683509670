// b200_flash_attn_paged_batch_q8: one query token for each of many sequences against an 8-bit paged cache.
//
// out_b = sum_j softmax_j(t_j) 2^ev_j vq_j over the keys j < seq_lens[b], t_j = scale 2^ek_j q_b . kq_j, with kq, vq in e4m3. Every
// cached row is read once (once per 16 query heads of its KV head), so HBM bounds the operator: 2 (D + 1) bytes and 4 D G flops a
// key and KV head.
//
//  * Work split, copies and joins as for the 16-bit caches (attention_paged_batch.cu): all key tiles of all (sequence,
//    KV head) pairs are one line cut into equal shares, each warp streams its own sub-tiles of 32 keys (8 KB of K and V at head_dim 128)
//    through a private ring, and few short pairs take one launch of clusters.
//  * Products are mma.sync m16n8k16 of F16 numbers for all query types: e4m3 is exact in F16. The order of the 16 dimensions of a
//    product is free, so a lane takes four neighbouring bytes of a key (ldmatrix) as the two halves of its fragment. V comes
//    transposed in pairs of dimensions; one byte permutation a word parts the even from the odd ones.
//  * A row of Q is scaled by a power of two to a largest magnitude in [2^14, 2^15) and enters as one F16 number (F16, BF16: exact, or
//    2^-39 of the row's largest) or as two (F32: 22 bits). Up to eight query heads the second takes the unused rows 8 .. 15
//    of the same product.
//  * The scales 2^ek multiply the scores. The scales 2^ev go into the weights: w_j = 2^(t_j log2 e - M + ev_j - N + 14), M the
//    running maximum of the scores and N the least whole number that no t_j log2 e - M + ev_j passes, as two F16 numbers. N is a
//    maximum of its own, so keys whose V is far larger than that of the heaviest key keep their bits; the sum of the weights goes
//    by M. At the end 2^(N - 14) takes both together. N counts from M, so that scores however large leave ev_j its bits, and is
//    whole, so that differences of N are exact.
// 64 BF16 sequences of 5 to 4069 keys, 32 / 8 heads of 128 (273 MB): 62 to 64 us with the join, 4.3 TB/s, 66 % of a large copy's
// rate; 16 F32 sequences of 1500 to 7548 keys, 16 / 8 heads (147 MB): 37.5 us, 3.9 TB/s. No unit is full (issue active 45 %,
// tensor pipe 29 %): eight warps an SM wait for the fixed latencies of one chain, and the start (3.6 us of dependent look-ups),
// the pairs' ends and the join (4 to 5 us) weigh twice at half the bytes a key.
// Rows past a sequence's end are not read; they and keys of invalid blocks get weight 0.
#include "paged_line.cuh"
#include "paged_q8.cuh"

namespace b200 {
namespace {

constexpr int kP8Warps = 4;
constexpr int kP8Threads = 32 * kP8Warps;
constexpr int kP8Ctas = 2;  // an SM (three, of 168 registers, spill: 92 us against 80)
constexpr int kP8MostCtas = 320;
constexpr int kP8JoinThreads = 256;
constexpr int kP8Cluster = 8;
constexpr int kP8ClusterKeys = 4096;
constexpr int kP8Sub = 32;                  // keys of a warp's sub-tile
constexpr int kP8Tile = kP8Sub * kP8Warps;  // keys of a tile
// Units of the line a tile and a pair's start and end take: 1.6 to 1.8 us against 2.4 (64 ragged sequences; shares of equal tiles ended
// between 50 and 69 us).
constexpr int kP8TileUnits = 2, kP8PairUnits = 3;
constexpr int kP8Top = 14;                  // weights are at most 2^14 (2^14.2), F16's largest power of two but one
constexpr float kP8Large = 1048576.f;       // scores from here on, in powers of two, hold 1/8 at best

struct P8Args {
    const void *q = nullptr;
    void *out = nullptr;
    int64_t q_seq = 0, q_head = 0, o_seq = 0, o_head = 0;  // elements
    const char *k = nullptr, *v = nullptr;
    const unsigned char *ke = nullptr, *ve = nullptr;
    int64_t block_stride = 0, tok_stride = 0, head_stride = 0;
    int64_t scale_block = 0, scale_tok = 0, scale_head = 0;
    int64_t n_blocks = 0;
    const int32_t *table = nullptr, *lens = nullptr;
    int64_t table_stride = 0;
    int64_t max_keys = 0;  // positions a table row covers (fits 31 bits)
    uint32_t bt = 1, bt_mul = 0, bt_shift = 0;  // x / bt = x bt_mul / 2^bt_shift for x < 2^31
    int n_seqs = 0, G = 0, VH = 0, HG = 0;  // query heads a KV head; (KV head, head group) pairs; groups a KV head
    float sl2 = 0.f;                        // scale * log2 e
    float *ws = nullptr;
    int32_t *status = nullptr;
};

template <int D, int HB>
struct P8Geometry {
    static constexpr int kStages = 2;  // (three: 1 us more)
    static constexpr int kChunks = D / 16;
    static constexpr int kHalf = kP8Sub * D;     // K (or V) bytes of a sub-tile
    static constexpr int kRec = HB * (D + 3);    // floats of a partial: o, then m, l, n
    static constexpr size_t kRing = static_cast<size_t>(kP8Warps) * kStages * 2 * kHalf;
    static constexpr size_t kStat = static_cast<size_t>(kP8Warps) * 3 * HB * 4;
    static constexpr size_t kScale = static_cast<size_t>(kP8Warps) * kStages * kP8Sub * 8;
    static constexpr size_t kSmem = kRing + kStat + kScale + kP8Warps * kStages * 4;
    static constexpr size_t kSmemCluster = kSmem + kRec * 4;
    static_assert(HB * D * 4 <= 2 * kHalf, "a warp's partial takes the place of its last sub-tile");
    static_assert(kP8Ctas * (kSmemCluster + 1024) <= 228 * 1024, "CTAs of an SM");
};

B200_DEVICE float p8_pow2(int e) { return __uint_as_float(static_cast<uint32_t>(max(-126, min(127, e)) + 127) << 23); }
// x 2^(n - 14) for a whole n; -inf: there was no weight, or only such as are no numbers
B200_DEVICE float p8_unscale(float x, float n) {
    const int e = static_cast<int>(fmaxf(n, -1000.f)) - kP8Top, half = e >> 1;  // 2^e may lie outside F32's range
    return x * p8_pow2(half) * p8_pow2(e - half);
}
// the smaller of x >= 0 and F32's largest; NaN stays
B200_DEVICE float p8_finite(float x) {
    float y;
    asm("min.NaN.f32 %0, %1, 0f7F7FFFFF;" : "=f"(y) : "f"(x));
    return y;
}
// m - M for running maxima of which both may be -inf
B200_DEVICE float p8_less(float m, float M) { return m - (M == -INFINITY ? 0.f : M); }

// Four columns of a head's output: o 2^(N - 14) / l; zeros where there is no weight.
template <typename T>
B200_DEVICE void p8_write(T *to, const float (&o)[4], float l, float n) {
    const float inv = l != 0.f ? 1.0f / l : 0.f;
    T x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = from_f32<T>(l != 0.f ? p8_unscale(o[j] * inv, n) : 0.f);
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4 *>(to) = *reinterpret_cast<const float4 *>(x);
    else *reinterpret_cast<uint2 *>(to) = *reinterpret_cast<const uint2 *>(x);
}

// One warp's running softmax: lane (g = lane / 4, t = lane % 4) holds head rows g (and g + 8 of 16), output columns
// 16 c + 4 t .. + 3.
template <typename T, int D, int HB>
struct P8State {
    static constexpr bool FULL = HB > 8, TWO = __is_same(T, float);
    static constexpr int R = FULL ? 2 : 1;  // head rows a lane holds
    // A fragments of Q. 16 heads: of 16 dimensions, and of their second terms. Up to 8 heads: rows 0 .. 7 and 8 .. 15 are the two terms
    // (TWO), or 16 dimensions and the next 16, of which a product with a key's 16 dimensions uses one half. Every fragment is four
    // registers in a row as the instruction wants them; zeros in half of them would have to be moved there each time.
    static constexpr int NQ = FULL || TWO ? D / 16 : D / 32;
    uint32_t q[NQ][4], ql[FULL && TWO ? NQ : 1][4];
    float o[D / 16][2][4];  // even and odd columns: rows g and g + 8; without FULL, row g's shares of the weights' two terms
    float m[R], l[R], n[R], qs[R];

    B200_DEVICE void begin(const P8Args &a, int b, int h0, int heads, int lane) {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            m[r] = n[r] = -INFINITY;
            l[r] = 0.f;
            const bool ok = g + 8 * r < heads;
            const T *row = static_cast<const T *>(a.q) + b * a.q_seq + (h0 + g + 8 * r) * a.q_head + 4 * t;
            float x[D / 16][4];
            uint32_t top = 0;  // the largest finite magnitude
#pragma unroll
            for (int s = 0; s < D / 16; ++s) {
                if constexpr (TWO) {
                    const float4 v = ok ? __ldg(reinterpret_cast<const float4 *>(row + 16 * s)) : make_float4(0.f, 0.f, 0.f, 0.f);
                    x[s][0] = v.x, x[s][1] = v.y, x[s][2] = v.z, x[s][3] = v.w;
                } else {
                    const uint2 v = ok ? __ldg(reinterpret_cast<const uint2 *>(row + 16 * s)) : make_uint2(0, 0);
                    const float2 lo = unpack2<T>(v.x), hi = unpack2<T>(v.y);
                    x[s][0] = lo.x, x[s][1] = lo.y, x[s][2] = hi.x, x[s][3] = hi.y;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t u = __float_as_uint(x[s][i]) & 0x7FFFFFFFu;
                    if (u < 0x7F800000u) top = max(top, u);
                }
            }
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int e = top ? max(-100, static_cast<int>(top >> 23) - 127) - 14 : 0;
            const float f = p8_pow2(-e);
            qs[r] = a.sl2 * p8_pow2(e);
#pragma unroll
            for (int s = 0; s < D / 16; ++s)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float y0 = x[s][2 * u] * f, y1 = x[s][2 * u + 1] * f;
                    const uint32_t hi = pack2<__half>(y0, y1);
                    uint32_t lo = 0;
                    if constexpr (TWO) {  // (the rest of an infinity or NaN would be NaN; it stays in the first)
                        const float2 h = unpack2<__half>(hi);
                        lo = pack2<__half>(fabsf(y0) < INFINITY ? y0 - h.x : 0.f, fabsf(y1) < INFINITY ? y1 - h.y : 0.f);
                    }
                    if constexpr (FULL) {
                        q[s][2 * u + r] = hi;
                        if constexpr (TWO) ql[s][2 * u + r] = lo;
                    } else if constexpr (TWO) {
                        q[s][2 * u] = hi, q[s][2 * u + 1] = lo;
                    } else {
                        q[s / 2][2 * u + s % 2] = hi;
                    }
                }
        }
#pragma unroll
        for (int c = 0; c < D / 16; ++c)
#pragma unroll
            for (int u = 0; u < 4; ++u) o[c][0][u] = o[c][1][u] = 0.f;
    }

    // 32 keys at sk / sv (rows of D bytes, chunks swizzled by `chunk_at`), their scales at `scales` (2^ek, ev); bit j of
    // `live`: key j takes part.
    B200_DEVICE void keys(uint32_t sk, uint32_t sv, uint32_t live, const float2 *scales, int lane) {
        const int mat = lane >> 3, rr = lane & 7, t2 = 2 * (lane & 3);
        constexpr int NS = FULL || TWO ? 1 : 2;  // sums: of even and odd 16 dimensions
        float s[NS][4][4];
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int u = 0; u < 4; ++u) s[i][j][u] = 0.f;
        const uint32_t row = (8 * mat + rr) * D;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            uint32_t kf[4];
            ldsm4(kf, sk + row + chunk_at(ks, rr));
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t b0, b1;
                e4m3x4_to_f16(kf[j], b0, b1);
                if constexpr (FULL) {
                    mma16<__half, true>(s[0][j], q[ks], b0, b1);
                    if constexpr (TWO) mma16<__half, true>(s[0][j], ql[ks], b0, b1);
                } else {
                    mma16<__half, true>(s[TWO ? 0 : ks % 2][j], q[TWO ? ks : ks / 2], b0, b1);
                }
            }
        }
        float ke[4][2], ve[4][2];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float4 x = *reinterpret_cast<const float4 *>(scales + 8 * j + t2);
            ke[j][0] = x.x, ve[j][0] = x.y, ke[j][1] = x.z, ve[j][1] = x.w;
        }
        uint32_t hi[2][2 * R], lo[2][2 * R];  // A fragments of the weights: 16 keys each, [key half][row]
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float x[4][2], mx = -INFINITY, nx = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float y = FULL ? s[0][j][2 * r + u] : s[0][j][u] + s[NS - 1][j][2 + u];
                    // (a large row of Q against small keys, or the inverse, stays in range; a score of 0 is one for any scales)
                    x[j][u] = y * p8_finite(qs[r] * ke[j][u]);
                    if (live != ~0u && !((live >> (8 * j + t2 + u)) & 1u)) x[j][u] = -INFINITY;
                    mx = fmaxf(mx, x[j][u]);
                    nx = fmaxf(nx, x[j][u] + ve[j][u]);
                }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            nx = fmaxf(nx, __shfl_xor_sync(0xffffffffu, nx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            nx = fmaxf(nx, __shfl_xor_sync(0xffffffffu, nx, 2));
            const float mn = fmaxf(m[r], mx), ms = mn == -INFINITY ? 0.f : mn, moved = m[r] - ms;
            float nn = ceilf(fmaxf(n[r] + moved, nx - ms));
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int u = 0; u < 2; ++u) x[j][u] -= ms;
            const bool large = fabsf(ms) >= kP8Large;
            if (__any_sync(0xffffffffu, mn > m[r] || nn > n[r] || large)) {
                if (__any_sync(0xffffffffu, large)) {  // ev is lost in such scores, not in their differences
                    nx = -INFINITY;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int u = 0; u < 2; ++u) nx = fmaxf(nx, x[j][u] + ve[j][u]);
                    nx = fmaxf(nx, __shfl_xor_sync(0xffffffffu, nx, 1));
                    nx = fmaxf(nx, __shfl_xor_sync(0xffffffffu, nx, 2));
                    nn = ceilf(fmaxf(n[r] + moved, nx));
                }
                l[r] *= exp2_approx(moved);
                const float f = exp2_approx(p8_less(n[r], nn) + moved);
#pragma unroll
                for (int c = 0; c < D / 16; ++c)
#pragma unroll
                    for (int u = FULL ? 2 * r : 0; u < (FULL ? 2 * r + 2 : 4); ++u) o[c][0][u] *= f, o[c][1][u] *= f;
            }
            m[r] = mn;
            n[r] = nn;
            const float ns = (nn == -INFINITY ? 0.f : nn) - static_cast<float>(kP8Top);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                l[r] += exp2_approx(x[j][0]) + exp2_approx(x[j][1]);
                const float w0 = exp2_approx(x[j][0] + (ve[j][0] - ns)), w1 = exp2_approx(x[j][1] + (ve[j][1] - ns));
                const uint32_t h = pack2<__half>(w0, w1);
                const float2 f = unpack2<__half>(h);
                hi[j >> 1][(j & 1) * R + r] = h;
                lo[j >> 1][(j & 1) * R + r] = pack2<__half>(w0 - f.x, w1 - f.y);
            }
        }
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
            uint32_t vf[4], x[4][2];
            ldsm4_t(vf, sv + row + chunk_at(c, rr));
#pragma unroll
            for (int j = 0; j < 4; ++j) {  // (key, column) bytes 00 01 10 11 as even and odd columns
                e4m3x4_to_f16(__byte_perm(vf[j], 0, 0x3120), x[j][0], x[j][1]);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    if constexpr (FULL) {
                        mma16<__half, true>(o[c][u], hi[h], x[2 * h][u], x[2 * h + 1][u]);
                        mma16<__half, true>(o[c][u], lo[h], x[2 * h][u], x[2 * h + 1][u]);
                    } else {  // the unused rows 8 .. 15 take the weights' second term
                        const uint32_t both[4] = {hi[h][0], lo[h][0], hi[h][1], lo[h][1]};
                        mma16<__half, true>(o[c][u], both, x[2 * h][u], x[2 * h + 1][u]);
                    }
                }
        }
    }
    // chunk c of a row whose number is rr modulo 8, so that eight rows' chunks fall into eight different bank groups
    static B200_DEVICE uint32_t chunk_at(int c, int rr) {
        return static_cast<uint32_t>(D == 128 ? (c ^ rr) : (c ^ (rr >> 1))) << 4;
    }

    // this warp's partial: o [HB][D], and m, l, n [HB] each
    B200_DEVICE void store(float *po, float *stat, int lane) {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            const int h = g + 8 * r;
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
                const float *e = o[c][0], *d = o[c][1];
                *reinterpret_cast<float4 *>(po + h * D + 16 * c + 4 * t) =
                    FULL ? make_float4(e[2 * r], d[2 * r], e[2 * r + 1], d[2 * r + 1])
                         : make_float4(e[0] + e[2], d[0] + d[2], e[1] + e[3], d[1] + d[3]);
            }
            if (t == 0) stat[h] = m[r], stat[HB + h] = l[r], stat[2 * HB + h] = n[r];
        }
    }
};

// CL: a cluster of kP8Cluster CTAs takes one pair, and writes its output.
template <typename T, int D, int HB, bool CL>
__global__ void __launch_bounds__(kP8Threads, kP8Ctas) paged_q8_kernel(const __grid_constant__ P8Args a) {
    using Ge = P8Geometry<D, HB>;
    extern __shared__ __align__(128) unsigned char p8_smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float *stat = reinterpret_cast<float *>(p8_smem + Ge::kRing);  // [warp][m, l, n][HB]
    float2 *scales = reinterpret_cast<float2 *>(p8_smem + Ge::kRing + Ge::kStat) + warp * Ge::kStages * kP8Sub;
    uint32_t *live = reinterpret_cast<uint32_t *>(p8_smem + Ge::kRing + Ge::kStat + Ge::kScale) + warp * Ge::kStages;
    float *own = reinterpret_cast<float *>(p8_smem + Ge::kSmem);  // CL: this CTA's record
    const uint32_t ring_at = warp * Ge::kStages * 2 * Ge::kHalf, ring = smem_addr(p8_smem) + ring_at;

    Place at = {};  // what is computed
    if constexpr (CL) {
        const int pair = blockIdx.x / kP8Cluster, rank = blockIdx.x % kP8Cluster;
        at.b = pair / a.VH;
        at.vh = pair % a.VH;
        at.len = seq_len(a, at.b);
        at.tiles = (at.len + kP8Tile - 1) / kP8Tile;
        at.t = at.tiles * rank / kP8Cluster;
        at.left = (at.tiles * (rank + 1) / kP8Cluster - at.t) * kP8TileUnits;
        if (rank == 0 && at.vh == 0 && threadIdx.x == 0) report_length(a, at.b);
        if (at.left == 0)  // no keys: nothing to add
            for (int i = threadIdx.x; i < Ge::kRec; i += kP8Threads)
                own[i] = i < HB * D || (i >= HB * (D + 1) && i < HB * (D + 2)) ? 0.f : -INFINITY;
    } else {
        grid_launch_dependents();  // the joining kernel waits for this grid's end
        const int64_t total = tiles_before<kP8Tile, kP8TileUnits, kP8PairUnits>(a, a.n_seqs) * a.VH;
        const int64_t ctas = min64(gridDim.x, total / kP8TileUnits);
        if (blockIdx.x >= ctas) return;
        const int64_t u0 = share_begin(total, blockIdx.x, ctas), u1 = share_begin(total, blockIdx.x + 1, ctas);
        at = place_at<kP8Tile, kP8TileUnits, kP8PairUnits>(a, u0, u1);
    }
    const Place start = at;
    Place in = at;  // what is loaded: one block lookup ahead of `issue`
    bool bad = false;

    // each lane looks up its key of the sub-tile at `in`
    uint32_t row_tok = 0;
    int32_t row_blk = -1, row_head = 0;
    bool row_in = false;
    const auto lookup = [&] {
        const int64_t key = static_cast<int64_t>(in.t) * kP8Tile + warp * kP8Sub + lane;
        row_in = in.left > 0 && key < in.len;
        if (row_in) {
            const uint32_t k32 = static_cast<uint32_t>(key);
            const uint32_t slot = static_cast<uint32_t>(static_cast<uint64_t>(k32) * a.bt_mul >> a.bt_shift);
            row_blk = __ldg(a.table + in.b * a.table_stride + slot);
            row_tok = k32 - slot * a.bt;
            row_head = a.HG == 1 ? in.vh : in.vh / a.HG;
        }
    };
    // Copies the looked-up sub-tile into `stage` and looks the next one up. Its scales are on their way to registers until the next
    // call, or `put`, writes them to the stage.
    uint32_t ke = 0, ve = 0;
    int scale_stage = -1;
    const auto put = [&] {
        if (scale_stage >= 0)
            scales[scale_stage * kP8Sub + lane] =
                make_float2(e8m0_value(ke), ve == 255u ? __uint_as_float(0x7FC00000u) : static_cast<float>(static_cast<int>(ve) - 127));
    };
    const auto issue = [&](int stage) {
        put();
        const bool ok = row_in && row_blk >= 0 && row_blk < a.n_blocks;
        bad |= row_in && !ok;
        const int64_t off = ok ? row_blk * a.block_stride + row_tok * a.tok_stride + row_head * a.head_stride : 0;
        const uint32_t mask = __ballot_sync(0xffffffffu, ok);
        if (lane == 0) live[stage] = mask;
        ke = ve = 0;
        scale_stage = stage;
        if (ok) {
            const int64_t se = row_blk * a.scale_block + row_tok * a.scale_tok + row_head * a.scale_head;
            ke = __ldg(a.ke + se);
            ve = __ldg(a.ve + se);
        }
        constexpr int RPI = 32 / Ge::kChunks;  // rows an instruction covers: row r0 + i RPI, chunk c
        const int c = lane % Ge::kChunks, r0 = lane / Ge::kChunks;
        const uint32_t dst = ring + stage * 2 * Ge::kHalf + r0 * D;
        const char *k = a.k + c * 16, *v = a.v + c * 16;
        if (mask == ~0u) {
#pragma unroll
            for (int i = 0; i < kP8Sub / RPI; ++i) {
                const int64_t o = __shfl_sync(0xffffffffu, off, r0 + i * RPI);
                const uint32_t d = dst + i * RPI * D + P8State<T, D, HB>::chunk_at(c, (r0 + i * RPI) & 7);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(k + o) : "memory");
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d + Ge::kHalf), "l"(v + o) : "memory");
            }
        } else if (mask) {  // rows that are not there are filled with zeros
#pragma unroll 1
            for (int i = 0; i < kP8Sub / RPI; ++i) {
                const int r = r0 + i * RPI, n = (mask >> r) & 1u ? 16 : 0;
                const int64_t o = __shfl_sync(0xffffffffu, off, r);
                const uint32_t d = dst + i * RPI * D + P8State<T, D, HB>::chunk_at(c, r & 7);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(k + o), "r"(n) : "memory");
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d + Ge::kHalf), "l"(v + o), "r"(n) : "memory");
            }
        }
        cp_async_commit();
        if (in.left > 0) place_next<kP8Tile, kP8TileUnits, kP8PairUnits>(a, in);
        lookup();
    };

    lookup();
#pragma unroll
    for (int s = 0; s < Ge::kStages - 1; ++s) issue(s);
    P8State<T, D, HB> st;
    int stage = 0;
    bool fresh = true;  // first tile of a part
    int part_t0 = 0, h0 = 0, heads = 0;  // of the part: its first tile and query head, its heads
#pragma unroll 1
    while (at.left > 0) {
        if (fresh) {
            h0 = (at.vh / a.HG) * a.G + (at.vh % a.HG) * HB;
            heads = min(HB, a.G - (at.vh % a.HG) * HB);
            st.begin(a, at.b, h0, heads, lane);
            part_t0 = at.t;
            fresh = false;
        }
        cp_async_wait<Ge::kStages - 2>();
        __syncwarp();  // every lane's copies have landed, and the previous stage has been read
        issue((stage + Ge::kStages - 1) % Ge::kStages);
        __syncwarp();  // the scales are there
        const uint32_t mask = live[stage];
        const uint32_t sk = ring + stage * 2 * Ge::kHalf;
        if (mask) st.keys(sk, sk + Ge::kHalf, mask, scales + stage * kP8Sub, lane);

        const bool pair_end = at.t + 1 == at.tiles;
        if (pair_end || at.left <= kP8TileUnits) {
            // the warps' partials, each in the place of its last sub-tile, joined in warp order
            __syncwarp();
            const uint32_t part_at = stage * 2 * Ge::kHalf;
            st.store(reinterpret_cast<float *>(p8_smem + ring_at + part_at), stat + warp * 3 * HB, lane);
            __syncthreads();
            const bool whole = !CL && pair_end && part_t0 == 0;
            // a CTA has at most two parts: one that begins within a pair, and one that begins with a pair
            float *rec = CL ? own : a.ws + (static_cast<int64_t>(blockIdx.x) * 2 + (part_t0 == 0)) * Ge::kRec;
            for (int i = 4 * threadIdx.x; i < heads * D; i += 4 * kP8Threads) {
                const int g = i / D;
                float M = -INFINITY, N = -INFINITY, ls = 0.f, os[4] = {};
#pragma unroll
                for (int w = 0; w < kP8Warps; ++w) M = fmaxf(M, stat[w * 3 * HB + g]);
#pragma unroll
                for (int w = 0; w < kP8Warps; ++w) N = fmaxf(N, stat[w * 3 * HB + 2 * HB + g] + p8_less(stat[w * 3 * HB + g], M));
                N = ceilf(N);
#pragma unroll
                for (int w = 0; w < kP8Warps; ++w) {
                    const float4 x =
                        *reinterpret_cast<const float4 *>(p8_smem + w * Ge::kStages * 2 * Ge::kHalf + part_at + i * 4);
                    const float moved = p8_less(stat[w * 3 * HB + g], M);
                    ls = fmaf(exp2_approx(moved), stat[w * 3 * HB + HB + g], ls);
                    const float f = exp2_approx(p8_less(stat[w * 3 * HB + 2 * HB + g], N) + moved);
                    os[0] = fmaf(f, x.x, os[0]), os[1] = fmaf(f, x.y, os[1]);
                    os[2] = fmaf(f, x.z, os[2]), os[3] = fmaf(f, x.w, os[3]);
                }
                if (whole) {
                    p8_write<T>(static_cast<T *>(a.out) + at.b * a.o_seq + (h0 + g) * a.o_head + (i - g * D), os, ls, N);
                } else {
                    *reinterpret_cast<float4 *>(rec + i) = make_float4(os[0], os[1], os[2], os[3]);
                    if (i == g * D) rec[HB * D + g] = M, rec[HB * (D + 1) + g] = ls, rec[HB * (D + 2) + g] = N;
                }
            }
            __syncthreads();  // the partials have been read
            fresh = true;
        }
        stage = (stage + 1) % Ge::kStages;
        place_next<kP8Tile, kP8TileUnits, kP8PairUnits>(a, at);
    }
    cp_async_wait<0>();
    if (bad) set_status(a.status, B200_DEV_BAD_POSITION);
    if constexpr (CL) {
        cluster_sync();  // every CTA's record is written
        const int rank = blockIdx.x % kP8Cluster;
        h0 = (start.vh / a.HG) * a.G + (start.vh % a.HG) * HB;
        heads = min(HB, a.G - (start.vh % a.HG) * HB);
        const int n = heads * D, i0 = n * rank / kP8Cluster, i1 = n * (rank + 1) / kP8Cluster;
        for (int i = i0 + threadIdx.x; i < i1; i += kP8Threads) {
            const int g = i / D;
            float m[kP8Cluster], l[kP8Cluster], s[kP8Cluster], o[kP8Cluster], M = -INFINITY, N = -INFINITY;
#pragma unroll
            for (int c = 0; c < kP8Cluster; ++c) {
                m[c] = ld_dsmem(dsmem_addr(own + HB * D + g, c));
                l[c] = ld_dsmem(dsmem_addr(own + HB * (D + 1) + g, c));
                s[c] = ld_dsmem(dsmem_addr(own + HB * (D + 2) + g, c));
                o[c] = ld_dsmem(dsmem_addr(own + i, c));
            }
#pragma unroll
            for (int c = 0; c < kP8Cluster; ++c) M = fmaxf(M, m[c]);
#pragma unroll
            for (int c = 0; c < kP8Cluster; ++c) m[c] = p8_less(m[c], M), N = fmaxf(N, s[c] + m[c]);
            N = ceilf(N);
            float ls = 0.f, os = 0.f;
#pragma unroll
            for (int c = 0; c < kP8Cluster; ++c) {
                ls = fmaf(exp2_approx(m[c]), l[c], ls);
                os = fmaf(exp2_approx(p8_less(s[c], N) + m[c]), o[c], os);
            }
            static_cast<T *>(a.out)[start.b * a.o_seq + (h0 + g) * a.o_head + (i - g * D)] =
                from_f32<T>(ls != 0.f ? p8_unscale(os / ls, N) : 0.f);
        }
        cluster_sync();  // no CTA's shared memory goes away while it is read
    }
}

// Joins the parts of each pair that more than one CTA took, and clears the rows of empty sequences. One CTA a pair, a thread four
// columns at a time; it asks for all of a few parts' numbers at once, so that their latency is paid once. (The registers of two CTAs an SM:
// with the compiler's own choice, 48, some loads wait for others; 16 F32 sequences 38.9 us against 37.4.)
template <typename T, int D, int HB>
__global__ void __launch_bounds__(kP8JoinThreads, 2) paged_q8_join_kernel(const __grid_constant__ P8Args a, const int64_t grid) {
    using Ge = P8Geometry<D, HB>;
    const int b = static_cast<int>(blockIdx.x / a.VH), vh = static_cast<int>(blockIdx.x % a.VH);
    const int64_t before = tiles_before<kP8Tile, kP8TileUnits, kP8PairUnits>(a, b);
    const int64_t total = tiles_before<kP8Tile, kP8TileUnits, kP8PairUnits>(a, a.n_seqs) * a.VH;
    const int64_t ctas = min64(grid, total / kP8TileUnits);  // as in the main kernel
    const int tiles = seq_tiles<kP8Tile>(a, b);
    const int h0 = (vh / a.HG) * a.G + (vh % a.HG) * HB;
    const int heads = min(HB, a.G - (vh % a.HG) * HB);
    T *out = static_cast<T *>(a.out) + b * a.o_seq + h0 * a.o_head;
    if (threadIdx.x == 0 && vh == 0) report_length(a, b);
    int64_t c0 = 0;
    int parts = 0;  // CTAs c0 .. c0 + parts - 1 hold parts
    if (tiles > 0) {
        const int64_t ua = before * a.VH + vh * units_of<kP8TileUnits, kP8PairUnits>(tiles);
        c0 = share_owner(total, ua, ctas);
        parts = static_cast<int>(share_owner(total, ua + (tiles - 1) * kP8TileUnits, ctas) - c0) + 1;
    }
    grid_wait();
    if (parts == 1) return;  // whole: written by its CTA
    const auto part = [&](int i) { return a.ws + ((c0 + i) * 2 + (i == 0)) * Ge::kRec; };
    constexpr int kAtOnce = 4;
    for (int j = 4 * threadIdx.x; j < heads * D; j += 4 * kP8JoinThreads) {
        const int g = j / D;
        float M = -INFINITY, N = -INFINITY, l = 0.f, o[4] = {};
        for (int i0 = 0; i0 < parts; i0 += kAtOnce) {
            float m[kAtOnce], n[kAtOnce], ls[kAtOnce], Mn = M;
            float4 x[kAtOnce];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                const float *p = part(min(i0 + i, parts - 1));
                x[i] = __ldcg(reinterpret_cast<const float4 *>(p + j));
                m[i] = __ldcg(p + HB * D + g);
                ls[i] = __ldcg(p + HB * (D + 1) + g);
                n[i] = __ldcg(p + HB * (D + 2) + g);
            }
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) Mn = fmaxf(Mn, m[i]);
            const float moved = p8_less(M, Mn);
            float Nn = N + moved;
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) m[i] = p8_less(m[i], Mn), Nn = fmaxf(Nn, n[i] + m[i]);
            Nn = ceilf(Nn);
            l *= exp2_approx(moved);
            const float f = exp2_approx(p8_less(N, Nn) + moved);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] *= f;
            M = Mn, N = Nn;
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                if (i0 + i >= parts) break;
                l = fmaf(exp2_approx(m[i]), ls[i], l);
                const float w = exp2_approx(p8_less(n[i], N) + m[i]);
                o[0] = fmaf(w, x[i].x, o[0]), o[1] = fmaf(w, x[i].y, o[1]);
                o[2] = fmaf(w, x[i].z, o[2]), o[3] = fmaf(w, x[i].w, o[3]);
            }
        }
        p8_write<T>(out + g * a.o_head + (j - g * D), o, l, N);
    }
}

int p8_max_ctas() { return device_sm_count() * kP8Ctas < kP8MostCtas ? device_sm_count() * kP8Ctas : kP8MostCtas; }

// Few pairs with short tables: a cluster each, no workspace.
bool p8_one_launch(int64_t pairs, int64_t max_keys) {
    return pairs * (kP8Cluster + 1) <= p8_max_ctas() && max_keys <= kP8ClusterKeys;
}

int p8_heads(int64_t G) { return G <= 8 ? 8 : 16; }  // heads a block handles

template <typename T, int D, int HB>
cudaError_t p8_launch(P8Args a, int64_t Hkv, cudaStream_t st) {
    using Ge = P8Geometry<D, HB>;
    a.HG = (a.G + HB - 1) / HB;
    a.VH = static_cast<int>(Hkv) * a.HG;
    const int64_t pairs = static_cast<int64_t>(a.n_seqs) * a.VH;
    if (pairs > INT32_MAX) return cudaErrorNotSupported;
    const auto allow = [](const void *kern, size_t bytes) {
        return once_per_device(kern, ATTR_SMEM, [&] {
            return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
        });
    };
    if (p8_one_launch(pairs, a.max_keys)) {
        auto kern = paged_q8_kernel<T, D, HB, true>;
        const cudaError_t e = allow(reinterpret_cast<const void *>(kern), Ge::kSmemCluster);
        if (e != cudaSuccess) return e;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(static_cast<unsigned>(pairs * kP8Cluster));
        cfg.blockDim = dim3(kP8Threads);
        cfg.dynamicSmemBytes = Ge::kSmemCluster;
        cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = kP8Cluster;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        return cudaLaunchKernelEx(&cfg, kern, a);
    }
    auto kern = paged_q8_kernel<T, D, HB, false>;
    cudaError_t e = allow(reinterpret_cast<const void *>(kern), Ge::kSmem);
    if (e != cudaSuccess) return e;
    const int64_t most = (a.max_keys + kP8Tile - 1) / kP8Tile;  // tiles of the longest possible sequence
    const int64_t ctas = min64(p8_max_ctas(), most > p8_max_ctas() ? p8_max_ctas() : pairs * most);
    e = b200_launch(kern, dim3(static_cast<unsigned>(ctas)), dim3(kP8Threads), Ge::kSmem, st, false, a);
    if (e != cudaSuccess) return e;
    return b200_launch(paged_q8_join_kernel<T, D, HB>, dim3(static_cast<unsigned>(pairs)), dim3(kP8JoinThreads), 0, st, true, a,
                       ctas);
}

template <typename T>
cudaError_t p8_by_dim(const P8Args &a, int64_t D, int64_t Hkv, cudaStream_t st) {
    if (p8_heads(a.G) == 8) return D == 128 ? p8_launch<T, 128, 8>(a, Hkv, st) : p8_launch<T, 64, 8>(a, Hkv, st);
    return D == 128 ? p8_launch<T, 128, 16>(a, Hkv, st) : p8_launch<T, 64, 16>(a, Hkv, st);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

size_t b200_flash_attn_paged_batch_q8_workspace_bytes(int64_t n_seqs, int64_t max_keys, int64_t D, int64_t Hq, int64_t Hkv) {
    if (n_seqs <= 0 || max_keys <= 0 || D <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv) return 0;
    const int64_t G = Hq / Hkv;
    const int hb = p8_heads(G);
    if (p8_one_launch(n_seqs * Hkv * ((G + hb - 1) / hb), max_keys)) return 0;
    // two partial records a CTA (its share's first and last part)
    return static_cast<size_t>(p8_max_ctas()) * 2 * hb * (D + 3) * 4;
}

int b200_flash_attn_paged_batch_q8(const void *q, int64_t q_seq_stride, int64_t q_head_stride, void *out,
                                   int64_t out_seq_stride, int64_t out_head_stride, int32_t dtype,
                                   const b200_kv_pool_q8 *pool, const int32_t *block_table, int64_t table_stride,
                                   int64_t max_blocks, const int32_t *seq_lens, int64_t n_seqs, int64_t Hq, float scale,
                                   void *workspace, size_t workspace_bytes, int32_t *dev_status, void *stream) {
    const int e = dtype_bytes(dtype);
    if (n_seqs < 0 || Hq <= 0 || !e) return B200_ERR_INVALID_ARGUMENT;
    const int rc = check_pool_q8(pool);
    if (rc != B200_OK) return rc;
    const int64_t D = pool->head_dim, Hkv = pool->n_head_kv;
    if (Hq % Hkv) return B200_ERR_INVALID_ARGUMENT;
    if (n_seqs == 0) return B200_OK;
    if (!q || !out || !block_table || !seq_lens || max_blocks <= 0 || table_stride < max_blocks)
        return B200_ERR_INVALID_ARGUMENT;
    if (n_seqs > kMostRows || Hq > 65536 || !rows_aligned16(q, q_seq_stride, q_head_stride, e) ||
        !rows_aligned16(out, out_seq_stride, out_head_stride, e))
        return B200_ERR_NOT_SUPPORTED;
    // a length and a tile past it fit 31 bits: the tail of a table of more positions is not used
    const int64_t max_keys =
        max_blocks > kMostKeys / pool->block_tokens ? kMostKeys : max_blocks * pool->block_tokens;
    const size_t need = b200_flash_attn_paged_batch_q8_workspace_bytes(n_seqs, max_keys, D, Hq, Hkv);
    if (need && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < need))
        return B200_ERR_INVALID_ARGUMENT;
    P8Args a;
    a.q = q;
    a.out = out;
    a.q_seq = q_seq_stride;
    a.q_head = q_head_stride;
    a.o_seq = out_seq_stride;
    a.o_head = out_head_stride;
    a.k = static_cast<const char *>(pool->k);
    a.v = static_cast<const char *>(pool->v);
    a.ke = static_cast<const unsigned char *>(pool->k_scale);
    a.ve = static_cast<const unsigned char *>(pool->v_scale);
    a.block_stride = pool->block_stride;
    a.tok_stride = pool->tok_stride;
    a.head_stride = pool->head_stride;
    a.scale_block = pool->scale_block_stride;
    a.scale_tok = pool->scale_tok_stride;
    a.scale_head = pool->scale_head_stride;
    a.n_blocks = pool->n_blocks;
    a.table = block_table;
    a.lens = seq_lens;
    a.table_stride = table_stride;
    a.bt = static_cast<uint32_t>(pool->block_tokens);
    reciprocal31(a.bt, a.bt_mul, a.bt_shift);
    a.max_keys = max_keys;
    a.n_seqs = static_cast<int>(n_seqs);
    a.G = static_cast<int>(Hq / Hkv);
    a.sl2 = (scale > 0.f ? scale : 1.0f / sqrtf(static_cast<float>(D))) * kLog2e;
    a.ws = static_cast<float *>(workspace);
    a.status = dev_status;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case B200_DTYPE_F16: return status_of(p8_by_dim<__half>(a, D, Hkv, st));
        case B200_DTYPE_BF16: return status_of(p8_by_dim<__nv_bfloat16>(a, D, Hkv, st));
    }
    return status_of(p8_by_dim<float>(a, D, Hkv, st));
}

}  // extern "C"
