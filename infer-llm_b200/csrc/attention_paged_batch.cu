// b200_flash_attn_paged_batch: one query token for each of many sequences against a paged
// K/V cache in F32, F16 or BF16.
//
// out_b = sum_j softmax_j(scale q_b . k_j) v_j over the keys j < seq_lens[b]. Every cached
// row is read once (once per 16 query heads of its KV head, of F32 per 8) and meets the query heads that share it, so
// HBM bounds the operator (2 G flops a byte at two bytes an element): what has to be had is
// many bytes in flight on every SM however ragged the lengths are.
//
//  * Work split: keys go in tiles of 4 sub-tiles (one a warp); all tiles of all
//    (sequence, KV head) pairs form one line, of which each CTA takes an equal share
//    (two CTAs an SM, one wave). A CTA's share may begin and end inside a pair: whole
//    pairs are written out directly, parts go to the workspace and a second small
//    kernel (programmatic launch) joins the parts of each cut pair in line order. The
//    shares come from the lengths alone, so results do not depend on timing. A grid
//    over (pair, fixed splits) instead leaves the SMs of short sequences idle.
//  * Few pairs with short contexts (kClusterKeys) take one launch instead: a cluster of eight
//    CTAs a pair, each an eighth of its tiles, joined through distributed shared memory (16 / 8
//    heads of 128, one launch against two: F32 301 keys 12.3 us against 13.3, 2000 keys 18.4
//    against 23.6, 4000 keys 24.6 against 25.6, 8000 keys 41 against 34; the caller also saves a launch).
//  * Each warp streams its own sub-tiles (16 keys of 2-byte elements, 8 of F32: 8 KB of K
//    and V at head_dim 128) through a private ring with cp.async, so no barrier is
//    taken while keys stream; block indices are read one sub-tile ahead of the copies
//    they address. Sub-tiles of the next pair are in flight while one is finished.
//  * 2-byte caches: S = Q K^T and O += P V are mma.sync m16n8k16 with the query heads of the
//    KV head as the 16 rows. Tensor throughput is no limit here (128 instructions per
//    32 KB of cache), which is why this is not a tcgen05 kernel: its M of 128 has no
//    rows to fill. P enters the second product as two terms, P = hi + lo (each rounded to the
//    element type), so P is not rounded to 8 or 11 bits; up to eight query heads the second
//    term takes the unused rows 8 .. 15 of the same product. Outputs that are no numbers are formed
//    again with P as one F32 number (output_again), so that an infinite V counts as the formula says.
//  * F32 caches: FFMA. For the scores a lane takes a quarter of head_dim of one of 8 keys;
//    for the output it takes head_dim / 32 columns of all 8.
// Measured: 64 ragged BF16 sequences (132 k keys, 32 / 8 heads of 128, 541 MB) 98 to 104 us by GPU, 5.2 to 5.5 TB/s,
// 79 to 84 % of a large copy's rate; 16 F32 sequences (587 MB) 99 us, 5.9 TB/s, 90 %. What is left is the join (~5 us)
// and, for BF16, the latency of a warp's chain from copy to product. Eight warps an SM issue in 40 % of
// the cycles.
// Rows past a sequence's end are not read; they and keys of invalid blocks get weight 0.
#include "batch.cuh"
#include "gemv.cuh"

namespace b200 {
namespace {

constexpr int kPbWarps = 4;
constexpr int kPbThreads = 32 * kPbWarps;
constexpr int kPbMostCtas = 320;
constexpr int kJoinThreads = 256;
constexpr int kCluster = 8;
constexpr int kClusterKeys = 4096;
constexpr int64_t kMostKeys = INT32_MAX - 256;

struct PbArgs {
    const void *q = nullptr;
    void *out = nullptr;
    int64_t q_seq = 0, q_head = 0, o_seq = 0, o_head = 0;  // elements
    const char *k = nullptr, *v = nullptr;
    int64_t block_stride = 0, tok_stride = 0, head_stride = 0;  // bytes
    int64_t n_blocks = 0;
    const int32_t *table = nullptr, *lens = nullptr;
    int64_t table_stride = 0;
    int64_t max_keys = 0;  // positions a table row covers (fits 31 bits)
    uint32_t bt = 1;
    int n_seqs = 0, G = 0, VH = 0, HG = 0;  // query heads a KV head; (KV head, head group) pairs; groups a KV head
    float sl2 = 0.f;                        // scale * log2 e
    float *ws = nullptr;
    int32_t *status = nullptr;
};

B200_DEVICE int seq_len(const PbArgs &a, int b) {
    const int64_t n = __ldg(a.lens + b);
    return static_cast<int>(n < 0 ? 0 : (n > a.max_keys ? a.max_keys : n));
}
B200_DEVICE void report_length(const PbArgs &a, int b) {
    const int64_t n = __ldg(a.lens + b);
    if (n < 0 || n > a.max_keys) set_status(a.status, B200_DEV_BAD_POSITION);
}
template <int TILE>
B200_DEVICE int seq_tiles(const PbArgs &a, int b) {
    return static_cast<int>((static_cast<int64_t>(seq_len(a, b)) + TILE - 1) / TILE);
}

// Tiles of the sequences before b (all sequences for b = n_seqs), by a whole warp.
template <int TILE>
B200_DEVICE int64_t tiles_before(const PbArgs &a, int b) {
    int64_t n = 0;
    for (int i = threadIdx.x & 31; i < b; i += 32) n += seq_tiles<TILE>(a, i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    return n;
}

// CTA c of n <= total takes the tiles [total c / n, total (c + 1) / n): at least one.
B200_DEVICE int64_t share_begin(int64_t total, int64_t c, int64_t n) { return total * c / n; }
B200_DEVICE int64_t share_owner(int64_t total, int64_t u, int64_t n) { return ((u + 1) * n - 1) / total; }

// A place in the line of tiles: tile t of (sequence b, virtual head vh).
struct Place {
    int b, vh, len, tiles, t;
    int64_t left;  // tiles of this CTA's share from here on
};

template <int TILE>
B200_DEVICE void place_next(const PbArgs &a, Place &p) {
    --p.left;
    if (++p.t < p.tiles || p.left == 0) return;
    p.t = 0;
    if (++p.vh < a.VH) return;
    p.vh = 0;
    do {  // the share has tiles left, so a sequence with some follows
        ++p.b;
        p.len = seq_len(a, p.b);
    } while (p.len == 0);
    p.tiles = (p.len + TILE - 1) / TILE;
}

template <int TILE>
B200_DEVICE Place place_at(const PbArgs &a, int64_t u0, int64_t u1) {
    const int lane = threadIdx.x & 31;
    int64_t before = 0;  // tiles of the sequences before `base`
    Place p = {};
    for (int base = 0; base < a.n_seqs; base += 32) {
        const int b = base + lane;
        const int64_t n = b < a.n_seqs ? seq_tiles<TILE>(a, b) : 0;
        int64_t incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        const unsigned past = __ballot_sync(0xffffffffu, (before + incl) * a.VH > u0);
        if (past) {
            const int l = __ffs(past) - 1;
            const int64_t excl = before + __shfl_sync(0xffffffffu, incl - n, l);
            p.b = base + l;
            p.len = seq_len(a, p.b);
            p.tiles = (p.len + TILE - 1) / TILE;
            const int64_t in = u0 - excl * a.VH;
            p.vh = static_cast<int>(in / p.tiles);
            p.t = static_cast<int>(in - static_cast<int64_t>(p.vh) * p.tiles);
            p.left = u1 - u0;
            break;
        }
        before += __shfl_sync(0xffffffffu, incl, 31);
    }
    return p;
}

template <typename T, int D, int HB>
struct Geometry {
    static constexpr int kSub = sizeof(T) == 4 ? 8 : 16;      // keys of a warp's sub-tile
    static constexpr int kTile = kSub * kPbWarps;             // keys of a tile
    static constexpr int kRow = D * static_cast<int>(sizeof(T));  // bytes of a cached row
    static constexpr int kChunks = kRow / 16;
    static constexpr int kHalf = kSub * kRow;                 // K (or V) bytes of a sub-tile
    // two CTAs an SM: the merge area of many heads leaves room for two stages
    static constexpr int kStages = HB > 8 || (sizeof(T) == 4 && HB > 2) ? 2 : 3;
    static constexpr int kRec = HB * (D + 2);                 // floats of a partial: o, m, l
    static constexpr int kQPad = D / 4 + 4;                   // F32: a quarter of a query row, padded
    static constexpr size_t kRing = static_cast<size_t>(kPbWarps) * kStages * 2 * kHalf;
    static constexpr size_t kMerge = static_cast<size_t>(kPbWarps) * kRec * 4;
    static constexpr size_t kQ = sizeof(T) == 4 ? static_cast<size_t>(kPbWarps) * HB * (4 * kQPad + 8) * 4 : 0;
    static constexpr size_t kSmem = kRing + kMerge + kQ + kPbWarps * kStages * 4;
};

B200_DEVICE void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
B200_DEVICE void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

// d += a . b, m16n8k16, F32 accumulators. Without FULL the rows 8..15 of A are zero and
// their accumulators are not kept.
template <typename T, bool FULL>
B200_DEVICE void mma16(float (&d)[FULL ? 4 : 2], const uint32_t (&a)[FULL ? 4 : 2], uint32_t b0, uint32_t b1) {
    if constexpr (FULL) {
        if constexpr (sizeof(T) == 2 && __is_same(T, __half))
            asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                         "{%0, %1, %2, %3};"
                         : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                         : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
        else
            asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, "
                         "%9}, {%0, %1, %2, %3};"
                         : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                         : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    } else {
        float x, y;  // rows 8..15: zero
        if constexpr (__is_same(T, __half))
            asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %5}, {%7, %8}, "
                         "{%0, %1, %9, %9};"
                         : "+f"(d[0]), "+f"(d[1]), "=f"(x), "=f"(y)
                         : "r"(a[0]), "r"(0), "r"(a[1]), "r"(b0), "r"(b1), "f"(0.f));
        else
            asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %5}, {%7, "
                         "%8}, {%0, %1, %9, %9};"
                         : "+f"(d[0]), "+f"(d[1]), "=f"(x), "=f"(y)
                         : "r"(a[0]), "r"(0), "r"(a[1]), "r"(b0), "r"(b1), "f"(0.f));
    }
}

template <typename T>
B200_DEVICE uint32_t pack2(float x, float y) {
    if constexpr (__is_same(T, __half)) {
        const __half2 h = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}
template <typename T>
B200_DEVICE float2 unpack2(uint32_t u) {
    if constexpr (__is_same(T, __half)) return __half22float2(*reinterpret_cast<const __half2 *>(&u));
    else return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&u));
}

// One warp's running softmax over 2-byte keys: lane (g = lane / 4, t = lane % 4) holds
// head rows g (and g + 8 with FULL), output columns 8 i + 2 t, + 1.
template <typename T, int D, int HB>
struct WarpState {
    static constexpr bool FULL = HB > 8;
    static constexpr int R = FULL ? 2 : 1;  // head rows a lane holds
    uint32_t q[D / 16][2 * R];
    float o[D / 8][4];  // head rows g and g + 8; without FULL, row g's shares of P's two terms
    float m[R], l[R];

    B200_DEVICE void begin(const PbArgs &a, const Place &p, int h0, int heads, float *, int lane) {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            m[r] = -INFINITY;
            l[r] = 0.f;
            const bool ok = g + 8 * r < heads;
            const T *row = static_cast<const T *>(a.q) + p.b * a.q_seq + (h0 + g + 8 * r) * a.q_head;
#pragma unroll
            for (int s = 0; s < D / 16; ++s)
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    q[s][u * R + r] = ok ? __ldg(reinterpret_cast<const uint32_t *>(row + 16 * s + 8 * u + 2 * t)) : 0u;
        }
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
#pragma unroll
            for (int u = 0; u < 4; ++u) o[i][u] = 0.f;
    }

    // 16 keys at sk / sv (rows of D elements, 16-byte chunk c of row r at c ^ (r & 7));
    // bit j of `live`: key j takes part.
    B200_DEVICE void keys(uint32_t sk, uint32_t sv, uint32_t live, float sl2, float *, int lane) {
        constexpr int RB = D * 2;
        float s[2][2 * R], odd[2][2 * R];  // two sums each: half as long a chain of dependent products
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int u = 0; u < 2 * R; ++u) s[j][u] = odd[j][u] = 0.f;
        const int mat = lane >> 3, rr = lane & 7;
        {
            const uint32_t row = sk + ((mat >> 1) * 8 + rr) * RB;
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
                uint32_t kf[4];
                ldsm4(kf, row + (((2 * ks + (mat & 1)) ^ rr) << 4));
                mma16<T, FULL>(ks & 1 ? odd[0] : s[0], q[ks], kf[0], kf[1]);
                mma16<T, FULL>(ks & 1 ? odd[1] : s[1], q[ks], kf[2], kf[3]);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int u = 0; u < 2 * R; ++u) s[j][u] += odd[j][u];
        }
        const int t2 = 2 * (lane & 3);
        uint32_t hi[2 * R], lo[2 * R];  // A fragments of P: [key half][row]
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float x[2][2];
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    x[j][u] = (live >> (8 * j + t2 + u)) & 1u ? s[j][2 * r + u] * sl2 : -INFINITY;
                    mx = fmaxf(mx, x[j][u]);
                }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float mn = fmaxf(m[r], mx);
            const float ms = mn == -INFINITY ? 0.f : mn;
            const float al = exp2_approx(m[r] - ms);
            if (__any_sync(0xffffffffu, mn > m[r])) {
                l[r] *= al;
#pragma unroll
                for (int i = 0; i < D / 8; ++i)
#pragma unroll
                    for (int u = FULL ? 2 * r : 0; u < (FULL ? 2 * r + 2 : 4); ++u) o[i][u] *= al;
            }
            m[r] = mn;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float p0 = exp2_approx(x[j][0] - ms), p1 = exp2_approx(x[j][1] - ms);
                l[r] += p0 + p1;
                hi[j * R + r] = pack2<T>(p0, p1);
                const float2 h = unpack2<T>(hi[j * R + r]);
                lo[j * R + r] = pack2<T>(p0 - h.x, p1 - h.y);
            }
        }
        const uint32_t row = sv + ((mat & 1) * 8 + rr) * RB;
#pragma unroll
        for (int np = 0; np < D / 16; ++np) {
            uint32_t vf[4];
            ldsm4_t(vf, row + (((2 * np + (mat >> 1)) ^ rr) << 4));
            if constexpr (FULL) {
                mma16<T, true>(o[2 * np], hi, vf[0], vf[1]);
                mma16<T, true>(o[2 * np], lo, vf[0], vf[1]);
                mma16<T, true>(o[2 * np + 1], hi, vf[2], vf[3]);
                mma16<T, true>(o[2 * np + 1], lo, vf[2], vf[3]);
            } else {  // the unused rows 8 .. 15 take P's second term
                const uint32_t both[4] = {hi[0], lo[0], hi[1], lo[1]};
                mma16<T, true>(o[2 * np], both, vf[0], vf[1]);
                mma16<T, true>(o[2 * np + 1], both, vf[2], vf[3]);
            }
        }
    }

    // this warp's partial: o [HB][D], m [HB], l [HB]
    B200_DEVICE void store(float *rec, int lane) {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            const int h = g + 8 * r;
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
                *reinterpret_cast<float2 *>(rec + h * D + 8 * i + 2 * t) =
                    FULL ? make_float2(o[i][2 * r], o[i][2 * r + 1]) : make_float2(o[i][0] + o[i][2], o[i][1] + o[i][3]);
            if (t == 0) {
                rec[HB * D + h] = m[r];
                rec[HB * D + HB + h] = l[r];
            }
        }
    }
};

// F32 keys: lane (key = lane % 8, quarter = lane / 8) scores a quarter of head_dim; the
// output columns are lane * (D / 32) ...
template <int D, int HB>
struct WarpState<float, D, HB> {
    static constexpr int E = D / 32;
    static constexpr int QP = Geometry<float, D, HB>::kQPad;
    float o[HB][E], m[HB], l[HB];

    B200_DEVICE void begin(const PbArgs &a, const Place &p, int h0, int heads, float *sq, int lane) {
        __syncwarp();  // the previous pair's reads of sq are done
#pragma unroll
        for (int g = 0; g < HB; ++g) {
            m[g] = -INFINITY;
            l[g] = 0.f;
            const float *row = static_cast<const float *>(a.q) + p.b * a.q_seq + (h0 + g) * a.q_head;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                o[g][e] = 0.f;
                const int d = lane + 32 * e;
                sq[(g * 4 + d / (D / 4)) * QP + d % (D / 4)] = g < heads ? __ldg(row + d) : 0.f;
            }
        }
        __syncwarp();
    }

    B200_DEVICE void keys(uint32_t sk, uint32_t sv, uint32_t live, float sl2, float *sq, int lane) {
        constexpr int RB = D * 4;
        const int key = lane & 7, quarter = lane >> 3;
        float s[HB];
#pragma unroll
        for (int g = 0; g < HB; ++g) s[g] = 0.f;
        const uint32_t krow = sk + key * RB;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            const float4 kx = lds4(krow + (((quarter * (D / 16) + i) ^ key) << 4));
#pragma unroll
            for (int g = 0; g < HB; ++g) {
                const float4 qx = *reinterpret_cast<const float4 *>(sq + (g * 4 + quarter) * QP + 4 * i);
                s[g] = fmaf(qx.x, kx.x, fmaf(qx.y, kx.y, fmaf(qx.z, kx.z, fmaf(qx.w, kx.w, s[g]))));
            }
        }
        float *sp = sq + HB * 4 * QP;  // [8 keys][HB]
        const bool on = (live >> key) & 1u;
#pragma unroll
        for (int g = 0; g < HB; ++g) {
            s[g] += __shfl_xor_sync(0xffffffffu, s[g], 8);
            s[g] += __shfl_xor_sync(0xffffffffu, s[g], 16);
            s[g] = on ? s[g] * sl2 : -INFINITY;
            float mx = s[g];
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            if (mx > m[g]) {
                const float al = exp2_approx(m[g] - mx);
                l[g] *= al;
#pragma unroll
                for (int e = 0; e < E; ++e) o[g][e] *= al;
                m[g] = mx;
            }
            const float p = exp2_approx(s[g] - (m[g] == -INFINITY ? 0.f : m[g]));
            l[g] += p;
            if (quarter == (g & 3)) sp[key * HB + g] = p;
        }
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            float vx[E];
            if constexpr (E == 4) {
                const float4 t = lds4(sv + k * RB + ((lane ^ k) << 4));
                vx[0] = t.x, vx[1] = t.y, vx[2] = t.z, vx[3] = t.w;
            } else {
                asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];"
                             : "=f"(vx[0]), "=f"(vx[1])
                             : "r"(sv + k * RB + (((lane >> 1) ^ k) << 4) + (lane & 1) * 8));
            }
#pragma unroll
            for (int g = 0; g < HB; ++g) {
                const float p = sp[k * HB + g];
#pragma unroll
                for (int e = 0; e < E; ++e) o[g][e] = fmaf(p, vx[e], o[g][e]);
            }
        }
        __syncwarp();
    }

    B200_DEVICE void store(float *rec, int lane) {
#pragma unroll
        for (int g = 0; g < HB; ++g) {
            float x = l[g];  // one quarter's lanes hold each key once
            x += __shfl_xor_sync(0xffffffffu, x, 1);
            x += __shfl_xor_sync(0xffffffffu, x, 2);
            x += __shfl_xor_sync(0xffffffffu, x, 4);
#pragma unroll
            for (int e = 0; e < E; ++e) rec[g * D + E * lane + e] = o[g][e];
            if (lane == 0) {
                rec[HB * D + g] = m[g];
                rec[HB * D + HB + g] = x;
            }
        }
    }
};

// Columns [c0, c1) of one query head's output once more, by WARPS warps (a key each in turn) with P as
// one F32 number. As two terms it is no factor for an infinite V: the second is often 0 or
// negative, and inf - inf or 0 inf is not P inf. Only for 16-bit outputs that are no numbers.
// smem: WARPS * (D + 2) floats.
template <typename T, int D, int WARPS>
__device__ __noinline__ void output_again(const PbArgs &a, int b, int head, int c0, int c1, float *smem) {
    constexpr int E = D / 32;  // columns lane * E ... of a lane
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, len = seq_len(a, b);
    const T *q = static_cast<const T *>(a.q) + b * a.q_seq + head * a.q_head + lane * E;
    float qx[E], o[E] = {}, m = -INFINITY, l = 0.f;
    for (int e = 0; e < E; ++e) qx[e] = to_f32<T>(q[e]);
    for (int64_t key = warp; key < len; key += WARPS) {
        const uint32_t k32 = static_cast<uint32_t>(key), slot = k32 / a.bt;
        const int32_t blk = __ldg(a.table + b * a.table_stride + slot);
        if (blk < 0 || blk >= a.n_blocks) continue;
        const int64_t off = blk * a.block_stride + static_cast<int64_t>(k32 - slot * a.bt) * a.tok_stride + (head / a.G) * a.head_stride;
        const T *k = reinterpret_cast<const T *>(a.k + off) + lane * E, *v = reinterpret_cast<const T *>(a.v + off) + lane * E;
        float s = 0.f;
        for (int e = 0; e < E; ++e) s = fmaf(qx[e], to_f32<T>(k[e]), s);
        s = warp_sum(s) * a.sl2;
        if (s > m) {
            const float al = exp2_approx(m - s);
            l *= al;
            for (int e = 0; e < E; ++e) o[e] *= al;
            m = s;
        }
        const float p = exp2_approx(s - (m == -INFINITY ? 0.f : m));
        l += p;
        for (int e = 0; e < E; ++e) o[e] = fmaf(p, to_f32<T>(v[e]), o[e]);
    }
    for (int e = 0; e < E; ++e) smem[warp * (D + 2) + lane * E + e] = o[e];
    if (lane == 0) smem[warp * (D + 2) + D] = m, smem[warp * (D + 2) + D + 1] = l;
    __syncthreads();
    for (int c = c0 + static_cast<int>(threadIdx.x); c < c1; c += 32 * WARPS) {
        float M = -INFINITY, ls = 0.f, os = 0.f;
        for (int w = 0; w < WARPS; ++w) M = fmaxf(M, smem[w * (D + 2) + D]);
        for (int w = 0; w < WARPS; ++w) {
            const float f = exp2_approx(smem[w * (D + 2) + D] - (M == -INFINITY ? 0.f : M));
            ls = fmaf(f, smem[w * (D + 2) + D + 1], ls);
            os = fmaf(f, smem[w * (D + 2) + c], os);
        }
        static_cast<T *>(a.out)[b * a.o_seq + head * a.o_head + c] = from_f32<T>(ls != 0.f ? os / ls : 0.f);
    }
    __syncthreads();  // smem is free again
}

// CL: a cluster of kCluster CTAs takes one pair, and writes its output.
template <typename T, int D, int HB, bool CL>
__global__ void __launch_bounds__(kPbThreads, 2) paged_batch_kernel(const __grid_constant__ PbArgs a) {
    using Ge = Geometry<T, D, HB>;
    extern __shared__ __align__(128) unsigned char pb_smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float *merge = reinterpret_cast<float *>(pb_smem + Ge::kRing);
    float *sq = reinterpret_cast<float *>(pb_smem + Ge::kRing + Ge::kMerge) +
                (sizeof(T) == 4 ? warp * HB * (4 * Ge::kQPad + 8) : 0);
    uint32_t *live = reinterpret_cast<uint32_t *>(pb_smem + Ge::kRing + Ge::kMerge + Ge::kQ) + warp * Ge::kStages;
    const uint32_t ring = smem_addr(pb_smem) + warp * Ge::kStages * 2 * Ge::kHalf;

    // CL: this CTA's record. It takes the ring's place once every warp has read its last sub-tile.
    float *own = reinterpret_cast<float *>(pb_smem);
    int64_t u0 = 0, u1 = 0;
    Place at = {};  // what is computed
    if constexpr (CL) {
        const int pair = blockIdx.x / kCluster, rank = blockIdx.x % kCluster;
        at.b = pair / a.VH;
        at.vh = pair % a.VH;
        at.len = seq_len(a, at.b);
        at.tiles = (at.len + Ge::kTile - 1) / Ge::kTile;
        at.t = at.tiles * rank / kCluster;
        at.left = at.tiles * (rank + 1) / kCluster - at.t;
        if (rank == 0 && at.vh == 0 && threadIdx.x == 0) report_length(a, at.b);
        if (at.left == 0)  // no keys: nothing to add
            for (int i = threadIdx.x; i < Ge::kRec; i += kPbThreads)
                own[i] = i >= HB * D && i < HB * D + HB ? -INFINITY : 0.f;
    } else {
        grid_launch_dependents();  // the joining kernel waits for this grid's end
        const int64_t total = tiles_before<Ge::kTile>(a, a.n_seqs) * a.VH;
        const int64_t ctas = min64(gridDim.x, total);
        if (blockIdx.x >= ctas) return;
        u0 = share_begin(total, blockIdx.x, ctas);
        u1 = share_begin(total, blockIdx.x + 1, ctas);
        at = place_at<Ge::kTile>(a, u0, u1);
    }
    const Place start = at;
    Place in = at;  // what is loaded: one block lookup ahead of `issue`
    bool bad = false;

    // lane r < kSub looks up key row r of the sub-tile at `in`
    int64_t row_off = -1;  // byte offset in the pool; -1: no row
    int32_t row_blk = -1;
    bool row_in = false;
    auto lookup = [&] {
        const int64_t key = static_cast<int64_t>(in.t) * Ge::kTile + warp * Ge::kSub + (lane & (Ge::kSub - 1));
        row_in = in.left > 0 && key < in.len;
        if (row_in) {
            const uint32_t k32 = static_cast<uint32_t>(key), slot = k32 / a.bt;
            row_blk = __ldg(a.table + in.b * a.table_stride + slot);
            row_off = static_cast<int64_t>(k32 - slot * a.bt) * a.tok_stride + (in.vh / a.HG) * a.head_stride;
        }
    };
    // copies the looked-up sub-tile into `stage` and looks the next one up
    auto issue = [&](int stage) {
        const bool ok = row_in && row_blk >= 0 && row_blk < a.n_blocks;
        bad |= row_in && !ok;
        const int64_t off = ok ? row_off + row_blk * a.block_stride : -1;
        const uint32_t mask = __ballot_sync(0xffffffffu, ok) & ((1u << Ge::kSub) - 1u);
        if (lane == 0) live[stage] = mask;
        const uint32_t dst = ring + stage * 2 * Ge::kHalf;
        constexpr int RPI = 32 / Ge::kChunks > 0 ? 32 / Ge::kChunks : 1;  // rows an instruction covers
        const int c = lane % Ge::kChunks, r0 = lane / Ge::kChunks;
        if (mask) {
#pragma unroll
            for (int i = 0; i < Ge::kSub / RPI; ++i) {
                const int r = r0 + i * RPI;
                const int64_t o = __shfl_sync(0xffffffffu, off, r);
                const uint32_t d = dst + r * Ge::kRow + ((c ^ (r & 7)) << 4);
                const int n = o >= 0 ? 16 : 0;
                const int64_t src = (o >= 0 ? o : 0) + c * 16;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(a.k + src), "r"(n) : "memory");
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d + Ge::kHalf), "l"(a.v + src), "r"(n)
                             : "memory");
            }
        }
        cp_async_commit();
        if (in.left > 0) place_next<Ge::kTile>(a, in);
        lookup();
    };

    lookup();
#pragma unroll
    for (int s = 0; s < Ge::kStages - 1; ++s) issue(s);
    WarpState<T, D, HB> st;
    int stage = 0;
    bool first = true, fresh = true;  // first tile of the share / of a part
    int part_t0 = 0;
#pragma unroll 1
    while (at.left > 0) {
        const int h0 = (at.vh / a.HG) * a.G + (at.vh % a.HG) * HB;  // first query head
        const int heads = min(HB, a.G - (at.vh % a.HG) * HB);
        if (fresh) {
            st.begin(a, at, h0, heads, sq, lane);
            part_t0 = at.t;
            fresh = false;
        }
        cp_async_wait<Ge::kStages - 2>();
        __syncwarp();  // every lane's copies have landed, and the previous stage has been read
        issue((stage + Ge::kStages - 1) % Ge::kStages);
        const uint32_t mask = live[stage];
        const uint32_t sk = ring + stage * 2 * Ge::kHalf;
        if (mask) st.keys(sk, sk + Ge::kHalf, mask, a.sl2, sq, lane);
        stage = (stage + 1) % Ge::kStages;

        const bool pair_end = at.t + 1 == at.tiles;
        if (pair_end || at.left == 1) {
            // the warps' partials, joined in warp order
            if (!first) __syncthreads();  // the previous part's partials have been read
            first = false;
            st.store(merge + warp * Ge::kRec, lane);
            __syncthreads();
            const bool whole = !CL && pair_end && part_t0 == 0;
            // parts: slot 0 begins with the CTA's share, slot 1 with a pair
            const int slot = part_t0 == 0 && at.left - 1 + (at.t + 1) != u1 - u0 ? 1 : 0;
            float *rec = CL ? own : a.ws + (static_cast<int64_t>(blockIdx.x) * 2 + slot) * Ge::kRec;
            for (int i = threadIdx.x; i < heads * D; i += kPbThreads) {
                const int g = i / D;
                float M = -INFINITY;
#pragma unroll
                for (int w = 0; w < kPbWarps; ++w) M = fmaxf(M, merge[w * Ge::kRec + HB * D + g]);
                const float ms = M == -INFINITY ? 0.f : M;
                float ls = 0.f, os = 0.f;
#pragma unroll
                for (int w = 0; w < kPbWarps; ++w) {
                    const float f = exp2_approx(merge[w * Ge::kRec + HB * D + g] - ms);
                    ls = fmaf(f, merge[w * Ge::kRec + HB * D + HB + g], ls);
                    os = fmaf(f, merge[w * Ge::kRec + i], os);
                }
                if (whole) {
                    static_cast<T *>(a.out)[at.b * a.o_seq + (h0 + g) * a.o_head + (i - g * D)] =
                        from_f32<T>(ls > 0.f || ls != ls ? os / ls : 0.f);
                } else {
                    rec[i] = os;
                    if (i == g * D) {
                        rec[HB * D + g] = M;
                        rec[HB * D + HB + g] = ls;
                    }
                }
            }
            fresh = true;
        }
        place_next<Ge::kTile>(a, at);
    }
    cp_async_wait<0>();
    if (bad) set_status(a.status, B200_DEV_BAD_POSITION);
    if constexpr (CL) {
        cluster_sync();  // every CTA's record is written
        const int rank = blockIdx.x % kCluster;
        const int h0 = (start.vh / a.HG) * a.G + (start.vh % a.HG) * HB, heads = min(HB, a.G - (start.vh % a.HG) * HB);
        const int n = heads * D, i0 = n * rank / kCluster, i1 = n * (rank + 1) / kCluster;
        bool odd = false;
        for (int i = i0 + threadIdx.x; i < i1; i += kPbThreads) {
            const int g = i / D;
            float m[kCluster], l[kCluster], o[kCluster], M = -INFINITY;
#pragma unroll
            for (int c = 0; c < kCluster; ++c) {
                m[c] = ld_dsmem(dsmem_addr(own + HB * D + g, c));
                l[c] = ld_dsmem(dsmem_addr(own + HB * D + HB + g, c));
                o[c] = ld_dsmem(dsmem_addr(own + i, c));
            }
#pragma unroll
            for (int c = 0; c < kCluster; ++c) M = fmaxf(M, m[c]);
            const float ms = M == -INFINITY ? 0.f : M;
            float ls = 0.f, os = 0.f;
#pragma unroll
            for (int c = 0; c < kCluster; ++c) {
                const float f = exp2_approx(m[c] - ms);
                ls = fmaf(f, l[c], ls);
                os = fmaf(f, o[c], os);
            }
            const float x = ls != 0.f ? os / ls : 0.f;
            odd |= !(fabsf(x) < INFINITY);
            static_cast<T *>(a.out)[start.b * a.o_seq + (h0 + g) * a.o_head + (i - g * D)] = from_f32<T>(x);
        }
        if constexpr (sizeof(T) == 2) {
            if (__syncthreads_or(odd))
                for (int g = i0 / D; g * D < i1; ++g)
                    output_again<T, D, kPbWarps>(a, start.b, h0 + g, max(0, i0 - g * D), min(D, i1 - g * D), merge);
        }
        cluster_sync();  // no CTA's shared memory goes away while it is read
    }
}

// Joins the parts of each pair that more than one CTA took, clears the rows of empty
// sequences, and looks for 16-bit outputs that are no numbers. One CTA a pair.
template <typename T, int D, int HB>
__global__ void __launch_bounds__(kJoinThreads) paged_batch_join_kernel(const __grid_constant__ PbArgs a, const int64_t grid) {
    using Ge = Geometry<T, D, HB>;
    __shared__ float factor[HB * kPbMostCtas], scale[HB];
    const int b = static_cast<int>(blockIdx.x / a.VH), vh = static_cast<int>(blockIdx.x % a.VH);
    const int64_t before = tiles_before<Ge::kTile>(a, b);
    const int64_t total = tiles_before<Ge::kTile>(a, a.n_seqs) * a.VH;
    const int64_t ctas = min64(grid, total);  // as in the main kernel
    const int tiles = seq_tiles<Ge::kTile>(a, b);
    const int h0 = (vh / a.HG) * a.G + (vh % a.HG) * HB;
    const int heads = min(HB, a.G - (vh % a.HG) * HB);
    T *out = static_cast<T *>(a.out) + b * a.o_seq + h0 * a.o_head;
    if (threadIdx.x == 0 && vh == 0) report_length(a, b);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int64_t c0 = 0;
    int parts = 0, slot0 = 0;  // CTAs c0 .. c0 + parts - 1 hold parts; only the first's may be a second part
    if (tiles > 0) {
        const int64_t ua = before * a.VH + static_cast<int64_t>(vh) * tiles;
        c0 = share_owner(total, ua, ctas);
        parts = static_cast<int>(share_owner(total, ua + tiles - 1, ctas) - c0) + 1;
        slot0 = share_begin(total, c0, ctas) >= ua ? 0 : 1;
    }
    grid_wait();
    const auto again = [&](bool odd) {
        if constexpr (sizeof(T) == 2) {
            if (__syncthreads_or(odd))
                for (int g = 0; g < heads; ++g) output_again<T, D, kJoinThreads / 32>(a, b, h0 + g, 0, D, factor);
        }
    };
    if (parts == 1) {  // whole: written by its CTA
        bool odd = false;
        if constexpr (sizeof(T) == 2)
            for (int i = tid; i < heads * D / 2; i += kJoinThreads) {
                const float2 x = unpack2<T>(__ldcg(reinterpret_cast<const uint32_t *>(out + (2 * i / D) * a.o_head + 2 * i % D)));
                odd |= !(fabsf(x.x) < INFINITY && fabsf(x.y) < INFINITY);
            }
        again(odd);
        return;
    }
    if (parts == 0) {
        for (int i = tid; i < heads * D; i += kJoinThreads) out[(i / D) * a.o_head + i % D] = from_f32<T>(0.f);
        return;
    }
    const float *first = a.ws + (c0 * 2 + slot0) * Ge::kRec, *rest = a.ws + c0 * 2 * Ge::kRec;
    const auto part = [&](int i) { return i == 0 ? first : rest + static_cast<int64_t>(i) * 2 * Ge::kRec; };
    // each part's factor 2^(m - M) / sum, a warp per head and a lane per part
    for (int g = warp; g < heads; g += kJoinThreads / 32) {
        float M = -INFINITY;
        for (int i = lane; i < parts; i += 32) {
            const float m = __ldcg(part(i) + HB * D + g);
            factor[g * kPbMostCtas + i] = m;
            M = fmaxf(M, m);
        }
        M = warp_max(M);
        const float ms = M == -INFINITY ? 0.f : M;
        float sum = 0.f;
        for (int i = lane; i < parts; i += 32) {
            const float f = exp2_approx(factor[g * kPbMostCtas + i] - ms);
            factor[g * kPbMostCtas + i] = f;
            sum = fmaf(f, __ldcg(part(i) + HB * D + HB + g), sum);
        }
        sum = warp_sum(sum);
        if (lane == 0) scale[g] = sum != 0.f ? 1.0f / sum : 0.f;
    }
    __syncthreads();
    bool odd = false;
    for (int j = tid; j < heads * D; j += kJoinThreads) {
        const int g = j / D;
        float acc = 0.f;
#pragma unroll 8
        for (int i = 0; i < parts; ++i) acc = fmaf(factor[g * kPbMostCtas + i], __ldcg(part(i) + j), acc);
        odd |= !(fabsf(acc * scale[g]) < INFINITY);
        out[g * a.o_head + (j - g * D)] = from_f32<T>(acc * scale[g]);
    }
    again(odd);
}

int pb_max_ctas() { return device_sm_count() * 2 < kPbMostCtas ? device_sm_count() * 2 : kPbMostCtas; }

// Few pairs with short tables: a cluster each, no workspace.
bool pb_one_launch(int64_t pairs, int64_t max_keys) {
    // at most the clusters that run at once: 32 on 148 SMs, as a GPC's last SMs hold no whole cluster
    return pairs * (kCluster + 1) <= pb_max_ctas() && max_keys <= kClusterKeys;
}

// heads a block handles: the next instantiated size
int pb_heads(int64_t G, bool f32) {
    if (!f32) return G <= 8 ? 8 : 16;
    return G <= 1 ? 1 : (G <= 2 ? 2 : (G <= 4 ? 4 : 8));
}

template <typename T, int D, int HB>
cudaError_t pb_launch(PbArgs a, int64_t Hkv, cudaStream_t st) {
    using Ge = Geometry<T, D, HB>;
    a.HG = (a.G + HB - 1) / HB;
    a.VH = static_cast<int>(Hkv) * a.HG;
    const int64_t pairs = static_cast<int64_t>(a.n_seqs) * a.VH;
    if (pairs > INT32_MAX) return cudaErrorNotSupported;
    const auto allow = [](const void *kern, size_t bytes) {
        return once_per_device(kern, ATTR_SMEM, [&] {
            return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
        });
    };
    if (pb_one_launch(pairs, a.max_keys)) {
        auto kern = paged_batch_kernel<T, D, HB, true>;
        const cudaError_t e = allow(reinterpret_cast<const void *>(kern), Ge::kSmem);
        if (e != cudaSuccess) return e;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(static_cast<unsigned>(pairs * kCluster));
        cfg.blockDim = dim3(kPbThreads);
        cfg.dynamicSmemBytes = Ge::kSmem;
        cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = kCluster;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        return cudaLaunchKernelEx(&cfg, kern, a);
    }
    auto kern = paged_batch_kernel<T, D, HB, false>;
    cudaError_t e = allow(reinterpret_cast<const void *>(kern), Ge::kSmem);
    if (e != cudaSuccess) return e;
    const int64_t most = (a.max_keys + Ge::kTile - 1) / Ge::kTile;  // tiles of the longest possible sequence
    const int64_t ctas = min64(pb_max_ctas(), most > pb_max_ctas() ? pb_max_ctas() : pairs * most);
    e = b200_launch(kern, dim3(static_cast<unsigned>(ctas)), dim3(kPbThreads), Ge::kSmem, st, false, a);
    if (e != cudaSuccess) return e;
    return b200_launch(paged_batch_join_kernel<T, D, HB>, dim3(static_cast<unsigned>(pairs)), dim3(kJoinThreads), 0, st, true,
                       a, ctas);
}

template <typename T, int D>
cudaError_t pb_by_heads(const PbArgs &a, int64_t Hkv, cudaStream_t st) {
    const int hb = pb_heads(a.G, sizeof(T) == 4);
    if constexpr (sizeof(T) == 4) {
        switch (hb) {
            case 1: return pb_launch<T, D, 1>(a, Hkv, st);
            case 2: return pb_launch<T, D, 2>(a, Hkv, st);
            case 4: return pb_launch<T, D, 4>(a, Hkv, st);
        }
        return pb_launch<T, D, 8>(a, Hkv, st);
    } else {
        return hb == 8 ? pb_launch<T, D, 8>(a, Hkv, st) : pb_launch<T, D, 16>(a, Hkv, st);
    }
}

template <typename T>
cudaError_t pb_by_dim(const PbArgs &a, int64_t Hkv, int64_t D, cudaStream_t st) {
    return D == 128 ? pb_by_heads<T, 128>(a, Hkv, st) : pb_by_heads<T, 64>(a, Hkv, st);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

size_t b200_flash_attn_paged_batch_workspace_bytes(int64_t n_seqs, int64_t max_keys, int64_t D, int64_t Hq, int64_t Hkv,
                                                   int32_t dtype) {
    if (n_seqs <= 0 || max_keys <= 0 || D <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || !dtype_bytes(dtype)) return 0;
    const int64_t G = Hq / Hkv;
    const int hb = pb_heads(G, dtype == B200_DTYPE_F32);
    if (pb_one_launch(n_seqs * Hkv * ((G + hb - 1) / hb), max_keys)) return 0;
    // two partial records a CTA (its share's first and last part)
    return static_cast<size_t>(pb_max_ctas()) * 2 * hb * (D + 2) * 4;
}

int b200_flash_attn_paged_batch(const void *q, int64_t q_seq_stride, int64_t q_head_stride, void *out,
                                int64_t out_seq_stride, int64_t out_head_stride, const b200_kv_pool *pool,
                                const int32_t *block_table, int64_t table_stride, int64_t max_blocks,
                                const int32_t *seq_lens, int64_t n_seqs, int64_t Hq, float scale, void *workspace,
                                size_t workspace_bytes, int32_t *dev_status, void *stream) {
    if (n_seqs < 0 || Hq <= 0) return B200_ERR_INVALID_ARGUMENT;
    const int rc = check_pool(pool);
    if (rc != B200_OK) return rc;
    const int64_t D = pool->head_dim, Hkv = pool->n_head_kv;
    if (Hq % Hkv) return B200_ERR_INVALID_ARGUMENT;
    if (n_seqs == 0) return B200_OK;
    if (!q || !out || !block_table || !seq_lens || max_blocks <= 0 || table_stride < max_blocks)
        return B200_ERR_INVALID_ARGUMENT;
    const int e = dtype_bytes(pool->dtype);
    if ((D != 64 && D != 128) || n_seqs > kMostRows || Hq > 65536 || !rows_aligned16(q, q_seq_stride, q_head_stride, e) ||
        !rows_aligned16(out, out_seq_stride, out_head_stride, e))
        return B200_ERR_NOT_SUPPORTED;
    // a length and a tile past it fit 31 bits: the tail of a table of more positions is not used
    const int64_t max_keys =
        max_blocks > kMostKeys / pool->block_tokens ? kMostKeys : max_blocks * pool->block_tokens;
    const size_t need = b200_flash_attn_paged_batch_workspace_bytes(n_seqs, max_keys, D, Hq, Hkv, pool->dtype);
    if (need && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < need))
        return B200_ERR_INVALID_ARGUMENT;
    PbArgs a;
    a.q = q;
    a.out = out;
    a.q_seq = q_seq_stride;
    a.q_head = q_head_stride;
    a.o_seq = out_seq_stride;
    a.o_head = out_head_stride;
    a.k = static_cast<const char *>(pool->k);
    a.v = static_cast<const char *>(pool->v);
    a.block_stride = pool->block_stride * e;
    a.tok_stride = pool->tok_stride * e;
    a.head_stride = pool->head_stride * e;
    a.n_blocks = pool->n_blocks;
    a.table = block_table;
    a.lens = seq_lens;
    a.table_stride = table_stride;
    a.bt = static_cast<uint32_t>(pool->block_tokens);
    a.max_keys = max_keys;
    a.n_seqs = static_cast<int>(n_seqs);
    a.G = static_cast<int>(Hq / Hkv);
    a.sl2 = (scale > 0.f ? scale : 1.0f / sqrtf(static_cast<float>(D))) * kLog2e;
    a.ws = static_cast<float *>(workspace);
    a.status = dev_status;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (pool->dtype) {
        case B200_DTYPE_F16: return status_of(pb_by_dim<__half>(a, Hkv, D, st));
        case B200_DTYPE_BF16: return status_of(pb_by_dim<__nv_bfloat16>(a, Hkv, D, st));
    }
    return status_of(pb_by_dim<float>(a, Hkv, D, st));
}

}  // extern "C"
