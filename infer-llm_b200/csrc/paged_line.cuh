// What the one-token attention kernels over paged caches share: the line of key tiles of all sequences and
// its even shares, and mma.sync fragments.
//
// An argument block A has lens (device lengths), max_keys (positions a table row covers, within 31 bits), n_seqs, VH (virtual heads: a KV
// head's groups of query heads, over all KV heads) and status.
#pragma once

#include "batch.cuh"
#include "gemv.cuh"

namespace b200 {

constexpr int64_t kMostKeys = INT32_MAX - 256;

template <typename A>
B200_DEVICE int seq_len(const A &a, int b) {
    const int64_t n = __ldg(a.lens + b);
    return static_cast<int>(n < 0 ? 0 : (n > a.max_keys ? a.max_keys : n));
}
template <typename A>
B200_DEVICE void report_length(const A &a, int b) {
    const int64_t n = __ldg(a.lens + b);
    if (n < 0 || n > a.max_keys) set_status(a.status, B200_DEV_BAD_POSITION);
}
template <int TILE, typename A>
B200_DEVICE int seq_tiles(const A &a, int b) {
    return static_cast<int>((static_cast<int64_t>(seq_len(a, b)) + TILE - 1) / TILE);
}

// The line's units: TU a tile and PU more a (sequence, virtual head), for what its start and end cost. A tile belongs to the share that
// has its first unit.
template <int TU, int PU>
B200_DEVICE int64_t units_of(int64_t tiles) { return tiles ? tiles * TU + PU : 0; }

// Units of a virtual head of the sequences before b (all sequences for b = n_seqs), by a whole warp.
template <int TILE, int TU = 1, int PU = 0, typename A>
B200_DEVICE int64_t tiles_before(const A &a, int b) {
    int64_t n = 0;
    for (int i = threadIdx.x & 31; i < b; i += 32) n += units_of<TU, PU>(seq_tiles<TILE>(a, i));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    return n;
}

// CTA c of n takes the units [total c / n, total (c + 1) / n): at least TU of them, so at least one tile of every pair that
// it lies within, if n <= total / TU.
B200_DEVICE int64_t share_begin(int64_t total, int64_t c, int64_t n) { return total * c / n; }
B200_DEVICE int64_t share_owner(int64_t total, int64_t u, int64_t n) { return ((u + 1) * n - 1) / total; }

// A place in the line of tiles: tile t of (sequence b, virtual head vh).
struct Place {
    int b, vh, len, tiles, t;
    int64_t left;  // units of this CTA's share from the tile's first on; none: past its end
};

// On to the first tile of the next virtual head, or sequence that has keys.
template <int TILE, typename A>
B200_DEVICE void place_pair(const A &a, Place &p) {
    p.t = 0;
    if (++p.vh < a.VH) return;
    p.vh = 0;
    do {  // the share has units left, so a sequence with some follows
        ++p.b;
        p.len = seq_len(a, p.b);
    } while (p.len == 0);
    p.tiles = (p.len + TILE - 1) / TILE;
}

template <int TILE, int TU = 1, int PU = 0, typename A>
B200_DEVICE void place_next(const A &a, Place &p) {
    p.left -= TU;
    if (++p.t < p.tiles || p.left <= 0) return;
    p.left -= PU;
    if (p.left > 0) place_pair<TILE>(a, p);
}

template <int TILE, int TU = 1, int PU = 0, typename A>
B200_DEVICE Place place_at(const A &a, int64_t u0, int64_t u1) {
    const int lane = threadIdx.x & 31;
    int64_t before = 0;  // units of the sequences before `base`
    Place p = {};
    for (int base = 0; base < a.n_seqs; base += 32) {
        const int b = base + lane;
        const int64_t n = b < a.n_seqs ? units_of<TU, PU>(seq_tiles<TILE>(a, b)) : 0;
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
            const int64_t in = u0 - excl * a.VH, pair = units_of<TU, PU>(p.tiles);
            p.vh = static_cast<int>(in / pair);
            const int64_t off = in - static_cast<int64_t>(p.vh) * pair;
            p.t = static_cast<int>((off + TU - 1) / TU);
            p.left = u1 - u0 - (static_cast<int64_t>(p.t) * TU - off);
            if (PU && p.t >= p.tiles) {  // behind the last tile's first unit: the next pair's
                p.left = u1 - u0 - (pair - off);
                if (p.left > 0) place_pair<TILE>(a, p);
            }
            break;
        }
        before += __shfl_sync(0xffffffffu, incl, 31);
    }
    return p;
}

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

}  // namespace b200
