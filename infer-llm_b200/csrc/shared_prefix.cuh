// Prefixes that groups of sequences share (b200_flash_attn_paged_shared): their kernels leave, for each part of a prefix's keys and each
// (sequence, query head) of its group, the normalised output of those keys with its maximum (in powers of two) and
// sum; the kernel of the sequences' own keys joins them.
#pragma once

#include "attention_packed.cuh"

namespace b200 {

struct PrefixArgs {
    const int32_t *cu = nullptr, *lens = nullptr, *table = nullptr;  // groups' sequences, lengths, blocks
    int64_t table_stride = 0, max_keys = 0, n_blocks = 0;            // max_keys: positions a table row covers (fits 31 bits)
    int64_t block_stride = 0, tok_stride = 0, head_stride = 0;       // of the pool, elements
    uint32_t bt = 1;
    int32_t n_groups = 0, n_seqs = 0, Hq = 0, parts = 0, tiles = 1;  // tiles: of rows, a CTA of the tensor-core kernel
    // F32 on the tensor cores: K and V as planes of F16 numbers with room for `room` positions a group (a multiple of 128), then exponents
    void *planes = nullptr;
    int64_t room = 0;
    // The prefixes' tiles: rows, rows a sequence counts for, and tiles that the grid has room for.
    int32_t tile_rows = 1, tile_heads = 1;
    int64_t tiles_run = 0;
    // CTAs of the own keys that run beside the prefixes' kernel, and how much longer than the others: units of their line of tiles, of the
    // prefix kernel's start and of each key tile of its longest part
    int32_t early = 0, gap_start = 0, gap_tile = 0;
    bool within = false;  // the own keys' kernel takes each sequence's prefix as its first keys; no other runs
    float *o = nullptr;    // [part][sequence][query head][D]
    float2 *ml = nullptr;  // [part][sequence][query head]: maximum, sum (-1: the group's prefix names a block out of range)
};

B200_DEVICE int prefix_len(const PrefixArgs &a, int group) {
    const int64_t n = __ldg(a.lens + group);
    return static_cast<int>(n < 0 ? 0 : (n > a.max_keys ? a.max_keys : n));
}
// The group of sequence b, by a whole warp: -1 if none names it, kSeveralGroups if more than one does, which takes offsets out of
// order. Their CTAs write the same places of the parts then, in any order, so such a row is cleared.
constexpr int kSeveralGroups = -2;
B200_DEVICE int prefix_group(const PrefixArgs &a, int b) {
    int group = -1, n = 0;
    for (int g = threadIdx.x & 31; g < a.n_groups; g += 32) {
        const int from = __ldg(a.cu + g), to = __ldg(a.cu + g + 1);
        if (from >= 0 && from <= b && b < to && to <= a.n_seqs) group = g, ++n;
    }
    n = __reduce_add_sync(0xffffffffu, n);
    group = __reduce_max_sync(0xffffffffu, group);
    return n > 1 ? kSeveralGroups : group;
}
// Where part i's numbers for (sequence b, query head h) are.
B200_DEVICE int64_t prefix_row(const PrefixArgs &a, int part, int64_t b, int h) {
    return (static_cast<int64_t>(part) * a.n_seqs + b) * a.Hq + h;
}
// Elements from the pool's start to KV head h of a prefix's position; -1: the block is out of range.
B200_DEVICE int64_t prefix_key(const PrefixArgs &a, int group, int h, int pos) {
    const uint32_t slot = static_cast<uint32_t>(pos) / a.bt;
    const int64_t blk = __ldg(a.table + group * a.table_stride + slot);
    if (blk < 0 || blk >= a.n_blocks) return -1;
    return blk * a.block_stride + static_cast<int64_t>(static_cast<uint32_t>(pos) - slot * a.bt) * a.tok_stride + h * a.head_stride;
}
// Whether one of the blocks of positions [from, to) is out of range, for lane `lane` of `lanes`.
B200_DEVICE bool prefix_bad(const PrefixArgs &a, int group, int from, int to, int lane, int lanes) {
    bool bad = false;
    if (from >= to) return bad;
    const int64_t last = static_cast<uint32_t>(to - 1) / a.bt;
    for (int64_t s = static_cast<uint32_t>(from) / a.bt + lane; s <= last; s += lanes) {
        const int32_t blk = __ldg(a.table + group * a.table_stride + s);
        bad |= blk < 0 || blk >= a.n_blocks;
    }
    return bad;
}
// At most so many tiles of M rows in all groups, a sequence being G rows.
inline int64_t most_prefix_tiles(int64_t n_groups, int64_t n_seqs, int64_t G, int64_t M) {
    const int64_t groups = min64(n_groups, n_seqs);
    return groups + (n_seqs * G - groups) / M;
}
// Tiles of the groups before `end`, by a whole warp. More than tiles_run only where offsets out of order make groups overlap.
B200_DEVICE int64_t prefix_tiles_before(const PrefixArgs &a, int end) {
    int64_t tiles = 0;
    for (int g = threadIdx.x & 31; g < end; g += 32) {
        int64_t first = 0;
        int n = 0;
        if (packed_range(a.cu, g, a.n_seqs, first, n))
            tiles += (static_cast<int64_t>(n) * a.tile_heads + a.tile_rows - 1) / a.tile_rows;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
    return tiles;
}
// Waits for the prefixes' grid; then, by one CTA, what it had no room for is marked as not to be used.
B200_DEVICE void prefixes_done(const PrefixArgs &a) {
    const int64_t tiles = a.parts > 0 ? prefix_tiles_before(a, a.n_groups) : 0;
    grid_wait();
    if (tiles <= a.tiles_run) return;
    for (int g = 0; g < a.n_groups; ++g) {
        int64_t first = 0;
        int n = 0;
        if (prefix_tiles_before(a, g + 1) <= a.tiles_run || !packed_range(a.cu, g, a.n_seqs, first, n)) continue;
        const int64_t rows = static_cast<int64_t>(n) * a.Hq;
        for (int part = 0; part < a.parts; ++part)
            for (int64_t i = threadIdx.x; i < rows; i += blockDim.x) a.ml[prefix_row(a, part, first, 0) + i] = make_float2(0.f, -1.f);
    }
}
// Tile `at` of M rows of the line of all groups' tiles, a row being a sequence with one of G heads; by a whole warp.
B200_DEVICE PackedTile find_prefix_tile(const PrefixArgs &a, int G, int M, int64_t at) {
    return find_tile(a.cu, a.n_groups, a.n_seqs, G, M, at, nullptr, [&](int s, int64_t &k0, int &nk) {
        k0 = s * a.room;
        nk = prefix_len(a, s);
        return true;
    });
}

// ffma_rows' keys of a prefix.
template <typename T>
struct PrefixKeys {
    const T *k, *v;
    const PrefixArgs &px;
    int group, kvh;
    B200_DEVICE PrefixKeys(const PackedArgs &a, const PrefixArgs &p, int g, int h)
        : k(static_cast<const T *>(a.k)), v(static_cast<const T *>(a.v)), px(p), group(g), kvh(h) {}
    B200_DEVICE bool operator()(int j, const T *&kr, const T *&vr) const {
        const int64_t at = prefix_key(px, group, kvh, j);
        kr = k + at, vr = v + at;
        return at >= 0;
    }
};

// Tensor-core kernel of the prefixes, F32 with `planes` of so many bytes; cudaErrorNotSupported (nothing launched) where it does not apply.
size_t prefix_planes_bytes(int64_t n_groups, int64_t room, int64_t D, int64_t Hkv);
cudaError_t prefix_tc_launch(const PackedArgs &a, const PrefixArgs &p, cudaStream_t st);
constexpr int kPrefixTcRows = 128;  // of a tile: whole sequences times the heads of a KV head

}  // namespace b200
