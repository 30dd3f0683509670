// b200_flash_attn_paged_shared: one query token for each of many sequences that share prefixes, against a paged K/V cache.
//
// out_b = softmax over the keys of the prefix of b's group and b's own keys, of the one pool. Three kernels, each of which may start
// while the one before ends:
//  * the prefixes: the rows of a group (its sequences times the query heads of a KV head) against its prefix in tiles, so that each key
//    is read once for up to 128 rows. 16-bit types: the packed attention's tensor-core kernel (attention_packed_tc.cu), whose K and V tiles
//    are copied block by block; F32 as three F16 products of planes that a kernel before writes from the blocks. Few F32 rows with short
//    prefixes, more than 128 query heads a KV head, or strides that a tensor map cannot hold: F32 FFMA (prefix_ffma_kernel). A prefix
//    is cut into parts, a CTA each (prefix_plan).
//  * the sequences' own keys, as in the batched decode (attention_paged_batch.cu);
//  * the join of all parts.
// Few short sequences take one launch of the batched decode instead, whose clusters read a prefix's keys as their sequence's first.
// 64 BF16 sequences of 32 / 8 heads of 128 behind one prefix of 8192 keys, with 33 k keys of their own (165 MB): 45 to 47 us, of which the
// join 5 to 6 after the own keys' end. A prefix CTA takes an SM's shared memory, so own keys run on the SMs that the plan leaves
// them (a small CTA beside theirs took 61 against 63, but 56 against 47 behind 16384 keys). 4 F32 sequences of 16 / 8 heads behind
// 301 keys: 12 us, one launch.
#include "attention_packed_ffma.cuh"
#include "paged_batch.cuh"

namespace b200 {
namespace {

constexpr int64_t kPrefixShort = 2048;
constexpr int64_t kPrefixParts = 32;  // at most: the join reads all of a row's

// A CTA: 64 rows (RT 4) or 16 (RT 1) of a group and KV head against a part of the prefix's keys.
template <typename T, int D, int RT>
__global__ void __launch_bounds__(kPkThreads, 2) prefix_ffma_kernel(const PackedArgs a, const PrefixArgs px) {
    extern __shared__ __align__(16) float pf_smem[];
    grid_launch_dependents();
    const int part = blockIdx.x % px.parts, kvh = blockIdx.x / px.parts % a.Hkv;
    const PackedTile p = find_prefix_tile(px, a.G, 16 * RT, blockIdx.x / (px.parts * a.Hkv));
    if (p.seq < 0) return;
    const int r0 = p.tile * 16 * RT, rows = min(16 * RT, p.nq * a.G - r0);
    const int64_t tiles = (static_cast<int64_t>(p.nk) + kPkKeys - 1) / kPkKeys;
    const int first = static_cast<int>(tiles * part / px.parts) * kPkKeys;
    const int end = static_cast<int>(min64(p.nk, tiles * (part + 1) / px.parts * kPkKeys));
    const auto row_of = [&](int r) { return prefix_row(px, part, p.q0 + (r0 + r) / a.G, kvh * a.G + (r0 + r) % a.G); };
    if (__syncthreads_or(prefix_bad(px, p.seq, first, end, threadIdx.x, kPkThreads))) {
        if (threadIdx.x == 0) set_status(a.status, B200_DEV_BAD_POSITION);
        if (threadIdx.x < rows) px.ml[row_of(threadIdx.x)] = make_float2(0.f, -1.f);  // the joining kernel clears the group's rows
        return;
    }
    ffma_rows<T, D, false, RT>(
        a, p, kvh, r0, rows, first, end, PrefixKeys<T>(a, px, p.seq, kvh), pf_smem, threadIdx.x, [] { __syncthreads(); },
        [&](int r, int c, const float (&x)[4], float m, float l) {
            const int64_t row = row_of(r);
            *reinterpret_cast<float4 *>(px.o + row * D + c) = make_float4(x[0], x[1], x[2], x[3]);
            if (c == 0) px.ml[row] = make_float2(m, l);
        });
}

// How the prefixes are cut: rows of a tile (sequences, or with FFMA sequences times heads), tiles a CTA, parts of the keys.
struct PrefixPlan {
    bool within = false;           // no kernel of their own
    bool tc = false, few = false;  // few: FFMA tiles of 16 rows
    int tiles = 1, parts = 0;
    int64_t room = 0;  // F32 on the tensor cores: positions a group in the planes
    int64_t early = 0;  // CTAs of the own keys that the prefixes' SMs leave room for
};
// Model of the tensor-core kernel and of the own keys' (us, kB a us): what a CTA's start and end and a tile of 128 keys take, and
// the rate of own keys on all SMs.
constexpr float kPxStart = 8.f, kPxStartF32 = 16.f, kPxTile = 2.5f, kPxTileF32 = 2.2f, kPxOwnRate = 4500.f;
// About the same start and tile, rounded down to whole units of the own keys' line (0.7 us).
constexpr int kGapStart = 10, kGapStartF32 = 20, kGapTile = 3;
constexpr size_t kPrefixMostPlanes = size_t(1) << 30;
PrefixPlan prefix_plan(int64_t n_seqs, int64_t max_keys, int64_t n_groups, int64_t max_prefix, int64_t D, int64_t G, int64_t Hkv,
                       int32_t dtype) {
    PrefixPlan p;
    if (n_groups <= 0 || n_seqs <= 0 || max_prefix <= 0) return p;
    // Few short pairs, prefixes included: one launch that reads a prefix once a sequence, from L2 after the first (4 sequences of
    // 16 / 8 heads of 128 behind 300, 2000 and 3500 keys, one launch against a kernel of the prefixes' and the own keys': F32 12
    // us against 19, 18.5 against 31, 24.6 against 45; BF16 12 against 17, 12.7 against 22.6, 16.6 against 24.5).
    p.within = paged_batch_one_launch(n_seqs, max_keys + max_prefix, G, Hkv, dtype);
    if (p.within) return p;
    // As if groups were alike, since the host knows neither lengths nor counts. (One of 32 sequences behind 8192 keys among 32 of
    // one sequence each takes one part: 147 us, against 45 with those 32 outside every group.)
    const int64_t groups = min64(n_groups, n_seqs), each = (n_seqs + groups - 1) / groups;
    p.few = each * G <= 16;
    p.tc = G <= kPrefixTcRows;
    if (dtype == B200_DTYPE_F32 && p.tc) {
        // F32 takes the tensor cores unless few rows meet short prefixes (16 / 8 heads of 128, whole calls, FFMA against tensor
        // cores: 16 rows of 2000 keys 30.8 us against 31.8, 8 of 8192 94 against 83; 32 rows of 1000 35 against 28.5, 40 of 300 35
        // against 28.7, 128 of 8192 180 against 86), or the planes, which are as long as the table, grow past a GiB.
        p.room = (max_prefix + 127) / 128 * 128;
        p.tc = !(p.few && max_prefix <= kPrefixShort) && n_groups <= INT32_MAX / p.room &&
               p.room * n_groups <= static_cast<int64_t>(kPrefixMostPlanes / 8) / (D * Hkv);
        if (!p.tc) p.room = 0;
    }
    int64_t rows = p.tc ? kPrefixTcRows / G : (p.few ? 16 : kPkRows);
    // 16-bit types: a group of more than one tile takes two a CTA, over the same keys.
    if (p.tc && dtype != B200_DTYPE_F32 && each > rows) p.tiles = 2;
    rows *= p.tiles;
    const int64_t ctas = groups * (((p.tc ? each : each * G) + rows - 1) / rows) * Hkv;
    // As many parts as the CTAs that run at once allow, of two key tiles at least (one, where two tiles of rows alternate or are few).
    const int64_t keys = p.tc ? 256 / p.tiles : (p.few ? kPkKeys : 2 * kPkKeys);
    const int64_t most = min64(kPrefixParts, (max_prefix + keys - 1) / keys);
    const int64_t sms = device_sm_count(), room = max64(1, min64(most, (p.tc ? sms * 3 / 4 : 2 * sms) / ctas));
    p.parts = static_cast<int>(room);
    if (!p.tc) return p;
    // Own keys run beside the prefixes on the SMs that these leave. The fewest parts with which the prefixes end before their
    // keys do, as if own lengths were half of what the table holds: fewer starts, and less to join. (Whole calls with all, 112,
    // 80, 56, 40 and 24 SMs for the prefixes, the rule's last: 64 BF16 sequences behind 8192 keys with 33 k of their own 57, 53,
    // 49.5, 49, 45, 61.5; 46. 16 behind 4096 with 16 k 37, 36, 33, 30, 29, 35; 29.6. 64 behind 16384 with one each 47, 41, 47, 57,
    // 73, 107; 41.)
    const float own = 0.5f * n_seqs * max_keys * Hkv * D * (dtype == B200_DTYPE_F32 ? 8 : 4) * 1e-3f / kPxOwnRate;
    const auto time = [&](int64_t parts) {
        const int64_t steps = ((max_prefix + 127) / 128 + parts - 1) / parts;
        return dtype == B200_DTYPE_F32 ? kPxStartF32 + kPxTileF32 * steps : kPxStart + kPxTile * steps;
    };
    for (int64_t parts = 1; parts < room; ++parts) {
        const float t = time(parts);
        // (twice the shortest time at most: tables may be far wider than their sequences are long)
        if (t > 0.9f * (own + t * ctas * parts / sms) || t > 2.f * time(room)) continue;
        p.parts = static_cast<int>(parts);
        break;
    }
    p.early = 2 * max64(0, sms - ctas * p.parts);
    return p;
}

// Bytes of the parts, and of the planes behind them. Several parts hold at most the rows of the CTAs that run at once, whatever the sizes
// are, so that room for them does for calls of fewer sequences too.
size_t prefix_parts_bytes(int64_t n_seqs, const PrefixPlan &p, int64_t D, int64_t Hq) {
    if (p.parts == 0) return 0;
    const int64_t sms = device_sm_count(), at_once = max64(sms * 3 / 4 * 2 * kPrefixTcRows, 2 * sms * kPkRows);
    return (static_cast<size_t>(max64(n_seqs * Hq, at_once)) * (D * 4 + 8) + 127) / 128 * 128;
}
size_t prefix_bytes(int64_t n_seqs, int64_t n_groups, const PrefixPlan &p, int64_t D, int64_t Hq, int64_t Hkv) {
    return prefix_parts_bytes(n_seqs, p, D, Hq) + (p.room ? prefix_planes_bytes(n_groups, p.room, D, Hkv) : 0);
}

template <typename T, int D, int RT>
cudaError_t prefix_ffma_launch(const PackedArgs &a, const PrefixArgs &px, cudaStream_t st) {
    auto kern = prefix_ffma_kernel<T, D, RT>;
    const cudaError_t e = once_per_device(reinterpret_cast<const void *>(kern), ATTR_SMEM, [&] {
        return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(ffma_smem<D>()));
    });
    if (e != cudaSuccess) return e;
    const int64_t ctas = px.tiles_run * a.Hkv * px.parts;
    if (ctas > INT32_MAX) return cudaErrorNotSupported;
    return b200_launch(kern, dim3(static_cast<unsigned>(ctas)), dim3(kPkThreads), ffma_smem<D>(), st, false, a, px);
}

template <typename T>
cudaError_t prefix_ffma_by_dim(const PackedArgs &a, const PrefixArgs &px, bool few, cudaStream_t st) {
    if (few) return a.D == 128 ? prefix_ffma_launch<T, 128, 1>(a, px, st) : prefix_ffma_launch<T, 64, 1>(a, px, st);
    return a.D == 128 ? prefix_ffma_launch<T, 128, 4>(a, px, st) : prefix_ffma_launch<T, 64, 4>(a, px, st);
}

cudaError_t prefix_ffma_by_type(const PackedArgs &a, const PrefixArgs &px, bool few, cudaStream_t st) {
    switch (a.dtype) {
        case B200_DTYPE_F16: return prefix_ffma_by_dim<__half>(a, px, few, st);
        case B200_DTYPE_BF16: return prefix_ffma_by_dim<__nv_bfloat16>(a, px, few, st);
    }
    return prefix_ffma_by_dim<float>(a, px, few, st);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

size_t b200_flash_attn_paged_shared_workspace_bytes(int64_t n_seqs, int64_t max_keys, int64_t n_groups, int64_t max_prefix,
                                                    int64_t D, int64_t Hq, int64_t Hkv, int32_t dtype) {
    if (n_seqs <= 0 || max_keys <= 0 || n_groups < 0 || max_prefix < 0 || D <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv ||
        !dtype_bytes(dtype))
        return 0;
    return prefix_bytes(n_seqs, n_groups, prefix_plan(n_seqs, max_keys, n_groups, max_prefix, D, Hq / Hkv, Hkv, dtype), D, Hq, Hkv) +
           paged_batch_prefix_bytes(n_seqs, max_keys, D, Hq / Hkv, Hkv, dtype);
}

int b200_flash_attn_paged_shared(const void *q, int64_t q_seq_stride, int64_t q_head_stride, void *out,
                                 int64_t out_seq_stride, int64_t out_head_stride, const b200_kv_pool *pool,
                                 const int32_t *prefix_table, int64_t prefix_stride, int64_t prefix_blocks,
                                 const int32_t *prefix_lens, const int32_t *cu_seqs, int64_t n_groups,
                                 const int32_t *block_table, int64_t table_stride, int64_t max_blocks,
                                 const int32_t *seq_lens, int64_t n_seqs, int64_t Hq, float scale, void *workspace,
                                 size_t workspace_bytes, int32_t *dev_status, void *stream) {
    if (n_seqs < 0 || n_groups < 0 || Hq <= 0) return B200_ERR_INVALID_ARGUMENT;
    const int rc = check_pool(pool);
    if (rc != B200_OK) return rc;
    const int64_t D = pool->head_dim, Hkv = pool->n_head_kv;
    if (Hq % Hkv) return B200_ERR_INVALID_ARGUMENT;
    if (n_seqs == 0) return B200_OK;
    if (!q || !out || !block_table || !seq_lens || max_blocks <= 0 || table_stride < max_blocks ||
        (n_groups > 0 && (!prefix_table || !prefix_lens || !cu_seqs || prefix_blocks <= 0 || prefix_stride < prefix_blocks)))
        return B200_ERR_INVALID_ARGUMENT;
    const int e = dtype_bytes(pool->dtype);
    if ((D != 64 && D != 128) || n_seqs > kMostRows || n_groups > kMostRows || Hq > 65536 ||
        !rows_aligned16(q, q_seq_stride, q_head_stride, e) || !rows_aligned16(out, out_seq_stride, out_head_stride, e))
        return B200_ERR_NOT_SUPPORTED;
    const auto positions = [&](int64_t blocks) {
        return blocks > kMostKeys / pool->block_tokens ? kMostKeys : blocks * pool->block_tokens;
    };
    const int64_t max_keys = positions(max_blocks), max_prefix = n_groups ? positions(prefix_blocks) : 0;
    const size_t need =
        b200_flash_attn_paged_shared_workspace_bytes(n_seqs, max_keys, n_groups, max_prefix, D, Hq, Hkv, pool->dtype);
    if (need && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < need))
        return B200_ERR_INVALID_ARGUMENT;
    const float sl2 = (scale > 0.f ? scale : 1.0f / sqrtf(static_cast<float>(D))) * kLog2e;
    PrefixArgs px;
    px.cu = cu_seqs;
    px.lens = prefix_lens;
    px.table = prefix_table;
    px.table_stride = prefix_stride;
    px.max_keys = max_prefix;
    px.n_blocks = pool->n_blocks;
    px.block_stride = pool->block_stride;
    px.tok_stride = pool->tok_stride;
    px.head_stride = pool->head_stride;
    px.bt = static_cast<uint32_t>(pool->block_tokens);
    px.n_groups = static_cast<int32_t>(n_groups);
    px.n_seqs = static_cast<int32_t>(n_seqs);
    px.Hq = static_cast<int32_t>(Hq);
    const PrefixPlan plan = prefix_plan(n_seqs, max_keys, n_groups, max_prefix, D, Hq / Hkv, Hkv, pool->dtype);
    px.parts = plan.parts;
    px.tiles = plan.tiles;
    px.within = plan.within;
    px.early = static_cast<int32_t>(plan.early);
    px.gap_start = pool->dtype == B200_DTYPE_F32 ? kGapStartF32 : kGapStart;
    px.gap_tile = kGapTile;
    px.o = static_cast<float *>(workspace);
    px.ml = reinterpret_cast<float2 *>(px.o + px.parts * n_seqs * Hq * D);
    px.room = plan.room;
    px.planes = plan.room ? static_cast<char *>(workspace) + prefix_parts_bytes(n_seqs, plan, D, Hq) : nullptr;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (px.parts > 0) {
        PackedArgs p;
        p.q = q;
        p.k = pool->k;
        p.v = pool->v;
        p.q_tok = q_seq_stride;
        p.q_head = q_head_stride;
        p.total_q = n_seqs;
        p.n_seqs = px.n_groups;
        p.Hq = px.Hq;
        p.Hkv = static_cast<int>(Hkv);
        p.G = static_cast<int>(Hq / Hkv);
        p.D = static_cast<int>(D);
        p.sl2 = sl2;
        p.dtype = pool->dtype;
        p.status = dev_status;
        px.tile_rows = static_cast<int32_t>(plan.tiles * (kPrefixTcRows / p.G));
        px.tiles_run = plan.tc ? most_prefix_tiles(n_groups, n_seqs, 1, px.tile_rows) : 0;
        cudaError_t rc2 = plan.tc ? prefix_tc_launch(p, px, st) : cudaErrorNotSupported;
        if (rc2 == cudaErrorNotSupported) {
            px.early = 0;
            px.tile_rows = plan.few ? 16 : kPkRows;
            px.tile_heads = p.G;
            px.tiles_run = most_prefix_tiles(n_groups, n_seqs, p.G, px.tile_rows);
            rc2 = prefix_ffma_by_type(p, px, plan.few, st);
        }
        if (rc2 != cudaSuccess) return status_of(rc2);
    }
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
    a.sl2 = sl2;
    a.status = dev_status;
    return status_of(paged_batch_prefix_launch(a, px, Hkv, D, pool->dtype,
                                               static_cast<char *>(workspace) + prefix_bytes(n_seqs, n_groups, plan, D, Hq, Hkv), st));
}

}  // extern "C"
