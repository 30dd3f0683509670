// Shared pieces of the batched serving operators: element types, the sequence that
// owns a packed row or tile, argument checks.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace b200 {

template <typename T>
B200_DEVICE float to_f32(T x);
template <>
B200_DEVICE float to_f32<float>(float x) { return x; }
template <>
B200_DEVICE float to_f32<__half>(__half x) { return __half2float(x); }
template <>
B200_DEVICE float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
B200_DEVICE T from_f32(float x);
template <>
B200_DEVICE float from_f32<float>(float x) { return x; }
template <>
B200_DEVICE __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
B200_DEVICE __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// 2^x (ex2.approx.ftz: relative error about 2^-22)
B200_DEVICE float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

constexpr float kLog2e = 1.4426950408889634f;

// Rows, keys and sequences of a call: numbers of a tile, or of 32 sequences, past the last one fit 31 bits.
constexpr int64_t kMostRows = INT32_MAX - 1024;

// The sequence s of [0, n) with cu[s] <= t < cu[s + 1], or -1. All lanes of a warp take
// part and get the answer: each round 32 probes narrow the range 32-fold, so the chain
// of dependent loads is log32(n) long. Offsets that are not ascending give some s or
// -1, never a read outside cu[0 .. n].
B200_DEVICE int warp_find_row(const int32_t *cu, int n, int64_t t) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = n + 1;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32;
        const int at = lo + lane * step;
        const bool le = at < hi && __ldg(cu + at) <= t;
        const unsigned b = __ballot_sync(0xffffffffu, le);
        if (!(b & 1u)) return -1;
        const int last = 31 - __clz(static_cast<int>(b));
        const int nlo = lo + last * step;
        hi = nlo + step < hi ? nlo + step : hi;
        lo = nlo;
    }
    return lo < n && __ldg(cu + lo) <= t && t < __ldg(cu + lo + 1) ? lo : -1;
}

// Packed sequences cut into tiles of M rows, a row being one query token with one of the
// G query heads of a KV head (row = token * G + head), so the heads that share keys share
// a tile.
struct PackedTile {
    int seq = -1;             // -1: no such tile
    int tile = 0;             // rows [tile * M, ...) of the sequence
    int nq = 0, nk = 0;       // its queries and keys
    int64_t q0 = 0, k0 = 0;   // its first row in q, in k / v
};

// nq of sequence s (0 where the offsets are not ascending within [0, total]), q0, nk, k0.
B200_DEVICE bool packed_range(const int32_t *cu, int s, int64_t total, int64_t &first, int &n) {
    const int64_t a = __ldg(cu + s), b = __ldg(cu + s + 1);
    const bool ok = a >= 0 && b >= a && b <= total;
    first = ok ? a : 0;
    n = ok ? static_cast<int>(b - a) : 0;
    return ok;
}

// Tile `at` of the line of all tiles (a sequence's last tiles, which see the most keys,
// first), found by a whole warp; each lane takes every 32nd sequence. keys(s, k0, nk) gives a sequence's keys, false: out of range.
template <typename Keys>
B200_DEVICE PackedTile find_tile(const int32_t *cu_q, int n_seqs, int64_t total_q, int G, int M, int64_t at, int32_t *status,
                                 Keys keys) {
    const int lane = threadIdx.x & 31;
    PackedTile p;
    int64_t before = 0;
    for (int base = 0; base < n_seqs; base += 32) {
        const int s = base + lane;
        int64_t q0 = 0, k0 = 0;
        int nq = 0, nk = 0;
        bool ok_k = true;  // (both ranges are read at once: one latency)
        if (s < n_seqs) {
            const bool ok_q = packed_range(cu_q, s, total_q, q0, nq);
            ok_k = keys(s, k0, nk);
            if (!ok_q) set_status(status, B200_DEV_BAD_POSITION);
        }
        // (rows fit 31 bits, with room for a tile)
        int64_t incl = (static_cast<unsigned>(nq) * static_cast<unsigned>(G) + static_cast<unsigned>(M) - 1u) / M;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        const unsigned past = __ballot_sync(0xffffffffu, before + incl > at);
        if (past) {
            const int l = __ffs(past) - 1;
            const int64_t end = before + __shfl_sync(0xffffffffu, incl, l);
            p.seq = base + l;
            p.tile = static_cast<int>(end - 1 - at);
            p.q0 = __shfl_sync(0xffffffffu, q0, l);
            p.nq = __shfl_sync(0xffffffffu, nq, l);
            p.k0 = __shfl_sync(0xffffffffu, k0, l);
            p.nk = __shfl_sync(0xffffffffu, nk, l);
            if (!__shfl_sync(0xffffffffu, static_cast<int>(ok_k), l)) {
                set_status(status, B200_DEV_BAD_POSITION);
                p.seq = -1;
            }
            return p;
        }
        before += __shfl_sync(0xffffffffu, incl, 31);
    }
    return p;
}
B200_DEVICE PackedTile find_packed_tile(const int32_t *cu_q, const int32_t *cu_k, int n_seqs, int64_t total_q,
                                        int64_t total_k, int G, int M, int64_t at, int32_t *status) {
    return find_tile(cu_q, n_seqs, total_q, G, M, at, status,
                     [&](int s, int64_t &k0, int &nk) { return packed_range(cu_k, s, total_k, k0, nk); });
}

// At most this many tiles, whatever the lengths are.
inline int64_t most_packed_tiles(int64_t n_seqs, int64_t total_q, int64_t G, int64_t M) {
    return total_q * G / M + min64(n_seqs, total_q);
}

// x / d = x mul / 2^shift for x < 2^31, d >= 1: for the least l with d <= 2^l, ceil(2^(31 + l) / d) is below 2^32 and
// its product exceeds the quotient by less than 1.
inline void reciprocal31(uint32_t d, uint32_t &mul, uint32_t &shift) {
    for (shift = 31; (1ull << (shift - 31)) < d;) ++shift;
    mul = static_cast<uint32_t>(((1ull << shift) + d - 1) / d);
}

inline bool rows_aligned16(const void *p, int64_t s0, int64_t s1, int elem_bytes) {
    return ((reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(s0 * elem_bytes) |
             static_cast<uintptr_t>(s1 * elem_bytes)) & 15) == 0;
}

inline int dtype_bytes(int32_t dtype) {
    return dtype == B200_DTYPE_F32 ? 4 : (dtype == B200_DTYPE_F16 || dtype == B200_DTYPE_BF16 ? 2 : 0);
}

inline int status_of(cudaError_t e) {
    if (e == cudaSuccess) return B200_OK;
    if (e == cudaErrorInvalidValue) return B200_ERR_INVALID_ARGUMENT;
    if (e == cudaErrorNotSupported) return B200_ERR_NOT_SUPPORTED;
    return B200_ERR_CUDA;
}

// Checks of a pool's description; B200_OK or the error.
inline int check_pool(const b200_kv_pool *p) {
    if (!p || !p->k || !p->v || p->n_blocks <= 0 || p->block_tokens <= 0 || p->n_head_kv <= 0 || p->head_dim <= 0)
        return B200_ERR_INVALID_ARGUMENT;
    const int e = dtype_bytes(p->dtype);
    if (!e) return B200_ERR_INVALID_ARGUMENT;
    if (p->n_blocks > INT32_MAX || p->block_tokens > INT32_MAX) return B200_ERR_NOT_SUPPORTED;
    if (!rows_aligned16(p->k, p->block_stride, p->tok_stride, e) || !rows_aligned16(p->v, p->head_stride, 0, e) ||
        (p->head_dim * e) % 16)
        return B200_ERR_NOT_SUPPORTED;
    return B200_OK;
}

}  // namespace b200
