// Causal attention of up to 64 packed rows with F32 FFMA: the kernel for short F32 calls, and what the
// tensor-core kernel does over for F32 tiles that two F16 numbers do not hold.
//
// out_i = sum_j softmax_j(scale q_i . k_j) v_j: 64 rows (tokens times the heads that share a KV head)
// against 64-key tiles, running maximum and sum, scores and output in registers as 4 x 4
// and 4 x D/16 blocks a thread. The FFMA rate bounds it.
#pragma once

#include "attention_packed.cuh"

namespace b200 {

constexpr int kPkRows = 64, kPkKeys = 64, kPkThreads = 256;
constexpr int kPkPad = kPkRows + 4;

B200_DEVICE void load4(const float *p, float (&x)[4]) {
    const float4 v = __ldg(reinterpret_cast<const float4 *>(p));
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
}
template <typename T>
B200_DEVICE void load4(const T *p, float (&x)[4]) {
    const uint2 v = __ldg(reinterpret_cast<const uint2 *>(p));
    const T *e = reinterpret_cast<const T *>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = to_f32<T>(e[i]);
}

template <int D>
constexpr size_t ffma_smem() {
    return (2 * static_cast<size_t>(D) * kPkPad + static_cast<size_t>(kPkKeys) * D) * 4;
}

// Rows [r0, r0 + rows) (row = token * G + head of the KV head's group; at most kPkRows) of sequence p against its
// keys [first, end), by kPkThreads threads, of which this is `tid`; sync() is their barrier and
// smem (16-byte aligned, ffma_smem<D>() bytes) theirs. store(row, column, x, m, l) gets each row's
// output four columns at a time, already over l, its maximum (in powers of two) and its sum.
template <typename T, int D, typename Sync, typename Store>
B200_DEVICE void ffma_rows(const PackedArgs &a, const PackedTile &p, int kvh, int r0, int rows, int first, int end,
                           float *smem, int tid, Sync sync, Store store) {
    float *qt = smem;                  // [D][row]
    float *kt = qt + D * kPkPad;       // [D][key]; then P [key][row]
    float *vs = kt + D * kPkPad;       // [key][D]
    const int ty = tid >> 4, tx = tid & 15;
    const T *q = static_cast<const T *>(a.q), *k = static_cast<const T *>(a.k), *v = static_cast<const T *>(a.v);
    // four elements a load; lanes take neighbouring rows, so the transposed stores do not collide
#pragma unroll
    for (int i0 = 0; i0 < kPkRows * D / 4; i0 += kPkThreads) {
        const int i = i0 + tid, r = i % kPkRows, d = i / kPkRows * 4;
        float x[4] = {0.f, 0.f, 0.f, 0.f};
        if (r < rows) {
            const int tok = (r0 + r) / a.G, h = kvh * a.G + (r0 + r) % a.G;
            load4(q + (p.q0 + tok) * a.q_tok + h * a.q_head + d, x);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) qt[(d + e) * kPkPad + r] = x[e];
    }
    end = min(end, p.nk - p.nq + (r0 + rows - 1) / a.G + 1);  // the keys the last row sees
    int last[4];  // last key each row sees (relative to the sequence)
#pragma unroll
    for (int i = 0; i < 4; ++i) last[i] = 4 * ty + i < rows ? min(end - 1, p.nk - p.nq + (r0 + 4 * ty + i) / a.G) : -1;
    float m[4], l[4], o[4][D / 16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int e = 0; e < D / 16; ++e) o[i][e] = 0.f;
    }
    for (int k0 = first; k0 < end; k0 += kPkKeys) {
        sync();
#pragma unroll
        for (int i0 = 0; i0 < kPkKeys * D / 4; i0 += kPkThreads) {
            const int i = i0 + tid, j = i % kPkKeys, d = i / kPkKeys * 4;
            const int64_t t = p.k0 + k0 + j;
            float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
            if (k0 + j < end) {
                load4(k + t * a.k_tok + kvh * a.k_head + d, x);
                load4(v + t * a.v_tok + kvh * a.v_head + d, y);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) kt[(d + e) * kPkPad + j] = x[e];
            *reinterpret_cast<float4 *>(vs + j * D + d) = make_float4(y[0], y[1], y[2], y[3]);
        }
        sync();
        float s[4][4] = {};
#pragma unroll 8
        for (int d = 0; d < D; ++d) {
            const float4 x = *reinterpret_cast<const float4 *>(qt + d * kPkPad + 4 * ty);
            const float4 y = *reinterpret_cast<const float4 *>(kt + d * kPkPad + 4 * tx);
            const float xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[i][j] = fmaf(xs[i], ys[j], s[i][j]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[i][j] = k0 + 4 * tx + j <= last[i] ? s[i][j] * a.sl2 : -INFINITY;
                mx = fmaxf(mx, s[i][j]);
            }
#pragma unroll
            for (int w = 1; w < 16; w <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
            const float mn = fmaxf(m[i], mx), ms = mn == -INFINITY ? 0.f : mn;
            const float al = exp2_approx(m[i] - ms);
            m[i] = mn;
            l[i] *= al;
#pragma unroll
            for (int e = 0; e < D / 16; ++e) o[i][e] *= al;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[i][j] = exp2_approx(s[i][j] - ms);
                l[i] += s[i][j];
            }
        }
        sync();  // the keys have been read
#pragma unroll
        for (int j = 0; j < 4; ++j)
            *reinterpret_cast<float4 *>(kt + (4 * tx + j) * kPkPad + 4 * ty) = make_float4(s[0][j], s[1][j], s[2][j], s[3][j]);
        sync();
        // a key that a row does not see has P = 0, and 0 times a V that is no number would
        // not be 0: such products are left out where the tile has hidden keys
        const bool all = k0 + kPkKeys - 1 <= min(end - 1, p.nk - p.nq + r0 / a.G);
#pragma unroll 4
        for (int j = 0; j < kPkKeys; ++j) {
            const float4 x = *reinterpret_cast<const float4 *>(kt + j * kPkPad + 4 * ty);
            const float xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
                const float4 y = *reinterpret_cast<const float4 *>(vs + j * D + 64 * c + 4 * tx);
                const float ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (all || k0 + j <= last[i]) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[i][4 * c + e] = fmaf(xs[i], ys[e], o[i][4 * c + e]);
                    }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = 4 * ty + i;
#pragma unroll
        for (int w = 1; w < 16; w <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], w);
        if (r >= rows) continue;
        const float inv = l[i] != 0.f ? 1.0f / l[i] : 0.f;  // no key, or scores of -inf alone: zeros
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
            const float x[4] = {o[i][4 * c] * inv, o[i][4 * c + 1] * inv, o[i][4 * c + 2] * inv, o[i][4 * c + 3] * inv};
            store(r, 64 * c + 4 * tx, x, m[i], l[i]);
        }
    }
}

}  // namespace b200
