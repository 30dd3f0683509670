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

// RT neighbouring numbers of shared memory.
template <int RT>
B200_DEVICE void read_rows(const float *p, float (&x)[RT]) {
    if constexpr (RT == 4) {
        const float4 v = *reinterpret_cast<const float4 *>(p);
        x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    } else {
        static_assert(RT == 1, "four rows a thread, or one");
        x[0] = *p;
    }
}

template <int D>
constexpr size_t ffma_smem() {
    return (2 * static_cast<size_t>(D) * kPkPad + static_cast<size_t>(kPkKeys) * D) * 4;
}

// Rows [r0, r0 + rows) of sequence p (row = token * G + head of the KV head's group) against its keys [first, end), with CAUSAL
// those that each row sees. kPkThreads threads take RT rows each, so rows is at most 16 RT (kPkRows with RT 4); this one is `tid`.
//  * key(j, k, v) points at key j's rows; false: it takes no part.
//  * sync() is the threads' barrier, smem (16-byte aligned, ffma_smem<D>() bytes) theirs.
//  * store(row, column, x, m, l) gets each row's output four columns at a time, already over l, its maximum (in powers of
//    two) and its sum.
template <typename T, int D, bool CAUSAL, int RT = 4, typename Key, typename Sync, typename Store>
B200_DEVICE void ffma_rows(const PackedArgs &a, const PackedTile &p, int kvh, int r0, int rows, int first, int end, Key key,
                           float *smem, int tid, Sync sync, Store store) {
    float *qt = smem;                  // [D][row]
    float *kt = qt + D * kPkPad;       // [D][key]; then P [key][row]
    float *vs = kt + D * kPkPad;       // [key][D]
    const int ty = tid >> 4, tx = tid & 15;
    const T *q = static_cast<const T *>(a.q);
    // four elements a load; lanes take neighbouring rows, so the transposed stores do not collide
#pragma unroll
    for (int i0 = 0; i0 < 16 * RT * D / 4; i0 += kPkThreads) {
        const int i = i0 + tid, r = i % (16 * RT), d = i / (16 * RT) * 4;
        float x[4] = {0.f, 0.f, 0.f, 0.f};
        if (r < rows) {
            const int tok = (r0 + r) / a.G, h = kvh * a.G + (r0 + r) % a.G;
            load4(q + (p.q0 + tok) * a.q_tok + h * a.q_head + d, x);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) qt[(d + e) * kPkPad + r] = x[e];
    }
    if (CAUSAL) end = min(end, p.nk - p.nq + (r0 + rows - 1) / a.G + 1);  // the keys the last row sees
    int last[RT];  // last key each row sees (relative to the sequence)
#pragma unroll
    for (int i = 0; i < RT; ++i)
        last[i] = RT * ty + i < rows ? (CAUSAL ? min(end - 1, p.nk - p.nq + (r0 + RT * ty + i) / a.G) : end - 1) : -1;
    float m[RT], l[RT], o[RT][D / 16];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int e = 0; e < D / 16; ++e) o[i][e] = 0.f;
    }
    for (int k0 = first; k0 < end; k0 += kPkKeys) {
        sync();
        static_assert(kPkThreads % kPkKeys == 0, "a thread loads of one key");
        const int j = tid % kPkKeys;
        const T *k = nullptr, *v = nullptr;
        const bool has = k0 + j < end && key(k0 + j, k, v);
#pragma unroll
        for (int i0 = 0; i0 < kPkKeys * D / 4; i0 += kPkThreads) {
            const int d = (i0 + tid) / kPkKeys * 4;
            float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
            if (has) {
                load4(k + d, x);
                load4(v + d, y);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) kt[(d + e) * kPkPad + j] = x[e];
            *reinterpret_cast<float4 *>(vs + j * D + d) = make_float4(y[0], y[1], y[2], y[3]);
        }
        sync();
        float s[RT][4] = {};
#pragma unroll 8
        for (int d = 0; d < D; ++d) {
            float xs[RT], ys[4];
            read_rows<RT>(qt + d * kPkPad + RT * ty, xs);
            read_rows<4>(kt + d * kPkPad + 4 * tx, ys);
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[i][j] = fmaf(xs[i], ys[j], s[i][j]);
        }
#pragma unroll
        for (int i = 0; i < RT; ++i) {
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
        for (int j = 0; j < 4; ++j) {
            float *to = kt + (4 * tx + j) * kPkPad + RT * ty;
            if constexpr (RT == 4) *reinterpret_cast<float4 *>(to) = make_float4(s[0][j], s[1][j], s[2][j], s[3][j]);
            else *to = s[0][j];
        }
        sync();
        // a key that a row does not see has P = 0, and 0 times a V that is no number would
        // not be 0: such products are left out where the tile has hidden keys
        const bool all = k0 + kPkKeys - 1 <= (CAUSAL ? min(end - 1, p.nk - p.nq + r0 / a.G) : end - 1);
#pragma unroll 4
        for (int j = 0; j < kPkKeys; ++j) {
            float xs[RT];
            read_rows<RT>(kt + j * kPkPad + RT * ty, xs);
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
                float ys[4];
                read_rows<4>(vs + j * D + 64 * c + 4 * tx, ys);
#pragma unroll
                for (int i = 0; i < RT; ++i)
                    if (all || k0 + j <= last[i]) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[i][4 * c + e] = fmaf(xs[i], ys[e], o[i][4 * c + e]);
                    }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int r = RT * ty + i;
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

// ffma_rows' keys of a packed sequence.
template <typename T>
struct PackedKeys {
    const T *k, *v;
    int64_t k_tok, v_tok;
    B200_DEVICE PackedKeys(const PackedArgs &a, const PackedTile &p, int kvh)
        : k(static_cast<const T *>(a.k) + p.k0 * a.k_tok + kvh * a.k_head),
          v(static_cast<const T *>(a.v) + p.k0 * a.v_tok + kvh * a.v_head), k_tok(a.k_tok), v_tok(a.v_tok) {}
    B200_DEVICE bool operator()(int j, const T *&kr, const T *&vr) const {
        kr = k + j * k_tok, vr = v + j * v_tok;
        return true;
    }
};

}  // namespace b200
