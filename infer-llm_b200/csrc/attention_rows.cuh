// One query token of each sequence against its cached keys, row by row: a CTA a (sequence, KV head), a warp a key in turn.
#pragma once

#include "batch.cuh"

namespace b200 {

constexpr int kArWarps = 8, kArHeads = 4;

// rows(key, lane, k, v): the lane's D / 32 elements of the key's rows; false: the key takes no part.
template <int D, typename Rows, typename Query, typename Store>
B200_DEVICE void attend_rows(int G, int64_t keys, float sl2, Rows rows, Query query, Store store) {
    constexpr int E = D / 32, R = D + 2;
    __shared__ float part[kArWarps * kArHeads * R];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int g0 = 0; g0 < G; g0 += kArHeads) {
        const int heads = min(kArHeads, G - g0);
        float q[kArHeads][E], o[kArHeads][E], m[kArHeads], l[kArHeads];
        for (int g = 0; g < kArHeads; ++g) {
            m[g] = -INFINITY, l[g] = 0.f;
            for (int e = 0; e < E; ++e) o[g][e] = 0.f, q[g][e] = g < heads ? query(g0 + g, lane * E + e) : 0.f;
        }
        for (int64_t j = warp; j < keys; j += kArWarps) {
            float k[E], v[E];
            if (!rows(j, lane, k, v)) continue;
            for (int g = 0; g < heads; ++g) {
                float s = 0.f;
                for (int e = 0; e < E; ++e) s = fmaf(q[g][e], k[e], s);
                s = warp_sum(s) * sl2;
                const float mn = fmaxf(m[g], s), ms = mn == -INFINITY ? 0.f : mn;
                const float al = exp2_approx(m[g] - ms), p = exp2_approx(s - ms);
                m[g] = mn;
                l[g] = l[g] * al + p;
                for (int e = 0; e < E; ++e) o[g][e] = fmaf(p, v[e], o[g][e] * al);
            }
        }
        __syncthreads();
        for (int g = 0; g < kArHeads; ++g) {
            float *r = part + (warp * kArHeads + g) * R;
            for (int e = 0; e < E; ++e) r[lane * E + e] = o[g][e];
            if (lane == 0) r[D] = m[g], r[D + 1] = l[g];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < heads * D; i += 32 * kArWarps) {
            const int g = i / D, d = i % D;
            float M = -INFINITY, ls = 0.f, os = 0.f;
            for (int w = 0; w < kArWarps; ++w) M = fmaxf(M, part[(w * kArHeads + g) * R + D]);
            for (int w = 0; w < kArWarps; ++w) {
                const float *r = part + (w * kArHeads + g) * R;
                const float f = exp2_approx(r[D] - (M == -INFINITY ? 0.f : M));
                ls = fmaf(f, r[D + 1], ls);
                os = fmaf(f, r[d], os);
            }
            store(g0 + g, d, ls != 0.f ? os / ls : 0.f);
        }
        __syncthreads();
    }
}

}  // namespace b200
