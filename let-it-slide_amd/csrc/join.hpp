// Joining the pieces that one row's keys were split into: out = sum_i acc_i 2^(m_i - M) / sum_i l_i 2^(m_i - M), M = max m_i.
#pragma once

#include "rptc_common.hpp"

namespace rptc {

constexpr int kJoinThreads = 256, kJoinMost = 128;

#ifdef __HIPCC__
// One workgroup, one row: acc [pieces][hd] and ml [pieces][2] (bound in log2 units and sum; sum 0 = the piece holds no key).
// Returns the numerator of dimension threadIdx.x (threads below hd); M and the denominator in every thread.  Every
// thread of the workgroup calls it.  256 / hd groups of threads take every so-manieth piece and are added up in a fixed
// order; the first 16 of a thread are asked for before the factors are worked out, one piece a thread, so that a row of
// up to 32 pieces at hd 128 costs one trip to memory (32 heads of 64 pieces: 6.5 us, with a thread per dimension walking over them 22.9).
__device__ __forceinline__ float join_pieces(const float *__restrict__ acc, const float *__restrict__ ml, int pieces, int hd,
                                             float &M, float &den)
{
    constexpr int kAhead = 16;
    __shared__ float s_f[kJoinMost], s_red[2 * kJoinThreads / 64], s_part[kJoinThreads];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int groups = kJoinThreads / hd, g = tid / hd, dim = tid - g * hd;
    float m = -INFINITY, l = 0.f, v[kAhead];
    if (tid < pieces) {
        const float2 w = reinterpret_cast<const float2 *>(ml)[tid];
        m = w.x;
        l = w.y;
    }
    auto ask = [&](int i0) {                   // (a piece past the last: the last once more, with factor 0)
#pragma unroll
        for (int u = 0; u < kAhead; u++) v[u] = acc[min(i0 + u * groups, pieces - 1) * hd + dim];
    };
    ask(g);
    float mx = m;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
    if (lane == 0) s_red[wave] = mx;
    __syncthreads();
    M = fmaxf(s_red[0], s_red[1]);             // pieces <= 128: the first two waves hold them
    // a sum of 0 takes part in nothing (its accumulators are 0); a bound of -inf with a sum is a row of not-a-numbers
    const float f = l == 0.f ? 0.f : m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - M);
    if (tid < kJoinMost) s_f[tid] = f;
    float d = l * f;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) d += __shfl_xor(d, off, 64);
    if (lane == 0) s_red[kJoinThreads / 64 + wave] = d;
    __syncthreads();
    den = s_red[kJoinThreads / 64] + s_red[kJoinThreads / 64 + 1];
    float num = 0.f;
    for (int i0 = g; i0 < pieces; i0 += kAhead * groups) {
        if (i0 != g) ask(i0);
#pragma unroll
        for (int u = 0; u < kAhead; u++)
            if (i0 + u * groups < pieces) num = fmaf(v[u], s_f[i0 + u * groups], num);
    }
    s_part[tid] = num;
    __syncthreads();
    if (tid < hd)
        for (int j = 1; j < groups; j++) num += s_part[tid + j * hd];
    return num;
}
#endif

}  // namespace rptc
