// Log probabilities of given tokens, the entropy of every row and its most likely tokens, from logits in one pass over them.
// (The reference's perplexity harness takes the cross entropy of whole windows with framework ops,
// contrib/eval_ppl.py:35-39.)
//
// With m the row's (running) maximum, d_i = x_i - m, l = sum exp(d_i), t = sum d_i exp(d_i):
//   log p(x_i) = d_i - ln l,   entropy = ln l - t / l.
// The difference comes before any factor, so rows at the type's lowest value are as good as others.  Sums are fp32: a
// thread's own, then over the workgroup in a fixed order.  A logit of -inf has probability 0 and adds nothing; +inf or a not-a-number makes
// the row's results not-a-number, and so does a row of -inf only, as a log-softmax does.
//
// The k most likely tokens need no second pass over the row: the k-th largest of 64 maxima (of the threads of a lane number) is a
// bound that at least k logits reach.  Every thread leaves the maxima of up to eight stretches of its logits in LDS;
// stretches that reach the bound (about as many as there are alternatives) are dealt out, one a thread, and read again; what
// reaches the bound there goes to a list (as value and id in one 64-bit key, so equal values order by the lowest id), and an
// entry's rank in the list is its place.  Where more logits reach the bound than the list holds (ties by the hundred, a row with
// nearly everything masked) the workgroup looks for one maximum after the other instead, reading the row again for each: 1 x 128257 with 10
// tokens left and 20 alternatives 303 us instead of 20, 2048 x 32000 490 instead of 47.
//
// 2048 x 128257 bf16 with 20 alternatives: 110 us, 4.8 TB/s (101 without them); 511 x 32000 fp32: 12.9 us, 5.1 TB/s, what a copy reaches.
// A single row is bound by its one compute unit's exponentials: 1 x 128257 bf16 14 us, of 1024 threads no less.
#include "rptc_common.hpp"

namespace rptc {

constexpr int kScoreThreads = 512;
constexpr int kScoreGroups = 64;
constexpr int kScoreList = 1024;
constexpr int kScoreUnits = 8;             // stretches of a thread's logits
constexpr int kScoreLoads = 4;             // 16-byte loads of a thread in flight
constexpr float kLog2E = 1.44269504088896f, kLn2 = 0.693147180559945f;

struct ScoreF16 {
    static constexpr int kEach = 8;            // logits of a 16-byte load
    typedef uint16_t elem;
    static __device__ __forceinline__ float one(elem b) { return half_bits_to_float(b); }
    static __device__ __forceinline__ void unpack(const uint4 &v, float *x)
    {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[2 * i] = half_bits_to_float((uint16_t)(w[i] & 0xFFFFu));
            x[2 * i + 1] = half_bits_to_float((uint16_t)(w[i] >> 16));
        }
    }
    static constexpr uint32_t kNone = 0xFC00FC00u;   // -inf
};
struct ScoreBf16 {
    static constexpr int kEach = 8;
    typedef uint16_t elem;
    static __device__ __forceinline__ float one(elem b) { return __builtin_bit_cast(float, (uint32_t)b << 16); }
    static __device__ __forceinline__ void unpack(const uint4 &v, float *x)
    {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[2 * i] = __builtin_bit_cast(float, w[i] << 16);
            x[2 * i + 1] = __builtin_bit_cast(float, w[i] & 0xFFFF0000u);
        }
    }
    static constexpr uint32_t kNone = 0xFF80FF80u;
};
struct ScoreF32 {
    static constexpr int kEach = 4;
    typedef float elem;
    static __device__ __forceinline__ float one(elem b) { return b; }
    static __device__ __forceinline__ void unpack(const uint4 &v, float *x)
    {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = __builtin_bit_cast(float, w[i]);
    }
    static constexpr uint32_t kNone = 0xFF800000u;
};

// Orders as the value does (-0 as 0, a not-a-number as -inf), then by the lowest id; never 0.
__device__ __forceinline__ uint64_t score_key(float x, uint32_t id)
{
    x = x != x ? -INFINITY : x + 0.f;
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    return (uint64_t)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (0xFFFFFFFFu - id);
}
__device__ __forceinline__ float score_value(uint64_t key)
{
    const uint32_t o = (uint32_t)(key >> 32);
    return __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}

struct ScoreArgs {
    const void *logits;
    const int64_t *tokens;
    float *logprob, *entropy, *top_logprobs;
    int64_t *top_ids;
    int64_t row_stride;
    int vocab, top;
};

template <class T>
__global__ __launch_bounds__(kScoreThreads) void token_logprobs_kernel(const ScoreArgs a)
{
    typedef typename T::elem elem;
    constexpr int kEach = T::kEach, kLoads = kScoreLoads, kWaves = kScoreThreads / 64;
    __shared__ float s_m[kWaves], s_l[kWaves], s_t[kWaves], s_big[kScoreThreads];
    __shared__ uint64_t s_list[kScoreList];
    __shared__ uint64_t s_best[kWaves];
    __shared__ float s_unit[kScoreUnits * kScoreThreads];
    __shared__ uint16_t s_found[kScoreList];
    __shared__ int s_count, s_found_count;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x;
    const elem *x = static_cast<const elem *>(a.logits) + row * a.row_stride;
    // 16-byte loads from the first aligned logit on; those in front and behind one by one
    const int head = min(a.vocab, (int)((16u - (uint32_t)(reinterpret_cast<uintptr_t>(x) & 15u)) & 15u) / (int)sizeof(elem));
    const int vecs = (a.vocab - head) / kEach, tail = head + vecs * kEach;
    const uint4 *xv = reinterpret_cast<const uint4 *>(x + head);
    const bool wants_token = a.logprob != nullptr;
    float x_tok = 0.f;
    bool tok_ok = false;
    if (wants_token && tid == 0) {
        const int64_t tok = a.tokens[row];
        tok_ok = tok >= 0 && tok < a.vocab;
        if (tok_ok) x_tok = T::one(x[tok]);
    }

    float big = -INFINITY;                     // the thread's largest logit
    float l = 0.f, t = 0.f;                    // sums relative to it
    auto rebase = [](float &l_, float &t_, float from, float to) {
        if (from != -INFINITY && from != to) {
            const float f = __builtin_amdgcn_exp2f((from - to) * kLog2E);
            t_ = f * fmaf(fmaxf(from - to, -1e30f), l_, t_);
            l_ *= f;
        }
    };
    auto raise = [&](float mx) {
        if (mx > big) {
            rebase(l, t, big, mx);
            big = mx;
        }
    };
    auto add = [&](float v, float base) {
        const float d = v - base;
        const float e = __builtin_amdgcn_exp2f(d * kLog2E);
        l += e;
        t = fmaf(fmaxf(d, -1e30f), e, t);      // (-inf * 0 is not a number)
    };
    for (int i = tid; i < head; i += kScoreThreads) {
        const float v = T::one(x[i]);
        raise(v);
        add(v, big == -INFINITY ? 0.f : big);
    }
    for (int i = tail + tid; i < a.vocab; i += kScoreThreads) {
        const float v = T::one(x[i]);
        raise(v);
        add(v, big == -INFINITY ? 0.f : big);
    }
    const int rounds = (vecs + kScoreThreads * kLoads - 1) / (kScoreThreads * kLoads);
    const int per_unit = (rounds + kScoreUnits - 1) / kScoreUnits;        // rounds of a stretch
    float unit_max = -INFINITY;
    for (int r = 0, in_unit = 0, unit = tid; r < rounds; r++) {
        const int v0 = r * kScoreThreads * kLoads + tid;
        uint4 raw[kLoads];
#pragma unroll
        for (int u = 0; u < kLoads; u++) {
            raw[u] = make_uint4(T::kNone, T::kNone, T::kNone, T::kNone);
            if (v0 + u * kScoreThreads < vecs) raw[u] = xv[v0 + u * kScoreThreads];
        }
#pragma unroll
        for (int u = 0; u < kLoads; u++) {
            float e[kEach];
            T::unpack(raw[u], e);
            float mx = e[0];
#pragma unroll
            for (int i = 1; i < kEach; i++) mx = fmaxf(mx, e[i]);
            raise(mx);
            unit_max = fmaxf(unit_max, mx);
            const float base = big == -INFINITY ? 0.f : big;
#pragma unroll
            for (int i = 0; i < kEach; i++) add(e[i], base);
        }
        if (++in_unit == per_unit || r == rounds - 1) {
            s_unit[unit] = unit_max;
            unit += kScoreThreads;
            unit_max = -INFINITY;
            in_unit = 0;
        }
    }

    // the workgroup's sums: the wave's by shuffles, the waves' through LDS, in a fixed order
    float M = big;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor(M, off, 64));
    rebase(l, t, big, M);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        l += __shfl_xor(l, off, 64);
        t += __shfl_xor(t, off, 64);
    }
    if (lane == 0) {
        s_m[wave] = M;
        s_l[wave] = l;
        s_t[wave] = t;
    }
    s_big[tid] = big;
    if (tid == 0) s_count = s_found_count = 0;
    __syncthreads();
    M = s_m[0];
#pragma unroll
    for (int w = 1; w < kWaves; w++) M = fmaxf(M, s_m[w]);
    l = 0.f;
    t = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
        float lw = s_l[w], tw = s_t[w];
        rebase(lw, tw, s_m[w], M);
        l += lw;
        t += tw;
    }
    const float base = M == -INFINITY ? 0.f : M;
    const bool none = l == 0.f;                // a row of -inf only
    // The results are differences of numbers of their own size, so ln l is held in two parts: with l = 2^k f, k ln 2 to 15 bits
    // (exact) and the rest, and a difference is rounded once, at its end (mean error 2.5 to 3.2e-8 of a log probability, 4.6 to 5.4e-8 of an
    // entropy; plain fp32 operations 2.7 to 3.4 and 4.7 to 5.5).
    const float k = (float)__builtin_amdgcn_frexp_expf(l);
    const float ln_hi = none ? __builtin_nanf("") : k * 0x1.62e4p-1f, ln_lo = fmaf(k, 0x1.7f7d1cp-20f, log2f(__builtin_amdgcn_frexp_mantf(l)) * kLn2);
    auto less_ln_l = [&](float d, float rest) {            // d + rest - ln l
        const float s = d - ln_hi, b = s - d;
        const float lost = (d - (s - b)) + (-ln_hi - b);
        return d == -INFINITY ? d - (ln_hi + ln_lo) : s + (lost + (rest - ln_lo));
    };
    auto logp = [&](float v) { return less_ln_l(v - base, 0.f); };
    if (tid == 0) {
        if (wants_token) a.logprob[row] = tok_ok ? logp(x_tok) : __builtin_nanf("");
        if (a.entropy) {
            const float mean = t / l;                      // of d; what its rounding left is added as well
            a.entropy[row] = -less_ln_l(mean, fmaf(-mean, l, t) / l);
        }
    }
    if (a.top == 0) return;

    // the top-th largest of the 64 maxima, in every wave: the one with top - 1 in front of it (equal ones in lane order)
    float own = s_big[lane];
#pragma unroll
    for (int w = 1; w < kWaves; w++) own = fmaxf(own, s_big[w * 64 + lane]);
    int front = 0;
#pragma unroll
    for (int i = 0; i < kScoreGroups; i++) {
        const float o = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, own), i));
        front += o > own || (o == own && i < lane);
    }
    const float bound = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, own), __builtin_ctzll(__ballot(front == a.top - 1))));
    // a bound of -inf says nothing (fewer lane numbers than wanted hold a logit above it): a row no longer than the list then
    // goes there whole, a longer one is searched below
    const bool all = bound == -INFINITY && a.vocab <= kScoreList;
    const bool listed = all || bound != -INFINITY;
    auto take = [&](float v, int id) {
        if (v >= bound || all) {
            const int at = atomicAdd(&s_count, 1);
            if (at < kScoreList) s_list[at] = score_key(v, (uint32_t)id);
        }
    };
    const int units = per_unit ? (rounds + per_unit - 1) / per_unit : 0;
    if (listed && (big >= bound || all)) {
        for (int i = tid; i < head; i += kScoreThreads) take(T::one(x[i]), i);
        for (int i = tail + tid; i < a.vocab; i += kScoreThreads) take(T::one(x[i]), i);
        for (int n = 0; n < units; n++)
            if (s_unit[n * kScoreThreads + tid] >= bound || all) {
                const int at = atomicAdd(&s_found_count, 1);
                if (at < kScoreList) s_found[at] = (uint16_t)(n * kScoreThreads + tid);
            }
    }
    __syncthreads();
    const int found = s_found_count;
    if (found <= kScoreList)
        for (int j = tid; j < found; j += kScoreThreads) {
            const int n = s_found[j] / kScoreThreads, owner = s_found[j] % kScoreThreads;
            for (int r = n * per_unit; r < min(rounds, (n + 1) * per_unit); r++) {
                const int v0 = r * kScoreThreads * kLoads + owner;
                uint4 raw[kLoads];
#pragma unroll
                for (int u = 0; u < kLoads; u++) raw[u] = xv[min(v0 + u * kScoreThreads, vecs - 1)];
#pragma unroll
                for (int u = 0; u < kLoads; u++) {
                    const int v = v0 + u * kScoreThreads;
                    if (v >= vecs) break;
                    float e[kEach];
                    T::unpack(raw[u], e);
#pragma unroll
                    for (int i = 0; i < kEach; i++) take(e[i], head + v * kEach + i);
                }
            }
        }
    __syncthreads();
    const int count = s_count;
    if (listed && found <= kScoreList && count <= kScoreList) {
        for (int j = tid; j < count; j += kScoreThreads) {
            const uint64_t key = s_list[j];
            int rank = 0;
            for (int i = 0; i < count; i++) rank += s_list[i] > key;
            if (rank < a.top) {
                if (a.top_ids) a.top_ids[row * a.top + rank] = 0xFFFFFFFFu - (uint32_t)key;
                if (a.top_logprobs) a.top_logprobs[row * a.top + rank] = logp(score_value(key));
            }
        }
        return;
    }
    auto each = [&](auto f) {                  // the thread's logits with their ids
        for (int i = tid; i < head; i += kScoreThreads) f(T::one(x[i]), i);
        for (int i = tail + tid; i < a.vocab; i += kScoreThreads) f(T::one(x[i]), i);
        for (int v = tid; v < vecs; v += kScoreThreads) {
            float e[kEach];
            T::unpack(xv[v], e);
#pragma unroll
            for (int i = 0; i < kEach; i++) f(e[i], head + v * kEach + i);
        }
    };
    // one after the other: the largest key below the last one taken
    uint64_t last = ~0ull;
    for (int r = 0; r < a.top; r++) {
        uint64_t best = 0;
        each([&](float v, int id) {
            const uint64_t key = score_key(v, (uint32_t)id);
            if (key < last && key > best) best = key;
        });
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            const uint64_t o = __shfl_xor(best, off, 64);
            if (o > best) best = o;
        }
        if (lane == 0) s_best[wave] = best;
        __syncthreads();
        best = s_best[0];
#pragma unroll
        for (int w = 1; w < kWaves; w++)
            if (s_best[w] > best) best = s_best[w];
        __syncthreads();
        last = best;
        if (tid == 0) {
            const uint32_t id = 0xFFFFFFFFu - (uint32_t)best;
            if (a.top_ids) a.top_ids[row * a.top + r] = id;
            if (a.top_logprobs) a.top_logprobs[row * a.top + r] = logp(T::one(x[id]));
        }
    }
}

}  // namespace rptc

using namespace rptc;

extern "C" int rptc_token_logprobs(const void *logits, int dtype, const int64_t *tokens, float *logprob, float *entropy,
                                   int64_t *top_ids, float *top_logprobs, int64_t rows, int64_t vocab, int64_t row_stride, int64_t top,
                                   void *stream, float *ms)
{
    if (!logits || (!logprob && !entropy && !top_ids && !top_logprobs) || (logprob && !tokens)) return RPTC_ENULL;
    if (dtype != RPTC_F16 && dtype != RPTC_BF16 && dtype != RPTC_F32) return RPTC_EMODE;
    if (rows < 1 || vocab < 1 || row_stride < 0 || top < 0 || top > vocab) return RPTC_ESHAPE;
    if ((top > 0) != (top_ids || top_logprobs)) return RPTC_ESHAPE;
    if (rows >= (int64_t)1 << 22 || vocab >= (int64_t)1 << 30 || row_stride >= (int64_t)1 << 34 || top > kScoreGroups) return RPTC_ELIMIT;
    const int64_t width = dtype == RPTC_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(logits) % width != 0) return RPTC_EALIGN;
    // what is read, then what is written: an output overlaps neither the one nor another
    const struct { const void *p; int64_t bytes; } part[6] = {{logits, ((rows - 1) * row_stride + vocab) * width}, {tokens, rows * 8},
                                                              {logprob, rows * 4}, {entropy, rows * 4}, {top_ids, rows * top * 8}, {top_logprobs, rows * top * 4}};
    for (int i = 2; i < 6; i++)
        for (int j = 0; j < i; j++) {
            const char *x = static_cast<const char *>(part[i].p), *y = static_cast<const char *>(part[j].p);
            if (x && y && x < y + part[j].bytes && y < x + part[i].bytes) return RPTC_EALIAS;
        }
    DeviceInfo *dev;
    int rc = device_info(&dev);
    if (rc) return rc;
    ScoreArgs a;
    a.logits = logits;
    a.tokens = tokens;
    a.logprob = logprob;
    a.entropy = entropy;
    a.top_logprobs = top_logprobs;
    a.top_ids = top_ids;
    a.row_stride = row_stride;
    a.vocab = (int)vocab;
    a.top = (int)top;
    hipStream_t s = static_cast<hipStream_t>(stream);
    Timer timer;
    if ((rc = timer.begin(dev, s, ms))) return rc;
    const dim3 grid((unsigned)rows), block(kScoreThreads);
    if (dtype == RPTC_F16) hipLaunchKernelGGL(token_logprobs_kernel<ScoreF16>, grid, block, 0, s, a);
    else if (dtype == RPTC_BF16) hipLaunchKernelGGL(token_logprobs_kernel<ScoreBf16>, grid, block, 0, s, a);
    else hipLaunchKernelGGL(token_logprobs_kernel<ScoreF32>, grid, block, 0, s, a);
    return timer.end();
}
