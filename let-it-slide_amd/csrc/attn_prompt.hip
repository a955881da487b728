// Attention of whole prompts: packed sequences of different lengths, causal or not, grouped heads, fp16 or bf16.
// (No counterpart in the reference, which generates with transformers on dense weights, quantize_hf.py:229-236.)
//
//   o_i = sum_j p_ij v_j / l_i,   p_ij = exp2(c q_i.k_j - m_i),   l_i = sum_j p_ij,   lse_i = (m_i + log2 l_i) ln 2
//
// with c = scale log2(e), over the keys j that query i sees, in one pass over the keys: m_i is a running bound of
// c q_i.k_j (raised, and the sums rescaled, only where a score exceeds it by more than 2^8, so p stays below 256).
// Scores, m, l and the output sums are fp32; p is rounded to the inputs' type for the matrix unit (relative 2^-12 or
// 2^-9, as the products need two operands of one type), l adds the unrounded p.
//
// A workgroup of four waves owns kRows = 128 query rows of one head, 32 a wave, and walks over its keys 64 at a time.
// The products are formed transposed, S^T = K Q^T and O^T = V^T P^T with 32x32x16 matrix instructions: a lane then holds
// scores of one query only (the row maximum is 31 maxima in the lane and one swap of the wave's halves), the scores'
// layout is, up to a renumbering of the keys that V follows, the layout the second product wants P in, and every
// factor of a row is a factor of a lane.  K and V come from memory straight into LDS (two buffers, 16 bytes a lane);
// V^T is read with the transposing LDS read.
#include "join.hpp"

namespace rptc {

constexpr int kPromptThreads = 256;
constexpr int kRows = 128;             // query rows of a workgroup
constexpr int kKeys = 64;              // keys of a step
constexpr float kLazy = 8.f;           // exponents of 2 a score may exceed the running bound by

typedef float float16_t __attribute__((ext_vector_type(16)));
typedef int int4_t __attribute__((ext_vector_type(4)));
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef short short8_t __attribute__((ext_vector_type(8)));
typedef float float2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

// the two element types: the matrix instruction, conversions
struct TypeF16 {
    static __device__ __forceinline__ float16_t mfma(short8_t a, short8_t b, float16_t c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b)
    {
        const float2_t v = {a, b};
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, half2_t));
    }
    static __device__ __forceinline__ float to_float(uint16_t b) { return half_bits_to_float(b); }
};
struct TypeBf16 {
    static __device__ __forceinline__ float16_t mfma(short8_t a, short8_t b, float16_t c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b)
    {
        const float2_t v = {a, b};
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2_t));
    }
    static __device__ __forceinline__ float to_float(uint16_t b) { return __builtin_bit_cast(float, (uint32_t)b << 16); }
};

struct PromptArgs {
    const uint16_t *q, *k, *v;
    uint16_t *out;
    float *lse;                        // [total_q][heads], may be null
    const int32_t *q_start, *k_start, *k_len;
    float *part_acc, *part_ml;         // splits > 1: [total_q][heads][split][hd] sums, [..][2] bound and sum of p
    rptc_prompt_strides st;
    int seqs, total_q, total_k, heads, kv_heads, tiles, splits, causal;
    float c;                           // scale * log2(e)
};

struct PromptTile {
    int seq, q_begin, q_end, row0;     // the sequence's query rows, the tile's first row
};

// A value every lane of the wave holds, as one the compiler knows to be such (scalar registers, scalar branches).
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// The sequence that holds tile `tile` when every sequence is cut into tiles of kRows query rows: 64 sequences at a time,
// a lane each.  A sequence's tiles are taken from its end (the longest rows of a causal prompt first).  The starts come
// from device memory: a sequence that does not lie inside the query rows has no tiles.
__device__ __forceinline__ bool find_tile(const PromptArgs &a, int tile, PromptTile &t)
{
    const int lane = threadIdx.x & 63;
    t.seq = -1;
    t.q_begin = t.q_end = t.row0 = 0;
    int in_front = 0;                      // tiles of the sequences in front (they do not overlap: at most a.tiles)
    for (int s0 = 0; s0 < a.seqs; s0 += 64) {
        const int s = s0 + lane;
        int begin = 0, end = 0;
        if (s < a.seqs) {
            begin = a.q_start ? a.q_start[s] : 0;
            end = a.q_start ? a.q_start[s + 1] : a.total_q;
        }
        const bool ok = begin >= 0 && end > begin && end <= a.total_q;
        const int n = ok ? (end - begin + kRows - 1) / kRows : 0;
        int incl = n;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int o = __shfl_up(incl, off, 64);
            if (lane >= off) incl += o;
        }
        const uint64_t hit = __ballot(in_front + incl > tile);
        if (hit) {
            const int f = __builtin_ctzll(hit);
            const int nf = __builtin_amdgcn_readlane(n, f);
            const int local = tile - (in_front + __builtin_amdgcn_readlane(incl, f) - nf);
            t.seq = s0 + f;
            t.q_begin = __builtin_amdgcn_readlane(begin, f);
            t.q_end = __builtin_amdgcn_readlane(end, f);
            t.row0 = t.q_begin + (nf - 1 - local) * kRows;
            break;
        }
        in_front += __builtin_amdgcn_readlane(incl, 63);
    }
    t.seq = uniform(t.seq);
    t.q_begin = uniform(t.q_begin);
    t.q_end = uniform(t.q_end);
    t.row0 = uniform(t.row0);
    return t.seq >= 0;
}

// The sequence's keys; false when they do not lie inside k and v (its rows are then left as they are).
__device__ __forceinline__ bool find_keys(const PromptArgs &a, const PromptTile &t, int &first, int &len)
{
    first = a.k_start ? a.k_start[t.seq] : a.q_start ? t.q_begin : 0;
    len = a.k_len ? a.k_len[t.seq] : a.q_start ? t.q_end - t.q_begin : a.total_k;
    first = uniform(first);
    len = uniform(len);
    return first >= 0 && len >= 0 && (int64_t)first + len <= a.total_k;
}

// 16 bytes a lane from `offset` of the buffer to LDS at `to` + 16 lane (no register receives anything: the request may
// stay in flight behind the statement).  As assembly because the compiler, which cannot tell the two buffers in LDS
// apart, waits for such a request in front of the next transposing LDS read, which reads the other buffer.  (m0 is
// reserved for such single uses: the compiler sets it in front of each of its own.)
__device__ __forceinline__ void load_to_lds(uint32_t offset, int4_t resource, uint32_t to)
{
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(offset), "s"(resource), "s"(to) : "memory");
}
__device__ __forceinline__ void wait_for_lds_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ uint32_t lds_address(const void *p)
{
    return (uint32_t)uniform((int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)p);
}

// x of the lane 32 away, in both halves of the wave: returns op(own, other)
__device__ __forceinline__ float halves_max(float x)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ __forceinline__ float halves_sum(float x)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
    return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}

// Rows of K and V in LDS, HD values each, cut into chunks of 16 bytes; the chunk that holds columns 8n .. 8n+7 of row r
// is chunk n ^ swizzle(r), so that the 16 lanes of a read's phase (16 rows of one column for K, four rows of 64 bytes
// for V) fall on different banks.
template <int HD>
__device__ __forceinline__ int swizzle_k(int row)
{
    return HD >= 128 ? row & 15 : HD == 64 ? (row >> 1) & 7 : (row >> 2) & 3;
}
template <int HD>
__device__ __forceinline__ int swizzle_v(int row)
{
    return HD >= 128 ? (row & 3) << 2 : HD == 64 ? (row >> 1 & 1) << 2 : 0;
}

// One wave's rows in plain fp32, one row after the other, keys [k_lo, k_hi) of those a row sees.  Taken when a sum of the
// matrix path came out infinite or not a number: that is right where the row sees such a value, and wrong where only
// a masked key or a masked row of V held it (0 * NaN is NaN), so the rows are worked out again without the masked ones.
template <int HD, class T>
__device__ __forceinline__ void prompt_rows_plain(const PromptArgs &a, const PromptTile &t, int row_first, int head, int kvh,
                                                            int ks, int lk, int k_lo, int k_hi, int split)
{
    const int lane = threadIdx.x & 63;
    const int lq = t.q_end - t.q_begin;
    constexpr int kOut = (HD + 63) / 64;
    for (int row = row_first; row < min(row_first + 32, t.q_end); row++) {
        const int see = a.causal ? lk - lq + 1 + (row - t.q_begin) : lk;
        const int end = min(see, k_hi);
        const uint16_t *q = a.q + (int64_t)row * a.st.q_token + (int64_t)head * a.st.q_head;
        auto score = [&](int j) {
            const uint16_t *k = a.k + (int64_t)(ks + j) * a.st.k_token + (int64_t)kvh * a.st.k_head;
            float s = 0.f;
            for (int d = 0; d < HD; d++) s = fmaf(T::to_float(q[d]), T::to_float(k[d]), s);
            return s;
        };
        float m = -INFINITY;
        for (int j = k_lo + lane; j < end; j += 64) m = fmaxf(m, score(j));
        for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
        const float mc = m == -INFINITY ? 0.f : m * a.c;
        float l = 0.f, acc[kOut];
        for (int u = 0; u < kOut; u++) acc[u] = 0.f;
        for (int j0 = k_lo; j0 < end; j0 += 64) {
            const float p = j0 + lane < end ? __builtin_amdgcn_exp2f(fmaf(score(j0 + lane), a.c, -mc)) : 0.f;
            l += p;
            for (int i = 0; i < min(64, end - j0); i++) {
                const float pi = __shfl(p, i, 64);
                const uint16_t *v = a.v + (int64_t)(ks + j0 + i) * a.st.v_token + (int64_t)kvh * a.st.v_head;
                for (int u = 0; u < kOut; u++)
                    if (lane + 64 * u < HD) acc[u] = fmaf(pi, T::to_float(v[lane + 64 * u]), acc[u]);
            }
        }
        for (int off = 32; off > 0; off >>= 1) l += __shfl_xor(l, off, 64);
        const int64_t at = (int64_t)row * a.heads + head;
        if (a.splits > 1) {
            const int64_t pa = at * a.splits + split;
            for (int u = 0; u < kOut; u++)
                if (lane + 64 * u < HD) a.part_acc[pa * HD + lane + 64 * u] = acc[u];
            if (lane == 0) {
                a.part_ml[2 * pa] = l == 0.f ? -INFINITY : mc;
                a.part_ml[2 * pa + 1] = l;
            }
            continue;
        }
        uint16_t *o = a.out + (int64_t)row * a.st.out_token + (int64_t)head * a.st.out_head;
        for (int u = 0; u < kOut; u++)
            if (lane + 64 * u < HD) o[lane + 64 * u] = (uint16_t)T::pack(l == 0.f ? 0.f : acc[u] / l, 0.f);
        if (a.lse && lane == 0) a.lse[at] = l == 0.f ? -INFINITY : (mc + log2f(l)) * 0.693147180559945f;
    }
}

template <int HD, class T>
__global__ __launch_bounds__(kPromptThreads, HD > 128 ? 1 : 2) void attn_prompt_kernel(const PromptArgs a)
{
    extern __shared__ __align__(16) uint16_t lds[];       // [2][K, V][kKeys][HD]
    constexpr int kTile = kKeys * HD;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int c = lane >> 5, col = lane & 31;

    // Workgroup -> (head, tile, split).  Consecutive workgroups go to the eight XCDs in turn, each with an L2 of its own:
    // the items are renumbered so that an XCD gets a run of them, heads of one group of queries (the same K and V) together.
    const int items = a.heads * a.tiles * a.splits, per_xcd = gridDim.x >> 3;
    const int item = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
    if (item >= items) return;
    const int head = item / (a.tiles * a.splits), rest = item - head * a.tiles * a.splits;
    const int tile = rest / a.splits, split = rest - tile * a.splits;
    PromptTile t;
    if (!find_tile(a, tile, t)) return;
    int ks, lk;
    if (!find_keys(a, t, ks, lk)) return;
    const int kvh = head / (a.heads / a.kv_heads);
    const int lq = t.q_end - t.q_begin;

    // keys a row sees: [0, see); of the tile's last row the most
    const int last = min(t.row0 + kRows, t.q_end) - 1;
    auto sees = [&](int row) { return a.causal ? max(0, lk - lq + 1 + (row - t.q_begin)) : lk; };
    const int k_most = uniform(sees(last));
    const int per_split = ((k_most + a.splits - 1) / a.splits + kKeys - 1) / kKeys * kKeys;
    const int k_lo = uniform((int)min((int64_t)k_most, (int64_t)split * per_split));
    const int k_hi = uniform((int)min((int64_t)k_most, (int64_t)k_lo + per_split));
    const int row_first = t.row0 + 32 * wave, row = row_first + col;
    const bool wave_live = row_first < t.q_end;
    const int see = row < t.q_end ? sees(row) : 0;
    // what all rows of the wave see, and what one of them sees
    const int see_least = uniform(wave_live ? min(sees(row_first), k_hi) : 0);
    const int see_most = uniform(wave_live ? min(sees(min(row_first + 31, t.q_end - 1)), k_hi) : 0);

    // K and V, 16 bytes a lane and request: a request covers 1024 bytes of LDS, the lane's source is chosen so that the
    // chunks land swizzled.  Past the sequence's last key the buffer's bounds check gives zeros.
    constexpr int kChunks = HD / 8, kRequests = kTile / 8 / kPromptThreads;
    static_assert(kTile % (8 * kPromptThreads) == 0, "whole requests");
    uint32_t k_off[kRequests], v_off[kRequests];
#pragma unroll
    for (int u = 0; u < kRequests; u++) {
        const int slot = (u * 4 + wave) * 64 + lane, r = slot / kChunks, ch = slot % kChunks;
        k_off[u] = (uint32_t)(r * a.st.k_token + (ch ^ swizzle_k<HD>(r)) * 8) * 2u;
        v_off[u] = (uint32_t)(r * a.st.v_token + (ch ^ swizzle_v<HD>(r)) * 8) * 2u;
    }
    const uint16_t *k_base = a.k + (int64_t)ks * a.st.k_token + (int64_t)kvh * a.st.k_head;
    const uint16_t *v_base = a.v + (int64_t)ks * a.st.v_token + (int64_t)kvh * a.st.v_head;
    // the descriptor of `rows` rows, in scalar registers; offsets at or past its end read as zero
    auto resource = [&](const uint16_t *base, int64_t token, int rows) {
        const uint64_t p = reinterpret_cast<uint64_t>(base);
        const int4_t r = {uniform((int)p), uniform((int)(p >> 32) & 0xFFFF), uniform(((rows - 1) * (int)token + HD) * 2), 0x00027000};
        return r;
    };
    const uint32_t lds_base = lds_address(lds) + (uint32_t)wave * 1024u;
    auto request = [&](int k0, int buf) {
        const int rows = min(lk - k0, kKeys);
        const int4_t kr = resource(k_base + (int64_t)k0 * a.st.k_token, a.st.k_token, rows);
        const int4_t vr = resource(v_base + (int64_t)k0 * a.st.v_token, a.st.v_token, rows);
        const uint32_t to = lds_base + (uint32_t)buf * (4u * kTile);
#pragma unroll
        for (int u = 0; u < kRequests; u++) load_to_lds(k_off[u], kr, to + u * 4096u);
#pragma unroll
        for (int u = 0; u < kRequests; u++) load_to_lds(v_off[u], vr, to + 2u * kTile + u * 4096u);
    };

    constexpr int kSteps = HD / 16, kDims = HD / 32;
    short8_t qf[kSteps];
    {
        // a lane without a row of its own takes the sequence's last (its results go nowhere)
        const uint16_t *q = a.q + (int64_t)min(row, t.q_end - 1) * a.st.q_token + (int64_t)head * a.st.q_head + 8 * c;
#pragma unroll
        for (int i = 0; i < kSteps; i++) qf[i] = *reinterpret_cast<const short8_t *>(q + 16 * i);
        // waited for here: a wait inside the loop would wait for the step's K and V as well
#pragma unroll
        for (int i = 0; i < kSteps; i++) asm volatile("" : "+v"(qf[i]));
    }
    float16_t acc[kDims];
#pragma unroll
    for (int d = 0; d < kDims; d++) acc[d] = (float16_t)(0.f);
    float m = -INFINITY, l = 0.f;           // running bound in units of c * score (log2), sum of p over the lane's keys

    if (k_lo < k_hi) request(k_lo, 0);
    int buf = 0;
    for (int k0 = k_lo; k0 < k_hi; k0 += kKeys, buf ^= 1) {
        wait_for_lds_loads();                              // this wave's part of the step is in LDS
        __syncthreads();                                   // everyone's is, and nobody reads the other buffer any more
        if (k0 + kKeys < k_hi) request(k0 + kKeys, buf ^ 1);
        if (k0 >= see_most) continue;
        const uint16_t *kt = lds + buf * 2 * kTile, *vt = kt + kTile;

        float16_t s[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            s[h] = (float16_t)(0.f);
            const int r = 32 * h + col;
#pragma unroll
            for (int i = 0; i < kSteps; i++) {
                const short8_t kf = *reinterpret_cast<const short8_t *>(kt + r * HD + ((2 * i + c) ^ swizzle_k<HD>(r)) * 8);
                s[h] = T::mfma(kf, qf[i], s[h]);
            }
        }
        if (k0 + kKeys > see_least) {                      // some row of the wave does not see all of the step's keys
            const int left = min(see, k_hi) - k0 - 4 * c;
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int r = 0; r < 16; r++)
                    if (32 * h + 8 * (r / 4) + r % 4 >= left) s[h][r] = -INFINITY;
        }
        float mx = s[0][0];
#pragma unroll
        for (int r = 1; r < 16; r++) mx = fmaxf(mx, s[0][r]);
#pragma unroll
        for (int r = 0; r < 16; r++) mx = fmaxf(mx, s[1][r]);
        mx = halves_max(mx) * a.c;
        if (__ballot(mx > m + kLazy)) {
            const float up = fmaxf(m, mx);
            const float f = up == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - up);
            l *= f;
#pragma unroll
            for (int d = 0; d < kDims; d++) acc[d] *= f;
            m = up;
        }
        const float mc = m == -INFINITY ? 0.f : m;
        uint32_t p[2][8];
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                const float p0 = __builtin_amdgcn_exp2f(fmaf(s[h][r], a.c, -mc)), p1 = __builtin_amdgcn_exp2f(fmaf(s[h][r + 1], a.c, -mc));
                l += p0;
                l += p1;
                p[h][r / 2] = T::pack(p0, p1);
            }
        // V^T: lane's dimension col of a tile of 32, keys in the order the scores' registers have them
        const int g16 = lane >> 4, rr = (lane & 15) >> 2, piece = lane & 3;
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int g = 0; g < 2; g++) {
                const uint4 pv = make_uint4(p[h][4 * g], p[h][4 * g + 1], p[h][4 * g + 2], p[h][4 * g + 3]);
                const int key = 32 * h + 16 * g + 4 * c + rr;
#pragma unroll
                for (int d = 0; d < kDims; d++) {
                    typedef __attribute__((address_space(3))) short4_t lds_short4;
                    const int ch = (4 * d + 2 * (g16 & 1) + piece / 2) ^ swizzle_v<HD>(key);   // key and key + 8: the same swizzle
                    const uint16_t *va = vt + key * HD + ch * 8 + (piece & 1) * 4;
                    const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4 *)va);
                    const short4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4 *)(va + 8 * HD));
                    acc[d] = T::mfma(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7), __builtin_bit_cast(short8_t, pv), acc[d]);
                }
            }
    }
    if (!wave_live) return;
    l = halves_sum(l);

    float bad = 0.f;
#pragma unroll
    for (int d = 0; d < kDims; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) bad = fmaf(acc[d][r], 0.f, bad);
    if (__ballot(bad != 0.f)) {                            // (not-a-number compares unequal)
        prompt_rows_plain<HD, T>(a, t, row_first, head, kvh, ks, lk, k_lo, k_hi, split);
        return;
    }
    const int64_t at = (int64_t)row * a.heads + head;
    if (a.splits > 1) {
        if (row >= t.q_end) return;
        const int64_t pa = at * a.splits + split;
        float *o = a.part_acc + pa * HD + 4 * c;
#pragma unroll
        for (int d = 0; d < kDims; d++)
#pragma unroll
            for (int b = 0; b < 4; b++)
                *reinterpret_cast<float4 *>(o + 32 * d + 8 * b) = make_float4(acc[d][4 * b], acc[d][4 * b + 1], acc[d][4 * b + 2], acc[d][4 * b + 3]);
        if (c == 0) *reinterpret_cast<float2 *>(a.part_ml + 2 * pa) = make_float2(l == 0.f ? -INFINITY : m, l);
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;            // a row that sees nothing: zeros
    uint16_t *o = a.out + (int64_t)min(row, t.q_end - 1) * a.st.out_token + (int64_t)head * a.st.out_head + 8 * c;
#pragma unroll
    for (int d = 0; d < kDims; d++)
#pragma unroll
        for (int b = 0; b < 4; b += 2) {
            // the lane's four dimensions of blocks b and b + 1 (8 dimensions each, the halves of the wave four): a swap of
            // the halves leaves eight consecutive ones of block b + c in each lane
            uint32_t x0 = T::pack(acc[d][4 * b] * inv, acc[d][4 * b + 1] * inv), x1 = T::pack(acc[d][4 * b + 2] * inv, acc[d][4 * b + 3] * inv);
            uint32_t y0 = T::pack(acc[d][4 * b + 4] * inv, acc[d][4 * b + 5] * inv), y1 = T::pack(acc[d][4 * b + 6] * inv, acc[d][4 * b + 7] * inv);
            const auto w0 = __builtin_amdgcn_permlane32_swap(x0, y0, false, false), w1 = __builtin_amdgcn_permlane32_swap(x1, y1, false, false);
            if (row < t.q_end)
                *reinterpret_cast<uint4 *>(o + 32 * d + 8 * b) = make_uint4((uint32_t)w0[0], (uint32_t)w1[0], (uint32_t)w0[1], (uint32_t)w1[1]);
        }
    if (a.lse && c == 0 && row < t.q_end) a.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.693147180559945f;
}

// Joins the pieces of a row, a workgroup per (row, head).  The rows are found as the kernel above found them: rows of no
// sequence have no pieces and stay as they are.
template <int HD, class T>
__global__ __launch_bounds__(kJoinThreads) void attn_prompt_merge_kernel(const PromptArgs a)
{
    const int head = blockIdx.y;
    PromptTile t;
    if (!find_tile(a, blockIdx.x / kRows, t)) return;
    int ks, lk;
    if (!find_keys(a, t, ks, lk)) return;
    const int row = t.row0 + blockIdx.x % kRows;
    if (row >= t.q_end) return;
    const int64_t at = (int64_t)row * a.heads + head;
    float M, l;
    const float num = join_pieces(a.part_acc + at * a.splits * HD, a.part_ml + 2 * at * a.splits, a.splits, HD, M, l);
    if (threadIdx.x < HD)
        a.out[(int64_t)row * a.st.out_token + (int64_t)head * a.st.out_head + threadIdx.x] = (uint16_t)T::pack(l == 0.f ? 0.f : num / l, 0.f);
    if (a.lse && threadIdx.x == 0) a.lse[at] = l == 0.f ? -INFINITY : (M + log2f(l)) * 0.693147180559945f;
}

template <int HD>
static constexpr size_t prompt_lds() { return (size_t)2 * 2 * kKeys * HD * 2; }

int prepare_attn_prompt()
{
    int rc;
    if ((rc = (int)hipFuncSetAttribute(reinterpret_cast<const void *>(&attn_prompt_kernel<128, TypeF16>), hipFuncAttributeMaxDynamicSharedMemorySize, prompt_lds<128>()))) return rc;
    if ((rc = (int)hipFuncSetAttribute(reinterpret_cast<const void *>(&attn_prompt_kernel<128, TypeBf16>), hipFuncAttributeMaxDynamicSharedMemorySize, prompt_lds<128>()))) return rc;
    if ((rc = (int)hipFuncSetAttribute(reinterpret_cast<const void *>(&attn_prompt_kernel<256, TypeF16>), hipFuncAttributeMaxDynamicSharedMemorySize, prompt_lds<256>()))) return rc;
    return (int)hipFuncSetAttribute(reinterpret_cast<const void *>(&attn_prompt_kernel<256, TypeBf16>), hipFuncAttributeMaxDynamicSharedMemorySize, prompt_lds<256>());
}

// Pieces a row's keys are cut into.  A call with fewer workgroups (128 rows of a head each) than compute units leaves
// most of the chip idle and its workgroups with long walks: the keys are then split so that about two workgroups a
// unit run, none with fewer than 256 keys of the longest sequence, and a second launch joins the pieces.
static int prompt_splits(int64_t tiles, int64_t heads, int64_t max_k, int cus)
{
    const int64_t groups = tiles * heads;
    if (groups >= cus) return 1;
    int64_t n = (2 * (int64_t)cus + groups - 1) / groups;
    if (n > max_k / 256) n = max_k / 256;
    return n < 1 ? 1 : n > 64 ? 64 : (int)n;
}

static int prompt_sizes(int64_t seqs, int64_t total_q, int64_t total_k, int64_t heads, int64_t kv_heads, int64_t hd)
{
    if (seqs < 1 || total_q < 1 || total_k < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0) return RPTC_ESHAPE;
    if (hd != 32 && hd != 64 && hd != 128 && hd != 256) return RPTC_ESHAPE;
    if (heads > 1024 || seqs > (1 << 20) || total_q > (1 << 24) || total_k >= ((int64_t)1 << 31) - 64) return RPTC_ELIMIT;
    if ((total_q / kRows + seqs) * heads >= (int64_t)1 << 23) return RPTC_ELIMIT;      // workgroups of one launch
    return 0;
}

template <int HD, class T>
static void launch_prompt(const PromptArgs &a, hipStream_t s)
{
    const int items = a.heads * a.tiles * a.splits;
    hipLaunchKernelGGL((attn_prompt_kernel<HD, T>), dim3((unsigned)((items + 7) / 8 * 8)), dim3(kPromptThreads), prompt_lds<HD>(), s, a);
    if (a.splits > 1)
        hipLaunchKernelGGL((attn_prompt_merge_kernel<HD, T>), dim3((unsigned)a.tiles * kRows, (unsigned)a.heads), dim3(kJoinThreads), 0, s, a);
}

}  // namespace rptc

using namespace rptc;

extern "C" int64_t rptc_attn_prompt_workspace_bytes(int64_t seqs, int64_t total_q, int64_t total_k, int64_t max_k, int64_t heads,
                                                    int64_t kv_heads, int64_t hd)
{
    int rc = prompt_sizes(seqs, total_q, total_k, heads, kv_heads, hd);
    if (rc) return rc;
    DeviceInfo *dev;
    if ((rc = device_info(&dev))) return rc < 0 ? rc : RPTC_EDEVICE;
    const int splits = prompt_splits(total_q / kRows + seqs, heads, max_k < total_k ? max_k : total_k, dev->cus);
    return splits > 1 ? (int64_t)splits * total_q * heads * (hd + 2) * 4 : 0;
}

extern "C" int rptc_attn_prompt(const uint16_t *q, const uint16_t *k, const uint16_t *v, uint16_t *out, float *lse,
                                const int32_t *q_start, const int32_t *k_start, const int32_t *k_len, int64_t seqs,
                                int64_t total_q, int64_t total_k, int64_t max_k, int64_t heads, int64_t kv_heads, int64_t hd,
                                const rptc_prompt_strides *strides, float scale, int causal, int dtype, void *workspace,
                                int64_t workspace_bytes, void *stream, float *ms)
{
    if (!q || !out || !strides || !k_start != !k_len) return RPTC_ENULL;
    if (total_k > 0 && (!k || !v)) return RPTC_ENULL;
    int rc = prompt_sizes(seqs, total_q, total_k, heads, kv_heads, hd);
    if (rc) return rc;
    if (dtype != RPTC_F16 && dtype != RPTC_BF16) return RPTC_EMODE;
    if ((!q_start && seqs != 1) || (q_start && !k_start && total_k != total_q)) return RPTC_ESHAPE;
    if (!(scale > 0.f) || !(scale < 1e30f) || max_k < 0) return RPTC_ESHAPE;
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out)) return RPTC_EALIGN;
    const int64_t st[8] = {strides->q_token, strides->q_head, strides->k_token, strides->k_head,
                           strides->v_token, strides->v_head, strides->out_token, strides->out_head};
    for (int i = 0; i < 8; i++) {
        if (st[i] < 0 || (i != 4 && i != 5 && i != 2 && i != 3 && st[i] == 0)) return RPTC_ESHAPE;
        if (st[i] % 8 != 0) return RPTC_EALIGN;
        if (i % 2 == 0 && st[i] > (1 << 23)) return RPTC_ELIMIT;     // 64 rows of a step inside 32-bit offsets
    }
    if (out == q || out == k || out == v) return RPTC_EALIAS;
    DeviceInfo *dev;
    if ((rc = device_info(&dev))) return rc;
    PromptArgs a;
    a.q = q;
    a.k = k;
    a.v = v;
    a.out = out;
    a.lse = lse;
    a.q_start = q_start;
    a.k_start = k_start;
    a.k_len = k_len;
    a.st = *strides;
    a.seqs = (int)seqs;
    a.total_q = (int)total_q;
    a.total_k = (int)total_k;
    a.heads = (int)heads;
    a.kv_heads = (int)kv_heads;
    a.tiles = (int)(total_q / kRows + seqs);
    a.splits = prompt_splits(a.tiles, heads, max_k < total_k ? max_k : total_k, dev->cus);
    a.causal = causal ? 1 : 0;
    a.c = scale * 1.44269504088896f;
    a.part_acc = a.part_ml = nullptr;
    if (a.splits > 1) {
        const int64_t n = (int64_t)a.splits * total_q * heads;
        if (!workspace) return RPTC_ENULL;
        if (!aligned16(workspace)) return RPTC_EALIGN;
        if (workspace_bytes < n * (hd + 2) * 4) return RPTC_ESHAPE;
        a.part_acc = static_cast<float *>(workspace);
        a.part_ml = a.part_acc + n * hd;
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    Timer timer;
    if ((rc = timer.begin(dev, s, ms))) return rc;
    const bool f16 = dtype == RPTC_F16;
    switch (hd) {
    case 32: f16 ? launch_prompt<32, TypeF16>(a, s) : launch_prompt<32, TypeBf16>(a, s); break;
    case 64: f16 ? launch_prompt<64, TypeF16>(a, s) : launch_prompt<64, TypeBf16>(a, s); break;
    case 128: f16 ? launch_prompt<128, TypeF16>(a, s) : launch_prompt<128, TypeBf16>(a, s); break;
    default: f16 ? launch_prompt<256, TypeF16>(a, s) : launch_prompt<256, TypeBf16>(a, s); break;
    }
    return timer.end();
}
