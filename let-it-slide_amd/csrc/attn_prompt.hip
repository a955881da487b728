// Attention of whole prompts: packed sequences of different lengths, causal or not, grouped heads, fp16 or bf16.
// (No counterpart in the reference, which generates with transformers on dense weights, quantize_hf.py:229-236.)
//
//   o_i = sum_j p_ij v_j / l_i,   p_ij = exp2(c q_i.k_j - m_i),   l_i = sum_j p_ij,   lse_i = (m_i + log2 l_i) ln 2
//
// with c = scale log2(e), over the keys j that query i sees, in one pass over the keys: m_i is a running bound of
// c q_i.k_j (raised, and the sums rescaled, only where a score exceeds it by more than 2^8, so p stays below 256; in fp16 all of
// them times 2^7, which the quotient takes off again).
// Scores, m, l and the output sums are fp32; p is rounded to the inputs' type for the matrix unit (by at most
// 2^-11 of it in fp16, 2^-8 in bf16: the products need two operands of one type), l adds the unrounded p.  Calls that leave the matrix unit
// idle put what the rounding left in as well (see prompt_plan).
//
// A workgroup of four waves owns 128 query rows of one head (64 or 32 in the forms for fewer rows), 32 a wave, and walks over its
// keys 64 at a time.
// The products are formed transposed, S^T = K Q^T and O^T = V^T P^T with 32x32x16 matrix instructions: a lane then holds
// scores of one query only (the row maximum is 31 maxima in the lane and one swap of the wave's halves), the scores'
// layout is, up to a renumbering of the keys that V follows, the layout the second product wants P in, and every
// factor of a row is a factor of a lane.  K and V come from memory straight into LDS (two buffers, 16 bytes a lane);
// V^T is read with the transposing LDS read.
//
// What bounds it: a SIMD's matrix and vector instructions hardly overlap (a step of 32 rows and 64 keys at hd 128: 0.47 us of one, 0.25 of
// the other, of 0.9 together), at the clock the power leaves.  8192 causal rows of 32 / 8 heads x 128, bf16: 503 to 530 us, 1.04 to 1.09
// PFLOP/s, the matrix unit busy for 62 % of it (a library product of 8192^3 1.22 PFLOP/s).  32 rows behind 8000, 32 heads x 128: 30 us
// for 132 MB, 4.4 TB/s, and 4 for joining the pieces.
#include "join.hpp"
#include "lds_load.hpp"

namespace rptc {

constexpr int kPromptThreads = 256;
constexpr int kWideRows = 128;         // query rows of a workgroup of the wide kernel
constexpr float kLazy = 8.f;           // exponents of 2 a score may exceed the running bound by

typedef float float16_t __attribute__((ext_vector_type(16)));
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
    static constexpr short kExponent = 0x7C00;
    // weights carry a factor 2^7: a weight far below the largest is held to 2^-31 of it instead of 2^-24 (many such ones behind one that outweighs
    // them would otherwise be lost), and the largest, 2^15, stays below 65504.  bf16 has fp32's exponents
    static constexpr float kWeightLog2 = 7.f, kWeightInverse = 0x1p-7f;
    // sum + 0 x for two values x: not a number where one of them is no finite number
    static __device__ __forceinline__ float zero_of(uint32_t w, float sum)
    {
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(half2_t, w), (half2_t)((_Float16)0.f), sum, false);
    }
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
    static constexpr short kExponent = 0x7F80;
    static constexpr float kWeightLog2 = 0.f, kWeightInverse = 1.f;
    static __device__ __forceinline__ float zero_of(uint32_t w, float sum)
    {
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w), (bf16x2_t)((__bf16)0.f), sum, false);
    }
};

struct PromptArgs {
    const uint16_t *q, *k, *v;
    uint16_t *out;
    float *lse;                        // [total_q][heads], may be null
    const int32_t *q_start, *k_start, *k_len;
    float *part_acc, *part_ml;         // splits > 1: [total_q][heads][split][hd] sums, [..][2] bound and sum of p
    int32_t *first_tile;               // [seqs], may be null: the tiles of the sequences in front of each
    rptc_prompt_strides st;
    int seqs, total_q, total_k, heads, kv_heads, tiles, splits, causal;
    int row_bits;                      // a tile has 2^row_bits query rows
    float c;                           // scale * log2(e)
};

struct PromptTile {
    int seq, q_begin, q_end, row0;     // the sequence's query rows, the tile's first row
    int k_first, k_len;                // and its keys
};

// Sequence s as device memory has it.  One that does not lie inside the query rows has no tiles.
struct PromptSequence {
    int begin, end, tiles, k_first, k_len;
};
__device__ __forceinline__ PromptSequence prompt_sequence(const PromptArgs &a, int s)
{
    PromptSequence r = {0, 0, 0, 0, 0};
    if (s >= a.seqs) return r;
    r.begin = a.q_start ? a.q_start[s] : 0;
    r.end = a.q_start ? a.q_start[s + 1] : a.total_q;
    r.k_first = a.k_start ? a.k_start[s] : a.q_start ? r.begin : 0;
    r.k_len = a.k_len ? a.k_len[s] : a.q_start ? r.end - r.begin : a.total_k;
    if (r.begin >= 0 && r.end > r.begin && r.end <= a.total_q) r.tiles = (r.end - r.begin + (1 << a.row_bits) - 1) >> a.row_bits;
    return r;
}

// The sequence that holds tile `tile` when every sequence is cut into tiles of 2^row_bits query rows: 64 sequences at a time, a
// lane each; of very many sequences by a search for the tile among their first ones, 64 of them at a time.  A sequence's
// tiles are taken from its end (the longest rows of a causal prompt first).  False for a tile past the last, and for one whose
// keys do not lie inside k and v (its rows are left as they are).
__device__ __forceinline__ bool find_tile(const PromptArgs &a, int tile, PromptTile &t)
{
    const int lane = threadIdx.x & 63;
    t.seq = -1;
    t.q_begin = t.q_end = t.row0 = t.k_first = t.k_len = 0;
    int in_front = 0, n = 0;               // tiles of the sequences in front (they do not overlap: at most a.tiles), of the sequence
    if (a.first_tile) {
        int s = 0;                         // first_tile[s] <= tile, the last such one in [s, s + range)
        for (int range = a.seqs; range > 1;) {
            const int stride = (range + 63) >> 6, at = lane * stride;
            const bool up_to = at < range && a.first_tile[s + at] <= tile;
            const int passed = (__builtin_popcountll(__ballot(up_to)) - 1) * stride;
            s += passed;
            range = min(stride, range - passed);
        }
        const PromptSequence r = prompt_sequence(a, s);
        in_front = a.first_tile[s];
        if (tile - in_front < r.tiles) {
            t.seq = s;
            t.q_begin = r.begin;
            t.q_end = r.end;
            t.k_first = r.k_first;
            t.k_len = r.k_len;
            n = r.tiles;
        }
    } else {
        for (int s0 = 0; s0 < a.seqs; s0 += 64) {
            const PromptSequence r = prompt_sequence(a, s0 + lane);
            int incl = r.tiles;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const int o = __shfl_up(incl, off, 64);
                if (lane >= off) incl += o;
            }
            const uint64_t hit = __ballot(in_front + incl > tile);
            if (hit) {
                const int f = __builtin_ctzll(hit);
                n = __builtin_amdgcn_readlane(r.tiles, f);
                in_front += __builtin_amdgcn_readlane(incl, f) - n;
                t.seq = s0 + f;
                t.q_begin = __builtin_amdgcn_readlane(r.begin, f);
                t.q_end = __builtin_amdgcn_readlane(r.end, f);
                t.k_first = __builtin_amdgcn_readlane(r.k_first, f);
                t.k_len = __builtin_amdgcn_readlane(r.k_len, f);
                break;
            }
            in_front += __builtin_amdgcn_readlane(incl, 63);
        }
    }
    if (t.seq < 0) return false;
    t.seq = uniform(t.seq);
    t.q_begin = uniform(t.q_begin);
    t.q_end = uniform(t.q_end);
    t.row0 = uniform(t.q_begin + ((n - 1 - (tile - in_front)) << a.row_bits));
    t.k_first = uniform(t.k_first);
    t.k_len = uniform(t.k_len);
    return t.k_first >= 0 && t.k_len >= 0 && (int64_t)t.k_first + t.k_len <= a.total_k;
}

// The tiles of the sequences in front of each, for calls of very many sequences: one workgroup, a thread a sequence at a time.  No more than
// a.tiles, the tiles there are room for (sequences that overlap, which is not a valid call, may have more).
constexpr int kTableThreads = 1024;
__global__ __launch_bounds__(kTableThreads) void attn_prompt_table_kernel(const PromptArgs a)
{
    __shared__ int s_waves[kTableThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int in_front = 0;
    for (int s0 = 0; s0 < a.seqs; s0 += kTableThreads) {
        const int n = prompt_sequence(a, s0 + tid).tiles;
        int incl = n;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int o = __shfl_up(incl, off, 64);
            if (lane >= off) incl += o;
        }
        if (lane == 63) s_waves[wave] = incl;
        __syncthreads();
        int before = in_front, all = 0;
        for (int w = 0; w < kTableThreads / 64; w++) {
            if (w < wave) before += s_waves[w];
            all += s_waves[w];
        }
        if (s0 + tid < a.seqs) a.first_tile[s0 + tid] = min(before + incl - n, a.tiles);
        in_front = min(in_front + all, a.tiles);
        __syncthreads();
    }
}

// keys a row sees: [0, sees)
__device__ __forceinline__ int prompt_sees(const PromptArgs &a, const PromptTile &t, int row)
{
    return a.causal ? max(0, t.k_len - (t.q_end - t.q_begin) + 1 + (row - t.q_begin)) : t.k_len;
}

// Workgroup -> (head, tile, split): tiles from the longest walks to the shortest, so that the last workgroups to start are
// short ones.  Consecutive workgroups go to the eight XCDs in turn, each with an L2 of its own: where the heads divide
// evenly an XCD gets a run of heads (those of a group read the same K and V) and walks over the tiles of all of them.
__device__ __forceinline__ void prompt_item(const PromptArgs &a, int &head, int &tile, int &split)
{
    const bool runs = a.heads % 8 == 0;
    const int run = runs ? a.heads >> 3 : a.heads, local = runs ? blockIdx.x >> 3 : blockIdx.x;
    const int rest = local / run;
    head = local - rest * run + (runs ? (blockIdx.x & 7) * run : 0);
    tile = rest / a.splits;
    split = rest - tile * a.splits;
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

// Values of V that are no finite numbers in a step where some row does not see some key (the last one or two of a walk): the weight is 0
// there, but 0 times infinity or not-a-number is none, and would reach a row that must not show it.  Where a wave's sums came out odd
// and its steps with masked keys hold such values, the walk is taken three times more: with a 1 in place of every value that is +infinity or
// not-a-number, a 0 of every other and equal weights, which marks the elements that see one; so for -infinity or not-a-number; and
// with 0 in place of all of them, in the first walk's order.  The elements then get what they saw, and one that saw none has the bits it
// has with zeros in V.  At most five times the time of a call without them (2000 rows of 32 heads x 128: 54 us, with an infinity in the
// first and the last values 244, nothing but not-a-numbers 275; the odd rows one after the other, with plain loads, took 11.5 ms and grew
// with the square of the rows).
enum { kUps, kDowns, kFiniteOnly, kWalks };
// whether rows [k0, k1) of V hold such values
template <int HD, class T>
__device__ __forceinline__ bool values_odd(const uint16_t *v, int64_t token, int k0, int k1)
{
    float none = 0.f;
    for (int i = 8 * (threadIdx.x & 63); i < (k1 - k0) * HD; i += 512) {
        const uint4 w = *reinterpret_cast<const uint4 *>(v + (k0 + i / HD) * token + i % HD);
        none = T::zero_of(w.w, T::zero_of(w.z, T::zero_of(w.y, T::zero_of(w.x, none))));
    }
    return __ballot(none != 0.f) != 0;
}
template <class T>
__device__ __forceinline__ void change_values(uint16_t *v, int walk)
{
    uint4 w = *reinterpret_cast<uint4 *>(v);
    uint32_t x[4] = {w.x, w.y, w.z, w.w};
    const uint32_t one = T::pack(1.f, 1.f);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t r = 0;
#pragma unroll
        for (int b = 0; b < 32; b += 16) {
            const uint32_t half = 0xFFFFu << b, value = x[i] & half, least = (uint32_t)T::kExponent << b, minus = least | 0x8000u << b;
            const bool finite = (value & least) != least;
            if (walk == kFiniteOnly) r |= finite ? value : 0u;
            else r |= !finite && value != (walk == kUps ? minus : least) ? one & half : 0u;
        }
        x[i] = r;
    }
    *reinterpret_cast<uint4 *>(v) = make_uint4(x[0], x[1], x[2], x[3]);
}

// What a wave holds of 32 query rows, and the parts of a step over KEYS keys (a multiple of 32).  Lane (col, c): row col; of
// every eight keys and of every eight dimensions the four from 4c on.
// TERMS = 2: p enters the product as the sum of two numbers of the type (its rounding and what that left), so that
// the output's own rounding is what is left: for the calls that leave the matrix unit idle (see prompt_plan).
template <int HD, class T, int KEYS, int TERMS>
struct PromptWave {
    static constexpr int kSteps = HD / 16, kDims = HD / 32, kBlocks = KEYS / 32;
    int tid;                               // the thread in its workgroup
    short8_t qf[kSteps];
    float16_t acc[kDims];
    float m, l;                            // running bound of c * score (log2 units), sum of p over the lane's keys

    __device__ __forceinline__ void begin(const PromptArgs &a, const PromptTile &t, int row, int head)
    {
        // a lane without a row of its own takes the sequence's last (its results go nowhere)
        const uint16_t *q = a.q + (int64_t)min(row, t.q_end - 1) * a.st.q_token + (int64_t)head * a.st.q_head + 8 * ((tid & 63) >> 5);
#pragma unroll
        for (int i = 0; i < kSteps; i++) qf[i] = *reinterpret_cast<const short8_t *>(q + 16 * i);
#pragma unroll
        for (int d = 0; d < kDims; d++) acc[d] = (float16_t)(0.f);
        m = -INFINITY;
        l = 0.f;
    }
    // the query is there: a wait inside the loop would wait for the step's K and V as well
    __device__ __forceinline__ void settle()
    {
#pragma unroll
        for (int i = 0; i < kSteps; i++) asm volatile("" : "+v"(qf[i]));
    }
    // S^T of the keys in LDS at kt
    __device__ __forceinline__ void scores(const uint16_t *kt, float16_t (&s)[kBlocks]) const
    {
        const int lane = tid & 63, c = lane >> 5, col = lane & 31;
#pragma unroll
        for (int h = 0; h < kBlocks; h++) {
            s[h] = (float16_t)(0.f);
            const int r = 32 * h + col;
#pragma unroll
            for (int i = 0; i < kSteps; i++) {
                const short8_t kf = *reinterpret_cast<const short8_t *>(kt + r * HD + ((2 * i + c) ^ swizzle_k<HD>(r)) * 8);
                s[h] = T::mfma(kf, qf[i], s[h]);
            }
        }
    }
    // the same for a walk taken again: where it marks, every key weighs the same
    __device__ __forceinline__ void scores_of(const uint16_t *kt, int walk, float16_t (&s)[kBlocks]) const
    {
        scores(kt, s);
        if (walk == kFiniteOnly) return;
#pragma unroll
        for (int h = 0; h < kBlocks; h++) s[h] = (float16_t)(0.f);
    }
    // keys from `left` on (counted from the step's first) are not the row's
    __device__ __forceinline__ void mask(float16_t (&s)[kBlocks], int left) const
    {
        left -= 4 * ((tid & 63) >> 5);
#pragma unroll
        for (int h = 0; h < kBlocks; h++)
#pragma unroll
            for (int r = 0; r < 16; r++)
                if (32 * h + 8 * (r / 4) + r % 4 >= left) s[h][r] = -INFINITY;
    }
    // raises the bound where a score exceeds it by more than 2^kLazy; returns what to take off of the scores times `scale`
    __device__ __forceinline__ float bound(float16_t (&s)[kBlocks], float &scale)
    {
        float mx = s[0][0];
#pragma unroll
        for (int h = 0; h < kBlocks; h++)
#pragma unroll
            for (int r = 0; r < 16; r++) mx = fmaxf(mx, s[h][r]);
        mx = halves_max(mx) * scale;
        const bool raise = mx > m + kLazy;                 // (each row by itself: its bits do not depend on the wave's others)
        if (__ballot(raise)) {
            const float up = raise ? mx : m;
            const float f = up == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - up);
            l *= f;
#pragma unroll
            for (int d = 0; d < kDims; d++) acc[d] *= f;
            m = up;
        }
        float off = (m == -INFINITY ? 0.f : m) - T::kWeightLog2;
        // the bound is a rounded product, and what the rounding left a factor of all weights: within 2^(1/32) of 1 below 2^20, but up to 2^32
        // at 2^30.  From 2^20 on the scores are multiplied and rounded as the bound was, and their differences to it taken
        const uint32_t size = __builtin_bit_cast(uint32_t, m) & 0x7FFFFFFFu;
        const bool far = size - 0x49800000u < 0x7F800000u - 0x49800000u;      // 2^20 <= |m| < infinity
        if (__ballot(far)) {
#pragma clang fp contract(off)
#pragma unroll
            for (int h = 0; h < kBlocks; h++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const float product = s[h][r] * scale;
                    s[h][r] = far ? product - m : s[h][r];
                }
            scale = far ? 1.f : scale;
            off = far ? -T::kWeightLog2 : off;
        }
        return off;
    }
    // p = exp2(c s - bound), packed in pairs of keys
    __device__ __forceinline__ void weights(const float16_t (&s)[kBlocks], float scale, float off, uint32_t (&p)[TERMS][kBlocks][8])
    {
#pragma unroll
        for (int h = 0; h < kBlocks; h++)
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                const float p0 = __builtin_amdgcn_exp2f(fmaf(s[h][r], scale, -off)), p1 = __builtin_amdgcn_exp2f(fmaf(s[h][r + 1], scale, -off));
                l += p0;
                l += p1;
                p[0][h][r / 2] = T::pack(p0, p1);
                if (TERMS > 1) {
                    const uint32_t w = p[0][h][r / 2];
                    p[TERMS - 1][h][r / 2] = T::pack(p0 - T::to_float((uint16_t)w), p1 - T::to_float((uint16_t)(w >> 16)));
                }
            }
    }
    // acc += V^T P^T, V in LDS at vt: the lane's dimension of a tile of 32, keys in the order the scores' registers have them
    __device__ __forceinline__ void product(const uint16_t *vt, const uint32_t (&p)[TERMS][kBlocks][8])
    {
        typedef __attribute__((address_space(3))) short4_t lds_short4;
        const int lane = tid & 63, c = lane >> 5, g16 = lane >> 4, rr = (lane & 15) >> 2, piece = lane & 3;
#pragma unroll
        for (int h = 0; h < kBlocks; h++)
#pragma unroll
            for (int g = 0; g < 2; g++) {
                uint4 pv[TERMS];
#pragma unroll
                for (int u = 0; u < TERMS; u++) pv[u] = make_uint4(p[u][h][4 * g], p[u][h][4 * g + 1], p[u][h][4 * g + 2], p[u][h][4 * g + 3]);
                const int key = 32 * h + 16 * g + 4 * c + rr;
#pragma unroll
                for (int d = 0; d < kDims; d++) {
                    const int ch = (4 * d + 2 * (g16 & 1) + piece / 2) ^ swizzle_v<HD>(key);   // key and key + 8: the same swizzle
                    const uint16_t *va = vt + key * HD + ch * 8 + (piece & 1) * 4;
                    const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4 *)va);
                    const short4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4 *)(va + 8 * HD));
#pragma unroll
                    for (int u = 0; u < TERMS; u++)
                        acc[d] = T::mfma(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7), __builtin_bit_cast(short8_t, pv[u]), acc[d]);
                }
            }
    }
    // whether a sum came out infinite or not a number, in any of the rows
    __device__ __forceinline__ bool odd() const
    {
        float bad = 0.f;
#pragma unroll
        for (int d = 0; d < kDims; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) bad = fmaf(acc[d][r], 0.f, bad);
        return __ballot(bad != 0.f) != 0;                  // (not-a-number compares unequal)
    }
    // which elements are above 0, a bit each
    static constexpr int kMarks = HD < 64 ? 1 : HD / 64;
    __device__ __forceinline__ void take_marks(uint32_t *marks) const
    {
#pragma unroll
        for (int i = 0; i < kMarks; i++) {
            uint32_t bits = 0;
#pragma unroll
            for (int d = 2 * i; d < 2 * i + 2 && d < kDims; d++)
#pragma unroll
                for (int r = 0; r < 16; r++) bits = bits << 1 | (acc[d][r] > 0.f ? 1u : 0u);
            marks[i * kPromptThreads] = bits;
        }
    }
    // the infinities (not-a-number where it is both) that the elements see
    __device__ __forceinline__ void put_marks(const uint32_t *ups, const uint32_t *downs)
    {
#pragma unroll
        for (int i = 0; i < kMarks; i++) {
            uint32_t up = ups[i * kPromptThreads], down = downs[i * kPromptThreads];
#pragma unroll
            for (int d = 2 * i + 1; d >= 2 * i; d--)
#pragma unroll
                for (int r = 15; r >= 0; r--) {
                    if (d >= kDims) continue;
                    if (up & 1u) acc[d][r] += INFINITY;
                    if (down & 1u) acc[d][r] -= INFINITY;
                    up >>= 1;
                    down >>= 1;
                }
        }
    }
};

// Many rows: 128 query rows of a head a workgroup, 32 a wave (G = 1); all waves walk over the same keys, which are brought to
// LDS once for the four of them, a step ahead.  G = 2: 64 query rows, two waves a row, one for the first and one for the second half of
// a step's 64 keys, joined at the end: twice the workgroups with half the walk, where the longest walk is what the call waits
// for; its keys may be cut into pieces as well (150 rows behind 8000, 32 / 8 heads x 128: 95 us whole, 46 in four).  64 keys a wave
// and a step of 128 need twice the LDS: 1024 rows of 32 heads x 128 29.4 us instead of 21.6; G = 1 with 32 keys a step meets
// twice as often: 8192 rows 567 us instead of 520.
template <int HD, int G>
constexpr int kWaveKeys = G == 2 ? 32 : 64;    // keys of a step and wave

// workgroups that a compute unit holds at once (by their registers; LDS has room for as many): said to the compiler as least and
// most, so that it uses the registers for operands asked for early instead of for more of them
// (two terms a weight: for calls that leave places free)
template <int HD, int G, int TERMS>
constexpr int kPlaces = HD > 128 ? 1 : HD == 128 || TERMS == 2 ? 2 : HD == 64 && G == 1 ? 3 : 4;

template <int HD, class T, int G, int TERMS>
__global__ __launch_bounds__(kPromptThreads) __attribute__((amdgpu_waves_per_eu(kPlaces<HD, G, TERMS>, kPlaces<HD, G, TERMS>))) void attn_prompt_kernel(const PromptArgs a)
{
    extern __shared__ __align__(16) uint16_t lds[];       // two buffers of K, two of V, [kKeys][HD] each
    constexpr int kMine = kWaveKeys<HD, G>, kKeys = G * kMine, kTile = kKeys * HD, kRows = kWideRows / G;
    static_assert(G == 1 || 2 * 32 * HD * 4 <= 4 * kTile * 2, "the sums of two waves fit where K and V were");
    __shared__ float s_ml[2][32][2];
    __shared__ uint32_t s_marks[2][PromptWave<HD, T, kMine, TERMS>::kMarks * kPromptThreads];
    __shared__ int s_again;
    int tid = threadIdx.x, lane = tid & 63, c = lane >> 5, col = lane & 31;
    const int wave = uniform(tid >> 6);
    int head, tile, split;
    prompt_item(a, head, tile, split);
    PromptTile t;
    if (!find_tile(a, tile, t)) return;
    const int kvh = head / (a.heads / a.kv_heads);

    const int k_most = uniform(prompt_sees(a, t, min(t.row0 + kRows, t.q_end) - 1));    // of the tile's last row: the most
    // this workgroup's piece of them, whole steps
    int k_lo = 0, k_hi = k_most;
    if (G == 2 && a.splits > 1) {
        const int per_split = ((k_most + a.splits - 1) / a.splits + kKeys - 1) / kKeys * kKeys;
        k_lo = uniform((int)min((int64_t)k_most, (int64_t)split * per_split));
        k_hi = uniform((int)min((int64_t)k_most, (int64_t)k_lo + per_split));
    }
    const int group = G == 2 ? wave >> 1 : 0, koff = group * kMine;
    const int row_first = t.row0 + 32 * (wave & (4 / G - 1));
    int row = row_first + col;
    const bool wave_live = row_first < t.q_end;
    int see = row < t.q_end ? prompt_sees(a, t, row) : 0;
    // what all rows of the wave see, and what one of them sees
    const int see_least = uniform(wave_live ? prompt_sees(a, t, row_first) : 0);
    const int see_most = uniform(wave_live ? prompt_sees(a, t, min(row_first + 31, t.q_end - 1)) : 0);

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
    const uint16_t *k_base = a.k + (int64_t)t.k_first * a.st.k_token + (int64_t)kvh * a.st.k_head;
    const uint16_t *v_base = a.v + (int64_t)t.k_first * a.st.v_token + (int64_t)kvh * a.st.v_head;
    const uint32_t lds_base = lds_address(lds) + (uint32_t)wave * 1024u;
    auto request_k = [&](int k0, int buf) {
        const int4_t r = buffer_resource(k_base + (int64_t)k0 * a.st.k_token, ((min(t.k_len - k0, kKeys) - 1) * (int)a.st.k_token + HD) * 2);
#pragma unroll
        for (int u = 0; u < kRequests; u++) load_to_lds(k_off[u], r, lds_base + (uint32_t)buf * (2u * kTile) + u * 4096u);
    };
    auto request_v = [&](int k0, int buf) {
        const int4_t r = buffer_resource(v_base + (int64_t)k0 * a.st.v_token, ((min(t.k_len - k0, kKeys) - 1) * (int)a.st.v_token + HD) * 2);
#pragma unroll
        for (int u = 0; u < kRequests; u++) load_to_lds(v_off[u], r, lds_base + (uint32_t)(2 + buf) * (2u * kTile) + u * 4096u);
    };

    if (k_lo < k_hi) {
        request_k(k_lo, 0);
        request_v(k_lo, 0);
        if (k_lo + kKeys < k_hi) request_k(k_lo + kKeys, 1);
    }
    PromptWave<HD, T, kMine, TERMS> w;
    w.tid = tid;
    w.begin(a, t, row, head);
    w.settle();
    if (tid == 0) s_again = 0;
    int masked_from = 0x7FFFFFFF;                          // the first step with a key that some row of the wave does not see
    // One step: the softmax of the scores s of the keys from k0 on and their product with V, while the matrix unit forms the
    // next step's scores (behind the last step these are of whatever the buffer holds, and nobody looks at them).
    auto step = [&](int k0, int buf, float16_t (&s)[kMine / 32], float16_t (&next)[kMine / 32]) {
        wait_for_lds_loads();                              // this wave's part of the next K and of this V is in LDS
        __syncthreads();                                   // everyone's is, and nobody reads what is requested over now
        if (k0 + 2 * kKeys < k_hi) request_k(k0 + 2 * kKeys, buf);
        if (k0 + kKeys < k_hi) request_v(k0 + kKeys, buf ^ 1);
        if (k0 + koff >= see_most) return;
        const bool masked = k0 + koff + kMine > see_least; // some row of the wave does not see all of its keys
        if (masked) {
            masked_from = min(masked_from, k0 + koff);
            w.mask(s, see - k0 - koff);
        }
        float scale = a.c;
        const float off = w.bound(s, scale);
        w.scores(lds + (buf ^ 1) * kTile + koff * HD, next);
        uint32_t p[TERMS][kMine / 32][8];
        w.weights(s, scale, off, p);
        w.product(lds + (2 + buf) * kTile + koff * HD, p);
    };
    if (k_lo < k_hi) {
        float16_t sa[kMine / 32], sb[kMine / 32];
        wait_for_lds_loads();
        __syncthreads();
        w.scores(lds + koff * HD, sa);
        for (int k0 = k_lo; k0 < k_hi; k0 += 2 * kKeys) {
            step(k0, 0, sa, sb);
            if (k0 + kKeys >= k_hi) break;
            step(k0 + kKeys, 1, sb, sa);
        }
        // what is known of the lane is worked out again for what follows: kept over the walk it would cost the registers that let
        // the loop ask for its operands early
        asm volatile("" : "+v"(tid));
        w.tid = tid;
        lane = tid & 63;
        c = lane >> 5;
        col = lane & 31;
        row = row_first + col;
        see = row < t.q_end ? prompt_sees(a, t, row) : 0;
        if (masked_from < k_hi && w.odd() && values_odd<HD, T>(v_base, a.st.v_token, masked_from, min(t.k_len, see_most + kMine))) s_again = 1;
    }
    auto finish = [&]() {
        float l = halves_sum(w.l);
        if (G == 2) {
            // sums of the second half's waves to the first's, a register of all lanes after the other
            float4 *sums = reinterpret_cast<float4 *>(lds) + (wave & 1) * (HD * 8) + lane;
            if (group == 1) {
#pragma unroll
                for (int d = 0; d < HD / 32; d++)
#pragma unroll
                    for (int b = 0; b < 4; b++)
                        sums[64 * (4 * d + b)] = make_float4(w.acc[d][4 * b], w.acc[d][4 * b + 1], w.acc[d][4 * b + 2], w.acc[d][4 * b + 3]);
                if (c == 0) {
                    s_ml[wave & 1][col][0] = w.m;
                    s_ml[wave & 1][col][1] = l;
                }
            }
            __syncthreads();
            if (group == 1) return;
            const float m1 = s_ml[wave][col][0], M = fmaxf(w.m, m1);
            const float f0 = w.m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(w.m - M), f1 = m1 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m1 - M);
            l = l * f0 + s_ml[wave][col][1] * f1;
            w.m = M;
#pragma unroll
            for (int d = 0; d < HD / 32; d++)
#pragma unroll
                for (int b = 0; b < 4; b++) {
                    const float4 o = sums[64 * (4 * d + b)];
                    w.acc[d][4 * b] = fmaf(o.x, f1, w.acc[d][4 * b] * f0);
                    w.acc[d][4 * b + 1] = fmaf(o.y, f1, w.acc[d][4 * b + 1] * f0);
                    w.acc[d][4 * b + 2] = fmaf(o.z, f1, w.acc[d][4 * b + 2] * f0);
                    w.acc[d][4 * b + 3] = fmaf(o.w, f1, w.acc[d][4 * b + 3] * f0);
                }
        }
        if (!wave_live) return;
        if (G == 2 && a.splits > 1) {
            if (row < t.q_end) {
                const int64_t pa = ((int64_t)row * a.heads + head) * a.splits + split;
                float *part = a.part_acc + pa * HD + 4 * c;
#pragma unroll
                for (int d = 0; d < HD / 32; d++)
#pragma unroll
                    for (int b = 0; b < 4; b++)
                        *reinterpret_cast<float4 *>(part + 32 * d + 8 * b) = make_float4(w.acc[d][4 * b], w.acc[d][4 * b + 1], w.acc[d][4 * b + 2], w.acc[d][4 * b + 3]);
                if (c == 0) *reinterpret_cast<float2 *>(a.part_ml + 2 * pa) = make_float2(l == 0.f ? -INFINITY : w.m, l);
            }
            return;
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;            // a row that sees nothing: zeros
        uint16_t *o = a.out + (int64_t)min(row, t.q_end - 1) * a.st.out_token + (int64_t)head * a.st.out_head + 8 * c;
#pragma unroll
        for (int d = 0; d < HD / 32; d++)
#pragma unroll
            for (int b = 0; b < 4; b += 2) {
                // the lane's four dimensions of blocks b and b + 1 (8 dimensions each, the halves of the wave four): a swap of
                // the halves leaves eight consecutive ones of block b + c in each lane
                const float16_t &x = w.acc[d];
                uint32_t x0 = T::pack(x[4 * b] * inv, x[4 * b + 1] * inv), x1 = T::pack(x[4 * b + 2] * inv, x[4 * b + 3] * inv);
                uint32_t y0 = T::pack(x[4 * b + 4] * inv, x[4 * b + 5] * inv), y1 = T::pack(x[4 * b + 6] * inv, x[4 * b + 7] * inv);
                const auto w0 = __builtin_amdgcn_permlane32_swap(x0, y0, false, false), w1 = __builtin_amdgcn_permlane32_swap(x1, y1, false, false);
                if (row < t.q_end)
                    *reinterpret_cast<uint4 *>(o + 32 * d + 8 * b) = make_uint4((uint32_t)w0[0], (uint32_t)w1[0], (uint32_t)w0[1], (uint32_t)w1[1]);
            }
        if (a.lse && c == 0 && row < t.q_end) a.lse[(int64_t)row * a.heads + head] = l == 0.f ? -INFINITY : (w.m + log2f(l * T::kWeightInverse)) * 0.693147180559945f;
    };
    // every wave has said whether to go again, and nobody reads K or V any more; one that need not wait for that has stored its rows
    if (G == 1) finish();
    __syncthreads();
    if (k_lo < k_hi && s_again) {
#pragma unroll 1
        for (int walk = kUps; walk < kWalks; walk++) {
            request_k(k_lo, 0);
            request_v(k_lo, 0);
            w.begin(a, t, row, head);
            w.settle();
#pragma unroll 1
            for (int k0 = k_lo, buf = 0; k0 < k_hi; k0 += kKeys, buf ^= 1) {
                wait_for_lds_loads();
                __syncthreads();
                if (k0 + kKeys < k_hi) {
                    request_k(k0 + kKeys, buf ^ 1);
                    request_v(k0 + kKeys, buf ^ 1);
                }
#pragma unroll 1
                for (int i = 8 * tid; i < kTile; i += 8 * kPromptThreads) change_values<T>(lds + (2 + buf) * kTile + i, walk);
                __syncthreads();
                if (k0 + koff >= see_most) continue;
                float16_t s[kMine / 32];
                uint32_t p[TERMS][kMine / 32][8];
                w.scores_of(lds + buf * kTile + koff * HD, walk, s);
                if (k0 + koff + kMine > see_least) w.mask(s, see - k0 - koff);
                float scale = a.c;
                const float off = w.bound(s, scale);
                w.weights(s, scale, off, p);
                w.product(lds + (2 + buf) * kTile + koff * HD, p);
            }
            if (walk != kFiniteOnly) w.take_marks(s_marks[walk - kUps] + tid);
            __syncthreads();                               // nobody reads K or V now
        }
        w.put_marks(s_marks[0] + tid, s_marks[1] + tid);
        if (G == 1) finish();
    }
    if (G == 2) finish();
}

// Few rows: 32 query rows of a head a workgroup; the four waves hold the same rows and take the steps over the keys (of this
// workgroup's piece of them) in turn, each with K and V of its own in LDS and no barrier until they join at the end: K of
// a wave's next step is on its way while it works on V, and the other way round.
constexpr int kNarrowRows = 32;
template <int HD>
constexpr int kNarrowKeys = HD > 128 ? 32 : 64;

template <int HD, class T>
__global__ __launch_bounds__(kPromptThreads, HD > 64 ? 1 : 2) void attn_prompt_narrow_kernel(const PromptArgs a)
{
    constexpr int kStep = kNarrowKeys<HD>, kTile = kStep * HD, kJoinRow = HD > 128 ? HD : HD + 4;
    static_assert(kNarrowRows * kJoinRow * 4 <= 2 * kTile * 2, "a wave's sums fit where its K and V were");
    extern __shared__ __align__(16) uint16_t lds[];       // [wave][K, V][kStep][HD]
    __shared__ float s_ml[4][kNarrowRows][2];
    __shared__ uint32_t s_marks[2][PromptWave<HD, T, kStep, 2>::kMarks * kPromptThreads];
    int tid = threadIdx.x, lane = tid & 63, c = lane >> 5, col = lane & 31;
    const int wave = uniform(tid >> 6);
    int head, tile, split;
    prompt_item(a, head, tile, split);
    PromptTile t;
    if (!find_tile(a, tile, t)) return;
    const int kvh = head / (a.heads / a.kv_heads);
    const int k_most = uniform(prompt_sees(a, t, min(t.row0 + kNarrowRows, t.q_end) - 1));
    const int per_split = ((k_most + a.splits - 1) / a.splits + kStep - 1) / kStep * kStep;
    const int k_lo = uniform((int)min((int64_t)k_most, (int64_t)split * per_split));
    const int k_hi = uniform((int)min((int64_t)k_most, (int64_t)k_lo + per_split));
    int row = t.row0 + col;
    int see = min(row < t.q_end ? prompt_sees(a, t, row) : 0, k_hi);
    const int see_least = uniform(min(prompt_sees(a, t, t.row0), k_hi));

    // a request is 1024 bytes: 512 / HD rows; the swizzles repeat every 16 rows (K) and every 4 (V)
    constexpr int kChunks = HD / 8, kRequests = kTile * 2 / 1024, kReqRows = 512 / HD;
    constexpr int kKOff = 16 / kReqRows < 1 ? 1 : 16 / kReqRows, kVOff = 4 / kReqRows < 1 ? 1 : 4 / kReqRows;
    uint32_t k_off[kKOff], v_off[kVOff];
#pragma unroll
    for (int u = 0; u < kKOff; u++) {
        const int r = u * kReqRows + lane / kChunks, ch = lane % kChunks;
        k_off[u] = (uint32_t)(r * a.st.k_token + (ch ^ swizzle_k<HD>(r)) * 8) * 2u;
        if (u < kVOff) v_off[u] = (uint32_t)(r * a.st.v_token + (ch ^ swizzle_v<HD>(r)) * 8) * 2u;
    }
    const uint16_t *k_base = a.k + (int64_t)t.k_first * a.st.k_token + (int64_t)kvh * a.st.k_head;
    const uint16_t *v_base = a.v + (int64_t)t.k_first * a.st.v_token + (int64_t)kvh * a.st.v_head;
    uint16_t *kt = lds + wave * 2 * kTile, *vt = kt + kTile;
    const uint32_t k_to = lds_address(kt), v_to = lds_address(vt);
    auto request_k = [&](int k0) {
        const int4_t r = buffer_resource(k_base + (int64_t)k0 * a.st.k_token, ((min(t.k_len - k0, kStep) - 1) * (int)a.st.k_token + HD) * 2);
#pragma unroll
        for (int u = 0; u < kRequests; u++)
            load_to_lds(k_off[u % kKOff] + (uint32_t)(u / kKOff * kKOff * kReqRows * (int)a.st.k_token * 2), r, k_to + u * 1024u);
    };
    auto request_v = [&](int k0) {
        const int4_t r = buffer_resource(v_base + (int64_t)k0 * a.st.v_token, ((min(t.k_len - k0, kStep) - 1) * (int)a.st.v_token + HD) * 2);
#pragma unroll
        for (int u = 0; u < kRequests; u++)
            load_to_lds(v_off[u % kVOff] + (uint32_t)(u / kVOff * kVOff * kReqRows * (int)a.st.v_token * 2), r, v_to + u * 1024u);
    };

    constexpr int kStride = 4 * kStep;
    const int k_first = k_lo + wave * kStep;
    if (k_first < k_hi) {
        request_k(k_first);
        request_v(k_first);
    }
    PromptWave<HD, T, kStep, 2> w;
    w.tid = tid;
    w.begin(a, t, row, head);
    w.settle();
    int masked_from = 0x7FFFFFFF;                          // as above
    for (int k0 = k_first; k0 < k_hi; k0 += kStride) {
        const bool more = k0 + kStride < k_hi;
        wait_for_lds_loads_but<kRequests>();               // K is there (V was asked for behind it)
        float16_t s[kStep / 32];
        w.scores(kt, s);
        wait_for_lds_reads();
        if (more) request_k(k0 + kStride);
        const bool masked = k0 + kStep > see_least;        // some row does not see all of the step's keys
        if (masked) {
            masked_from = min(masked_from, k0);
            w.mask(s, see - k0);
        }
        float scale = a.c;
        const float off = w.bound(s, scale);
        uint32_t p[2][kStep / 32][8];
        w.weights(s, scale, off, p);
        if (more) wait_for_lds_loads_but<kRequests>();     // V is there (the next K was asked for behind it)
        else wait_for_lds_loads();
        w.product(vt, p);
        wait_for_lds_reads();
        if (more) request_v(k0 + kStride);
    }
    asm volatile("" : "+v"(tid));                        // as above
    w.tid = tid;
    lane = tid & 63;
    c = lane >> 5;
    col = lane & 31;
    row = t.row0 + col;
    see = min(row < t.q_end ? prompt_sees(a, t, row) : 0, k_hi);
    if (masked_from < k_hi && w.odd() && values_odd<HD, T>(v_base, a.st.v_token, masked_from, min(t.k_len, k_hi + kStep))) {
#pragma unroll 1
        for (int walk = kUps; walk < kWalks; walk++) {
            w.begin(a, t, row, head);
            w.settle();
#pragma unroll 1
            for (int k0 = k_first; k0 < k_hi; k0 += kStride) {
                request_k(k0);
                request_v(k0);
                wait_for_lds_loads();
#pragma unroll 1
                for (int i = 8 * lane; i < kTile; i += 512) change_values<T>(vt + i, walk);
                wait_for_lds_reads();
                float16_t s[kStep / 32];
                uint32_t p[2][kStep / 32][8];
                w.scores_of(kt, walk, s);
                if (k0 + kStep > see_least) w.mask(s, see - k0);
                float scale = a.c;
                const float off = w.bound(s, scale);
                w.weights(s, scale, off, p);
                w.product(vt, p);
                wait_for_lds_reads();
            }
            if (walk != kFiniteOnly) w.take_marks(s_marks[walk - kUps] + tid);
        }
        w.put_marks(s_marks[0] + tid, s_marks[1] + tid);
    }

    // the waves join: sums to where K and V were, row by row (four floats of padding where there is room: rows on different banks)
    float *mine = reinterpret_cast<float *>(kt);
    const float l = halves_sum(w.l);
#pragma unroll
    for (int d = 0; d < HD / 32; d++)
#pragma unroll
        for (int b = 0; b < 4; b++)
            *reinterpret_cast<float4 *>(mine + col * kJoinRow + 32 * d + 8 * b + 4 * c) =
                make_float4(w.acc[d][4 * b], w.acc[d][4 * b + 1], w.acc[d][4 * b + 2], w.acc[d][4 * b + 3]);
    if (c == 0) {
        s_ml[wave][col][0] = l == 0.f ? -INFINITY : w.m;
        s_ml[wave][col][1] = l;
    }
    __syncthreads();
    constexpr int kRowChunks = HD / 8;
    for (int i = tid; i < kNarrowRows * kRowChunks; i += kPromptThreads) {
        const int r = i / kRowChunks, d = i % kRowChunks * 8;
        if (t.row0 + r >= t.q_end) break;
        const float M = fmaxf(fmaxf(s_ml[0][r][0], s_ml[1][r][0]), fmaxf(s_ml[2][r][0], s_ml[3][r][0]));
        float den = 0.f, num[8];
#pragma unroll
        for (int u = 0; u < 8; u++) num[u] = 0.f;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float mj = s_ml[j][r][0];
            const float f = mj == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mj - M);
            den = fmaf(s_ml[j][r][1], f, den);
            const float *src = reinterpret_cast<const float *>(lds + j * 2 * kTile) + r * kJoinRow + d;
#pragma unroll
            for (int u = 0; u < 8; u++) num[u] = fmaf(src[u], f, num[u]);
        }
        const int64_t at = (int64_t)(t.row0 + r) * a.heads + head;
        if (a.splits > 1) {
            const int64_t pa = at * a.splits + split;
            float4 *o = reinterpret_cast<float4 *>(a.part_acc + pa * HD + d);
            o[0] = make_float4(num[0], num[1], num[2], num[3]);
            o[1] = make_float4(num[4], num[5], num[6], num[7]);
            if (d == 0) *reinterpret_cast<float2 *>(a.part_ml + 2 * pa) = make_float2(M, den);
            continue;
        }
        const float inv = den == 0.f ? 0.f : 1.f / den;
        *reinterpret_cast<uint4 *>(a.out + (int64_t)(t.row0 + r) * a.st.out_token + (int64_t)head * a.st.out_head + d) =
            make_uint4(T::pack(num[0] * inv, num[1] * inv), T::pack(num[2] * inv, num[3] * inv), T::pack(num[4] * inv, num[5] * inv), T::pack(num[6] * inv, num[7] * inv));
        if (a.lse && d == 0) a.lse[at] = den == 0.f ? -INFINITY : (M + log2f(den * T::kWeightInverse)) * 0.693147180559945f;
    }
}

// Joins the pieces of a row, a workgroup per (row, head), for more pieces than the kernel below takes.  The rows are found as the kernel above found them: rows of no
// sequence have no pieces and stay as they are.
template <int HD, class T>
__global__ __launch_bounds__(kJoinThreads) void attn_prompt_merge_kernel(const PromptArgs a)
{
    const int head = blockIdx.y;
    PromptTile t;
    if (!find_tile(a, blockIdx.x >> a.row_bits, t)) return;
    const int row = t.row0 + (blockIdx.x & ((1 << a.row_bits) - 1));
    if (row >= t.q_end) return;
    const int64_t at = (int64_t)row * a.heads + head;
    float M, l;
    const float num = join_pieces(a.part_acc + at * a.splits * HD, a.part_ml + 2 * at * a.splits, a.splits, HD, M, l);
    if (threadIdx.x < HD)
        a.out[(int64_t)row * a.st.out_token + (int64_t)head * a.st.out_head + threadIdx.x] = (uint16_t)T::pack(l == 0.f ? 0.f : num / l, 0.f);
    if (a.lse && threadIdx.x == 0) a.lse[at] = l == 0.f ? -INFINITY : (M + log2f(l * T::kWeightInverse)) * 0.693147180559945f;
}

// The same for at most kFewPieces pieces: a wave per (row, head), eight pieces asked for at once (2300 rows of 8 heads in two pieces: 6 us
// where a workgroup a row took 28; a branch a piece in place of the clamped index: 45).
constexpr int kFewPieces = 16;
template <int HD, class T>
__global__ __launch_bounds__(256) void attn_prompt_merge_few_kernel(const PromptArgs a)
{
    constexpr int kEach = HD / 64 < 1 ? 1 : HD / 64;       // dimensions of a lane (hd 32: the lanes from 32 on repeat the others)
    typedef float vec __attribute__((ext_vector_type(kEach)));
    const int lane = threadIdx.x & 63, head = blockIdx.y * 4 + uniform((int)threadIdx.x >> 6);
    if (head >= a.heads) return;
    PromptTile t;
    if (!find_tile(a, blockIdx.x >> a.row_bits, t)) return;
    const int row = t.row0 + (blockIdx.x & ((1 << a.row_bits) - 1));
    if (row >= t.q_end) return;
    const int64_t at = (int64_t)row * a.heads + head;
    const int dim = kEach * lane % HD;
    const float *acc = a.part_acc + at * a.splits * HD + dim;
    vec v[8];
    auto ask = [&](int i0) {                               // (a piece past the last: the last once more, with factor 0)
#pragma unroll
        for (int u = 0; u < 8; u++) v[u] = *reinterpret_cast<const vec *>(acc + min(i0 + u, a.splits - 1) * HD);
    };
    ask(0);
    float m = -INFINITY, l = 0.f;
    if (lane < a.splits) {
        const float2 w = reinterpret_cast<const float2 *>(a.part_ml)[at * a.splits + lane];
        m = w.x;
        l = w.y;
    }
    float M = m;
#pragma unroll
    for (int off = kFewPieces / 2; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor(M, off, 64));
    // a sum of 0 takes part in nothing (its sums are 0); a bound of -inf with a sum is a row of not-a-numbers
    const float f = l == 0.f ? 0.f : m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - M);
    vec num = (vec)(0.f);
    float den = l * f;
#pragma unroll
    for (int off = kFewPieces / 2; off > 0; off >>= 1) den += __shfl_xor(den, off, 64);
    den = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, den)));   // (of the first 16 lanes)
    for (int i0 = 0;; i0 += 8) {
#pragma unroll
        for (int u = 0; u < 8; u++) {
            const float fi = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), i0 + u));
            num += i0 + u < a.splits ? v[u] * fi : (vec)(0.f);
        }
        if (i0 + 8 >= a.splits) break;
        ask(i0 + 8);
    }
    const float inv = den == 0.f ? 0.f : 1.f / den;
    uint16_t *o = a.out + (int64_t)row * a.st.out_token + (int64_t)head * a.st.out_head + dim;
    if (kEach * lane < HD) {
        if (kEach == 1) *o = (uint16_t)T::pack(num[0] * inv, 0.f);
        else {
#pragma unroll
            for (int u = 0; u + 1 < kEach; u += 2) *reinterpret_cast<uint32_t *>(o + u) = T::pack(num[u] * inv, num[(u + 1) % kEach] * inv);
        }
    }
    if (a.lse && lane == 0) a.lse[at] = den == 0.f ? -INFINITY : (M + log2f(den * T::kWeightInverse)) * 0.693147180559945f;
}

template <int HD, int G>
static constexpr size_t prompt_lds() { return (size_t)2 * 2 * G * kWaveKeys<HD, G> * HD * 2; }
template <int HD>
static constexpr size_t narrow_lds() { return (size_t)4 * 2 * kNarrowKeys<HD> * HD * 2; }

template <int HD, class T>
static int prepare_prompt()
{
    int rc = (int)hipFuncSetAttribute(reinterpret_cast<const void *>(&attn_prompt_kernel<HD, T, 1, 1>), hipFuncAttributeMaxDynamicSharedMemorySize, prompt_lds<HD, 1>());
    if (rc) return rc;
    rc = (int)hipFuncSetAttribute(reinterpret_cast<const void *>(&attn_prompt_kernel<HD, T, 2, 1>), hipFuncAttributeMaxDynamicSharedMemorySize, prompt_lds<HD, 2>());
    if (rc) return rc;
    rc = (int)hipFuncSetAttribute(reinterpret_cast<const void *>(&attn_prompt_kernel<HD, T, 2, 2>), hipFuncAttributeMaxDynamicSharedMemorySize, prompt_lds<HD, 2>());
    if (rc) return rc;
    return (int)hipFuncSetAttribute(reinterpret_cast<const void *>(&attn_prompt_narrow_kernel<HD, T>), hipFuncAttributeMaxDynamicSharedMemorySize, narrow_lds<HD>());
}

int prepare_attn_prompt()
{
    int rc;
    if ((rc = prepare_prompt<64, TypeF16>())) return rc;
    if ((rc = prepare_prompt<64, TypeBf16>())) return rc;
    if ((rc = prepare_prompt<128, TypeF16>())) return rc;
    if ((rc = prepare_prompt<128, TypeBf16>())) return rc;
    if ((rc = prepare_prompt<256, TypeF16>())) return rc;
    return prepare_prompt<256, TypeBf16>();
}

struct PromptPlan {
    int rows;                              // query rows of a workgroup: 128 or 64 (the wide kernel), 32 (the narrow one)
    int tiles, splits;
    int terms;                             // of a weight in the second product
};

// sequences cut into tiles: at most so many (whatever the sequences' lengths are)
static int64_t prompt_tiles(int64_t seqs, int64_t total_q, int64_t rows) { return (total_q + seqs * (rows - 1)) / rows; }

// Which form and how many pieces of the keys: the cheapest by an estimate (us) that fits the measurements below.  A workgroup takes
// `alone` a step of 64 keys by itself; w workgroups a compute unit take `busy` a step and workgroup (the walks of a causal prompt are
// half as long on average, those of a chunk behind a long context all alike: `even`), the first round of them (`places` run on a unit
// at once) costs `start`, the others half of it where the steps of another place hide them.  Pieces (of 512 keys and more) shorten the walk, but their sums go to memory and back and a second launch joins them.
// Measured 128 / 64 / 32 rows a workgroup, us: hd 128: 1024 rows of 32 heads 25.8 / 21.6 / 42, 2048 rows 52.2 / 55.9 / 117, 8192 rows of
// 32 / 8 520 / 609 / 1153, 2300 rows of 8 heads 44 / 34 / 43, of 2 heads 43 / 31 / 24; hd 64: 2000 rows of 16 heads 30 / 22 / 28, 2400
// of 4 33 / 23 / 18, 8192 of 16 177 / 188 / 287; hd 256: 2000 rows of 16 heads 105 / 88 / 113, 3000 143 / 175 / 195, 700 of 8 40 / 31 / 23.  Behind 8000
// keys, 32 / 8 heads x 128, 1 / 2 / 4 / 8 pieces: 150 rows in 64s 95 / 60 / 46 / 46, 512 rows 103 / 96 / 100 / 116, 8 rows in 32s
// 64 / 40 / 26 / 20.
// Two terms a weight (the output's own rounding is then what is left, 1.00 times it, with one term 1.2 to 1.33) in the 32-row form, and in the
// 64-row form where at most half of the compute units have a workgroup: the matrix unit idles there.  One / two, us: 37 rows of 32 heads x 128
// 7.1 / 7.2, 130 of 32 / 8 8.1 / 8.4; with more it is the time of the products: 512 rows of 32 heads 12.7 / 14.0, 200 behind 4000 38 / 44,
// packed 1 .. 2049 rows of 16 heads x 64 29 / 36, and in the 128-row form 2048 rows of 32 heads 51 / 65, 8192 of 32 / 8 508 / 688.
static PromptPlan prompt_plan(int64_t seqs, int64_t total_q, int64_t total_k, int64_t heads, int64_t hd, int64_t max_k, int cus)
{
    struct Form { int rows, places; double start, alone, busy; };
    static const Form forms[3][3] = {{{kWideRows, 3, 6, 0.73, 0.56}, {kWideRows / 2, 4, 5.5, 0.47, 0.32}, {kNarrowRows, 2, 6, 0.34, 0.25}},
                                     {{kWideRows, 2, 6, 1.10, 0.92}, {kWideRows / 2, 2, 6, 0.75, 0.60}, {kNarrowRows, 1, 8, 0.43, 0.43}},
                                     {{kWideRows, 1, 6, 2.90, 2.10}, {kWideRows / 2, 1, 7, 2.10, 1.75}, {kNarrowRows, 1, 14, 0.70, 0.90}}};
    static const int pieces[12] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64};
    // the longest walk: no longer than max_k, and where that is no more than all rows, likely not over twice the average sequence's
    const double longest = (double)(max_k < 2 * total_k / seqs ? max_k : 2 * total_k / seqs), s = (longest + 63) / 64;
    const double even = total_k > total_q ? 1 - 0.5 * (double)total_q / (double)total_k : 0.5;
    PromptPlan best = {kWideRows, 0, 1, 1};
    double least = 0;
    for (const Form &f : forms[hd <= 64 ? 0 : hd == 128 ? 1 : 2]) {
        const int64_t tiles = prompt_tiles(seqs, total_q, f.rows);
        for (const int n : pieces) {
            // (128 rows a workgroup: whole walks; 64: what the join of few pieces takes)
            if (n > 1 && (f.rows == kWideRows || s < 8 * n || (f.rows != kNarrowRows && n > kFewPieces))) break;
            const double w = (double)tiles * heads * n / cus, rounds = w <= f.places ? 1 : f.places == 1 ? w : 0.5 + 0.5 * w / f.places;
            const double busy = f.busy * (even * w + 1 - even);
            double us = f.start * rounds + s / n * (busy > f.alone ? busy : f.alone);
            if (n > 1) us += 3.5 + (double)total_q * heads * n * hd * (8 / 4.5e6);
            if (best.tiles && us >= least) continue;
            best = {f.rows, (int)tiles, n, f.rows == kNarrowRows || (f.rows < kWideRows && 2 * tiles * heads * n <= cus) ? 2 : 1};
            least = us;
        }
    }
    return best;
}

// More sequences than this are looked up in a table that a launch in front works out: a workgroup's walk over all of them grows with their
// square.  Walk / table, us: 128 sequences of 5 rows, 32 / 8 heads x 128: 46 / 45; 200 of 30, 8 heads x 64: 14.2 / 14.7; 256 of 30, 32 / 8
// heads x 128: 114 / 93; 4096 of 30, 8 heads x 64: 1082 / 223.
constexpr int64_t kTableSeqs = 128;

// The workspace: the pieces' sums and bounds, then the table.
struct PromptRoom {
    int64_t sums, bounds, table;           // bytes, multiples of 16
};
static PromptRoom prompt_room(const PromptPlan &plan, int64_t seqs, int64_t total_q, int64_t heads, int64_t hd)
{
    const int64_t parts = plan.splits > 1 ? plan.splits * total_q * heads : 0;
    return {parts * hd * 4, (parts * 8 + 15) / 16 * 16, seqs > kTableSeqs ? (seqs * 4 + 15) / 16 * 16 : 0};
}

static int prompt_sizes(int64_t seqs, int64_t total_q, int64_t total_k, int64_t heads, int64_t kv_heads, int64_t hd)
{
    if (seqs < 1 || total_q < 1 || total_k < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0) return RPTC_ESHAPE;
    if (hd != 32 && hd != 64 && hd != 128 && hd != 256) return RPTC_ESHAPE;
    if (heads > 1024 || seqs > (1 << 20) || total_q > (1 << 24) || total_k >= ((int64_t)1 << 31) - 1024) return RPTC_ELIMIT;
    if (prompt_tiles(seqs, total_q, kNarrowRows) * heads >= (int64_t)1 << 23) return RPTC_ELIMIT;      // workgroups of one launch
    return 0;
}

template <int HD, class T>
static void launch_prompt(const PromptArgs &a, const PromptPlan &plan, hipStream_t s)
{
    if (a.first_tile) hipLaunchKernelGGL(attn_prompt_table_kernel, dim3(1), dim3(kTableThreads), 0, s, a);
    const dim3 grid((unsigned)(a.heads * a.tiles * a.splits));
    const dim3 block(kPromptThreads);
    if (plan.rows == kWideRows) hipLaunchKernelGGL((attn_prompt_kernel<HD, T, 1, 1>), grid, block, (prompt_lds<HD, 1>()), s, a);
    else if (plan.rows == kNarrowRows) hipLaunchKernelGGL((attn_prompt_narrow_kernel<HD, T>), grid, block, narrow_lds<HD>(), s, a);
    else if (plan.terms == 2) hipLaunchKernelGGL((attn_prompt_kernel<HD, T, 2, 2>), grid, block, (prompt_lds<HD, 2>()), s, a);
    else hipLaunchKernelGGL((attn_prompt_kernel<HD, T, 2, 1>), grid, block, (prompt_lds<HD, 2>()), s, a);
    if (a.splits == 1) return;
    const unsigned tile_rows = (unsigned)a.tiles << a.row_bits;
    if (a.splits <= kFewPieces) hipLaunchKernelGGL((attn_prompt_merge_few_kernel<HD, T>), dim3(tile_rows, (unsigned)(a.heads + 3) / 4), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((attn_prompt_merge_kernel<HD, T>), dim3(tile_rows, (unsigned)a.heads), dim3(kJoinThreads), 0, s, a);
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
    const PromptPlan plan = prompt_plan(seqs, total_q, total_k, heads, hd, max_k < total_k ? max_k : total_k, dev->cus);
    const PromptRoom room = prompt_room(plan, seqs, total_q, heads, hd);
    return room.sums + room.bounds + room.table;
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
        if (st[i] < 0 || (i >= 6 && st[i] == 0)) return RPTC_ESHAPE;     // (what is read may repeat)
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
    const PromptPlan plan = prompt_plan(seqs, total_q, total_k, heads, hd, max_k < total_k ? max_k : total_k, dev->cus);
    a.tiles = plan.tiles;
    a.splits = plan.splits;
    a.causal = causal ? 1 : 0;
    a.c = scale * 1.44269504088896f;
    a.row_bits = __builtin_ctz((unsigned)plan.rows);
    a.part_acc = a.part_ml = nullptr;
    a.first_tile = nullptr;
    const PromptRoom room = prompt_room(plan, seqs, total_q, heads, hd);
    if (const int64_t need = room.sums + room.bounds + room.table) {
        if (!workspace) return RPTC_ENULL;
        if (!aligned16(workspace)) return RPTC_EALIGN;
        if (workspace_bytes < need) return RPTC_ESHAPE;
        char *p = static_cast<char *>(workspace);
        if (room.sums) {
            a.part_acc = reinterpret_cast<float *>(p);
            a.part_ml = reinterpret_cast<float *>(p + room.sums);
        }
        if (room.table) a.first_tile = reinterpret_cast<int32_t *>(p + room.sums + room.bounds);
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    Timer timer;
    if ((rc = timer.begin(dev, s, ms))) return rc;
    const bool f16 = dtype == RPTC_F16;
    switch (hd) {
    case 32: f16 ? launch_prompt<32, TypeF16>(a, plan, s) : launch_prompt<32, TypeBf16>(a, plan, s); break;
    case 64: f16 ? launch_prompt<64, TypeF16>(a, plan, s) : launch_prompt<64, TypeBf16>(a, plan, s); break;
    case 128: f16 ? launch_prompt<128, TypeF16>(a, plan, s) : launch_prompt<128, TypeBf16>(a, plan, s); break;
    default: f16 ? launch_prompt<256, TypeF16>(a, plan, s) : launch_prompt<256, TypeBf16>(a, plan, s); break;
    }
    return timer.end();
}
