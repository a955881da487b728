// A key/value cache held in 4 bits: appending rows, reading them back, and the attention of one token per sequence over it.
// (No counterpart in the reference, which generates with transformers on dense weights and caches, quantize_hf.py:229-236.)
//
// A row is one position of one head, hd fp16 values in groups of 32:
//   m = min x,  s = fp16((max x - min x) / 15), or the number below it where fp16(15 s + m) would be infinite,
//   code = clamp(rint((x - m) / s), 0, 15) (0 where s = 0),  the value a code stands for = fp16(code * s + m), one rounding
// (the quotients in fp32, correctly rounded; a group that holds a value which is no finite number reads as not-a-number).
// hd / 2 bytes of codes, then s and m of every group: hd / 2 + hd / 8 bytes, 80 against 256 at hd = 128.  Word w of a row
// holds the values 8w .. 8w+7, nibble t the value 8w + 2t and nibble t + 4 the value 8w + 2t + 1: one mask of a word gives a
// pair of neighbours in the two halves of a register.
#include "join.hpp"
#include "lds_load.hpp"

namespace rptc {

constexpr int kKv4Group = 32;
constexpr int kKv4Tile = 32;                // positions a wave takes at a time
typedef float float2v_t __attribute__((ext_vector_type(2)));
typedef float float4v_t __attribute__((ext_vector_type(4)));
typedef _Float16 half8v_t __attribute__((ext_vector_type(8)));

constexpr int kv4_row_bytes(int hd) { return hd / 2 + hd / kKv4Group * 4; }

__device__ __forceinline__ half2_t as_half2(uint32_t w) { return __builtin_bit_cast(half2_t, w); }
__device__ __forceinline__ uint32_t low_halves(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ uint32_t high_halves(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// A byte 0000cccc read as an fp8 number (e4m3) is c / 512, denormal or not, so the conversion of two fp8 numbers with the scale
// 512 gives two codes as fp16, exactly, in one instruction (against three: into a power's mantissa by mask and or, the
// power taken off).
template <bool HIGH>
__device__ __forceinline__ half2_t byte_codes(uint32_t w)
{
    return __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 512.f, HIGH));
}

// The eight values of a word, in the order of its bytes' nibbles: 0, 4, 1, 5, 2, 6, 3, 7 (kWordOrder).
__device__ __forceinline__ void word_values(uint32_t w, uint32_t par, half2_t (&r)[4])
{
    const half2_t s = as_half2(low_halves(par, par)), m = as_half2(high_halves(par, par));
    const uint32_t even = w & 0x0F0F0F0Fu, odd = (w >> 4) & 0x0F0F0F0Fu;
    r[0] = __builtin_elementwise_fma(byte_codes<false>(even), s, m);
    r[1] = __builtin_elementwise_fma(byte_codes<true>(even), s, m);
    r[2] = __builtin_elementwise_fma(byte_codes<false>(odd), s, m);
    r[3] = __builtin_elementwise_fma(byte_codes<true>(odd), s, m);
}
__device__ __forceinline__ half8v_t as_half8(const half2_t (&r)[4])
{
    const half8v_t v = {r[0].x, r[0].y, r[1].x, r[1].y, r[2].x, r[2].y, r[3].x, r[3].y};
    return v;
}

// The codes of a lane's eight values and its group's parameters (four consecutive lanes hold a group).
__device__ __forceinline__ void quantize_word(const float (&x)[8], uint32_t &code, uint32_t &par)
{
    float lo = x[0], hi = x[0], odd = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
        odd = fmaf(x[i], 0.f, odd);            // 0, or not a number
    }
#define RPTC_QUAD(v, ctrl) __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0u, __builtin_bit_cast(uint32_t, v), ctrl, 0xF, 0xF, true))
    lo = fminf(lo, RPTC_QUAD(lo, 0xB1));       // quad_perm [1, 0, 3, 2]
    hi = fmaxf(hi, RPTC_QUAD(hi, 0xB1));
    odd += RPTC_QUAD(odd, 0xB1);
    lo = fminf(lo, RPTC_QUAD(lo, 0x4E));       // quad_perm [2, 3, 0, 1]
    hi = fmaxf(hi, RPTC_QUAD(hi, 0x4E));
    odd += RPTC_QUAD(odd, 0x4E);
#undef RPTC_QUAD
    code = 0;
    if (odd != 0.f) {
        par = 0x7E007E00u;
        return;
    }
    uint16_t sb = float_to_half_bits((hi - lo) / 15.f);
    const uint16_t mb = float_to_half_bits(lo);
    // the scale's rounding may take the largest code past 65504: the scale below it does not
    const _Float16 top = __builtin_elementwise_fma((_Float16)15.f, __builtin_bit_cast(_Float16, sb), __builtin_bit_cast(_Float16, mb));
    if (__builtin_bit_cast(uint16_t, top) == 0x7C00u) sb--;
    const float s = half_bits_to_float(sb);
    par = (uint32_t)mb << 16 | sb;
    if (s == 0.f) return;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float q = fminf(fmaxf(rintf((x[i] - lo) / s), 0.f), 15.f);
        code |= (uint32_t)q << (4 * (i / 2) + 16 * (i % 2));
    }
}

// ---------------------------------------------------------------- append and read

struct Kv4AppendArgs {
    const uint16_t *k, *v;
    uint8_t *k_cache, *v_cache;
    const int64_t *pos;
    const int32_t *q_start;                // may be null: rows_each rows a sequence
    int64_t k_token, k_head, v_token, v_head, max_len;
    int seqs, total, rows_each, kv_heads;
};

// A lane takes eight values of a row; the rows of consecutive tokens of a head are consecutive in the cache, so a wave
// writes a run of memory.  512 rows of 32 heads x 128: 6.8 us for 11 MB, a launch (2.6) and one round of loads and stores, all of
// them in flight at once; the quotients are not what it waits for (by a reciprocal, with the near ones divided: 7.0 us).
template <int HD>
__global__ __launch_bounds__(256) void kv4_append_kernel(const Kv4AppendArgs a)
{
    constexpr int kWords = HD / 8;
    const int word = threadIdx.x % kWords, token = blockIdx.x * (256 / kWords) + threadIdx.x / kWords;
    if (token >= a.total) return;          // (whole rows: the lanes of a group stay together)
    const bool is_v = blockIdx.y >= a.kv_heads;
    const int head = blockIdx.y - (is_v ? a.kv_heads : 0);
    int seq, start;
    if (a.q_start) {
        // the last sequence that starts at or in front of the token
        int lo = 0, hi = a.seqs;           // q_start[lo] <= token < q_start[hi] where the starts rise
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.q_start[mid] <= token) lo = mid;
            else hi = mid;
        }
        seq = lo;
        start = a.q_start[seq];
        if (token < start || token >= a.q_start[seq + 1]) return;
    } else {
        seq = token / a.rows_each;
        start = seq * a.rows_each;
    }
    const int64_t first = a.pos[seq];
    // a sequence that begins outside the cache is not written, nor what lies past its end
    if (first < 0 || first >= a.max_len) return;
    const int64_t p = first + ((int64_t)token - start);
    if (p >= a.max_len) return;
    const uint16_t *src = is_v ? a.v + (int64_t)token * a.v_token + (int64_t)head * a.v_head
                               : a.k + (int64_t)token * a.k_token + (int64_t)head * a.k_head;
    const uint4 raw = *reinterpret_cast<const uint4 *>(src + 8 * word);
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[2 * i] = half_bits_to_float((uint16_t)(w[i] & 0xFFFFu));
        x[2 * i + 1] = half_bits_to_float((uint16_t)(w[i] >> 16));
    }
    uint32_t code, par;
    quantize_word(x, code, par);
    uint8_t *row = (is_v ? a.v_cache : a.k_cache) + (((int64_t)seq * a.kv_heads + head) * a.max_len + p) * kv4_row_bytes(HD);
    *reinterpret_cast<uint32_t *>(row + 4 * word) = code;
    if (word % 4 == 0) *reinterpret_cast<uint32_t *>(row + HD / 2 + word) = par;
}

struct Kv4ReadArgs {
    const uint8_t *k_cache, *v_cache;
    uint16_t *k, *v;
    int64_t k_token, k_head, v_token, v_head, max_len;
    int rows, kv_heads;
};

// A lane gives eight values of a row: 923 rows of 32 heads x 128 in 5.4 us, 3.7 TB/s with the launch.
template <int HD>
__global__ __launch_bounds__(256) void kv4_read_kernel(const Kv4ReadArgs a)
{
    constexpr int kWords = HD / 8;
    const int word = threadIdx.x % kWords, p = blockIdx.x * (256 / kWords) + threadIdx.x / kWords;
    if (p >= a.rows) return;
    const bool is_v = blockIdx.y >= a.kv_heads;
    const int head = blockIdx.y - (is_v ? a.kv_heads : 0), seq = blockIdx.z;
    const uint8_t *row = (is_v ? a.v_cache : a.k_cache) + (((int64_t)seq * a.kv_heads + head) * a.max_len + p) * kv4_row_bytes(HD);
    const uint32_t code = *reinterpret_cast<const uint32_t *>(row + 4 * word);
    const uint32_t par = *reinterpret_cast<const uint32_t *>(row + HD / 2 + word / 4 * 4);
    const int64_t token = (int64_t)seq * a.rows + p;
    uint16_t *out = is_v ? a.v + token * a.v_token + (int64_t)head * a.v_head : a.k + token * a.k_token + (int64_t)head * a.k_head;
    half2_t r[4];
    word_values(code, par, r);
    // from the order 0, 4, 1, 5, 2, 6, 3, 7 to the natural one
    const half2_t v[4] = {{r[0].x, r[1].x}, {r[2].x, r[3].x}, {r[0].y, r[1].y}, {r[2].y, r[3].y}};
    *reinterpret_cast<half8v_t *>(out + 8 * word) = as_half8(v);
}

// One token of a decode step: rotates the (2i, 2i+1) pairs of q and k by the angle of the token's position (the fp16
// arithmetic of rptc_rope_cache), writes q_out and appends k and v.  qkv rows are [q | k | v].
__global__ __launch_bounds__(256) void kv4_rope_append_kernel(const uint16_t *__restrict__ qkv, const uint16_t *__restrict__ cos_t,
                                                              const uint16_t *__restrict__ sin_t, const int64_t *__restrict__ pos,
                                                              uint16_t *__restrict__ q_out, uint8_t *__restrict__ k_cache,
                                                              uint8_t *__restrict__ v_cache, int heads, int kv_heads, int hd,
                                                              int64_t max_len, int items)
{
#pragma clang fp contract(off)
    const int id = blockIdx.x * 256 + threadIdx.x, words = hd >> 3;
    if (id >= items) return;
    const int seq = blockIdx.y, word = id % words, h = id / words;      // h: heads of q, then of k, then of v
    const int64_t p = pos[seq];
    if (p < 0 || p >= max_len) return;
    const uint16_t *src = qkv + (int64_t)seq * (heads + 2 * kv_heads) * hd + (int64_t)h * hd + 8 * word;
    const uint4 raw = *reinterpret_cast<const uint4 *>(src);
    uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    if (h < heads + kv_heads) {
        const uint2 cr = *reinterpret_cast<const uint2 *>(cos_t + p * (hd >> 1) + 4 * word);
        const uint2 sr = *reinterpret_cast<const uint2 *>(sin_t + p * (hd >> 1) + 4 * word);
        const uint32_t cw[2] = {cr.x, cr.y}, sw[2] = {sr.x, sr.y};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const half2_t ab = as_half2(w[i]);
            const _Float16 c = as_half2(cw[i / 2])[i % 2], s = as_half2(sw[i / 2])[i % 2];
            const _Float16 ac = ab.x * c, bs = ab.y * s, as = ab.x * s, bc = ab.y * c;
            const half2_t r = {(_Float16)(ac - bs), (_Float16)(as + bc)};
            w[i] = __builtin_bit_cast(uint32_t, r);
        }
    }
    if (h < heads) {
        *reinterpret_cast<uint4 *>(q_out + ((int64_t)seq * heads + h) * hd + 8 * word) = make_uint4(w[0], w[1], w[2], w[3]);
        return;
    }
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[2 * i] = half_bits_to_float((uint16_t)(w[i] & 0xFFFFu));
        x[2 * i + 1] = half_bits_to_float((uint16_t)(w[i] >> 16));
    }
    uint32_t code, par;
    quantize_word(x, code, par);
    const bool is_v = h >= heads + kv_heads;
    const int kh = h - heads - (is_v ? kv_heads : 0);
    uint8_t *row = (is_v ? v_cache : k_cache) + (((int64_t)seq * kv_heads + kh) * max_len + p) * kv4_row_bytes(hd);
    *reinterpret_cast<uint32_t *>(row + 4 * word) = code;
    if (word % 4 == 0) *reinterpret_cast<uint32_t *>(row + hd / 2 + word) = par;
}

// ---------------------------------------------------------------- attention of one token per sequence
//
//   out[h] = sum_j p_j v_j / sum_j p_j,  p_j = exp2(c q[h].k_j - m), over positions 0..pos, in one pass (m a running bound
//   that is raised only where a score exceeds it by more than 2^8).
// A wave takes 32 positions of one key head at a time, for up to 16 query heads of its group, and needs nothing from
// another lane but the maxima: S^T = K q^T with 16x16x32 matrix instructions, the lane holding one quarter of a row's
// words as the row operand; its result has, in a lane, scores of one head for four positions of each of two tiles, which is,
// with the positions renumbered accordingly, the operand P of O^T = V^T P^T; V^T's operand wants eight positions of one
// dimension in a lane, so the lane reads one word (eight dimensions) of its eight rows and pairs the positions up with byte
// permutes.  Values are formed in fp16, as stored; p enters the product rounded to fp16, and what that left enters as well:
// through the free columns with at most eight heads, by a second product with more (one term alone: error 1.32 to 1.39 times that of the
// output's own rounding instead of 1.00, for
// 0 to 6 % of the time: 32 sequences of 3000, 32 / 2 heads x 128, 19.9 us, 8 of 2000, 48 / 4 x 256, 30.1 -> 31.6).
// The 32 rows are a run of memory, and come straight into LDS, two stages a wave in flight (10 KB of them at hd 128, up to
// 160 KB a compute unit); the row length in words (20 at hd 128) puts the lanes of every LDS read on different banks.
// The matrix unit is mostly idle (15 of 16 columns with one query head a key head); what counts is the vector unit's work of
// unpacking, about three instructions a pair of values, and memory: one sequence of 131007, 32 / 8 heads x 128, 35.5 us for 168 MB,
// 4.7 TB/s; 64 of 4000 66 us, 5.0.  A short sequence is a chain: of 601 positions, 32 heads, 6.1 us behind the launch, 1.4 until the
// first rows are there, 2.6 for three tiles a wave, 1.4 for the join, 0.7 for the store (asking for the first tiles before the
// position is known and a join with two barriers less: no change).
struct Kv4AttnArgs {
    const uint16_t *q;
    const uint8_t *k_cache, *v_cache;
    const int64_t *pos;
    uint16_t *out;
    float *part;                            // pieces: [head][slot][hd] sums, then [head][slot][2] bound and sum of p
    int64_t q_token, max_len, part_ml;      // part_ml: where the second part begins
    int seqs, heads, kv_heads, group, head_blocks;
    int slots;                              // workgroups a key head (block): every sequence takes one a piece
    int want, least;                        // the pieces of all sequences together that fill the chip; tiles of the shortest
    float c;                                // scale * log2(e)
};

// How the sequences' positions are cut into pieces, a workgroup each (and key head): pieces of one length, whatever the
// sequences' own, so that the workgroups of a batch of unequal sequences end together and few are without a piece (one
// of those holds its place for about 2 us).  The positions come from device memory: every wave works the cut out for
// itself, a lane a sequence, 64 at a time.  Lengths in tiles of 32 positions (at most 1024 sequences of 2^21).
struct Kv4Piece {
    int seq, len, pieces, piece, slot0;     // the sequence, its positions and pieces, which of them, the slot of its first
};
__device__ __forceinline__ int kv4_length(const Kv4AttnArgs &a, int s)
{
    const int64_t p = s < a.seqs ? a.pos[s] : -1;
    return p >= 0 && p < a.max_len ? (int)p + 1 : 0;       // a position outside the cache: no piece, nothing is read or written
}
// sums over lanes 0 .. own, by DPP (see wave_sum)
__device__ __forceinline__ uint32_t scan64(uint32_t v)
{
#define RPTC_DPP_ADD(ctrl, row_mask) v += __builtin_amdgcn_update_dpp(0u, v, ctrl, row_mask, 0xF, false)
    RPTC_DPP_ADD(0x111, 0xF);
    RPTC_DPP_ADD(0x112, 0xF);
    RPTC_DPP_ADD(0x114, 0xF);
    RPTC_DPP_ADD(0x118, 0xF);
    RPTC_DPP_ADD(0x142, 0xA);
    RPTC_DPP_ADD(0x143, 0xC);
#undef RPTC_DPP_ADD
    return v;
}

// The piece of slot `slot`, or (by_seq) the first piece of sequence `slot`.  False: there is none.
__device__ __forceinline__ bool kv4_find(const Kv4AttnArgs &a, int slot, bool by_seq, Kv4Piece &r)
{
    r.piece = 0;
    if (a.want == 1) {                                     // nothing is cut
        r.seq = r.slot0 = slot;
        r.len = uniform(kv4_length(a, slot));
        r.pieces = 1;
        return r.len > 0;
    }
    const int lane = threadIdx.x & 63;
    uint32_t total = 0;
    int len = 0;
    for (int s0 = 0; s0 < a.seqs; s0 += 64) {
        len = kv4_length(a, s0 + lane);
        total += (uint32_t)(len + kKv4Tile - 1) / kKv4Tile;
    }
    total = (uint32_t)__builtin_amdgcn_readlane((int)scan64(total), 63);
    uint32_t size = max((uint32_t)a.least, (total + (uint32_t)a.want - 1) / (uint32_t)a.want);      // so at most seqs + want - 1 pieces
    if (a.seqs > 1 && a.seqs <= 64) {
        // where the sequences' last pieces make it more than wanted, some compute units would have two: longer ones, until they
        // do not (measured without / with: 12 sequences of 1 .. 8191, 8 key heads x 128, 26.7 / 23.6 us; 12 of 3191 26.9 / 23.2;
        // 3 of 30000 44.6 / 32.9)
        const uint32_t want = (uint32_t)a.want;
        for (int u = 0; u < 4; u++) {
            const uint32_t count = (uint32_t)__builtin_amdgcn_readlane((int)scan64(((uint32_t)(len + kKv4Tile - 1) / kKv4Tile + size - 1) / size), 63);
            if (count <= want || size >= total / 2) break;
            // size count / want, rounded up: in 32 bits, as size < 2^26 and count <= want + 63
            size = min(total, size / want * count + (size % want * count + want - 1) / want);
        }
    }
    uint32_t in_front = 0;
    r.seq = -1;
    r.len = r.pieces = r.slot0 = 0;
    for (int s0 = 0; s0 < a.seqs; s0 += 64) {
        if (a.seqs > 64) len = kv4_length(a, s0 + lane);
        const uint32_t n = ((uint32_t)(len + kKv4Tile - 1) / kKv4Tile + size - 1) / size;      // at most a.want of one sequence
        const uint32_t incl = scan64(n);
        const uint64_t hit = __ballot(by_seq ? s0 + lane == slot : in_front + incl > (uint32_t)slot);
        if (hit) {
            const int f = __builtin_ctzll(hit);
            r.seq = s0 + f;
            r.len = __builtin_amdgcn_readlane(len, f);
            r.pieces = __builtin_amdgcn_readlane((int)n, f);
            r.slot0 = (int)in_front + __builtin_amdgcn_readlane((int)incl, f) - r.pieces;
            break;
        }
        in_front += (uint32_t)__builtin_amdgcn_readlane((int)incl, 63);
    }
    r.seq = uniform(r.seq);
    r.len = uniform(r.len);
    r.pieces = uniform(r.pieces);
    r.slot0 = uniform(r.slot0);
    r.piece = by_seq ? 0 : slot - r.slot0;
    return r.seq >= 0 && r.pieces > 0;
}

__device__ __forceinline__ float rows_max(float x)
{
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    const float y = fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
    const uint32_t d = __builtin_bit_cast(uint32_t, y);
    const auto s = __builtin_amdgcn_permlane32_swap(d, d, false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)s[0]), __builtin_bit_cast(float, (uint32_t)s[1]));
}
__device__ __forceinline__ float rows_sum(float x)
{
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    const float y = __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
    const uint32_t d = __builtin_bit_cast(uint32_t, y);
    const auto s = __builtin_amdgcn_permlane32_swap(d, d, false, false);
    return __builtin_bit_cast(float, (uint32_t)s[0]) + __builtin_bit_cast(float, (uint32_t)s[1]);
}

constexpr int kKv4Stages = 2;               // of them on their way or in LDS
constexpr float kKv4Lazy = 8.f;
// weights carry a factor 2^7, which the quotient takes off again: one far below the largest is held to 2^-31 of it instead of 2^-24 (many such
// ones behind one that outweighs them would otherwise be lost), and the largest, 2^15, stays below 65504
constexpr float kKv4WeightLog2 = 7.f;
template <int HD>
constexpr int kKv4Waves = HD > 128 ? 4 : 8;
template <int HD>
constexpr int kKv4Stage = kKv4Tile * kv4_row_bytes(HD);     // bytes of K, and of V, of a stage: 640, 1280, 2560, 5120
template <int HD>
constexpr int kv4_lds(int live)
{
    // the stages, later the waves' sums [wave][column][HD + 4] and [wave][16][2]
    const int columns = live <= 8 ? 2 * live : live;
    const int ring = kKv4Waves<HD> * kKv4Stages * 2 * kKv4Stage<HD>, sums = (kKv4Waves<HD> * columns * (HD + 4) + kKv4Waves<HD> * 32) * 4;
    return ring > sums ? ring : sums;
}

template <int HD>
__global__ __launch_bounds__(64 * kKv4Waves<HD>, HD > 128 ? 2 : 4) void kv4_attn_kernel(const Kv4AttnArgs a)
{
    extern __shared__ __align__(16) uint8_t lds4[];
    constexpr int kRow = kv4_row_bytes(HD), kStage = kKv4Stage<HD>, kWaves = kKv4Waves<HD>;
    constexpr int kRequests = (kStage + 1023) / 1024, kLastLanes = (kStage % 1024) / 16;      // of a wave's 1024 bytes; lanes of a part of one
    constexpr int kW = HD / 32;                            // words of a row a lane holds of K
    constexpr int kE = HD / 16;                            // dimensions of a row a lane holds of V
    constexpr int kVW = HD >= 128 ? HD / 128 : 1;          // words of that
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int n = lane & 15, c = lane >> 4;
    // the heads of a piece together, the slots without a piece at the end: workgroups with one fall on different compute units
    const int groups = a.kv_heads * a.head_blocks, slot = blockIdx.x / groups, group = blockIdx.x - slot * groups;
    const int kvh = group / a.head_blocks, hb = group - kvh * a.head_blocks;
    const int live = min(16, a.group - 16 * hb);           // query heads of this workgroup
    const int head0 = kvh * a.group + 16 * hb;
    Kv4Piece r;
    if (!kv4_find(a, slot, false, r)) return;
    const int per = ((r.len + r.pieces - 1) / r.pieces + kKv4Tile - 1) / kKv4Tile * kKv4Tile;
    const int lo = (int)min((int64_t)r.len, (int64_t)r.piece * per), hi = min(r.len, lo + per);
    const int64_t head_base = ((int64_t)r.seq * a.kv_heads + kvh) * a.max_len;
    const uint8_t *k_base = a.k_cache + head_base * kRow, *v_base = a.v_cache + head_base * kRow;

    // this wave's tiles: from lo + 32 wave on, every kWaves-th; rows past the piece's end come as zeros
    const int first = lo + wave * kKv4Tile, tiles = uniform(first < hi ? (hi - first + kWaves * kKv4Tile - 1) / (kWaves * kKv4Tile) : 0);
    uint8_t *ring = lds4 + wave * (kKv4Stages * 2 * kStage);
    const uint32_t ring_to = lds_address(ring);
    auto request = [&](int i) {
        const int j0 = first + i * kWaves * kKv4Tile, bytes = min(kKv4Tile, hi - j0) * kRow;
        const int4_t kr = buffer_resource(k_base + (int64_t)j0 * kRow, bytes), vr = buffer_resource(v_base + (int64_t)j0 * kRow, bytes);
        const uint32_t to = ring_to + (uint32_t)(i % kKv4Stages) * (2u * kStage);
#pragma unroll
        for (int u = 0; u < kStage / 1024; u++) load_to_lds(lane * 16u + u * 1024u, kr, to + u * 1024u);
#pragma unroll
        for (int u = 0; u < kStage / 1024; u++) load_to_lds(lane * 16u + u * 1024u, vr, to + kStage + u * 1024u);
        if (lane < kLastLanes) {
            load_to_lds(lane * 16u + kStage / 1024 * 1024u, kr, to + kStage / 1024 * 1024u);
            load_to_lds(lane * 16u + kStage / 1024 * 1024u, vr, to + kStage + kStage / 1024 * 1024u);
        }
    };
#pragma unroll
    for (int i = 0; i < kKv4Stages; i++)
        if (i < tiles) request(i);
    // Column n of the products is head n; with at most eight heads the columns from 8 on hold them once more, and take
    // what the rounding of p to fp16 leaves.
    const bool twice = live <= 8, second = twice && n >= 8;
    const int column = second ? n - 8 : n;
    half8v_t qf[kW];
#pragma unroll
    for (int w = 0; w < kW; w++) {
        half8v_t q = (half8v_t)((_Float16)0.f);
        if (column < live)
            q = *reinterpret_cast<const half8v_t *>(a.q + r.seq * a.q_token + (int64_t)(head0 + column) * HD + 8 * (c * kW + w));
        qf[w] = __builtin_shufflevector(q, q, 0, 4, 1, 5, 2, 6, 3, 7);     // as word_values orders a word
    }
    // the queries are there: a wait inside the loop would wait for rows on their way as well
#pragma unroll
    for (int w = 0; w < kW; w++) asm volatile("" : "+v"(qf[w]));

    // hd 64, 32: the lane's four or two dimensions are nibbles of two bytes of the word (hd 32: of one parity)
    const uint32_t v_bytes = 0x06020400u + 0x01010101u * (uint32_t)(HD == 64 ? n & 1 : n >> 1 & 1);
    const int v_shift = HD == 32 ? 4 * (n & 1) : 0;
    float4v_t acc[kE];
#pragma unroll
    for (int e = 0; e < kE; e++) acc[e] = (float4v_t)(0.f);
    float m = -INFINITY, l = 0.f;
    for (int i = 0; i < tiles; i++) {
        if (i + 1 < tiles) wait_for_lds_loads_but<(kKv4Stages - 1) * 2 * kRequests>();
        else wait_for_lds_loads();
        static_assert(kKv4Stages == 2, "the wait above");
        const uint8_t *ks = ring + (i % kKv4Stages) * 2 * kStage, *vs = ks + kStage;
        uint32_t kw[2][kW], kp[2][(kW + 3) / 4], vw[8][kVW], vp[8];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const uint8_t *r = ks + (16 * t + n) * kRow;
#pragma unroll
            for (int w = 0; w < kW; w++) kw[t][w] = *reinterpret_cast<const uint32_t *>(r + 4 * (c * kW + w));
#pragma unroll
            for (int g = 0; g < (kW + 3) / 4; g++) kp[t][g] = *reinterpret_cast<const uint32_t *>(r + HD / 2 + 4 * (c * kW / 4 + g));
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint8_t *r = vs + (16 * (j / 4) + 4 * c + j % 4) * kRow;
#pragma unroll
            for (int w = 0; w < kVW; w++) vw[j][w] = *reinterpret_cast<const uint32_t *>(r + 4 * (HD >= 128 ? n * kVW + w : n * kE / 8));
            vp[j] = *reinterpret_cast<const uint32_t *>(r + HD / 2 + 4 * (n * kE / 32));
        }
        wait_for_lds_reads();
        if (i + kKv4Stages < tiles) request(i + kKv4Stages);

        float4v_t s[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            s[t] = (float4v_t)(0.f);
#pragma unroll
            for (int w = 0; w < kW; w++) {
                half2_t v[4];
                word_values(kw[t][w], kp[t][w / 4], v);
                s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_half8(v), qf[w], s[t], 0, 0, 0);
            }
        }
        const int left = hi - (first + i * kWaves * kKv4Tile);
        if (left < kKv4Tile) {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (16 * (j / 4) + 4 * c + j % 4 >= left) s[j / 4][j % 4] = -INFINITY;
        }
        float mx = s[0][0];
#pragma unroll
        for (int j = 1; j < 8; j++) mx = fmaxf(mx, s[j / 4][j % 4]);
        mx = rows_max(mx) * a.c;
        if (__ballot(mx > m + kKv4Lazy)) {
            const float up = fmaxf(m, mx);
            const float f = up == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - up);
            l *= f;
#pragma unroll
            for (int e = 0; e < kE; e++) acc[e] *= f;
            m = up;
        }
        float mc = (m == -INFINITY ? 0.f : m) - kKv4WeightLog2, scale = a.c;
        // the bound is a rounded product, and what the rounding left a factor of all weights: within 2^(1/32) of 1 below 2^20, but up to 2^32
        // at 2^30.  From 2^20 on the scores are multiplied and rounded as the bound was, and their differences to it taken
        const uint32_t size = __builtin_bit_cast(uint32_t, m) & 0x7FFFFFFFu;
        const bool far = size - 0x49800000u < 0x7F800000u - 0x49800000u;      // 2^20 <= |m| < infinity
        if (__ballot(far)) {
#pragma clang fp contract(off)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float product = s[j / 4][j % 4] * scale;
                s[j / 4][j % 4] = far ? product - m : s[j / 4][j % 4];
            }
            scale = far ? 1.f : scale;
            mc = far ? -kKv4WeightLog2 : mc;
        }
        half2_t p2[4], rest[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int r = 2 * j;
            const float x = __builtin_amdgcn_exp2f(fmaf(s[r / 4][r % 4], scale, -mc)), y = __builtin_amdgcn_exp2f(fmaf(s[r / 4][r % 4 + 1], scale, -mc));
            l += x;
            l += y;
            const float2v_t xy = {x, y};
            p2[j] = __builtin_convertvector(xy, half2_t);
            const float2v_t left_over = {x - (float)p2[j].x, y - (float)p2[j].y};
            rest[j] = __builtin_convertvector(left_over, half2_t);
            p2[j] = second ? rest[j] : p2[j];
        }
        const half8v_t p = as_half8(p2);
        // V: the same byte of two positions' words side by side, then the nibbles of a dimension of both in one register
        half2_t val[kE][4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const half2_t sc = as_half2(low_halves(vp[2 * j], vp[2 * j + 1])), mn = as_half2(high_halves(vp[2 * j], vp[2 * j + 1]));
#pragma unroll
            for (int w = 0; w < kVW; w++) {
                const uint32_t x = vw[2 * j][w], y = vw[2 * j + 1][w];
                if (kE >= 8) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const uint32_t xy = __builtin_amdgcn_perm(y, x, h ? 0x07030602u : 0x05010400u);
                        const uint32_t even = xy & 0x0F0F0F0Fu, odd = (xy >> 4) & 0x0F0F0F0Fu;
                        val[8 * w + h][j] = __builtin_elementwise_fma(byte_codes<false>(even), sc, mn);
                        val[8 * w + 4 + h][j] = __builtin_elementwise_fma(byte_codes<true>(even), sc, mn);
                        val[8 * w + 2 + h][j] = __builtin_elementwise_fma(byte_codes<false>(odd), sc, mn);
                        val[8 * w + 6 + h][j] = __builtin_elementwise_fma(byte_codes<true>(odd), sc, mn);
                    }
                } else {
                    const uint32_t xy = __builtin_amdgcn_perm(y, x, v_bytes) >> v_shift;
                    const uint32_t even = xy & 0x0F0F0F0Fu;
                    val[0][j] = __builtin_elementwise_fma(byte_codes<false>(even), sc, mn);
                    val[1][j] = __builtin_elementwise_fma(byte_codes<true>(even), sc, mn);
                    if (kE > 2) {
                        const uint32_t odd = (xy >> 4) & 0x0F0F0F0Fu;
                        val[2 % kE][j] = __builtin_elementwise_fma(byte_codes<false>(odd), sc, mn);
                        val[3 % kE][j] = __builtin_elementwise_fma(byte_codes<true>(odd), sc, mn);
                    }
                }
            }
        }
#pragma unroll
        for (int e = 0; e < kE; e++) acc[e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_half8(val[e]), p, acc[e], 0, 0, 0);
        if (!twice) {                                      // no free columns: a second product
            const half8v_t left_over = as_half8(rest);
#pragma unroll
            for (int e = 0; e < kE; e++) acc[e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_half8(val[e]), left_over, acc[e], 0, 0, 0);
        }
    }

    // The waves join through LDS: lane (column n, quarter c) holds the dimensions 4 kE c .. 4 kE (c + 1) of its column, a run of
    // floats; a column has four floats of padding, so that the columns' runs begin on different banks.
    __syncthreads();                                       // nobody reads a stage any more
    constexpr int kColumn = HD + 4;
    float *sums = reinterpret_cast<float *>(lds4);
    const int columns = twice ? 2 * live : live, wave_sums = columns * kColumn;
    float *w_ml = sums + (size_t)kWaves * wave_sums;       // [wave][16][2]: bound and sum, later the wave's factor and the sum by it
    l = rows_sum(l);
    if (column < live) {
        float4 *to = reinterpret_cast<float4 *>(sums + (size_t)wave * wave_sums + (second ? live + column : n) * kColumn + 4 * kE * c);
#pragma unroll
        for (int i = 0; i < kE; i++)                       // float i * 4 + k of the run: dimension e = (4 i + k) % kE of row r = (4 i + k) / kE
            to[i] = make_float4(acc[(4 * i) % kE][(4 * i) / kE], acc[(4 * i + 1) % kE][(4 * i + 1) / kE], acc[(4 * i + 2) % kE][(4 * i + 2) / kE],
                                acc[(4 * i + 3) % kE][(4 * i + 3) / kE]);
        if (c == 0 && !second) {
            w_ml[2 * (wave * 16 + n)] = m;
            w_ml[2 * (wave * 16 + n) + 1] = l;
        }
    }
    __syncthreads();
    float M = -INFINITY, f = 0.f, lw = 0.f;                // thread (head, wave) of the first 16 kWaves
    if (tid < 16 * kWaves && tid / kWaves < live) {
        const int h = tid / kWaves, w = tid % kWaves;
        const float mw = w_ml[2 * (w * 16 + h)];
        lw = w_ml[2 * (w * 16 + h) + 1];
#pragma unroll
        for (int i = 0; i < kWaves; i++) M = fmaxf(M, w_ml[2 * (i * 16 + h)]);
        // a wave without a position has sum 0 (and accumulators 0); a bound of -inf with a sum is not-a-numbers
        f = lw == 0.f ? 0.f : mw == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mw - M);
    }
    __syncthreads();
    if (tid < 16 * kWaves && tid / kWaves < live) {
        const int h = tid / kWaves, w = tid % kWaves;
        w_ml[2 * (w * 16 + h)] = f;
        w_ml[2 * (w * 16 + h) + 1] = lw * f;
        if (r.pieces > 1 && w == 0) a.part[a.part_ml + 2 * ((int64_t)(head0 + h) * a.slots + slot)] = M;
    }
    __syncthreads();
    for (int i = tid; i < live * HD; i += 64 * kWaves) {
        const int h = i / HD, d = i % HD;
        float num = 0.f, den = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            float part = sums[(size_t)w * wave_sums + h * kColumn + d];
            if (twice) part += sums[(size_t)w * wave_sums + (live + h) * kColumn + d];
            num = fmaf(part, w_ml[2 * (w * 16 + h)], num);
            den += w_ml[2 * (w * 16 + h) + 1];
        }
        if (r.pieces == 1) {
            a.out[((int64_t)r.seq * a.heads + head0 + h) * HD + d] = float_to_half_bits(num / den);
        } else {
            const int64_t at = (int64_t)(head0 + h) * a.slots + slot;
            a.part[at * HD + d] = num;
            if (d == 0) a.part[a.part_ml + 2 * at + 1] = den;
        }
    }
}

// Joins the pieces of a head, a workgroup per (head, sequence).
template <int HD>
__global__ __launch_bounds__(kJoinThreads) void kv4_merge_kernel(const Kv4AttnArgs a)
{
    const int head = blockIdx.x, seq = blockIdx.y;
    Kv4Piece r;
    if (!kv4_find(a, seq, true, r) || r.pieces == 1) return;
    const int64_t at = (int64_t)head * a.slots + r.slot0;
    float M, den;
    const float num = join_pieces(a.part + at * HD, a.part + a.part_ml + 2 * at, r.pieces, HD, M, den);
    if (threadIdx.x < HD) a.out[((int64_t)seq * a.heads + head) * HD + threadIdx.x] = float_to_half_bits(num / den);
}

int prepare_kv4()
{
    int rc;
    if ((rc = (int)hipFuncSetAttribute(reinterpret_cast<const void *>(&kv4_attn_kernel<64>), hipFuncAttributeMaxDynamicSharedMemorySize, kv4_lds<64>(16)))) return rc;
    if ((rc = (int)hipFuncSetAttribute(reinterpret_cast<const void *>(&kv4_attn_kernel<128>), hipFuncAttributeMaxDynamicSharedMemorySize, kv4_lds<128>(16)))) return rc;
    return (int)hipFuncSetAttribute(reinterpret_cast<const void *>(&kv4_attn_kernel<256>), hipFuncAttributeMaxDynamicSharedMemorySize, kv4_lds<256>(16));
}

static int kv4_sizes(int64_t seqs, int64_t kv_heads, int64_t hd, int64_t max_len)
{
    if (seqs < 1 || kv_heads < 1 || max_len < 1) return RPTC_ESHAPE;
    if (hd != 32 && hd != 64 && hd != 128 && hd != 256) return RPTC_ESHAPE;
    if (seqs > 65535 || kv_heads > 1024 || max_len > (int64_t)1 << 26) return RPTC_ELIMIT;
    return 0;
}

struct Kv4Plan {
    int slots, want, least;
};

// groups: workgroups a piece has (key heads, times blocks of 16 query heads).  Cut into pieces, so that about one workgroup
// a compute unit runs, and joined by a second launch (4 us): caches of 2048 positions and more (a workgroup walks 1024 in
// 4 steps of its waves, 2 us) with fewer sequences and heads than compute units, and of 8192 and more up to four times as
// many, for what one long sequence among short ones would cost.  Pieces are no shorter than 512 positions.  Measured, uncut /
// cut, heads x 128: one sequence of 1024, 32 heads: 10.4 / 11.3 us; of 8192, 32 heads: 34 / 18; 32 of 2000, 8 heads x 64: 14.4 / 17.3.
// One key head would take a piece a compute unit, but joining more than 128 costs more than the shorter walks give: one sequence of 131072, one
// head x 128, 128 / 256 pieces: 19.3 / 22.9 us.
static Kv4Plan kv4_plan(int64_t seqs, int64_t groups, int64_t max_len, int cus)
{
    Kv4Plan p = {(int)seqs, 1, 512 / kKv4Tile};
    if (max_len < 2048 || seqs > 1024 || seqs * groups >= (max_len >= 8192 ? 4 : 1) * (int64_t)cus) return p;
    p.want = (int)((cus + groups - 1) / groups);
    if (p.want < 2) p.want = 2;
    if (p.want > kJoinMost) p.want = kJoinMost;
    p.slots = (int)seqs + p.want - 1;          // pieces of one length: fewer than want whole ones and one more a sequence
    return p;
}

}  // namespace rptc

using namespace rptc;

extern "C" int64_t rptc_kv4_row_bytes(int64_t hd) { return hd == 32 || hd == 64 || hd == 128 || hd == 256 ? kv4_row_bytes((int)hd) : RPTC_ESHAPE; }

extern "C" int rptc_kv4_append(const uint16_t *k, const uint16_t *v, uint8_t *k_cache, uint8_t *v_cache, const int64_t *pos,
                               const int32_t *q_start, int64_t seqs, int64_t total, int64_t kv_heads, int64_t hd, int64_t max_len,
                               int64_t k_token, int64_t k_head, int64_t v_token, int64_t v_head, void *stream, float *ms)
{
    if (!k || !v || !k_cache || !v_cache || !pos) return RPTC_ENULL;
    int rc = kv4_sizes(seqs, kv_heads, hd, max_len);
    if (rc) return rc;
    if (total < 1 || (!q_start && total % seqs != 0) || k_token < 0 || k_head < 0 || v_token < 0 || v_head < 0) return RPTC_ESHAPE;
    if (total > (1 << 24)) return RPTC_ELIMIT;
    if (!aligned16(k) || !aligned16(v) || !aligned16(k_cache) || !aligned16(v_cache)) return RPTC_EALIGN;
    if (k_token % 8 || k_head % 8 || v_token % 8 || v_head % 8) return RPTC_EALIGN;
    auto rows = [&](const void *c) { return c == k || c == v; };
    if (k_cache == v_cache || rows(k_cache) || rows(v_cache)) return RPTC_EALIAS;
    DeviceInfo *dev;
    if ((rc = device_info(&dev))) return rc;
    Kv4AppendArgs a;
    a.k = k;
    a.v = v;
    a.k_cache = k_cache;
    a.v_cache = v_cache;
    a.pos = pos;
    a.q_start = q_start;
    a.k_token = k_token;
    a.k_head = k_head;
    a.v_token = v_token;
    a.v_head = v_head;
    a.max_len = max_len;
    a.seqs = (int)seqs;
    a.total = (int)total;
    a.rows_each = (int)(total / seqs);
    a.kv_heads = (int)kv_heads;
    const int per = 256 / (int)(hd / 8);       // rows of a workgroup
    const dim3 grid((unsigned)((total + per - 1) / per), (unsigned)(2 * kv_heads));
    hipStream_t s = static_cast<hipStream_t>(stream);
    Timer timer;
    if ((rc = timer.begin(dev, s, ms))) return rc;
    switch (hd) {
    case 32: hipLaunchKernelGGL(kv4_append_kernel<32>, grid, dim3(256), 0, s, a); break;
    case 64: hipLaunchKernelGGL(kv4_append_kernel<64>, grid, dim3(256), 0, s, a); break;
    case 128: hipLaunchKernelGGL(kv4_append_kernel<128>, grid, dim3(256), 0, s, a); break;
    default: hipLaunchKernelGGL(kv4_append_kernel<256>, grid, dim3(256), 0, s, a); break;
    }
    return timer.end();
}

extern "C" int rptc_kv4_read(const uint8_t *k_cache, const uint8_t *v_cache, uint16_t *k, uint16_t *v, int64_t seqs, int64_t rows,
                             int64_t kv_heads, int64_t hd, int64_t max_len, int64_t k_token, int64_t k_head, int64_t v_token,
                             int64_t v_head, void *stream, float *ms)
{
    if (!k || !v || !k_cache || !v_cache) return RPTC_ENULL;
    int rc = kv4_sizes(seqs, kv_heads, hd, max_len);
    if (rc) return rc;
    if (rows < 1 || rows > max_len || k_token < 0 || k_head < 0 || v_token < 0 || v_head < 0) return RPTC_ESHAPE;
    if ((seqs * rows > 1 && (k_token == 0 || v_token == 0)) || (kv_heads > 1 && (k_head == 0 || v_head == 0))) return RPTC_ESHAPE;      // rows over rows
    if (!aligned16(k) || !aligned16(v) || !aligned16(k_cache) || !aligned16(v_cache)) return RPTC_EALIGN;
    if (k_token % 8 || k_head % 8 || v_token % 8 || v_head % 8) return RPTC_EALIGN;
    auto cache = [&](const void *o) { return o == k_cache || o == v_cache; };
    if (k == v || cache(k) || cache(v)) return RPTC_EALIAS;
    DeviceInfo *dev;
    if ((rc = device_info(&dev))) return rc;
    Kv4ReadArgs a;
    a.k_cache = k_cache;
    a.v_cache = v_cache;
    a.k = k;
    a.v = v;
    a.k_token = k_token;
    a.k_head = k_head;
    a.v_token = v_token;
    a.v_head = v_head;
    a.max_len = max_len;
    a.rows = (int)rows;
    a.kv_heads = (int)kv_heads;
    const int per = 256 / (int)(hd / 8);       // rows of a workgroup
    const dim3 grid((unsigned)((rows + per - 1) / per), (unsigned)(2 * kv_heads), (unsigned)seqs);
    hipStream_t s = static_cast<hipStream_t>(stream);
    Timer timer;
    if ((rc = timer.begin(dev, s, ms))) return rc;
    switch (hd) {
    case 32: hipLaunchKernelGGL(kv4_read_kernel<32>, grid, dim3(256), 0, s, a); break;
    case 64: hipLaunchKernelGGL(kv4_read_kernel<64>, grid, dim3(256), 0, s, a); break;
    case 128: hipLaunchKernelGGL(kv4_read_kernel<128>, grid, dim3(256), 0, s, a); break;
    default: hipLaunchKernelGGL(kv4_read_kernel<256>, grid, dim3(256), 0, s, a); break;
    }
    return timer.end();
}

extern "C" int rptc_kv4_rope_append(const uint16_t *qkv, const uint16_t *cos_t, const uint16_t *sin_t, const int64_t *pos,
                                    uint16_t *q_out, uint8_t *k_cache, uint8_t *v_cache, int64_t seqs, int64_t heads, int64_t kv_heads,
                                    int64_t hd, int64_t max_len, void *stream, float *ms)
{
    if (!qkv || !cos_t || !sin_t || !pos || !q_out || !k_cache || !v_cache) return RPTC_ENULL;
    int rc = kv4_sizes(seqs, kv_heads, hd, max_len);
    if (rc) return rc;
    if (heads < 1 || heads % kv_heads != 0) return RPTC_ESHAPE;
    if (heads > 1024) return RPTC_ELIMIT;
    if (!aligned16(qkv) || !aligned16(cos_t) || !aligned16(sin_t) || !aligned16(q_out) || !aligned16(k_cache) || !aligned16(v_cache)) return RPTC_EALIGN;
    auto cache = [&](const void *p) { return p == k_cache || p == v_cache; };
    if (q_out == qkv || k_cache == v_cache || cache(q_out) || cache(qkv)) return RPTC_EALIAS;
    DeviceInfo *dev;
    if ((rc = device_info(&dev))) return rc;
    const int items = (int)((heads + 2 * kv_heads) * (hd / 8));
    hipStream_t s = static_cast<hipStream_t>(stream);
    Timer timer;
    if ((rc = timer.begin(dev, s, ms))) return rc;
    hipLaunchKernelGGL(kv4_rope_append_kernel, dim3((unsigned)((items + 255) / 256), (unsigned)seqs), dim3(256), 0, s, qkv, cos_t, sin_t, pos,
                       q_out, k_cache, v_cache, (int)heads, (int)kv_heads, (int)hd, max_len, items);
    return timer.end();
}

extern "C" int64_t rptc_kv4_attn_decode_workspace_bytes(int64_t seqs, int64_t heads, int64_t kv_heads, int64_t hd, int64_t max_len)
{
    int rc = kv4_sizes(seqs, kv_heads, hd, max_len);
    if (rc) return rc;
    if (heads < 1 || heads % kv_heads != 0) return RPTC_ESHAPE;
    if (heads > 1024 || seqs * kv_heads * ((heads / kv_heads + 15) / 16) >= (int64_t)1 << 22) return RPTC_ELIMIT;
    DeviceInfo *dev;
    if ((rc = device_info(&dev))) return rc < 0 ? rc : RPTC_EDEVICE;
    const Kv4Plan plan = kv4_plan(seqs, kv_heads * ((heads / kv_heads + 15) / 16), max_len, dev->cus);
    return plan.want > 1 ? heads * plan.slots * (hd + 2) * 4 : 0;
}

template <int HD>
static void launch_kv4_attn(const Kv4AttnArgs &a, hipStream_t s)
{
    const int live = a.group < 16 ? a.group : 16;
    hipLaunchKernelGGL(kv4_attn_kernel<HD>, dim3((unsigned)(a.slots * a.kv_heads * a.head_blocks)), dim3(64 * kKv4Waves<HD>),
                       kv4_lds<HD>(live), s, a);
    if (a.want > 1)
        hipLaunchKernelGGL(kv4_merge_kernel<HD>, dim3((unsigned)a.heads, (unsigned)a.seqs), dim3(kJoinThreads), 0, s, a);
}

extern "C" int rptc_kv4_attn_decode(const uint16_t *q, const uint8_t *k_cache, const uint8_t *v_cache, const int64_t *pos, uint16_t *out,
                                    int64_t seqs, int64_t heads, int64_t kv_heads, int64_t hd, int64_t max_len, int64_t q_token,
                                    float scale, void *workspace, int64_t workspace_bytes, void *stream, float *ms)
{
    if (!q || !k_cache || !v_cache || !pos || !out) return RPTC_ENULL;
    int rc = kv4_sizes(seqs, kv_heads, hd, max_len);
    if (rc) return rc;
    if (heads < 1 || heads % kv_heads != 0 || q_token < 0 || !(scale > 0.f) || !(scale < 1e30f)) return RPTC_ESHAPE;
    if (heads > 1024 || seqs * kv_heads * ((heads / kv_heads + 15) / 16) >= (int64_t)1 << 22) return RPTC_ELIMIT;
    if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out) || q_token % 8) return RPTC_EALIGN;
    auto read = [&](const void *o) { return o == q || o == k_cache || o == v_cache; };
    if (read(out)) return RPTC_EALIAS;
    DeviceInfo *dev;
    if ((rc = device_info(&dev))) return rc;
    Kv4AttnArgs a;
    a.q = q;
    a.k_cache = k_cache;
    a.v_cache = v_cache;
    a.pos = pos;
    a.out = out;
    a.q_token = q_token;
    a.max_len = max_len;
    a.heads = (int)heads;
    a.kv_heads = (int)kv_heads;
    a.group = (int)(heads / kv_heads);
    a.head_blocks = (a.group + 15) / 16;
    const Kv4Plan plan = kv4_plan(seqs, kv_heads * a.head_blocks, max_len, dev->cus);
    a.seqs = (int)seqs;
    a.slots = plan.slots;
    a.want = plan.want;
    a.least = plan.least;
    a.c = scale * 1.44269504088896f;
    a.part = nullptr;
    a.part_ml = heads * a.slots * hd;
    if (a.want > 1) {
        if (!workspace) return RPTC_ENULL;
        if (!aligned16(workspace)) return RPTC_EALIGN;
        if (workspace_bytes < heads * a.slots * (hd + 2) * 4) return RPTC_ESHAPE;
        a.part = static_cast<float *>(workspace);
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    Timer timer;
    if ((rc = timer.begin(dev, s, ms))) return rc;
    switch (hd) {
    case 32: launch_kv4_attn<32>(a, s); break;
    case 64: launch_kv4_attn<64>(a, s); break;
    case 128: launch_kv4_attn<128>(a, s); break;
    default: launch_kv4_attn<256>(a, s); break;
    }
    return timer.end();
}
