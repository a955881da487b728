// A key/value cache held in 4 bits: appending rows, reading them back, and the attention of one token per sequence over it.
// (No counterpart in the reference, which generates with transformers on dense weights and caches, quantize_hf.py:229-236.)
//
// A row is one position of one head, hd fp16 values in groups of 32:
//   m = min x,  s = fp16((max x - min x) / 15),  code = clamp(rint((x - m) / s), 0, 15) (0 where s = 0),
//   the value a code stands for = fp16(code * s + m), one rounding
// (the quotients in fp32, correctly rounded; a group that holds a value which is no finite number reads as not-a-number).
// hd / 2 bytes of codes, then s and m of every group: hd / 2 + hd / 8 bytes, 80 against 256 at hd = 128.  Word w of a row
// holds the values 8w .. 8w+7, nibble t the value 8w + 2t and nibble t + 4 the value 8w + 2t + 1: one mask of a word gives a
// pair of neighbours in the two halves of a register.
#include "join.hpp"

namespace rptc {

constexpr int kKv4Group = 32;
typedef float float4v_t __attribute__((ext_vector_type(4)));
typedef _Float16 half8v_t __attribute__((ext_vector_type(8)));

constexpr int kv4_row_bytes(int hd) { return hd / 2 + hd / kKv4Group * 4; }

__device__ __forceinline__ half2_t as_half2(uint32_t w) { return __builtin_bit_cast(half2_t, w); }
__device__ __forceinline__ uint32_t low_halves(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ uint32_t high_halves(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// Nibbles 0, 1, 2, 3 of both halves of w as pairs of fp16 numbers: the bits of a code are put into the mantissa of 1024 (at
// its lowest bits) or of 64 (four bits up, so without a shift), and the power taken off again, exactly.
template <int N>
__device__ __forceinline__ void nibble_pairs(uint32_t w, half2_t *c)
{
    const half2_t k1024 = {(_Float16)1024.f, (_Float16)1024.f}, k64 = {(_Float16)64.f, (_Float16)64.f};
    c[0] = as_half2((w & 0x000F000Fu) | 0x64006400u) - k1024;
    if (N > 1) c[1] = as_half2((w & 0x00F000F0u) | 0x54005400u) - k64;
    if (N > 2) {
        const uint32_t v = w >> 8;
        c[2] = as_half2((v & 0x000F000Fu) | 0x64006400u) - k1024;
        c[3] = as_half2((v & 0x00F000F0u) | 0x54005400u) - k64;
    }
}

// the eight values of a word, in order
__device__ __forceinline__ half8v_t word_values(uint32_t w, uint32_t par)
{
    const half2_t s = as_half2(low_halves(par, par)), m = as_half2(high_halves(par, par));
    half2_t c[4];
    nibble_pairs<4>(w, c);
#pragma unroll
    for (int t = 0; t < 4; t++) c[t] = __builtin_elementwise_fma(c[t], s, m);
    half8v_t r;
#pragma unroll
    for (int t = 0; t < 4; t++) {
        r[2 * t] = c[t].x;
        r[2 * t + 1] = c[t].y;
    }
    return r;
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
    const uint16_t sb = float_to_half_bits((hi - lo) / 15.f);
    const float s = half_bits_to_float(sb);
    par = (uint32_t)float_to_half_bits(lo) << 16 | sb;
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
// writes a run of memory.
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
    // a position outside the cache is not written
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
    *reinterpret_cast<half8v_t *>(out + 8 * word) = word_values(code, par);
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
// words as the row operand (16 bytes of 16 consecutive rows: a run of memory); its result has, in a lane, scores of one head
// for four positions of each of two tiles, which is, with the positions renumbered accordingly, the operand P of
// O^T = V^T P^T; V^T's operand wants eight positions of one dimension in a lane, so the lane reads one word (eight
// dimensions) of its eight rows and pairs the positions up with byte permutes.  Values are formed in fp16, as stored.
// The matrix unit is mostly idle (15 of 16 columns with one query head a key head); what counts is the vector unit's work of
// unpacking, 4 instructions a pair of values, which stays under the time of the bytes.
struct Kv4AttnArgs {
    const uint16_t *q;
    const uint8_t *k_cache, *v_cache;
    const int64_t *pos;
    uint16_t *out;
    float *part;                            // splits > 1: [seq][head][split][hd] sums, then [seq][head][split][2] bound and sum of p
    int64_t q_token, max_len, part_ml;      // part_ml: where the second part begins
    int heads, kv_heads, group, head_blocks, splits;
    float c;                                // scale * log2(e)
};

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

constexpr int kKv4Waves = 8;
constexpr int kKv4Tile = 32;                // positions a wave takes at a time
constexpr float kKv4Lazy = 8.f;

template <int HD>
__global__ __launch_bounds__(64 * kKv4Waves) void kv4_attn_kernel(const Kv4AttnArgs a)
{
    extern __shared__ __align__(16) float lds4[];          // [wave][head][HD], then [wave][16][2]
    constexpr int kRow = kv4_row_bytes(HD);
    constexpr int kW = HD / 32;                            // words of a row a lane holds of K
    constexpr int kE = HD / 16;                            // dimensions of a row a lane holds of V
    constexpr int kVW = HD >= 128 ? HD / 128 : 1;          // words of that
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, c = lane >> 4;
    const int split = blockIdx.x, kvh = blockIdx.y / a.head_blocks, hb = blockIdx.y % a.head_blocks, seq = blockIdx.z;
    const int64_t pos = a.pos[seq];
    // a position outside the cache: nothing is read or written
    if (pos < 0 || pos >= a.max_len) return;
    const int64_t len = pos + 1;
    const int64_t per = ((len + a.splits - 1) / a.splits + kKv4Tile - 1) / kKv4Tile * kKv4Tile;
    const int64_t lo = split * per, hi = min(len, lo + per);
    const int live = min(16, a.group - 16 * hb);           // query heads of this workgroup
    const int head0 = kvh * a.group + 16 * hb;
    const int64_t head_base = ((int64_t)seq * a.kv_heads + kvh) * a.max_len;

    half8v_t qf[kW];
#pragma unroll
    for (int w = 0; w < kW; w++) {
        qf[w] = (half8v_t)((_Float16)0.f);
        if (n < live)
            qf[w] = *reinterpret_cast<const half8v_t *>(a.q + seq * a.q_token + (int64_t)(head0 + n) * HD + 8 * (c * kW + w));
    }
    float4v_t acc[kE];
#pragma unroll
    for (int e = 0; e < kE; e++) acc[e] = (float4v_t)(0.f);
    float m = -INFINITY, l = 0.f;

    for (int64_t j0 = lo + wave * kKv4Tile; j0 < hi; j0 += kKv4Waves * kKv4Tile) {
        // rows past the piece: its last row, masked below (its values count with p = 0)
        const uint8_t *kb = a.k_cache + (head_base + j0) * kRow, *vb = a.v_cache + (head_base + j0) * kRow;
        const int left = (int)min((int64_t)kKv4Tile, hi - j0);
        uint32_t kw[2][kW], kp[2][(kW + 3) / 4], vw[8][kVW], vp[8];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const uint8_t *r = kb + min(16 * t + n, left - 1) * kRow;
#pragma unroll
            for (int w = 0; w < kW; w++) kw[t][w] = *reinterpret_cast<const uint32_t *>(r + 4 * (c * kW + w));
#pragma unroll
            for (int g = 0; g < (kW + 3) / 4; g++) kp[t][g] = *reinterpret_cast<const uint32_t *>(r + HD / 2 + 4 * (c * kW / 4 + g));
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint8_t *r = vb + min(16 * (i / 4) + 4 * c + i % 4, left - 1) * kRow;
#pragma unroll
            for (int w = 0; w < kVW; w++) vw[i][w] = *reinterpret_cast<const uint32_t *>(r + 4 * (HD >= 128 ? n * kVW + w : n * kE / 8));
            vp[i] = *reinterpret_cast<const uint32_t *>(r + HD / 2 + 4 * (n * kE / 32));
        }
        float4v_t s[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            s[t] = (float4v_t)(0.f);
#pragma unroll
            for (int w = 0; w < kW; w++) s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(word_values(kw[t][w], kp[t][w / 4]), qf[w], s[t], 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (16 * (i / 4) + 4 * c + i % 4 >= left) s[i / 4][i % 4] = -INFINITY;
        float mx = s[0][0];
#pragma unroll
        for (int i = 1; i < 8; i++) mx = fmaxf(mx, s[i / 4][i % 4]);
        mx = rows_max(mx) * a.c;
        if (__ballot(mx > m + kKv4Lazy)) {
            const float up = fmaxf(m, mx);
            const float f = up == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - up);
            l *= f;
#pragma unroll
            for (int e = 0; e < kE; e++) acc[e] *= f;
            m = up;
        }
        const float mc = m == -INFINITY ? 0.f : m;
        half8v_t p;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float x = __builtin_amdgcn_exp2f(fmaf(s[i / 4][i % 4], a.c, -mc));
            l += x;
            p[i] = (_Float16)x;
        }
        // V: the positions in pairs, the nibbles of a dimension of both in one register
        half2_t val[kE][4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const half2_t sc = as_half2(low_halves(vp[2 * i], vp[2 * i + 1])), mn = as_half2(high_halves(vp[2 * i], vp[2 * i + 1]));
#pragma unroll
            for (int w = 0; w < kVW; w++) {
                uint32_t x = vw[2 * i][w], y = vw[2 * i + 1][w];
                constexpr int kN = kE >= 8 ? 4 : kE / 2;   // pairs of dimensions of the word that are the lane's
                if (kE < 8) {
                    x >>= 2 * kE * (n % (8 / kE));
                    y >>= 2 * kE * (n % (8 / kE));
                }
                half2_t even[4], oddv[4];
                nibble_pairs<kN>(low_halves(x, y), even);
                nibble_pairs<kN>(high_halves(x, y), oddv);
#pragma unroll
                for (int t = 0; t < kN; t++) {
                    val[8 * w + 2 * t][i] = __builtin_elementwise_fma(even[t], sc, mn);
                    val[8 * w + 2 * t + 1][i] = __builtin_elementwise_fma(oddv[t], sc, mn);
                }
            }
        }
#pragma unroll
        for (int e = 0; e < kE; e++) {
            const half8v_t v8 = {val[e][0].x, val[e][0].y, val[e][1].x, val[e][1].y, val[e][2].x, val[e][2].y, val[e][3].x, val[e][3].y};
            acc[e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8, p, acc[e], 0, 0, 0);
        }
    }

    // the waves join through LDS: lane (head n, quarter c) holds the dimensions 4 kE c .. 4 kE (c + 1)
    float *w_acc = lds4 + (size_t)wave * live * HD, *w_ml = lds4 + (size_t)kKv4Waves * live * HD;
    l = rows_sum(l);
    if (n < live) {
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int e = 0; e < kE; e++) w_acc[n * HD + kE * (4 * c + r) + e] = acc[e][r];
        if (c == 0) {
            w_ml[2 * (wave * 16 + n)] = m;
            w_ml[2 * (wave * 16 + n) + 1] = l;
        }
    }
    __syncthreads();
    for (int i = tid; i < live * HD; i += 64 * kKv4Waves) {
        const int h = i / HD, d = i % HD;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kKv4Waves; w++) M = fmaxf(M, w_ml[2 * (w * 16 + h)]);
        float num = 0.f, den = 0.f;
#pragma unroll
        for (int w = 0; w < kKv4Waves; w++) {
            const float mw = w_ml[2 * (w * 16 + h)], lw = w_ml[2 * (w * 16 + h) + 1];
            if (lw == 0.f) continue;                       // the wave had no position
            const float f = mw == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mw - M);
            num = fmaf(lds4[(size_t)w * live * HD + i], f, num);
            den = fmaf(lw, f, den);
        }
        const int64_t at = (int64_t)seq * a.heads + head0 + h;
        if (a.splits == 1) {
            a.out[at * HD + d] = float_to_half_bits(num / den);
        } else {
            a.part[(at * a.splits + split) * HD + d] = num;
            if (d == 0) *reinterpret_cast<float2 *>(a.part + a.part_ml + 2 * (at * a.splits + split)) = make_float2(M, den);
        }
    }
}

// Joins the pieces of a head, a workgroup per (sequence, head).
__global__ __launch_bounds__(kJoinThreads) void kv4_merge_kernel(const float *__restrict__ part, int64_t part_ml, const int64_t *__restrict__ pos,
                                                                 uint16_t *__restrict__ out, int heads, int hd, int splits, int64_t max_len)
{
    const int head = blockIdx.x, seq = blockIdx.y;
    if (pos[seq] < 0 || pos[seq] >= max_len) return;
    const int64_t at = (int64_t)seq * heads + head;
    float M, den;
    const float num = join_pieces(part + at * splits * hd, part + part_ml + 2 * at * splits, splits, hd, M, den);
    if (threadIdx.x < hd) out[at * hd + threadIdx.x] = float_to_half_bits(num / den);
}

template <int HD>
static size_t kv4_lds(int live) { return ((size_t)kKv4Waves * live * HD + kKv4Waves * 32) * 4; }

int prepare_kv4()
{
    int rc;
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

static int64_t kv4_splits(int64_t groups, int64_t max_len, int cus)
{
    int64_t n = (2 * (int64_t)cus + groups - 1) / groups;
    if (n > max_len / (2 * kKv4Waves * kKv4Tile)) n = max_len / (2 * kKv4Waves * kKv4Tile);
    return n < 1 ? 1 : n > 128 ? 128 : n;
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
    if (k_cache == v_cache) return RPTC_EALIAS;
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
    if (!aligned16(k) || !aligned16(v) || !aligned16(k_cache) || !aligned16(v_cache)) return RPTC_EALIGN;
    if (k_token % 8 || k_head % 8 || v_token % 8 || v_head % 8) return RPTC_EALIGN;
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
    if (q_out == qkv || k_cache == v_cache) return RPTC_EALIAS;
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
    if (heads > 1024) return RPTC_ELIMIT;
    DeviceInfo *dev;
    if ((rc = device_info(&dev))) return rc < 0 ? rc : RPTC_EDEVICE;
    const int64_t splits = kv4_splits(seqs * kv_heads * ((heads / kv_heads + 15) / 16), max_len, dev->cus);
    return splits > 1 ? seqs * heads * splits * (hd + 2) * 4 : 0;
}

template <int HD>
static void launch_kv4_attn(const Kv4AttnArgs &a, int seqs, hipStream_t s)
{
    const int live = a.group < 16 ? a.group : 16;
    hipLaunchKernelGGL(kv4_attn_kernel<HD>, dim3((unsigned)a.splits, (unsigned)(a.kv_heads * a.head_blocks), (unsigned)seqs),
                       dim3(64 * kKv4Waves), kv4_lds<HD>(live), s, a);
}

extern "C" int rptc_kv4_attn_decode(const uint16_t *q, const uint8_t *k_cache, const uint8_t *v_cache, const int64_t *pos, uint16_t *out,
                                    int64_t seqs, int64_t heads, int64_t kv_heads, int64_t hd, int64_t max_len, int64_t q_token,
                                    float scale, void *workspace, int64_t workspace_bytes, void *stream, float *ms)
{
    if (!q || !k_cache || !v_cache || !pos || !out) return RPTC_ENULL;
    int rc = kv4_sizes(seqs, kv_heads, hd, max_len);
    if (rc) return rc;
    if (heads < 1 || heads % kv_heads != 0 || q_token < 0 || !(scale > 0.f) || !(scale < 1e30f)) return RPTC_ESHAPE;
    if (heads > 1024) return RPTC_ELIMIT;
    if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out) || q_token % 8) return RPTC_EALIGN;
    if (out == q) return RPTC_EALIAS;
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
    a.splits = (int)kv4_splits(seqs * kv_heads * a.head_blocks, max_len, dev->cus);
    a.c = scale * 1.44269504088896f;
    a.part = nullptr;
    a.part_ml = seqs * heads * a.splits * hd;
    if (a.splits > 1) {
        if (!workspace) return RPTC_ENULL;
        if (!aligned16(workspace)) return RPTC_EALIGN;
        if (workspace_bytes < seqs * heads * a.splits * (hd + 2) * 4) return RPTC_ESHAPE;
        a.part = static_cast<float *>(workspace);
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    Timer timer;
    if ((rc = timer.begin(dev, s, ms))) return rc;
    switch (hd) {
    case 32: launch_kv4_attn<32>(a, (int)seqs, s); break;
    case 64: launch_kv4_attn<64>(a, (int)seqs, s); break;
    case 128: launch_kv4_attn<128>(a, (int)seqs, s); break;
    default: launch_kv4_attn<256>(a, (int)seqs, s); break;
    }
    if (a.splits > 1)
        hipLaunchKernelGGL(kv4_merge_kernel, dim3((unsigned)heads, (unsigned)seqs), dim3(kJoinThreads), 0, s, a.part, a.part_ml, pos, out, (int)heads,
                           (int)hd, a.splits, max_len);
    return timer.end();
}
