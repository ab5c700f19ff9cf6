// Keys and values held in 4 bits: the format, and what the kernels that write, read and attend to it share.
//
// A pool is [pages, kv_heads, page, dim · 9 / 16] bytes. What a page holds of a head is one piece: first the codes of its keys (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign; two in a
// byte, the earlier dimension in the low half), dim / 2 bytes each, then their scales (e4m3), one per 16 dimensions. A value is code · scale · factor, with an f32 factor per head (1 where none are
// given). code · scale has six significant bits at most and lies between 2^-10 and 2688: f16 holds it exactly, so matrix instructions multiply what is stored, not a rounding of it.
//
// Stored is, of y = x / factor in f32 and a = max |y| over 16 dimensions, scale = e4m3(a / 6) and code = e2m1(y / scale), both to the nearest, ties to even, at most 448 and 6. Where the
// scale comes out as 0 so do the codes; where one of the 16 is no number the scale is none, and all 16 read as NaN. The code of 0 has no sign.
#pragma once
#include "paged_util.cuh"
#include "quotient.hpp"

namespace oxk {

constexpr int kPack = 16;  // dimensions of a scale
constexpr float kNone = -3.402823466e38f;  // below every score, and finite: differences stay numbers

struct PackP {
    const void* proj;            // [rows, ld]
    const float* turns;          // [2, half]
    unsigned char *keys, *values;  // [pages, kv_heads, page, dim | vdim times 9 / 16]
    void* q;                     // prepared queries [rows, heads, dim]: f32, or f16 for the prompt kernel
    float* q_mul;                // [rows, heads]: what products with f16 queries are multiplied by, in base 2; the sign of `mul2` is in the queries
    void* out;                   // [rows, heads · vdim]
    const int* seqs;             // [R, 4]
    const int* table;            // [R, width]
    const float *key_factors, *value_factors;  // [kv_heads], or null: 1
    float* part;                 // partial results of single tokens
    unsigned* counters;
    ErrWord* err;
    long long rows, ld, q_off, k_off, v_off;
    int n_seqs, width, n_pages, shift /* log2 of the page */, heads, kv_heads, dim, vdim, half, window, node;
    float scale, cap;            // scores in natural units
    float mul2, cap2;            // base 2: cap2 = 0: score2 = mul2 · q·k, otherwise cap2 · tanh with mul2 = 2 log2 e · scale / cap
    double eps;
    int norm, sink, append;
    int singles;                 // sequences with one new token are for these kernels too
    unsigned by_rep, by_units, by_runs;  // for over(): heads of a key head, units of eight pairs or dimensions of a query or key, runs of eight dimensions of a value
    unsigned by_key, by_value, by_eighths;  // the same: scales of a key, of a value, runs of eight dimensions of a key
    int by8;                     // the parts of a projection row begin on 16 bytes
    int pieces;                  // single tokens: CTAs per sequence and group of query heads; 0: CTAs share them all evenly
    int raw_slots;               // prompts: copies of 64 keys or values under way
    int only;                    // no rows for prompts: as many rows as sequences, none of which may have more than one new token
};

// n / d for 0 ≤ n ≤ most: `by` is by_of(d, most)
__device__ __forceinline__ int over(int n, unsigned by) { return by ? (int)__umulhi((unsigned)n, by) : n; }

__device__ __forceinline__ float key_factor(const PackP& p, int g) { return p.key_factors ? p.key_factors[g] : 1.f; }
__device__ __forceinline__ float value_factor(const PackP& p, int g) { return p.value_factors ? p.value_factors[g] : 1.f; }

// Where page `pg` holds head g's codes and, behind them, scales, for keys or values of `dim` dimensions.
template <class P> __device__ __forceinline__ unsigned char* held(const P& p, unsigned char* pool, long long pg, int g, int dim) {
    return pool + ((pg * p.kv_heads + g) << p.shift) * (dim / kPack) * 9;
}
template <class P> __device__ __forceinline__ unsigned char* codes_of(const P& p, unsigned char* held, int pos, int dim) { return held + (pos & ((1 << p.shift) - 1)) * (dim / 2); }
template <class P> __device__ __forceinline__ unsigned char* scales_of(const P& p, unsigned char* held, int pos, int dim) {
    return held + ((dim / 2) << p.shift) + (pos & ((1 << p.shift) - 1)) * (dim / kPack);
}

// ── the format ──
__device__ __forceinline__ unsigned bits(__half2 v) { return *reinterpret_cast<unsigned*>(&v); }
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// The scale of sixteen values whose largest magnitude is `a`, as it is stored.
__device__ __forceinline__ unsigned scale_code(float a) {
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(a / 6.f));
    return r & 0xFFu;
}
__device__ __forceinline__ __half2 scales_f16(unsigned two) {
    unsigned r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((unsigned short)two));
    return *reinterpret_cast<__half2*>(&r);
}
__device__ __forceinline__ float scale_value(unsigned code) { return __low2float(scales_f16(code)); }
// A value over its scale; 0 where that is 0 or no number.
__device__ __forceinline__ float over_scale(float y, float scale) { return scale > 0.f ? y / scale : 0.f; }
// The same for a value of eight significant bits (bf16), by the scale's reciprocal `by`: y / scale is halfway between two codes (a multiple of 1/4 up to 5), or 2^-10 away from it and more. The sum
// with 2560 rounds to a multiple of 2^-12: what is halfway comes out so, the rest stays on its side.
__device__ __forceinline__ float near_scale(float y, float by) { return __fadd_rn(__fmaf_rn(y, by, 2560.f), -2560.f); }
__device__ __forceinline__ unsigned without_signs_of_0(unsigned codes) { return codes & (0x77777777u | (((codes & 0x77777777u) + 0x77777777u) & 0x88888888u)); }
// Eight values over their scale as codes, the first one lowest.
__device__ __forceinline__ unsigned codes8(const float (&r)[8]) {
    unsigned v;
    asm("{\n .reg .b8 a, b, c, d;\n"
        " cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
        " mov.b32 %0, {a, b, c, d};\n}\n"
        : "=r"(v)
        : "f"(r[0]), "f"(r[1]), "f"(r[2]), "f"(r[3]), "f"(r[4]), "f"(r[5]), "f"(r[6]), "f"(r[7]));
    return without_signs_of_0(v);
}
__device__ __forceinline__ unsigned code_of(float r) {
    unsigned v;
    asm("{\n .reg .b8 a, b;\n cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n mov.b32 %0, {a, a, a, a};\n}\n" : "=r"(v) : "f"(r), "f"(0.f));
    v &= 15u;
    return v == 8u ? 0u : v;
}
// What the four bytes of a word stand for, two dimensions each, without their scale.
__device__ __forceinline__ void units8(unsigned word, __half2 (&v)[4]) {
    unsigned a, b, c, d;
    asm("{\n .reg .b8 e, f, g, h;\n mov.b32 {e, f, g, h}, %4;\n"
        " cvt.rn.f16x2.e2m1x2 %0, e;\n cvt.rn.f16x2.e2m1x2 %1, f;\n cvt.rn.f16x2.e2m1x2 %2, g;\n cvt.rn.f16x2.e2m1x2 %3, h;\n}\n"
        : "=r"(a), "=r"(b), "=r"(c), "=r"(d)
        : "r"(word));
    v[0] = *reinterpret_cast<__half2*>(&a);
    v[1] = *reinterpret_cast<__half2*>(&b);
    v[2] = *reinterpret_cast<__half2*>(&c);
    v[3] = *reinterpret_cast<__half2*>(&d);
}

// ── a batch step ──
// Keys are counted in 32 bits, 128 at a time: a sequence ends this far in front of their end.
constexpr long long kMostKeys = (1ll << 31) - 128;
// Sequence r of the batch. One whose rows are not the batch's, or whose positions the page table has no place for, is reported and has no rows.
template <class P> __device__ __forceinline__ SeqRow checked_seq(const P& p, int r) {
    SeqRow s = load_seq(p.seqs, r);
    if (s.len != 0 && (s.start < 0 || s.len < 0 || s.past < 0 || s.start + (long long)s.len > p.rows || s.past + (long long)s.len > min((long long)p.width << p.shift, kMostKeys))) {
        report(p.err, ERR_BATCH_SEQ, p.node, r, s.past + (long long)s.len);
        s.len = 0;
    }
    return s;
}
// By the CTA of the batch's first row: what is wrong with a sequence that no row belongs to.
template <class P> __device__ __forceinline__ void check_others(const P& p, int row, int tid, int threads) {
    if (row == 0)
        for (int i = tid; i < p.n_seqs; i += threads) checked_seq(p, i);
}
// The tile of `tq` tokens a CTA works on, counted over the sequences with `least` new tokens and more, and the sequence that it belongs to.
template <class P> __device__ __forceinline__ bool locate_rows(const P& p, int tile, int tq, int least, int* seq, int* first, SeqRow* row) {
    const int lane = threadIdx.x & 31;
    int before = 0;
    for (int r0 = 0; r0 < p.n_seqs; r0 += 32) {
        const SeqRow mine = r0 + lane < p.n_seqs ? checked_seq(p, r0 + lane) : SeqRow{0, 0, 0, 0};
        const int n = mine.len >= least ? (mine.len + tq - 1) / tq : 0;
        int inc = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, before + inc > tile);
        if (hit) {
            const int at = __ffs(hit) - 1;
            *seq = r0 + at;
            *first = (tile - before - (__shfl_sync(0xffffffffu, inc, at) - __shfl_sync(0xffffffffu, n, at))) * tq;
            *row = SeqRow{__shfl_sync(0xffffffffu, mine.start, at), __shfl_sync(0xffffffffu, mine.len, at), __shfl_sync(0xffffffffu, mine.past, at), 0};
            return true;
        }
        before += __shfl_sync(0xffffffffu, inc, 31);
    }
    return false;
}
template <class P> __device__ __forceinline__ int first_key(const P& p, int pos) { return p.window > 0 ? max(0, pos - p.window + 1) : 0; }
// Cosine and sine of every pair at a position, by `threads` threads, in 64 bits: what one step stores is the rounding of the key itself, which any other way to compute it finds too.
template <class P> __device__ __forceinline__ void exact_angles(const P& p, int pos, double* cs, double* sn, int tid, int threads) {
    for (int i = tid; i < p.half; i += threads) {
        const double t = (double)pos * ((double)p.turns[i] + (double)p.turns[p.half + i]) * 2.0;
        sincospi(t - 2.0 * rint(0.5 * t), sn + i, cs + i);
    }
}
// The same of one pair in 32 bits, for queries, which f16 holds to 2^-11. Turns are reduced to quarters in 64 bits: what is left is small and loses little as f32.
__device__ __forceinline__ void short_angle(int pos, double turns, float* cs, float* sn) {
    const double t = (double)pos * turns * 4.0, whole = rint(t);
    const int quarter = (int)((long long)whole & 3);
    float s, c;
    sincospif(0.5f * (float)(t - whole), &s, &c);
    *cs = quarter == 0 ? c : quarter == 1 ? -s : quarter == 2 ? -c : s;
    *sn = quarter == 0 ? s : quarter == 1 ? c : quarter == 2 ? -s : -c;
}
// Dimension i of a query or key whose leading 2 · half dimensions turn, i with i + half.
template <typename T> __device__ __forceinline__ double turned(int half, const T* x, const double* cs, const double* sn, int i) {
    const double v = (double)to_f(x[i]);
    if (i >= 2 * half) return v;
    return i < half ? v * cs[i] - (double)to_f(x[i + half]) * sn[i] : v * cs[i - half] + (double)to_f(x[i - half]) * sn[i - half];
}
// The sum of squares of a query or key in 64 bits, by one warp, and 1 / root mean square
template <typename T> __device__ __forceinline__ double square_sum(const PackP& p, const T* x) {
    double ss = 0.0;
    for (int i = threadIdx.x & 31; i < p.dim; i += 32) ss += (double)to_f(x[i]) * (double)to_f(x[i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    return ss;
}
__device__ __forceinline__ double norm_of(const PackP& p, double ss) { return 1.0 / sqrt(ss / p.dim + p.eps); }
template <typename T> __device__ __forceinline__ double norm_factor(const PackP& p, const T* x) { return p.norm ? norm_of(p, square_sum(p, x)) : 1.0; }

// The power of two that brings the largest element of a query, `top`, next to 1, as its exponent field: queries are f16 times it, so that none is too large and what is rounded is 2^-11 of an element, of those
// below 2^-14 of the largest 2^-25 of that.
__device__ __forceinline__ int query_exponent(float top) { return min(max((int)(__float_as_uint(top) >> 23), 1), 253); }
__device__ __forceinline__ float power_down(int e) { return __uint_as_float((unsigned)(254 - e) << 23); }
__device__ __forceinline__ float power_up(int e) { return __uint_as_float((unsigned)e << 23); }
// Weights of a softmax are f16 against a reference that the largest score so far lies kLeast to kMost above (in base 2): a sum of values is rescaled where it moves, which is dear. Down to
// 2^-(14 + kLeast) of the largest weight f16 holds 11 bits of them, below it has steps of 2^-(24 + kLeast) of that: a first key that has nearly all weight, and a value that adds little, leaves the others
// what they are. A closer reference costs prompts more moves: 4096 tokens of 32 heads over 16 take 187 us with 8, 194 with 11, 206 with 13.
constexpr float kLeast = 8.f, kMost = 15.f;
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// cap2 · tanh(u), x = 2 log2 e · u. tanh u = 1 - 2 / (1 + e^2u) is off by 4e-7: for a cap2 up to kWideCap less than queries in f16 move a score. Beyond (WIDE) what lies within a quarter of the cap is a series,
// u (1 - u²/3 + 2u⁴/15 - 17u⁶/315 + 62u⁸/2835 - ...), which leaves out 4e-7 of the score itself. (Rows of scores on both sides of the quarter have either: every element is chosen for.)
constexpr float kWideCap = 256.f, kTwiceLog2e = 2.f * kLog2e;
__device__ __forceinline__ float cap_series(float cap2, float z) {  // z = u²: what u is multiplied by
    return __fmaf_rn(__fmaf_rn(__fmaf_rn(cap2 * (-17.f / 315.f), z, cap2 * (2.f / 15.f)), z, cap2 * (-1.f / 3.f)), z, cap2);
}
template <bool WIDE> __device__ __forceinline__ float capped_score(float cap2, float x) {
    const float far = cap2 - __fdividef(2.f * cap2, 1.f + exp2_fast(x)), u = x * (1.f / kTwiceLog2e);
    return WIDE && fabsf(u) <= 0.25f ? u * cap_series(cap2, u * u) : far;
}
// 32 values of a head by one warp, the lane's `value` dimension c + lane: codes and scales to where they are held. Values from n on are nobody's.
__device__ __forceinline__ void put_32(unsigned char* codes, unsigned char* scales, int c, int n, float factor, float value) {
    const int lane = threadIdx.x & 31, i = c + lane;
    const float y = i < n ? value / factor : 0.f;
    float a = fabsf(y);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
    const unsigned s = scale_code(a), code = code_of(over_scale(y, scale_value(s))), next = __shfl_down_sync(0xffffffffu, code, 1);
    if (i < n && lane % 2 == 0) codes[i / 2] = (unsigned char)(code | next << 4);
    if (i < n && lane % kPack == 0) scales[i / kPack] = (unsigned char)s;
}
template <class F> __device__ __forceinline__ void put_head(unsigned char* codes, unsigned char* scales, int n, float factor, F&& value) {
    for (int c = 0; c < n; c += 32) put_32(codes, scales, c, n, factor, c + (int)(threadIdx.x & 31) < n ? value(c + (int)(threadIdx.x & 31)) : 0.f);
}

// Single tokens in bf16 (packed_decode.cu), keys and values of 256 dimensions at most.
using PackKernel = void (*)(const PackP);
struct PackedDecode {
    PackKernel kernel;
    int smem, part;          // bytes; floats of a partial result
    int resident, heads, step, pieces;  // CTAs of an SM; query heads and keys that a CTA takes at a time; the most CTAs that may share a sequence
};
PackedDecode packed_decode_of(int64_t dim, int64_t vdim);
// Prompts in bf16 (packed_prefill.cu), keys and values of 256 dimensions at most, 128 query heads of a key head at most.
struct PackedPrefill {
    PackKernel kernel;
    int smem, rows, threads, slots;  // bytes; (token, head) rows of a CTA; copies of 64 keys or values under way
};
PackedPrefill packed_prefill_of(int64_t dim, int64_t vdim, int64_t rows, int64_t kv_heads, int64_t rep, float cap2);

}  // namespace oxk
