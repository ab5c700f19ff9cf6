// What the kernels of differential attention share: their parameters.
#pragma once
#include "paged_util.cuh"

namespace oxk {

struct DiffP {
    const void* proj;            // [rows, ld]
    const float* turns;          // [2, half]
    void *keys, *values;         // [pages, kv_heads, page, 2 · dim | vdim]
    void* q;                     // prepared queries: [rows, heads, map, dim] of the pools' type, or, as the prefill kernel copies them, [kv_heads, rows, heads of a key head, map, high and low part, dim]
    void* out;                   // [rows, heads · vdim]
    const int* seqs;             // [R, 4]
    const int* table;            // [R, width]
    const float* lambda;         // [heads]
    const float* gain;           // [vdim], or null: results as they are
    float* part;                 // partial results of single tokens
    unsigned* counters;
    ErrWord* err;
    long long rows, ld, q_off, k_off, v_off;
    int n_seqs, width, n_pages, shift /* log2 of the page */, heads, kv_heads, dim, vdim, half, window, splits, node;
    float scale, cap, eps, head_eps;
    float mul2, cap2;            // base 2: cap2 = 0: score2 = mul2 · q·k, otherwise cap2 · tanh with mul2 = 2 log2 e · scale / cap
    int norm, sink;
    int singles;                 // sequences with one new token are for these kernels too
    int parts;                   // prepare: queries in two parts, times mul2
    int by8;                     // the parts of a projection row begin on 16 bytes
    int only;                    // no rows for prompts: with as many rows as sequences none may have more than one new token, with fewer those are differential_several's
    int low;                     // weights are the sum of two bf16
    int rep;                     // heads of a key head
    unsigned by_rep, by_units, by_lanes;  // 2^32 / (heads of a key head, units of a query, sixteen bytes of a value), rounded up; 0: of one
};

// Sequence r of the batch. One whose rows are not the batch's, or whose positions the page table has no place for, is reported and has no rows.
__device__ __forceinline__ SeqRow checked_seq(const DiffP& p, int r) {
    SeqRow s = load_seq(p.seqs, r);
    if (s.len != 0 && (s.start < 0 || s.len < 0 || s.past < 0 || s.start + (long long)s.len > p.rows || s.past + (long long)s.len > (long long)p.width << p.shift)) {
        report(p.err, ERR_BATCH_SEQ, p.node, r, s.past + (long long)s.len);
        s.len = 0;
    }
    return s;
}
// By the CTA of the batch's first row: what is wrong with a sequence that no row belongs to.
__device__ __forceinline__ void check_others(const DiffP& p, int row, int tid, int threads) {
    if (row == 0)
        for (int i = tid; i < p.n_seqs; i += threads) checked_seq(p, i);
}
__device__ __forceinline__ int first_key(const DiffP& p, int pos) { return p.window > 0 ? max(0, pos - p.window + 1) : 0; }
// log2 e · score of a dot product; tanh x = 1 − 2 / (1 + e^2x) is off by a few 1e-7 of the cap
__device__ __forceinline__ float score2(const DiffP& p, float d) {
    const float x = d * p.mul2;
    return p.cap2 > 0.f ? p.cap2 - __fdividef(2.f * p.cap2, 1.f + exp2f(x)) : x;
}
// Cosine and sine of every pair at a position, by `threads` threads, in 64 bits: a key is stored once and read for as long as its sequence lives, and in 64 bits it is the rounding of its
// value (with whole turns as f32, 1.6 times as many keys are a rounding off as with f32 products of 64-bit angles).
__device__ __forceinline__ void exact_angles(const DiffP& p, int pos, double* cs, double* sn, int tid, int threads) {
    for (int i = tid; i < p.half; i += threads) {
        const double t = (double)pos * ((double)p.turns[i] + (double)p.turns[p.half + i]) * 2.0;
        sincospi(t - 2.0 * rint(0.5 * t), sn + i, cs + i);
    }
}
// The same in 32 bits for queries, whose low part ends at 2^-18. Turns are reduced to quarters in 64 bits: what is left is small and loses little as f32.
__device__ __forceinline__ void short_angles(const DiffP& p, int pos, float* cs, float* sn, int tid, int threads) {
    for (int i = tid; i < p.half; i += threads) {
        const double t = (double)pos * ((double)p.turns[i] + (double)p.turns[p.half + i]) * 4.0, whole = rint(t);
        const int quarter = (int)((long long)whole & 3);
        float s, c;
        sincospif(0.5f * (float)(t - whole), &s, &c);
        cs[i] = quarter == 0 ? c : quarter == 1 ? -s : quarter == 2 ? -c : s;
        sn[i] = quarter == 0 ? s : quarter == 1 ? c : quarter == 2 ? -s : -c;
    }
}
// Dimension i of a query or key whose leading 2 · half dimensions turn, i with i + half.
template <typename T> __device__ __forceinline__ double turned(const DiffP& p, const T* x, const double* cs, const double* sn, int i) {
    const double v = (double)to_f(x[i]);
    if (i >= 2 * p.half) return v;
    return i < p.half ? v * cs[i] - (double)to_f(x[i + p.half]) * sn[i] : v * cs[i - p.half] + (double)to_f(x[i - p.half]) * sn[i - p.half];
}
// A query as the sum of two bf16. Rounded to one, it alone puts results 2.7e-3 from those of an f32 query (one token, 520 keys, scores of spread 1.5), more than the rounding
// of the weights (1.1e-3) and of the results (1.7e-3) together.
__device__ __forceinline__ bf16 low_part(float v, bf16 high) { return __float2bfloat16_rn(v - __bfloat162float(high)); }
// 1 / root mean square of a map's query or key, by one warp
template <typename T> __device__ __forceinline__ float map_factor(const DiffP& p, const T* x) {
    if (!p.norm) return 1.f;
    float ss = 0.f;
    for (int i = threadIdx.x & 31; i < p.dim; i += 32) {
        const float v = to_f(x[i]);
        ss = fmaf(v, v, ss);
    }
    return 1.f / sqrtf(warp_sum(ss) / (float)p.dim + p.eps);
}

// locate_tile, and the sequence that the tile belongs to: its row of the batch description comes with the count.
__device__ __forceinline__ bool locate_rows(const DiffP& p, int tile, int tq, int least, int* seq, int* first, SeqRow* row) {
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

// n / d for n < 2^32 / d
__device__ __forceinline__ int over(int n, unsigned by) { return by ? (int)__umulhi((unsigned)n, by) : n; }
// Where the high part of query h (2 · head + map) of a row is, for the prefill kernel.
__device__ __forceinline__ bf16* part_row(const DiffP& p, int row, int h) {
    const int g = over(h >> 1, p.by_rep);
    return (bf16*)p.q + ((((g * p.rows + row) * p.rep + (h >> 1) - g * p.rep) * 2 + (h & 1)) * 2) * p.dim;
}

// Prompts on tcgen05 (differential_prefill.cu); queries come from `q` (part_row) in units of base 2; `ptrs`: fields of DiffP by their offset.
bool differential_prefill_fits(const DiffP&, const TRef& keys, const TRef& values, int64_t out_off);
void emit_differential_prefill(Emitter&, const DiffP&, const TRef& keys, const TRef& values, std::initializer_list<std::pair<size_t, Buf>> ptrs);

}  // namespace oxk
