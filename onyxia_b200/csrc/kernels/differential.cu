// Differential attention of a ragged batch over paged pools of keys and values (Ye et al., "Differential Transformer", 2024): a head has two queries, its
// key head two keys per token and one value, and the second softmax map is taken from the first before the values are added up,
//
//   score_m(i, j) = cap(scale · q_i,m · k_j,m) for 0 ≤ i − j < window,  m = 0, 1,  cap(s) = c · tanh(s / c),
//   w_m(i, j) = exp(score_m) / ([exp(0)] + Σ_j exp(score_m)),   o_i = Σ_j (w_0(i, j) − λ w_1(i, j)) v_j,
//   out_i = gain · o_i / sqrt(mean(o_i²) + eps)     (or o_i)
//
// Queries and keys rotate and are normed as in paged_kv_attention.cu, each map by itself. A pool's key is the two maps' side by side.
//
//   differential_prepare   rotated, normed queries; the new keys and values go to the pools
//   differential_prefill   sequences with several new tokens in bf16 (differential_prefill.cu)
//   differential_decode    sequences with one new token: their keys split over CTAs and warps, all of the above in one launch
//   differential_simt      any shape, f32 and bf16
//   differential_several   sequences with several new tokens beside empty ones, in batches of fewer rows than sequences
//
// Decode reads min(past, window) · kv_heads · (2 · dim + vdim) · 2 bytes per sequence.
#include <cmath>

#include "differential.cuh"

namespace oxk {

namespace {

// One CTA per row, one warp per query or key of a map.
template <typename T> __global__ void __launch_bounds__(128) differential_prepare(const DiffP p) {
    extern __shared__ double angle[];  // cos[half], sin[half]
    pdl_enter();
    const int row = blockIdx.x, s = find_seq(p.seqs, p.n_seqs, row), lane = threadIdx.x & 31;
    const SeqRow sq = checked_seq(p, s);
    check_others(p, row, threadIdx.x, 128);
    const int pos = sq.past + row - sq.start;
    if (row < sq.start || row >= sq.start + sq.len || (sq.len == 1 && !p.singles)) return;
    exact_angles(p, pos, angle, angle + p.half, threadIdx.x, 128);
    __syncthreads();
    const T* x = (const T*)p.proj + (long long)row * p.ld;
    const long long pg = page_of(p, s, pos);
    for (int h = threadIdx.x >> 5; h < 2 * (p.heads + p.kv_heads); h += 4) {
        const int k = h - 2 * p.heads;
        const T* src = k < 0 ? x + p.q_off + (long long)h * p.dim : x + p.k_off + (long long)k * p.dim;
        T* dst = k < 0 ? (T*)p.q + ((long long)row * p.heads * 2 + h) * p.dim : (T*)p.keys + (key_row(p, pg, k >> 1, pos) * 2 + (k & 1)) * p.dim;
        const float f = map_factor(p, src);
        if constexpr (sizeof(T) == 2)
            if (k < 0 && p.parts) {
                bf16* to = part_row(p, row, h);
                for (int i = lane; i < p.dim; i += 32) {
                    const float v = (float)turned(p, src, angle, angle + p.half, i) * f * p.mul2;
                    const bf16 high = __float2bfloat16_rn(v);
                    to[i] = high;
                    to[p.dim + i] = low_part(v, high);
                }
                continue;
            }
        for (int i = lane; i < p.dim; i += 32) dst[i] = from_f<T>((float)(turned(p, src, angle, angle + p.half, i) * f));
    }
    for (int i = threadIdx.x; i < p.kv_heads * p.vdim; i += 128) ((T*)p.values)[key_row(p, pg, i / p.vdim, pos) * p.vdim + i % p.vdim] = x[p.v_off + i];
}

// The same in bf16 eight elements at a time, where heads, rotated halves and rows allow it: a unit is eight pairs that turn or eight elements that do not. 4096 tokens with 64 queries and
// 32 keys of 64 and 16 values of 128 (167 MB in and out): 40 us, with divisions by what only the host knows and nothing asked for before the angles 54; the kernel above 146.
__global__ void __launch_bounds__(128, 8) differential_prepare8(const DiffP p) {
    extern __shared__ double angle[];  // cos[half], sin[half], both again as f32 (for the queries), with norms [2 · (heads + kv_heads)] factors as f32
    pdl_enter();
    const int row = blockIdx.x, tid = threadIdx.x;
    // the row's queries, keys and values are on their way while its sequence is looked up and its angles are made
    const bf16* x = (const bf16*)p.proj + (long long)row * p.ld;
    auto fetch = [&](long long at, int n) {
        for (int i = tid * 64; i < n; i += 128 * 64) asm volatile("prefetch.global.L1 [%0];" ::"l"(x + at + i) : "memory");
    };
    fetch(p.q_off, 2 * p.heads * p.dim);
    fetch(p.k_off, 2 * p.kv_heads * p.dim);
    fetch(p.v_off, p.kv_heads * p.vdim);
    const int s = find_seq(p.seqs, p.n_seqs, row);
    const SeqRow sq = checked_seq(p, s);
    check_others(p, row, tid, 128);
    const int pos = sq.past + row - sq.start, maps = 2 * (p.heads + p.kv_heads);
    if (row < sq.start || row >= sq.start + sq.len || (sq.len == 1 && !p.singles)) return;
    float* short_angle = reinterpret_cast<float*>(angle + 2 * p.half);
    exact_angles(p, pos, angle, angle + p.half, tid, 128);
    for (int i = tid; i < p.half; i += 128) short_angle[i] = (float)angle[i], short_angle[p.half + i] = (float)angle[p.half + i];  // (its own)
    auto source = [&](int h) { return h < 2 * p.heads ? x + p.q_off + (long long)h * p.dim : x + p.k_off + (long long)(h - 2 * p.heads) * p.dim; };
    float* factor = short_angle + 2 * p.half;
    if (p.norm)
        for (int h = tid >> 5; h < maps; h += 4) {
            const float f = map_factor(p, source(h));
            if ((tid & 31) == 0) factor[h] = f;
        }
    __syncthreads();
    const long long pg = page_of(p, s, pos);
    const int turned = p.half / 8, units = p.dim / 8 - turned, lanes = p.vdim / 8;
    const long long key0 = key_row(p, pg, 0, pos), page = 1ll << p.shift;
    auto wide = [](uint4 u, float (&v)[8]) {
        const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; e++) v[2 * e] = __uint_as_float(w[e] << 16), v[2 * e + 1] = __uint_as_float(w[e] & 0xFFFF0000u);
    };
    auto put = [&](bf16* to, const float (&v)[8], bool parts) {
        unsigned w[4];
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = pack_bf16(v[2 * e], v[2 * e + 1]);
        *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
        if (!parts) return;
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = pack_bf16(v[2 * e] - __uint_as_float(w[e] << 16), v[2 * e + 1] - __uint_as_float(w[e] & 0xFFFF0000u));
        *reinterpret_cast<uint4*>(to + p.dim) = make_uint4(w[0], w[1], w[2], w[3]);
    };
    for (int u = tid; u < 2 * p.heads * units; u += 128) {
        const int h = over(u, p.by_units), i = u - h * units;
        const bool turns = i < turned;
        const int at = turns ? i * 8 : (i + turned) * 8;
        const bf16* src = x + p.q_off + h * p.dim + at;
        bf16* to = (p.parts ? part_row(p, row, h) : (bf16*)p.q + ((long long)row * p.heads * 2 + h) * p.dim) + at;
        const float f = (p.norm ? factor[h] : 1.f) * (p.parts ? p.mul2 : 1.f);
        float a[8], b[8], o[8];
        wide(*reinterpret_cast<const uint4*>(src), a);
        if (!turns) {
#pragma unroll
            for (int e = 0; e < 8; e++) o[e] = a[e] * f;
            put(to, o, p.parts);
            continue;
        }
        wide(*reinterpret_cast<const uint4*>(src + p.half), b);
        const float *c = short_angle + at, *n = c + p.half;
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] = (a[e] * c[e] - b[e] * n[e]) * f;
        put(to, o, p.parts);
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] = (b[e] * c[e] + a[e] * n[e]) * f;
        put(to + p.half, o, p.parts);
    }
    for (int u = tid; u < 2 * p.kv_heads * units; u += 128) {
        const int k = over(u, p.by_units), i = u - k * units;
        const bool turns = i < turned;
        const int at = turns ? i * 8 : (i + turned) * 8;
        const bf16* src = x + p.k_off + k * p.dim + at;
        bf16* to = (bf16*)p.keys + ((key0 + (k >> 1) * page) * 2 + (k & 1)) * p.dim + at;
        const float f = p.norm ? factor[2 * p.heads + k] : 1.f;
        float a[8], b[8], o[8];
        wide(*reinterpret_cast<const uint4*>(src), a);
        if (!turns) {
#pragma unroll
            for (int e = 0; e < 8; e++) o[e] = a[e] * f;
            put(to, o, false);
            continue;
        }
        wide(*reinterpret_cast<const uint4*>(src + p.half), b);
        const double *c = angle + at, *n = c + p.half;
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] = (float)(((double)a[e] * c[e] - (double)b[e] * n[e]) * f);
        put(to, o, false);
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] = (float)(((double)b[e] * c[e] + (double)a[e] * n[e]) * f);
        put(to + p.half, o, false);
    }
    for (int u = tid; u < p.kv_heads * lanes; u += 128) {
        const int g = over(u, p.by_lanes);
        *reinterpret_cast<uint4*>((bf16*)p.values + (key0 + g * page) * p.vdim + (u - g * lanes) * 8) = *reinterpret_cast<const uint4*>(x + p.v_off + u * 8);
    }
}

// A row's head by 128 threads: chunks of 128 keys, a thread per key, then a thread per value dimension. `sm`: q[2][dim] (there), acc[2][vdim], w[2][128].
template <typename T> __device__ __forceinline__ void attend_row(const DiffP& p, int s, int pos, int row, int h, float* sm, float* red) {
    const int tid = threadIdx.x, g = h / (p.heads / p.kv_heads);
    float *q = sm, *acc = sm + 2 * p.dim, *w = acc + 2 * p.vdim;
    for (int i = tid; i < 2 * p.vdim; i += kAnyKeys) acc[i] = 0.f;
    // a sink is a score of 0 that has no value; without one the sums begin below every score, at a number: differences stay numbers
    float m[2], l[2];
    m[0] = m[1] = p.sink ? 0.f : -1e30f;
    l[0] = l[1] = p.sink ? 1.f : 0.f;
    __syncthreads();
    for (int j0 = first_key(p, pos); j0 <= pos; j0 += kAnyKeys) {
        const int j = j0 + tid;
        float keep[2];
        const T* k = j <= pos ? (const T*)p.keys + key_row(p, page_of(p, s, j), g, j) * 2 * p.dim : nullptr;
        for (int e = 0; e < 2; e++) {
            float sc = -INFINITY;
            if (k) {
                sc = dot_in_order(q + e * p.dim, k + e * p.dim, p.dim, 0.f) * p.scale;
                if (p.cap > 0.f) sc = p.cap * tanhf(sc / p.cap);
            }
            const float top = fmaxf(m[e], block_max(sc, red)), x = expf(sc - top);
            w[e * kAnyKeys + tid] = x;
            keep[e] = expf(m[e] - top);
            l[e] = l[e] * keep[e] + block_sum(x, red);  // (its barriers order the stores to w)
            m[e] = top;
        }
        const int live = min(kAnyKeys, pos + 1 - j0);
        for (int i = tid; i < 2 * p.vdim; i += kAnyKeys) {
            const int e = i >= p.vdim;
            acc[i] = weigh_in_order(p, (const T*)p.values, s, g, j0, live, p.vdim, i - e * p.vdim, w + e * kAnyKeys, acc[i] * keep[e]);
        }
        __syncthreads();
    }
    const float f0 = 1.f / l[0], f1 = p.lambda[h] / l[1];
    float ss = 0.f;
    for (int i = tid; i < p.vdim; i += kAnyKeys) {
        const float o = acc[i] * f0 - acc[p.vdim + i] * f1;
        acc[i] = o;
        ss = fmaf(o, o, ss);
    }
    const float f = p.gain ? 1.f / sqrtf(block_sum(ss, red) / (float)p.vdim + p.head_eps) : 1.f;
    for (int i = tid; i < p.vdim; i += kAnyKeys) ((T*)p.out)[((long long)row * p.heads + h) * p.vdim + i] = from_f<T>(p.gain ? acc[i] * f * p.gain[i] : acc[i]);
}

template <typename T> __global__ void __launch_bounds__(kAnyKeys) differential_simt(const DiffP p) {
    extern __shared__ float sm[];
    __shared__ float red[32];
    pdl_enter();
    const int row = blockIdx.x, h = blockIdx.y, s = find_seq(p.seqs, p.n_seqs, row);
    const SeqRow sq = checked_seq(p, s);
    if (row < sq.start || row >= sq.start + sq.len || (sq.len == 1 && !p.singles)) return;
    for (int i = threadIdx.x; i < 2 * p.dim; i += kAnyKeys) sm[i] = to_f(((const T*)p.q)[((long long)row * p.heads + h) * 2 * p.dim + i]);
    attend_row<T>(p, s, sq.past + row - sq.start, row, h, sm, red);
}

// The sequences of several new tokens in a batch of fewer rows than sequences, whose single tokens differential_decode takes: a CTA per key head and sequence stores the keys and values, then
// goes through the rows. (64 sequences behind 2000, 16 heads of 2 x 64 over 4, four of
// them without new tokens: 4 us of a call of 77; the launches for prompts in its place took 24.)
__global__ void __launch_bounds__(kAnyKeys) differential_several(const DiffP p) {
    extern __shared__ float sm[];  // what attend_row has, cosines and sines behind it
    __shared__ float red[32];
    pdl_enter();
    const int g = blockIdx.x, seq = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rep = p.heads / p.kv_heads;
    const SeqRow sq = checked_seq(p, seq);
    if (sq.len < 2) return;
    double *cs = reinterpret_cast<double*>(sm + 2 * (p.dim + p.vdim + kAnyKeys)), *sn = cs + p.half;
    bf16 *keys = (bf16*)p.keys, *values = (bf16*)p.values;
    for (int t = 0; t < sq.len; t++) {
        const int pos = sq.past + t;
        const bf16* x = (const bf16*)p.proj + (long long)(sq.start + t) * p.ld;
        const long long at = key_row(p, page_of(p, seq, pos), g, pos);
        exact_angles(p, pos, cs, sn, tid, kAnyKeys);
        __syncthreads();
        if (warp < 2) {
            const bf16* k = x + p.k_off + (long long)(g * 2 + warp) * p.dim;
            const float f = map_factor(p, k);
            for (int i = lane; i < p.dim; i += 32) keys[(at * 2 + warp) * p.dim + i] = __float2bfloat16_rn((float)(turned(p, k, cs, sn, i) * f));
        }
        for (int i = tid; i < p.vdim; i += kAnyKeys) values[at * p.vdim + i] = x[p.v_off + (long long)g * p.vdim + i];
        __syncthreads();
    }
    for (int t = 0; t < sq.len; t++) {
        const int pos = sq.past + t;
        const bf16* x = (const bf16*)p.proj + (long long)(sq.start + t) * p.ld;
        exact_angles(p, pos, cs, sn, tid, kAnyKeys);
        for (int h = g * rep; h < (g + 1) * rep; h++) {
            __syncthreads();
            if (warp < 2) {
                const bf16* q = x + p.q_off + (long long)(h * 2 + warp) * p.dim;
                const float f = map_factor(p, q);
                for (int i = lane; i < p.dim; i += 32) sm[warp * p.dim + i] = (float)(turned(p, q, cs, sn, i) * f);
            }
            attend_row<bf16>(p, seq, pos, sq.start + t, h, sm, red);
        }
        __syncthreads();
    }
}

// ───────────────────────────── single tokens ────────────────────────────
constexpr int kDecWarps = 4, kDecThreads = kDecWarps * 32, kDecPages = 256, kDecHeads = 8, kDecKeys = 16;
constexpr float kNoScore = -1e30f;  // below every score, and finite: differences stay numbers

// DM, DV: dimensions of a map and of a value, padded
template <int DM, int DV> struct DecSmem {
    static constexpr int stages = DM <= 64 && DV <= 128 ? 3 : 2;
    static constexpr int q_stride = DM * 2 + 16, k_stride = DM * 4 + 16, v_stride = DV * 2 + 16;
    static constexpr int tile = kDecKeys * (k_stride + v_stride);  // keys, then values
    static constexpr int q = 0;                                    // [map][high, low][8 heads]
    static constexpr int kv = 4 * kDecHeads * q_stride;            // [warps][stages][tile]
    static constexpr int ring = kDecWarps * stages * tile;
    static constexpr int part = part_size(2 * kDecHeads, DV);      // floats of one partial result, rows [map][8 heads]
    static constexpr int merge = kDecWarps * part * 4;             // reuses the ring after the last key
    static constexpr int angle = kv + (ring > merge ? ring : merge);
    static constexpr int raw = angle + DM * 12;                    // the token's queries of 8 heads, then its two keys, as they come
    static constexpr int total = raw + 18 * DM * 2;
};

// The difference of the two maps' results, from `n` partial results ([n][map][8 heads][DV + 2]: maximum, sum, accumulator), a warp per head.
template <int DV> __device__ void merge_maps(const DiffP& p, const float* part, int n, int h0, int heads, bf16* out) {
    constexpr int size = part_size(2 * kDecHeads, DV), C = (DV + 31) / 32;
    const int lane = threadIdx.x & 31;
    for (int r = threadIdx.x >> 5; r < heads; r += kDecWarps) {
        float o[C] = {}, f0[2], f1[2];
        const float* head[2] = {part + r * (DV + 2), part + (kDecHeads + r) * (DV + 2)};
#pragma unroll
        for (int m = 0; m < 2; m++) {
            // lane i weighs parts i and i + 32 (n ≤ 64); a part that saw no key has the maximum kNoScore, sum and values 0
            float pm[2], pl[2];
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const bool in = k * 32 + lane < n;
                pm[k] = in ? head[m][(long long)(k * 32 + lane) * size] : kNoScore;
                pl[k] = in ? head[m][(long long)(k * 32 + lane) * size + 1] : 0.f;
            }
            float top = warp_max(fmaxf(pm[0], pm[1]));
            if (p.sink) top = fmaxf(top, 0.f);
            f0[m] = exp2f(pm[0] - top), f1[m] = exp2f(pm[1] - top);
            const float l = warp_sum(fmaf(pl[0], f0[m], pl[1] * f1[m])) + (p.sink ? exp2f(-top) : 0.f);
            const float f = m ? -p.lambda[h0 + r] / l : 1.f / l;
            f0[m] *= f, f1[m] *= f;
        }
#pragma unroll(DV <= 128 ? 8 : 4)
        for (int i = 0; i < n; i++) {
            const float w0 = __shfl_sync(0xffffffffu, i < 32 ? f0[0] : f1[0], i & 31), w1 = __shfl_sync(0xffffffffu, i < 32 ? f0[1] : f1[1], i & 31);
#pragma unroll
            for (int c = 0; c < C; c++)
                if (c * 32 + lane < DV) o[c] = fmaf(head[1][(long long)i * size + 2 + c * 32 + lane], w1, fmaf(head[0][(long long)i * size + 2 + c * 32 + lane], w0, o[c]));
        }
        float f = 1.f;
        if (p.gain) {
            float ss = 0.f;
#pragma unroll
            for (int c = 0; c < C; c++) ss = fmaf(o[c], o[c], ss);  // dimensions that are padding are 0
            f = 1.f / sqrtf(warp_sum(ss) / (float)p.vdim + p.head_eps);
        }
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int i = c * 32 + lane;
            if (i < p.vdim) out[r * p.vdim + i] = __float2bfloat16_rn(p.gain ? o[c] * f * p.gain[i] : o[c]);
        }
    }
}

// Grid: (splits, kv_heads · groups of 8 query heads, sequences). Both maps of eight heads of one key head share each tile of 16 keys and values, which a warp copies for itself.
template <int DM, int DV, bool LOW> __global__ void __launch_bounds__(kDecThreads) differential_decode(const DiffP p) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ unsigned arrived;
    __shared__ int page_s[kDecPages];  // this CTA's pages, checked
    using L = DecSmem<DM, DV>;
    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g8 = lane >> 2, t4 = lane & 3;
    // no launch of a step writes the batch description or the keys and values of earlier steps (where the module computes the
    // former, this launch does not begin early): they may be read while the launches before this one finish
    const int seq = blockIdx.z;
    const SeqRow sq = checked_seq(p, seq);
    const int rep = p.heads / p.kv_heads, groups = (rep + kDecHeads - 1) / kDecHeads, g = blockIdx.y / groups, h0 = g * rep + (blockIdx.y % groups) * kDecHeads;
    const int n_heads = min(kDecHeads, (g + 1) * rep - h0), pos = sq.past, dim = p.dim, vdim = p.vdim;
    const bf16* x = (const bf16*)p.proj + (long long)sq.start * p.ld;
    bf16 *keys = (bf16*)p.keys, *values = (bf16*)p.values;
    const unsigned sm0 = smem_u32(smem);
    double *cs = reinterpret_cast<double*>(smem + L::angle), *sn = cs + DM / 2;

    // keys of this CTA: whole tiles of all four warps, so that a split never cuts a tile
    constexpr int step = kDecKeys * kDecWarps;
    const int low = first_key(p, pos), base = low / step, blocks = sq.len == 1 ? pos / step + 1 - base : 0;
    const int b0 = base + (int)((long long)blocks * blockIdx.x / p.splits), b1 = base + (int)((long long)blocks * (blockIdx.x + 1) / p.splits);
    const int lo = b0 * step, hi = min(b1 * step, pos + 1), from = max(lo, low);  // pages in front of the window may be anybody's
    const int page0 = from >> p.shift, n_pages = from < hi ? ((hi - 1) >> p.shift) - page0 + 1 : 0;
    for (int i = tid; i < min(n_pages, kDecPages); i += kDecThreads) page_s[i] = (int)page_of(p, seq, (page0 + i) << p.shift);
    const bool newest = hi == pos + 1 && lo < hi;  // this CTA's keys include the new one
    __syncthreads();
    auto page_at = [&](int j) {
        const int i = (j >> p.shift) - page0;
        return i < kDecPages ? (long long)page_s[i] : page_of(p, seq, j);
    };
    const unsigned ring = sm0 + L::kv + warp * L::stages * L::tile;
    const int first = lo + warp * kDecKeys, tiles = first < hi ? (hi - first + step - 1) / step : 0;
    auto load_tile = [&](int i) {
        const int j0 = first + i * step;
        if (i < tiles) {
            const unsigned dst = ring + (i % L::stages) * L::tile;
            const bool whole = (1 << p.shift) >= kDecKeys;  // a tile lies in one page
            const long long row0 = whole && j0 + kDecKeys > from ? key_row(p, page_at(max(j0, from)), g, j0) : 0;
            constexpr int k_ch = DM / 4, v_ch = DV / 8;  // 16-byte pieces of a key and of a value
            if (whole && dim == DM && vdim == DV) {      // contiguous runs: a lane's copies are evenly spaced
                const bf16 *k = keys + row0 * 2 * DM + lane * 8, *v = values + row0 * DV + lane * 8;
#pragma unroll
                for (int c = 0; c < kDecKeys * k_ch / 32; c++) {
                    const int at = c * 32 + lane, j = j0 + at / k_ch;
                    const bool live = j >= from && j < hi;
                    cp_async16(dst + at / k_ch * L::k_stride + at % k_ch * 16, live ? k + c * 256 : keys, live);
                }
#pragma unroll
                for (int c = 0; c < kDecKeys * v_ch / 32; c++) {
                    const int at = c * 32 + lane, j = j0 + at / v_ch;
                    const bool live = j >= from && j < hi;
                    cp_async16(dst + kDecKeys * L::k_stride + at / v_ch * L::v_stride + at % v_ch * 16, live ? v + c * 256 : values, live);
                }
            } else {  // key by key, a lane per piece (what is padding was cleared before)
                const int pieces = dim / 8;
                const bool has_k = lane < 2 * pieces, has_v = lane < vdim / 8;
                const unsigned k_to = dst + lane * 16 + (lane >= pieces ? DM * 2 - dim * 2 : 0), v_to = dst + kDecKeys * L::k_stride + lane * 16;
#pragma unroll 4
                for (int key = 0; key < kDecKeys; key++) {
                    const int j = j0 + key;
                    const bool live = j >= from && j < hi;
                    const long long row = !live ? 0 : whole ? row0 + key : key_row(p, page_at(j), g, j);
                    if (has_k) cp_async16(k_to + key * L::k_stride, live ? keys + row * 2 * dim + lane * 8 : keys, live);
                    if (has_v) cp_async16(v_to + key * L::v_stride, live ? values + row * vdim + lane * 8 : values, live);
                }
            }
        }
        cp_async_commit();
    };
    if (dim != DM || vdim != DV) {  // what is padding stays 0
        for (int u = tid; u < kDecWarps * L::stages * L::tile / 16; u += kDecThreads) reinterpret_cast<uint4*>(smem + L::kv)[u] = make_uint4(0, 0, 0, 0);
        __syncthreads();
    }
    auto fill = [&]() {
#pragma unroll
        for (int i = 0; i < L::stages - 1; i++) load_tile(i);
    };
    // The first tiles are on their way while the launch before this one ends, unless the new key is among them.
    const bool late = newest && (pos - lo) / step < L::stages - 1;
    if (!late) fill();
    float *short_cs = reinterpret_cast<float*>(sn + DM / 2), *short_sn = short_cs + DM / 2;
    if (sq.len == 1 && warp < 2) short_angles(p, pos, short_cs, short_sn, tid, 64);
    if (newest && warp >= 2) exact_angles(p, pos, cs, sn, tid - 64, 64);
    pdl_wait();
    if (sq.len != 1) {
        if (p.only && sq.len > 1 && p.rows == p.n_seqs && tid == 0) report(p.err, ERR_BATCH_ROWS, p.node, seq, sq.len);
        return;
    }
    // all that comes from the projection at once
    bf16* raw = reinterpret_cast<bf16*>(smem + L::raw);
    const int q_rows = 2 * n_heads, raw_rows = q_rows + (newest ? 2 : 0);
    const long long row = newest ? key_row(p, page_at(pos), g, pos) : 0;
    auto source = [&](int r) { return r < q_rows ? x + p.q_off + (long long)(h0 * 2 + r) * dim : x + p.k_off + (long long)(g * 2 + r - q_rows) * dim; };
    if (p.by8) {
        const int chunks = dim / 8;
        for (int u = tid; u < raw_rows * chunks; u += kDecThreads) {
            const int r = u / chunks, c = u - r * chunks;
            reinterpret_cast<uint4*>(raw)[r * (DM / 8) + c] = reinterpret_cast<const uint4*>(source(r))[c];
        }
        if (newest)
            for (int u = tid; u < vdim / 8; u += kDecThreads) reinterpret_cast<uint4*>(values + row * vdim)[u] = reinterpret_cast<const uint4*>(x + p.v_off + (long long)g * vdim)[u];
    } else {
        for (int r = warp; r < raw_rows; r += kDecWarps)
            for (int i = lane; i < dim; i += 32) raw[r * DM + i] = source(r)[i];
        if (newest)
            for (int i = tid; i < vdim; i += kDecThreads) values[row * vdim + i] = x[p.v_off + (long long)g * vdim + i];
    }
    __syncthreads();
    if (newest) {
        // (where a key head has several groups of queries, each CTA that needs the new key writes it: the same bits)
        const int m = warp >> 1;  // two warps per map
        const bf16* k = raw + (q_rows + m) * DM;
        const float f = map_factor(p, k);
        for (int i = lane + (warp & 1) * 32; i < dim; i += 64) keys[(row * 2 + m) * dim + i] = __float2bfloat16_rn((float)(turned(p, k, cs, sn, i) * f));
        __syncthreads();
        if (late) fill();
    }
    auto put = [&](bf16* to, int i, float v) {
        const bf16 high = __float2bfloat16_rn(v);
        to[i] = high;
        to[kDecHeads * L::q_stride / 2 + i] = low_part(v, high);
    };
#pragma unroll
    for (int k = 0; k < 2 * kDecHeads / kDecWarps; k++) {
        const int r = k * kDecWarps + warp, m = r & 1, h = r >> 1;
        const bool live = h < n_heads;
        const bf16* q = raw + (live ? r : 0) * DM;
        const float f = live ? map_factor(p, q) : 0.f;
        bf16* to = reinterpret_cast<bf16*>(smem + L::q + (2 * m * kDecHeads + h) * L::q_stride);
        for (int i = lane; i < p.half; i += 32) {
            const float a = to_f(q[i]), b = to_f(q[i + p.half]), c = short_cs[i], n = short_sn[i];
            put(to, i, live ? (a * c - b * n) * f : 0.f);
            put(to, i + p.half, live ? (b * c + a * n) * f : 0.f);
        }
        for (int i = 2 * p.half + lane; i < DM; i += 32) put(to, i, live && i < dim ? to_f(q[i]) * f : 0.f);
    }
    __syncthreads();

    // Keys are the rows of both products (S^T = K q^T, O^T = V^T P^T): a lane holds scores of keys g, g + 8 and heads 2t, 2t + 1.
    float o[2][DV / 16][4];
    float top[2][2], l[2][2];
#pragma unroll
    for (int m = 0; m < 2; m++) {
        top[m][0] = top[m][1] = kNoScore;
        l[m][0] = l[m][1] = 0.f;
#pragma unroll
        for (int n = 0; n < DV / 16; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[m][n][e] = 0.f;
    }
    for (int i = 0; i < tiles; i++) {
        cp_async_wait<L::stages - 2>();
        __syncwarp();
        load_tile(i + L::stages - 1);  // the slot was read in the previous iteration
        const unsigned ks = ring + (i % L::stages) * L::tile, vs = ks + kDecKeys * L::k_stride;
        const int j0 = first + i * step;
        float s[2][4];
#pragma unroll
        for (int m = 0; m < 2; m++) {
#pragma unroll
            for (int e = 0; e < 4; e++) s[m][e] = 0.f;
#pragma unroll
            for (int kk = 0; kk < DM / 32; kk++) {
                unsigned high[4], low4[4];
                const unsigned at = sm0 + L::q + (2 * m * kDecHeads + (lane & 7)) * L::q_stride + kk * 64 + (lane >> 3) * 16;
                ldmatrix_x4(high, at);
                ldmatrix_x4(low4, at + kDecHeads * L::q_stride);
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    unsigned ka[4];
                    ldmatrix_x4(ka, ks + (lane & 15) * L::k_stride + m * DM * 2 + kk * 64 + half * 32 + (lane >> 4) * 16);
                    mma_bf16(s[m], ka[0], ka[1], ka[2], ka[3], high[2 * half], high[2 * half + 1]);
                    mma_bf16(s[m], ka[0], ka[1], ka[2], ka[3], low4[2 * half], low4[2 * half + 1]);
                }
            }
        }
        const bool edge = j0 + kDecKeys > hi || j0 < low;
        bool moved = false;
        float now[2][2];
#pragma unroll
        for (int m = 0; m < 2; m++) {
            now[m][0] = top[m][0];
            now[m][1] = top[m][1];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int j = j0 + g8 + 8 * (e >> 1);
                s[m][e] = edge && (j >= hi || j < low) ? -INFINITY : score2(p, s[m][e]);
                now[m][e & 1] = fmaxf(now[m][e & 1], s[m][e]);
            }
#pragma unroll
            for (int e = 0; e < 2; e++) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) now[m][e] = fmaxf(now[m][e], __shfl_xor_sync(0xffffffffu, now[m][e], d));
                moved |= now[m][e] != top[m][e];
            }
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const float keep = exp2f(top[m][e] - now[m][e]);
                    top[m][e] = now[m][e];
                    l[m][e] *= keep;
#pragma unroll
                    for (int n = 0; n < DV / 16; n++) {
                        o[m][n][e] *= keep;
                        o[m][n][e + 2] *= keep;
                    }
                }
        }
        unsigned pb[2][2], rest[2][2];
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const float w0 = exp2f(s[m][2 * r] - top[m][0]), w1 = exp2f(s[m][2 * r + 1] - top[m][1]);
                const unsigned w = pack_bf16(w0, w1);
                const float h0 = __uint_as_float(w << 16), h1 = __uint_as_float(w & 0xFFFF0000u);
                // the sums of the weights as they are multiplied: the rounding of a weight that stands out is in both
                l[m][0] += LOW ? w0 : h0;
                l[m][1] += LOW ? w1 : h1;
                pb[m][r] = transpose8x8(w);
                if constexpr (LOW) rest[m][r] = transpose8x8(pack_bf16(w0 - h0, w1 - h1));
            }
#pragma unroll
        for (int n = 0; n < DV / 16; n++) {
            unsigned va[4];
            ldmatrix_x4_trans(va, vs + ((lane >> 4) * 8 + (lane & 7)) * L::v_stride + n * 32 + ((lane >> 3) & 1) * 16);
#pragma unroll
            for (int m = 0; m < 2; m++) {
                mma_bf16(o[m][n], va[0], va[1], va[2], va[3], pb[m][0], pb[m][1]);
                if constexpr (LOW) mma_bf16(o[m][n], va[0], va[1], va[2], va[3], rest[m][0], rest[m][1]);
            }
        }
        __syncwarp();
    }
    cp_async_wait<0>();
    __syncthreads();  // the ring becomes the merge area
    float* parts = reinterpret_cast<float*>(smem + L::kv);
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) l[m][e] += __shfl_xor_sync(0xffffffffu, l[m][e], d);
            float* to = parts + warp * L::part + (m * kDecHeads + t4 * 2 + e) * (DV + 2);
            if (g8 == 0) {
                to[0] = top[m][e];
                to[1] = l[m][e];
            }
#pragma unroll
            for (int n = 0; n < DV / 16; n++) {
                to[2 + n * 16 + g8] = o[m][n][e];
                to[2 + n * 16 + g8 + 8] = o[m][n][e + 2];
            }
        }
    __syncthreads();
    bf16* out = (bf16*)p.out + ((long long)sq.start * p.heads + h0) * vdim;
    if (p.splits == 1) {
        merge_maps<DV>(p, parts, kDecWarps, h0, n_heads, out);
        return;
    }
    const long long cell = (long long)blockIdx.z * gridDim.y + blockIdx.y;
    for (int m = 0; m < 2; m++)
        merge_parts<DV, 2 * kDecHeads, kDecWarps>(parts + m * kDecHeads * (DV + 2), kDecWarps, n_heads, vdim, 0.f, nullptr, p.part + (cell * p.splits + blockIdx.x) * L::part + m * kDecHeads * (DV + 2));
    __threadfence();
    __syncthreads();
    if (tid == 0) arrived = atomicAdd(&p.counters[cell], 1u);
    __syncthreads();
    if (arrived != (unsigned)p.splits - 1) return;
    __threadfence();
    if (tid == 0) p.counters[cell] = 0;
    merge_maps<DV>(p, p.part + cell * p.splits * L::part, p.splits, h0, n_heads, out);
}

using DiffKernel = void (*)(const DiffP);
struct DecChoice {
    DiffKernel kernel;
    int smem, part;
};
template <int DM, int DV> DecChoice choice(bool low) { return {low ? differential_decode<DM, DV, true> : differential_decode<DM, DV, false>, DecSmem<DM, DV>::total, DecSmem<DM, DV>::part}; }
template <int DM> DecChoice choice(int64_t vdim, bool low) { return vdim <= 64 ? choice<DM, 64>(low) : vdim <= 128 ? choice<DM, 128>(low) : choice<DM, 256>(low); }

}  // namespace

void emit_differential(Emitter& em, const DifferentialDesc& d, const TRef& proj, const TRef& turns, const TRef& keys, const TRef& values, const TRef& seqs,
                       const TRef& pages, const TRef& lambda, const TRef* gain, const TRef& out) {
    const int64_t rows = proj.shape[0], n_seqs = seqs.shape[0];
    if (rows == 0 || n_seqs == 0) return;
    if (keys.shape[0] == 0) throw std::runtime_error("differential attention: new tokens, and pools without a page");
    DiffP p{};
    p.rows = rows;
    p.ld = proj.shape[1];
    p.q_off = d.q_off;
    p.k_off = d.k_off;
    p.v_off = d.v_off;
    p.n_seqs = (int)n_seqs;
    p.width = (int)pages.shape[1];
    p.n_pages = (int)keys.shape[0];
    while ((int64_t)1 << p.shift < d.page) p.shift++;
    p.heads = (int)d.heads;
    p.kv_heads = (int)d.kv_heads;
    p.dim = (int)d.dim;
    p.vdim = (int)d.vdim;
    p.half = (int)(d.rot_dims / 2);
    p.window = (int)d.window;
    p.node = em.node;
    p.scale = (float)d.scale;
    p.cap = (float)d.softcap;
    p.eps = (float)d.eps;
    p.head_eps = (float)d.head_eps;
    p.norm = d.norm;
    p.sink = d.sink;
    p.cap2 = (float)(d.softcap * (double)kLog2e);
    p.mul2 = (float)(d.softcap > 0 ? 2.0 * (double)kLog2e * d.scale / d.softcap : (double)kLog2e * d.scale);
    p.splits = 1;
    const bool bf = proj.dtype == DT_BF16;
    // 16-byte copies of key and value rows
    const bool tc = bf && d.dim % 8 == 0 && d.vdim % 8 == 0 && d.dim <= 128 && d.vdim <= 256 && keys.buf.off % 16 == 0 && values.buf.off % 16 == 0 && n_seqs <= 65535;
    p.only = tc && rows <= n_seqs;                     // every sequence has one new token, or none; with fewer rows than sequences some may have more (differential_several)
    p.singles = !tc || (!p.only && n_seqs == 1);       // a lone token with rows of nobody behind it
    const bool prefill = tc && !p.only && differential_prefill_fits(p, keys, values, out.buf.off);
    p.parts = prefill;
    // Weights as the sum of two bf16 where scores are known not to spread: of queries and keys that are normed (their products spread by dim^1/2) or of a tight cap. Nearly equal weights of two maps cancel,
    // their roundings do not. Off from 64-bit results with one bf16 → with two (1 500 keys): normed, scores of a spread of 1 2.5e-3 → 1.66e-3 (prompts), 2.3e-3 → 1.66e-3 (tokens), which is the results' own
    // rounding; of 1.25 2.4e-3, of 2 2.2e-3, without a norm and of 1.5 2.3e-3; capped at 1 2.66e-3, at 2 2.64e-3. Time, one after the other: 4096 tokens, 32 heads of 2 x 64 over 16 393 → 475 us,
    // normed 464 → 528; 2048, 16 over 4 79 → 86, normed 92 → 104; 1999 capped and normed behind 1000, 4 heads of 2 x 128 77 → 89; 64 tokens behind 2047, 32 over 16 212 → 224, other tokens 1 %.
    p.low = (d.norm && std::fabs(d.scale) * std::sqrt((double)d.dim) <= 1.25) || (d.softcap > 0 && d.softcap <= 3.0);
    auto by = [](int64_t d) { return d > 1 ? (unsigned)(((1ull << 32) + d - 1) / d) : 0u; };
    p.rep = d.heads / d.kv_heads;
    p.by_rep = by(p.rep);
    p.by_units = by(d.dim / 8 - d.rot_dims / 16);
    p.by_lanes = by(d.vdim / 8);
    p.by8 = p.ld % 8 == 0 && d.q_off % 8 == 0 && d.k_off % 8 == 0 && d.v_off % 8 == 0 && proj.buf.off % 16 == 0;
    const Buf none{kSlotNull, 0}, q = p.only ? none : em.scratch((size_t)rows * d.heads * 2 * d.dim * (bf && !prefill ? 2 : 4));
    auto launch = [&](DiffKernel k, dim3 grid, unsigned block, unsigned smem, Buf part, const char* label) {
        em.launch(k, grid, dim3(block), smem, p,
                  {{&p.proj, proj.buf}, {&p.turns, turns.buf}, {&p.keys, keys.buf}, {&p.values, values.buf}, {&p.q, q}, {&p.out, out.buf}, {&p.seqs, seqs.buf}, {&p.table, pages.buf},
                   {&p.lambda, lambda.buf}, {&p.gain, gain ? gain->buf : none}, {&p.part, part}, {&p.counters, Buf{kSlotCounters, 0}}, {&p.err, Buf{kSlotErr, 0}}},
                  label, /*pdl=*/true);
    };
    if (!p.only) {
        const int64_t eight = d.rot_dims * 12 + (d.norm ? 2 * (d.heads + d.kv_heads) : 0) * 4;  // bytes that the kernel for eight at a time shares; a block may have 48 KB
        if (tc && p.by8 && d.rot_dims % 16 == 0 && d.heads <= 4096 && eight <= 48 * 1024) launch(differential_prepare8, dim3((unsigned)rows), 128, (unsigned)eight, none, "differential_prepare");
        else {
            const DiffKernel prepare = bf ? differential_prepare<bf16> : differential_prepare<float>;
            ensure_max_dynamic_smem((const void*)prepare, 8192 * 8);
            launch(prepare, dim3((unsigned)rows), 128, (unsigned)(d.rot_dims * 8), none, "differential_prepare");
        }
        if (prefill) {
            emit_differential_prefill(em, p, keys, values,
                                      {{offsetof(DiffP, q), q}, {offsetof(DiffP, out), out.buf}, {offsetof(DiffP, seqs), seqs.buf}, {offsetof(DiffP, table), pages.buf},
                                       {offsetof(DiffP, lambda), lambda.buf}, {offsetof(DiffP, gain), gain ? gain->buf : none}, {offsetof(DiffP, err), Buf{kSlotErr, 0}}});
        } else {
            const DiffKernel k = bf ? differential_simt<bf16> : differential_simt<float>;
            ensure_max_dynamic_smem((const void*)k, 220 * 1024);
            launch(k, dim3((unsigned)rows, (unsigned)d.heads), kAnyKeys, (unsigned)((d.dim + d.vdim + kAnyKeys) * 8), none, "differential_simt");
        }
    }
    if (p.only && rows > 1 && rows < n_seqs) launch(differential_several, dim3((unsigned)d.kv_heads, (unsigned)n_seqs), kAnyKeys, (unsigned)((d.dim + d.vdim + kAnyKeys) * 8 + d.rot_dims * 8), none, "differential_several");
    if (tc && (p.only || n_seqs > 1)) {
        const DecChoice dc = d.dim <= 32 ? choice<32>(d.vdim, p.low) : d.dim <= 64 ? choice<64>(d.vdim, p.low) : choice<128>(d.vdim, p.low);
        const int64_t groups = d.kv_heads * ((d.heads / d.kv_heads + kDecHeads - 1) / kDecHeads), cells = n_seqs * groups;
        // Splits of the most keys a sequence can see: whole waves of resident CTAs, and the pieces have to be merged. A CTA's beginning and end cost as much as 200 KB of keys and values
        // (64 sequences behind 2047, 32 heads of 2 x 64 over 16, us for 1, 2, 4, 8 splits: 223, 246, 291, 369; four that see 4096 keys: 90, 60, 52, 58).
        const int64_t resident = std::max<int64_t>(1, std::min<int64_t>(3, 224 * 1024 / (dc.smem + 2560))), slots = resident * sm_count();
        int64_t seen = (int64_t)p.width * d.page;
        if (d.window > 0) seen = std::min<int64_t>(seen, d.window + 64);
        int64_t splits = 1;
        const double fixed = 100.0 * 1024.0 / (2 * d.dim + d.vdim);
        double best = 1e300;
        for (int64_t sp = 1; sp <= 64 && sp * 64 <= std::max<int64_t>(seen, 64); sp++) {
            const double us = (double)((cells * sp + slots - 1) / slots) * ((double)seen / sp + fixed) + 4.0 * sp;
            if (us < best) {
                best = us;
                splits = sp;
            }
        }
        if (cells > (int64_t)kCounterWords) splits = 1;
        p.splits = (int)splits;
        const Buf part = splits > 1 ? em.scratch((size_t)cells * splits * dc.part * 4) : none;
        ensure_max_dynamic_smem((const void*)dc.kernel, dc.smem);
        launch(dc.kernel, dim3((unsigned)splits, (unsigned)groups, (unsigned)n_seqs), kDecThreads, (unsigned)dc.smem, part, "differential_decode");
    }
}

}  // namespace oxk
