// Keys and values in 4 bits over paged pools (packed_cache.cuh has the format): written, read back, and attended to by ragged batches.
//
//   score(i, j) = cap(scale · q_i · k_j) for 0 ≤ i − j < window,  cap(s) = c · tanh(s / c),
//   out_i = Σ_j exp(score) v_j / ([exp(0)] + Σ_j exp(score))
//
// with k_j and v_j as they are stored, those of the step itself too. Queries and keys rotate and are normed as in paged_kv_attention.cu.
//
//   packed_write   a batch's keys (rotated, normed) and values go to the pools; its queries, where there are any, are prepared
//   packed_read    the keys and values of given places, side by side
//   packed_decode  sequences with one new token in bf16, all of the above in one launch (packed_decode.cu)
//   packed_prefill sequences with several new tokens in bf16 (packed_prefill.cu)
//   packed_simt    attention of any shape, f32 and bf16
#include <cfloat>
#include <cmath>

#include "packed_cache.cuh"

namespace oxk {

namespace {

// One CTA per row, one warp per query, key or value of a head. For f32, and for bf16 of odd widths or offsets: angles, rotation and norms in 64 bits, which bound it (4096 tokens of 32 + 16 heads of 128: 206 us; packed_write8 42).
template <typename T> __global__ void __launch_bounds__(128) packed_write(const PackP p) {
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
    const long long pg = p.append ? page_of(p, s, pos) : 0;
    for (int h = threadIdx.x >> 5; h < p.heads + (p.append ? 2 * p.kv_heads : 0); h += 4) {
        const int g = h - p.heads;
        if (g < 0) {
            const T* src = x + p.q_off + (long long)h * p.dim;
            const long long at = (long long)row * p.heads + h;
            const double f = norm_factor(p, src);
            auto value = [&](int i) { return (float)(turned(p.half, src, angle, angle + p.half, i) * f); };
            if (p.q_mul) {
                float top = 0.f;
                for (int i = lane; i < p.dim; i += 32) top = fmaxf(top, fabsf(value(i)));
                const int e = query_exponent(warp_max(top));
                __half* q = (__half*)p.q + at * p.dim;
                for (int i = lane; i < p.dim; i += 32) q[i] = __float2half_rn(copysignf(1.f, p.mul2) * value(i) * power_down(e));
                if (lane == 0) p.q_mul[at] = fabsf(p.mul2) * power_up(e) * key_factor(p, h / (p.heads / p.kv_heads));
            } else {
                for (int i = lane; i < p.dim; i += 32) ((float*)p.q)[at * p.dim + i] = value(i);
            }
        } else if (g < p.kv_heads) {
            const T* src = x + p.k_off + (long long)g * p.dim;
            unsigned char* to = held(p, p.keys, pg, g, p.dim);
            const double f = norm_factor(p, src);
            put_head(codes_of(p, to, pos, p.dim), scales_of(p, to, pos, p.dim), p.dim, key_factor(p, g),
                     [&](int i) { return to_f(from_f<T>((float)(turned(p.half, src, angle, angle + p.half, i) * f))); });
        } else {
            const T* src = x + p.v_off + (long long)(g - p.kv_heads) * p.vdim;
            unsigned char* to = held(p, p.values, pg, g - p.kv_heads, p.vdim);
            put_head(codes_of(p, to, pos, p.vdim), scales_of(p, to, pos, p.vdim), p.vdim, value_factor(p, g - p.kv_heads), [&](int i) { return to_f(src[i]); });
        }
    }
}

// The same in bf16 eight elements at a time, where heads, rotated halves and rows allow it: a unit is eight pairs that turn (all of them, ALL) or eight elements that do not, two neighbours share their
// scales. Angles, and keys where that says which bf16 they are, in 32 bits. 4096 tokens of 32 + 16 + 16 heads of 128: 67 MB read, 51 MB written in 42 us (2.8 TB/s; by the device's clock, events have 45); without queries (read 33.6 MB, 9.4 written) 29 us. The 1560
// instructions of a warp take 62 % of the issue slots, the rest is the chain from the sequence's lookup over angles to scales.
template <bool ALL, bool NORM> __global__ void __launch_bounds__(128, 8) packed_write8(const PackP p) {
    extern __shared__ __align__(16) float cs[];  // cosines [half], sines [half], norms of keys [kv_heads] in 64 bits, of queries [heads], with queries as f16 their largest elements [heads]
    pdl_enter();
    const int row = blockIdx.x, tid = threadIdx.x;
    // the row's queries, keys and values are on their way while its sequence is looked up and its angles are made
    const bf16* x = (const bf16*)p.proj + (long long)row * p.ld;
    const bf16 *from_q = x + p.q_off, *from_k = x + p.k_off, *from_v = x + p.v_off;
    auto fetch = [&](const bf16* from, int n) {
        for (int i = tid * 64; i < n; i += 128 * 64) asm volatile("prefetch.global.L1 [%0];" ::"l"(from + i) : "memory");
    };
    fetch(from_q, p.heads * p.dim);
    if (p.append) fetch(from_k, p.kv_heads * p.dim), fetch(from_v, p.kv_heads * p.vdim);
    const int s = find_seq(p.seqs, p.n_seqs, row);
    const SeqRow sq = checked_seq(p, s);
    check_others(p, row, tid, 128);
    const int pos = sq.past + row - sq.start, kv = p.append ? p.kv_heads : 0, half = p.half;
    if (row < sq.start || row >= sq.start + sq.len || (sq.len == 1 && !p.singles)) return;
    float* sn = cs + half;
    double* norms = reinterpret_cast<double*>(sn + half);
    float* query_norm = reinterpret_cast<float*>(norms + p.kv_heads);
    unsigned* query_top = reinterpret_cast<unsigned*>(query_norm + p.heads);
    for (int i = tid; i < half; i += 128) short_angle(pos, (double)p.turns[i] + (double)p.turns[half + i], cs + i, sn + i);
    const int turned = half / 8, units = p.dim / 8 - turned, runs = p.vdim / 8, eighths = p.dim / 8;
    if (NORM)
        for (int h0 = tid >> 5; h0 < p.heads + kv; h0 += 4 * 32) {  // a warp sums up to 32 heads, then has a root and a quotient for each lane
            const int h = h0 + 4 * (tid & 31);
            double mine = 0.0;
#pragma unroll 4
            for (int j = 0; j < 32; j++) {
                const int other = h0 + 4 * j;
                if (other >= p.heads + kv) break;
                const double ss = square_sum(p, other < p.heads ? from_q + other * p.dim : from_k + (other - p.heads) * p.dim);
                if (j == (tid & 31)) mine = ss;
            }
            if (h < p.heads + kv) {
                const double f = norm_of(p, mine);
                h < p.heads ? (void)(query_norm[h] = (float)f) : (void)(norms[h - p.heads] = f);
            }
        }
    auto wide = [](const bf16* from, float (&v)[8]) {
        const uint4 u = *reinterpret_cast<const uint4*>(from);
        const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; e++) v[2 * e] = __uint_as_float(w[e] << 16), v[2 * e + 1] = __uint_as_float(w[e] & 0xFFFF0000u);
    };
    if (p.q_mul) {  // (a rotation makes no element larger than sqrt 2 times the largest)
        for (int h = tid; h < p.heads; h += 128) query_top[h] = 0;
        __syncthreads();
        for (int u = tid; u < p.heads * eighths; u += 128) {
            const uint4 v = *reinterpret_cast<const uint4*>(from_q + u * 8);
            auto most = [](unsigned a, unsigned b) { return __vmaxu2(a & 0x7FFF7FFFu, b & 0x7FFF7FFFu); };  // magnitudes are ordered as their bits
            const unsigned m = __vmaxu2(most(v.x, v.y), most(v.z, v.w));
            atomicMax(query_top + over(u, p.by_eighths), max(m << 16, m & 0xFFFF0000u));
        }
    }
    __syncthreads();
    for (int u = tid; u < p.heads * units; u += 128) {
        const int h = over(u, p.by_units), i = u - h * units;
        const bool turns = ALL || i < turned;
        const int at = turns ? i * 8 : (i + turned) * 8;
        const bf16* src = from_q + h * p.dim + at;
        const long long to = ((long long)row * p.heads + h) * p.dim + at;
        float f = NORM ? query_norm[h] : 1.f;
        if (p.q_mul) {
            const int e = query_exponent(__uint_as_float(query_top[h]) * f);
            f *= copysignf(power_down(e), p.mul2);
            if (i == 0) p.q_mul[(long long)row * p.heads + h] = fabsf(p.mul2) * power_up(e) * key_factor(p, over(h, p.by_rep));
        }
        auto put = [&](long long at, const float (&v)[8]) {
            if (p.q_mul) {
                unsigned w[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const __half2 two = __floats2half2_rn(v[2 * e], v[2 * e + 1]);
                    w[e] = *reinterpret_cast<const unsigned*>(&two);
                }
                *reinterpret_cast<uint4*>((__half*)p.q + at) = make_uint4(w[0], w[1], w[2], w[3]);
            } else {
                float4* q = reinterpret_cast<float4*>((float*)p.q + at);
                q[0] = make_float4(v[0], v[1], v[2], v[3]);
                q[1] = make_float4(v[4], v[5], v[6], v[7]);
            }
        };
        float a[8], b[8], o[8];
        wide(src, a);
#pragma unroll
        for (int e = 0; e < 8; e++) a[e] *= f;
        if (!turns) {
            put(to, a);
            continue;
        }
        wide(src + half, b);
        const float4 *c4 = reinterpret_cast<const float4*>(cs + at), *n4 = reinterpret_cast<const float4*>(sn + at);
        const float4 c0 = c4[0], c1 = c4[1], n0 = n4[0], n1 = n4[1];
        const float c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w}, n[8] = {n0.x, n0.y, n0.z, n0.w, n1.x, n1.y, n1.z, n1.w};
#pragma unroll
        for (int e = 0; e < 8; e++) b[e] *= f, o[e] = a[e] * c[e] - b[e] * n[e];
        put(to, o);
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] = b[e] * c[e] + a[e] * n[e];
        put(to + half, o);
    }
    if (!p.append) return;
    const long long pg = page_of(p, s, pos);
    const int off = pos & ((1 << p.shift) - 1), key_head = (p.dim / kPack * 9) << p.shift, value_head = (p.vdim / kPack * 9) << p.shift;
    unsigned char *keys = p.keys + pg * p.kv_heads * key_head, *values = p.values + pg * p.kv_heads * value_head;
    // eight dimensions from `at` on; the lane next to this one has the other eight of their scale
    auto store = [&](unsigned char* to, int dim, int at, float (&v)[8], float factor, bool in) {
        const bool plain = factor == 1.f;
        if (!plain)
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] /= factor;
        float a = 0.f;
#pragma unroll
        for (int e = 0; e < 8; e++) a = max_nan(a, fabsf(v[e]));
        const unsigned code = scale_code(max_nan(a, __shfl_xor_sync(0xffffffffu, a, 1)));
        const float scale = scale_value(code);
        // (an infinite value over a scale that is none would be no number)
        if (plain && scale > 0.f) {
            const float by = __frcp_rn(scale);
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = near_scale(v[e], by);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = over_scale(v[e], scale);
        }
        if (!in) return;
        *reinterpret_cast<unsigned*>(to + (off * dim + at) / 2) = codes8(v);
        if (at % kPack == 0) to[((dim / 2) << p.shift) + (off * dim + at) / kPack] = (unsigned char)code;
    };
    for (int u0 = 0; u0 < kv * units; u0 += 128) {
        const bool in = u0 + tid < kv * units;
        const int u = in ? u0 + tid : tid & 1, g = over(u, p.by_units), i = u - g * units;
        const bool turns = ALL || i < turned;
        const int at = turns ? i * 8 : (i + turned) * 8;
        const bf16* src = from_k + g * p.dim + at;
        unsigned char* to = keys + g * key_head;
        const double f = NORM ? norms[g] : 1.0;
        const float factor = key_factor(p, g), short_f = (float)f;
        float a[8], b[8], second[8] = {}, size[8];
        wide(src, a);
        // In 32 bits a key is off by less than 2^-21 of its pair; where that leaves open which bf16 it is, or the pair is infinite, 64 bits say. (One element of 4000.)
        auto rounded = [&](float (&v)[8], auto&& exact) {
            unsigned open = 0;
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const unsigned less = pack_bf16(__fmaf_rn(size[e], -0x1p-21f, v[e]), __fmaf_rn(size[e + 1], -0x1p-21f, v[e + 1]));
                const unsigned more = pack_bf16(__fmaf_rn(size[e], 0x1p-21f, v[e]), __fmaf_rn(size[e + 1], 0x1p-21f, v[e + 1]));
                const unsigned other = less ^ more;
                open |= (other & 0xFFFFu ? 1u << e : 0u) | (other >> 16 ? 2u << e : 0u);
                v[e] = __uint_as_float(less << 16);
                v[e + 1] = __uint_as_float(less & 0xFFFF0000u);
            }
            if (open) {
#pragma unroll 1
                for (int e = 0; e < 8; e++) {
                    if (!(open >> e & 1)) continue;
                    const float w = __bfloat162float(__float2bfloat16_rn((float)exact(e)));
#pragma unroll
                    for (int k = 0; k < 8; k++)
                        if (k == e) v[k] = w;
                }
            }
        };
        auto turn = [&](int e, double* c, double* n) {
            const double t = (double)pos * ((double)p.turns[at + e] + (double)p.turns[half + at + e]) * 2.0;
            sincospi(t - 2.0 * rint(0.5 * t), n, c);
        };
        if (turns) {
            wide(src + half, b);
            const float4 *c4 = reinterpret_cast<const float4*>(cs + at), *n4 = reinterpret_cast<const float4*>(sn + at);
            const float4 c0 = c4[0], c1 = c4[1], n0 = n4[0], n1 = n4[1];
            const float c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w}, n[8] = {n0.x, n0.y, n0.z, n0.w, n1.x, n1.y, n1.z, n1.w};
            if (NORM)
#pragma unroll
                for (int e = 0; e < 8; e++) a[e] *= short_f, b[e] *= short_f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float first = a[e] * c[e] - b[e] * n[e];
                size[e] = fabsf(a[e]) + fabsf(b[e]);
                second[e] = b[e] * c[e] + a[e] * n[e];
                a[e] = first;
            }
            rounded(a, [&](int e) {
                double ec, en;
                turn(e, &ec, &en);
                return ((double)to_f(src[e]) * ec - (double)to_f(src[e + half]) * en) * f;
            });
            rounded(second, [&](int e) {
                double ec, en;
                turn(e, &ec, &en);
                return ((double)to_f(src[e + half]) * ec + (double)to_f(src[e]) * en) * f;
            });
        } else if (NORM) {
#pragma unroll
            for (int e = 0; e < 8; e++) size[e] = fabsf(a[e]) * short_f, a[e] *= short_f;
            rounded(a, [&](int e) { return (double)to_f(src[e]) * f; });
        }
        // (all lanes come)
        store(to, p.dim, at, a, factor, in);
        if (ALL || turned > 0) store(to, p.dim, at + half, second, factor, in && turns);
    }
    for (int u0 = 0; u0 < kv * runs; u0 += 128) {
        const bool in = u0 + tid < kv * runs;
        const int u = in ? u0 + tid : tid & 1, g = over(u, p.by_runs), at = (u - g * runs) * 8;
        float a[8];
        wide(from_v + u * 8, a);
        store(values + g * value_head, p.vdim, at, a, value_factor(p, g), in);
    }
}

// ── reading back ──
struct ReadP {
    unsigned char *keys, *values;
    const int* places;  // [rows, 2]: row of the page table, position
    const int* table;   // [R, width]
    void* out;          // [rows, kv_heads · (dim + vdim)]
    const float *key_factors, *value_factors;
    ErrWord* err;
    long long rows;
    int n_seqs, width, n_pages, shift, kv_heads, dim, vdim, node;
    int per;                              // places of a CTA
    unsigned by_all, by_key, by_value;    // for over(): blocks of 16 dimensions of a place, of a key, of a value
};
constexpr int kReadThreads = 256, kReadRows = 64;

// A CTA has a run of places, a thread sixteen dimensions at a time: two stores of 16 bytes in bf16. 32768 places of 16 heads of 128 + 128: 75 MB read, 268 MB written in 60 us, calls one behind the other (5.7 TB/s; a launch between events 73); stores
// element by element took 791.
template <typename T> __global__ void __launch_bounds__(kReadThreads) packed_read(const ReadP p) {
    __shared__ int page_s[kReadRows], pos_s[kReadRows];
    pdl_enter();
    const long long row0 = (long long)blockIdx.x * p.per;
    const int rows = (int)min((long long)p.per, p.rows - row0), keys = p.kv_heads * (p.dim / kPack), all = keys + p.kv_heads * (p.vdim / kPack);
    for (int r = threadIdx.x; r < rows; r += kReadThreads) {
        const int2 at = reinterpret_cast<const int2*>(p.places)[row0 + r];
        int pg = -1;
        if ((unsigned)at.x >= (unsigned)p.n_seqs || at.y < 0) report(p.err, ERR_GATHER_OOB, p.node, (unsigned)at.x >= (unsigned)p.n_seqs ? at.x : at.y, p.n_seqs);
        else {
            const int i = at.y >> p.shift, given = i < p.width ? p.table[(long long)at.x * p.width + i] : -1;
            if ((unsigned)given >= (unsigned)p.n_pages) report(p.err, ERR_GATHER_OOB, p.node, given, p.n_pages);
            else pg = given;
        }
        page_s[r] = pg;
        pos_s[r] = at.y;
    }
    __syncthreads();
    T* out = (T*)p.out + row0 * all * kPack;
#pragma unroll 4
    for (int u = threadIdx.x; u < rows * all; u += kReadThreads) {
        const int r = over(u, p.by_all), v = u - r * all, pg = page_s[r], pos = pos_s[r];
        const bool of_key = v < keys;
        const int dim = of_key ? p.dim : p.vdim, w = of_key ? v : v - keys, g = over(w, of_key ? p.by_key : p.by_value), b = w - g * (dim / kPack);
        uint2 codes = make_uint2(0, 0);
        unsigned scale = 0;
        float f = 1.f;
        if (pg >= 0) {
            unsigned char* from = held(p, of_key ? p.keys : p.values, pg, g, dim);
            codes = reinterpret_cast<const uint2*>(codes_of(p, from, pos, dim))[b];
            scale = scales_of(p, from, pos, dim)[b];
            const float* factors = of_key ? p.key_factors : p.value_factors;
            if (factors) f = factors[g];
        }
        const __half2 s = __low2half2(scales_f16(scale));
        uint4* to = reinterpret_cast<uint4*>(out + (long long)u * kPack);
#pragma unroll
        for (int k = 0; k < 2; k++) {
            __half2 h[4];
            units8(k ? codes.y : codes.x, h);
            float2 x[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                x[e] = __half22float2(__hmul2(h[e], s));  // exact
                x[e].x *= f;
                x[e].y *= f;
            }
            if constexpr (sizeof(T) == 2) {
                to[k] = make_uint4(pack_bf16(x[0].x, x[0].y), pack_bf16(x[1].x, x[1].y), pack_bf16(x[2].x, x[2].y), pack_bf16(x[3].x, x[3].y));
            } else {
                auto four = [](float2 a, float2 b) { return make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y)); };
                to[2 * k] = four(x[0], x[1]);
                to[2 * k + 1] = four(x[2], x[3]);
            }
        }
    }
}

// ── attention of any shape ──
// A row's head by 128 threads: chunks of 128 keys, a thread per key, then a thread per value dimension. Nothing is shared between rows or heads: it is right for f32, dimensions beyond 256, more than 128 heads of a key and scales beyond
// 1024, where the tensor cores' f16 queries and weights would not hold the results. Slow where there is much to do (us a call, beside pools in f32 with onyxia.PagedKVAttention): 2048 tokens of 16 heads of 128 over 4 in f32 7200 (5900),
// one behind 8191 1400 (1500), 16 behind 8191 2500 (3500).
template <typename T> __global__ void __launch_bounds__(kAnyKeys) packed_simt(const PackP p) {
    extern __shared__ float sm[];  // q[dim], acc[vdim], w[128]
    __shared__ float red[32];
    __shared__ long long page_s[kAnyKeys];  // of each key of the chunk
    pdl_enter();
    const int row = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, s = find_seq(p.seqs, p.n_seqs, row), g = h / (p.heads / p.kv_heads);
    const SeqRow sq = checked_seq(p, s);
    if (row < sq.start || row >= sq.start + sq.len || (sq.len == 1 && !p.singles)) return;
    const int pos = sq.past + row - sq.start;
    float *q = sm, *acc = sm + p.dim, *w = acc + p.vdim;
    for (int i = tid; i < p.dim; i += kAnyKeys) q[i] = ((const float*)p.q)[((long long)row * p.heads + h) * p.dim + i];
    for (int i = tid; i < p.vdim; i += kAnyKeys) acc[i] = 0.f;
    // a sink is a score of 0 that has no value; without one the sums begin below every score
    float m = p.sink ? 0.f : kNone, l = p.sink ? 1.f : 0.f;
    const float scale = p.scale * key_factor(p, g);
    __syncthreads();
    for (int j0 = first_key(p, pos); j0 <= pos; j0 += kAnyKeys) {
        const int j = j0 + tid;
        float sc = -INFINITY;
        if (j <= pos) {
            const long long pg = page_of(p, s, j);
            page_s[tid] = pg;
            unsigned char* from = held(p, p.keys, pg, g, p.dim);
            const uint2* codes = reinterpret_cast<const uint2*>(codes_of(p, from, j, p.dim));
            const unsigned char* scales = scales_of(p, from, j, p.dim);
            float d = 0.f;
            for (int b = 0; b < p.dim / kPack; b++) {
                const uint2 c = codes[b];
                float one = 0.f;
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    __half2 v[4];
                    units8(k ? c.y : c.x, v);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float2 u = __half22float2(v[e]);
                        one = fmaf(q[b * kPack + k * 8 + 2 * e + 1], u.y, fmaf(q[b * kPack + k * 8 + 2 * e], u.x, one));
                    }
                }
                d = fmaf(one, scale_value(scales[b]), d);
            }
            sc = d * scale;
            if (p.cap > 0.f) sc = p.cap * tanhf(sc / p.cap);
        }
        const float top = fmaxf(m, block_max(sc, red)), x = expf(sc - top), keep = expf(m - top);
        w[tid] = x;
        l = l * keep + block_sum(x, red);  // (its barriers order the stores to w and to the pages)
        m = top;
        const int live = min(kAnyKeys, pos + 1 - j0);
        for (int i = tid; i < p.vdim; i += kAnyKeys) {
            float a = acc[i] * keep;
#pragma unroll 4
            for (int jj = 0; jj < live; jj++) {
                unsigned char* from = held(p, p.values, page_s[jj], g, p.vdim);
                const unsigned byte = codes_of(p, from, j0 + jj, p.vdim)[i / 2];
                __half2 v[4];
                units8(i & 1 ? byte >> 4 : byte & 15u, v);
                a = fmaf(w[jj], __low2float(v[0]) * scale_value(scales_of(p, from, j0 + jj, p.vdim)[i / kPack]), a);
            }
            acc[i] = a;
        }
        __syncthreads();
    }
    const float f = value_factor(p, g) / l;
    for (int i = tid; i < p.vdim; i += kAnyKeys) ((T*)p.out)[((long long)row * p.heads + h) * p.vdim + i] = from_f<T>(acc[i] * f);
}

}  // namespace

void emit_packed_attention(Emitter& em, const PackedDesc& d, const TRef& proj, const TRef& turns, const TRef& keys, const TRef& values, const TRef& seqs, const TRef& pages,
                           const TRef* key_factors, const TRef* value_factors, const TRef* out) {
    const int64_t rows = proj.shape[0], n_seqs = seqs.shape[0];
    if (rows == 0 || n_seqs == 0) return;
    if (keys.shape[0] == 0) throw std::runtime_error("packed keys and values: new tokens, and pools without a page");
    if (keys.buf.off % 16 || values.buf.off % 16) throw std::runtime_error("packed keys and values: pools begin on 16 bytes");
    PackP p{};
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
    // (a cap that f32 does not hold is the least that it does: 0 would be none)
    const double cap = d.softcap > 0 ? std::max(d.softcap, (double)FLT_MIN) : 0.0;
    p.cap = (float)cap;
    p.eps = d.eps;
    p.norm = d.norm;
    p.sink = d.sink;
    p.append = d.append;
    p.cap2 = (float)(cap * (double)kLog2e);
    p.mul2 = (float)(d.softcap > 0 ? 2.0 * (double)kLog2e * d.scale / d.softcap : (double)kLog2e * d.scale);
    // (rows of a prompt's CTA, scales of 64 keys)
    const int64_t most_heads = std::max(d.heads, d.kv_heads), units = d.dim / 8 - d.rot_dims / 16, cta_rows = 256, cta_keys = 64;
    p.by_rep = by_of(d.heads ? d.heads / d.kv_heads : 1, std::max(d.heads, cta_rows));
    p.by_units = by_of(units, most_heads * units);
    p.by_runs = by_of(d.vdim / 8, d.kv_heads * d.vdim / 8);
    p.by_key = by_of(d.dim / kPack, std::max(cta_keys * d.dim / kPack, cta_rows));
    p.by_value = by_of(d.vdim / kPack, std::max(cta_keys * d.vdim / kPack, cta_rows));
    p.by_eighths = by_of(d.dim / 8, d.heads * d.dim / 8);
    const bool bf = proj.dtype == DT_BF16, tc = out && bf && d.dim <= 256 && d.vdim <= 256 && n_seqs <= 65535 && n_seqs * d.heads <= INT32_MAX;
    p.only = tc && rows == n_seqs;
    // Prompts subtract a rounded score from products that are not: beyond 2^28 that leaves weights below f16's. Rounding them first costs 1.4 % of 4096 tokens of 32 heads over 16; what has a scale that
    // leads there is left to the other kernel.
    const bool prefill = tc && !p.only && (d.softcap > 0 || std::fabs(d.scale) <= 1024.0) && d.heads / d.kv_heads <= 128 && out->buf.off % 16 == 0 && rows * d.heads / 64 + n_seqs * d.kv_heads <= INT32_MAX;
    p.singles = !tc || (!p.only && n_seqs == 1);  // a lone token with rows of nobody behind it
    const Buf none{kSlotNull, 0}, q = out && !p.only ? em.scratch((size_t)rows * d.heads * d.dim * (prefill ? 2 : 4)) : none, q_mul = prefill ? em.scratch((size_t)rows * d.heads * 4) : none;
    auto launch = [&](PackKernel k, dim3 grid, unsigned block, unsigned smem, Buf part, const char* label) {
        em.launch(k, grid, dim3(block), smem, p,
                  {{&p.proj, proj.buf}, {&p.turns, turns.buf}, {&p.keys, keys.buf}, {&p.values, values.buf}, {&p.q, q}, {&p.q_mul, q_mul}, {&p.out, out ? out->buf : none}, {&p.seqs, seqs.buf},
                   {&p.table, pages.buf}, {&p.key_factors, key_factors ? key_factors->buf : none}, {&p.value_factors, value_factors ? value_factors->buf : none}, {&p.part, part},
                   {&p.counters, Buf{kSlotCounters, 0}}, {&p.err, Buf{kSlotErr, 0}}},
                  label, /*pdl=*/true);
    };
    p.by8 = p.ld % 8 == 0 && d.q_off % 8 == 0 && d.k_off % 8 == 0 && d.v_off % 8 == 0 && proj.buf.off % 16 == 0;
    if (!p.only) {
        // bytes that the kernel for eight at a time shares, of which a block may have 48 KB; it counts a page's bytes in 32 bits
        const int64_t eight = d.kv_heads * 8 + d.rot_dims * 4 + d.heads * 8;
        if (bf && p.by8 && d.rot_dims % 32 == 0 && eight <= 48 * 1024 && d.kv_heads * d.page * std::max(d.dim, d.vdim) < (int64_t)1 << 31) {
            const bool turns = d.rot_dims == d.dim;
            launch(d.norm ? (turns ? packed_write8<true, true> : packed_write8<false, true>) : turns ? packed_write8<true, false> : packed_write8<false, false>, dim3((unsigned)rows), 128, (unsigned)eight,
                   none, "packed_write");
        } else {
            const PackKernel write = bf ? packed_write<bf16> : packed_write<float>;
            ensure_max_dynamic_smem((const void*)write, 8192 * 8);
            launch(write, dim3((unsigned)rows), 128, (unsigned)(d.rot_dims * 8), none, "packed_write");
        }
        if (!out) return;
        if (prefill) {
            const int64_t rep = d.heads / d.kv_heads;
            const PackedPrefill pf = packed_prefill_of(d.dim, d.vdim, rows, d.kv_heads, rep, p.cap2);
            const int64_t tq = pf.rows / rep;
            p.raw_slots = pf.slots;
            ensure_max_dynamic_smem((const void*)pf.kernel, pf.smem);
            launch(pf.kernel, dim3((unsigned)(((rows + tq - 1) / tq + n_seqs) * d.kv_heads)), (unsigned)pf.threads, (unsigned)pf.smem, none, "packed_prefill");
        } else {
            const PackKernel k = bf ? packed_simt<bf16> : packed_simt<float>;
            ensure_max_dynamic_smem((const void*)k, 220 * 1024);
            launch(k, dim3((unsigned)rows, (unsigned)d.heads), kAnyKeys, (unsigned)((d.dim + d.vdim + kAnyKeys) * 4), none, "packed_simt");
        }
    }
    if (tc && (p.only || n_seqs > 1)) {
        const PackedDecode dc = packed_decode_of(d.dim, d.vdim);
        const int64_t groups = d.kv_heads * ((d.heads / d.kv_heads + dc.heads - 1) / dc.heads), cells = n_seqs * groups;
        // Pieces of the same number for every cell leave nobody a second one, which costs as much as a dozen blocks of 128 keys. With more cells than places, or places that would stay empty, CTAs share
        // all blocks evenly, but for cells without a counter each. us a call with pieces, shares, one behind the other (alone): 64 sequences up to 8192 long of 4 cells 57, 62 (101, 99); behind 8191 of 16 cells
        // each, 16 sequences 68, 71 (123, 114), 30 123, 128 (198, 175), 37 150, 150, 37 up to 8192 long 133, 140 (186, 198); 20 up to 8192 long, where this shares, 84, 83 (141, 128); 64, one CTA a cell, 290, 267.
        const int64_t places = (int64_t)dc.resident * sm_count(), blocks = ((int64_t)p.width * d.page + dc.step - 1) / dc.step + 1;
        const int64_t pieces = std::min<int64_t>({places / cells, blocks, dc.pieces});
        p.pieces = (int)(cells > (int64_t)kCounterWords ? 1 : pieces * cells * 5 >= places * 4 || pieces == blocks || pieces == dc.pieces ? pieces : 0);
        const int64_t ctas = p.pieces ? cells * p.pieces : std::min(places, cells * blocks);
        const Buf part = p.pieces == 1 ? none : em.scratch((size_t)ctas * 2 * dc.part * 4);
        ensure_max_dynamic_smem((const void*)dc.kernel, dc.smem);
        launch(dc.kernel, dim3((unsigned)ctas), 128, (unsigned)dc.smem, part, "packed_decode");
    }
}

void emit_packed_read(Emitter& em, const PackedDesc& d, const TRef& keys, const TRef& values, const TRef& places, const TRef& pages, const TRef* key_factors, const TRef* value_factors,
                      const TRef& out) {
    const int64_t rows = places.shape[0];
    if (rows == 0) return;
    if (keys.buf.off % 16 || values.buf.off % 16) throw std::runtime_error("packed keys and values: pools begin on 16 bytes");
    ReadP p{};
    p.rows = rows;
    p.n_seqs = (int)pages.shape[0];
    p.width = (int)pages.shape[1];
    p.n_pages = (int)keys.shape[0];
    while ((int64_t)1 << p.shift < d.page) p.shift++;
    p.kv_heads = (int)d.kv_heads;
    p.dim = (int)d.dim;
    p.vdim = (int)d.vdim;
    p.node = em.node;
    const int64_t blocks = d.kv_heads * (d.dim + d.vdim) / kPack;
    // eight blocks a thread, fewer where that leaves SMs without a CTA
    p.per = (int)std::max<int64_t>(1, std::min<int64_t>({kReadRows, 8 * kReadThreads / blocks, (rows + 2 * sm_count() - 1) / (2 * sm_count())}));
    p.by_all = p.per > 1 ? by_of(blocks, p.per * blocks) : 1u;  // (1: the quotient is 0, however many blocks the one place has)
    p.by_key = by_of(d.dim / kPack, d.kv_heads * d.dim / kPack);
    p.by_value = by_of(d.vdim / kPack, d.kv_heads * d.vdim / kPack);
    const Buf none{kSlotNull, 0};
    em.launch(out.dtype == DT_BF16 ? packed_read<bf16> : packed_read<float>, dim3((unsigned)((rows + p.per - 1) / p.per)), dim3(kReadThreads), 0, p,
              {{&p.keys, keys.buf}, {&p.values, values.buf}, {&p.places, places.buf}, {&p.table, pages.buf}, {&p.out, out.buf}, {&p.key_factors, key_factors ? key_factors->buf : none},
               {&p.value_factors, value_factors ? value_factors->buf : none}, {&p.err, Buf{kSlotErr, 0}}},
              "packed_read", /*pdl=*/true);
}

}  // namespace oxk
