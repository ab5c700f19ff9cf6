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
#include <cmath>

#include "packed_cache.cuh"

namespace oxk {

namespace {

// One CTA per row, one warp per query, key or value of a head.
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
                for (int i = lane; i < p.dim; i += 32) q[i] = __float2half_rn(value(i) * power_down(e));
                if (lane == 0) p.q_mul[at] = p.mul2 * power_up(e) * key_factor(p, h / (p.heads / p.kv_heads));
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
};

// A CTA per place, a thread per sixteen dimensions.
template <typename T> __global__ void __launch_bounds__(128) packed_read(const ReadP p) {
    pdl_enter();
    const long long row = blockIdx.x;
    const int seq = p.places[2 * row], pos = p.places[2 * row + 1], keys = p.kv_heads * p.dim / kPack, values = p.kv_heads * p.vdim / kPack;
    long long pg = -1;
    if ((unsigned)seq >= (unsigned)p.n_seqs || pos < 0) report(p.err, ERR_GATHER_OOB, p.node, seq < 0 || seq >= p.n_seqs ? seq : pos, p.n_seqs);
    else {
        const int i = pos >> p.shift;
        const int at = i < p.width ? p.table[(long long)seq * p.width + i] : -1;
        if ((unsigned)at >= (unsigned)p.n_pages) report(p.err, ERR_GATHER_OOB, p.node, at, p.n_pages);
        else pg = at;
    }
    T* out = (T*)p.out + row * (keys + values) * kPack;
    for (int u = threadIdx.x; u < keys + values; u += 128) {
        const bool of_key = u < keys;
        const int dim = of_key ? p.dim : p.vdim, v = of_key ? u : u - keys, g = v / (dim / kPack), b = v % (dim / kPack);
        float x[kPack];
        if (pg < 0) {
            for (int i = 0; i < kPack; i++) x[i] = 0.f;
        } else {
            unsigned char* from = held(p, of_key ? p.keys : p.values, pg, g, dim);
            const float* factors = of_key ? p.key_factors : p.value_factors;
            const float f = factors ? factors[g] : 1.f, s = scale_value(scales_of(p, from, pos, dim)[b]);
            const uint2 w = reinterpret_cast<const uint2*>(codes_of(p, from, pos, dim))[b];
#pragma unroll
            for (int k = 0; k < 2; k++) {
                __half2 h[4];
                units8(k ? w.y : w.x, h);
#pragma unroll
                for (int e = 0; e < 4; e++) x[k * 8 + 2 * e] = __low2float(h[e]) * s * f, x[k * 8 + 2 * e + 1] = __high2float(h[e]) * s * f;
            }
        }
#pragma unroll
        for (int i = 0; i < kPack; i++) out[u * kPack + i] = from_f<T>(x[i]);
    }
}

// ── attention of any shape ──
// A row's head by 128 threads: chunks of 128 keys, a thread per key, then a thread per value dimension.
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
    // a sink is a score of 0 that has no value; without one the sums begin below every score, at a number: differences stay numbers
    float m = p.sink ? 0.f : -1e30f, l = p.sink ? 1.f : 0.f;
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
    p.cap = (float)d.softcap;
    p.eps = d.eps;
    p.norm = d.norm;
    p.sink = d.sink;
    p.append = d.append;
    p.cap2 = (float)(d.softcap * (double)kLog2e);
    p.mul2 = (float)(d.softcap > 0 ? 2.0 * (double)kLog2e * d.scale / d.softcap : (double)kLog2e * d.scale);
    p.splits = 1;
    const bool bf = proj.dtype == DT_BF16, tc = out && bf && d.dim <= 256 && d.vdim <= 256 && n_seqs <= 65535;
    p.only = tc && rows == n_seqs;
    const bool prefill = tc && !p.only && d.heads / d.kv_heads <= 128 && out->buf.off % 16 == 0;
    p.singles = !tc || (!p.only && n_seqs == 1);  // a lone token with rows of nobody behind it
    const Buf none{kSlotNull, 0}, q = out && !p.only ? em.scratch((size_t)rows * d.heads * d.dim * (prefill ? 2 : 4)) : none, q_mul = prefill ? em.scratch((size_t)rows * d.heads * 4) : none;
    auto launch = [&](PackKernel k, dim3 grid, unsigned block, unsigned smem, Buf part, const char* label) {
        em.launch(k, grid, dim3(block), smem, p,
                  {{&p.proj, proj.buf}, {&p.turns, turns.buf}, {&p.keys, keys.buf}, {&p.values, values.buf}, {&p.q, q}, {&p.q_mul, q_mul}, {&p.out, out ? out->buf : none}, {&p.seqs, seqs.buf},
                   {&p.table, pages.buf}, {&p.key_factors, key_factors ? key_factors->buf : none}, {&p.value_factors, value_factors ? value_factors->buf : none}, {&p.part, part},
                   {&p.counters, Buf{kSlotCounters, 0}}, {&p.err, Buf{kSlotErr, 0}}},
                  label, /*pdl=*/true);
    };
    if (!p.only) {
        const PackKernel write = bf ? packed_write<bf16> : packed_write<float>;
        ensure_max_dynamic_smem((const void*)write, 8192 * 8);
        launch(write, dim3((unsigned)rows), 128, (unsigned)(d.rot_dims * 8), none, "packed_write");
        if (!out) return;
        if (prefill) {
            const int64_t rep = d.heads / d.kv_heads;
            const PackedPrefill pf = packed_prefill_of(d.dim, d.vdim, rows, d.kv_heads, rep);
            const int64_t tq = pf.rows / rep;
            ensure_max_dynamic_smem((const void*)pf.kernel, pf.smem);
            launch(pf.kernel, dim3((unsigned)((rows + tq - 1) / tq + n_seqs), (unsigned)d.kv_heads), (unsigned)pf.threads, (unsigned)pf.smem, none, "packed_prefill");
        } else {
            const PackKernel k = bf ? packed_simt<bf16> : packed_simt<float>;
            ensure_max_dynamic_smem((const void*)k, 220 * 1024);
            launch(k, dim3((unsigned)rows, (unsigned)d.heads), kAnyKeys, (unsigned)((d.dim + d.vdim + kAnyKeys) * 4), none, "packed_simt");
        }
    }
    if (tc && (p.only || n_seqs > 1)) {
        const PackedDecode dc = packed_decode_of(d.dim, d.vdim);
        const int64_t groups = d.kv_heads * ((d.heads / d.kv_heads + dc.heads - 1) / dc.heads), cells = n_seqs * groups;
        // Splits of the most keys a sequence can see: whole waves of resident CTAs, each with a beginning and an end, and the pieces have to be merged.
        const int64_t slots = (int64_t)dc.resident * sm_count();
        int64_t seen = (int64_t)p.width * d.page;
        if (d.window > 0) seen = std::min<int64_t>(seen, d.window + dc.step);
        int64_t splits = 1;
        const double fixed = 64.0 * 1024.0 / (d.dim + d.vdim);
        double best = 1e300;
        for (int64_t sp = 1; sp <= 64 && sp * dc.step <= std::max<int64_t>(seen, dc.step); sp++) {
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
        launch(dc.kernel, dim3((unsigned)splits, (unsigned)groups, (unsigned)n_seqs), 128, (unsigned)dc.smem, part, "packed_decode");
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
    const Buf none{kSlotNull, 0};
    em.launch(out.dtype == DT_BF16 ? packed_read<bf16> : packed_read<float>, dim3((unsigned)rows), dim3(128), 0, p,
              {{&p.keys, keys.buf}, {&p.values, values.buf}, {&p.places, places.buf}, {&p.table, pages.buf}, {&p.out, out.buf}, {&p.key_factors, key_factors ? key_factors->buf : none},
               {&p.value_factors, value_factors ? value_factors->buf : none}, {&p.err, Buf{kSlotErr, 0}}},
              "packed_read", /*pdl=*/true);
}

}  // namespace oxk
