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
//   differential_simt      any shape, f32 and bf16
#include "differential.cuh"

namespace oxk {

namespace {

// One CTA per row, one warp per query or key of a map.
template <typename T> __global__ void __launch_bounds__(128) differential_prepare(const DiffP p) {
    extern __shared__ float angle[];  // cos[half], sin[half]
    pdl_enter();
    const int row = blockIdx.x, s = find_seq(p.seqs, p.n_seqs, row), lane = threadIdx.x & 31;
    const SeqRow sq = load_seq(p.seqs, s);
    const int pos = sq.past + row - sq.start;
    if (row < sq.start || row >= sq.start + sq.len || (sq.len == 1 && !p.singles)) return;
    angles(p.turns, p.half, pos, angle, angle + p.half, threadIdx.x, 128);
    __syncthreads();
    const T* x = (const T*)p.proj + (long long)row * p.ld;
    const long long pg = page_of(p, s, pos);
    for (int h = threadIdx.x >> 5; h < 2 * (p.heads + p.kv_heads); h += 4) {
        const int k = h - 2 * p.heads;
        const T* src = k < 0 ? x + p.q_off + (long long)h * p.dim : x + p.k_off + (long long)k * p.dim;
        T* dst = k < 0 ? (T*)p.q + ((long long)row * p.heads * 2 + h) * p.dim : (T*)p.keys + (key_row(p, pg, k >> 1, pos) * 2 + (k & 1)) * p.dim;
        const float f = map_factor(p, src);
        for (int i = lane; i < p.dim; i += 32) dst[i] = from_f<T>(rotated(p.half, 0, src, angle, angle + p.half, i) * f);
    }
    for (int i = threadIdx.x; i < p.kv_heads * p.vdim; i += 128) ((T*)p.values)[key_row(p, pg, i / p.vdim, pos) * p.vdim + i % p.vdim] = x[p.v_off + i];
}

// One CTA per (row, head); chunks of 128 keys, a thread per key, then a thread per value dimension.
template <typename T> __global__ void __launch_bounds__(kAnyKeys) differential_simt(const DiffP p) {
    extern __shared__ float sm[];  // q[2][dim], acc[2][vdim], w[2][128]
    __shared__ float red[32];
    pdl_enter();
    const int row = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, s = find_seq(p.seqs, p.n_seqs, row);
    const SeqRow sq = load_seq(p.seqs, s);
    if (row < sq.start || row >= sq.start + sq.len) return;
    const int pos = sq.past + row - sq.start, g = h / (p.heads / p.kv_heads);
    float *q = sm, *acc = sm + 2 * p.dim, *w = acc + 2 * p.vdim;
    for (int i = tid; i < 2 * p.dim; i += kAnyKeys) q[i] = to_f(((const T*)p.q)[((long long)row * p.heads + h) * 2 * p.dim + i]);
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

using DiffKernel = void (*)(const DiffP);

}  // namespace

void emit_differential(Emitter& em, const DifferentialDesc& d, const TRef& proj, const TRef& turns, const TRef& keys, const TRef& values, const TRef& seqs,
                       const TRef& pages, const TRef& lambda, const TRef* gain, const TRef& out) {
    const int64_t rows = proj.shape[0], n_seqs = seqs.shape[0];
    if (rows == 0 || n_seqs == 0) return;
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
    p.singles = 1;
    const bool bf = proj.dtype == DT_BF16;
    const Buf none{kSlotNull, 0}, q = em.scratch((size_t)rows * d.heads * 2 * d.dim * (bf ? 2 : 4));
    auto launch = [&](DiffKernel k, dim3 grid, unsigned block, unsigned smem, const char* label) {
        em.launch(k, grid, dim3(block), smem, p,
                  {{&p.proj, proj.buf}, {&p.turns, turns.buf}, {&p.keys, keys.buf}, {&p.values, values.buf}, {&p.q, q}, {&p.out, out.buf}, {&p.seqs, seqs.buf}, {&p.table, pages.buf},
                   {&p.lambda, lambda.buf}, {&p.gain, gain ? gain->buf : none}, {&p.err, Buf{kSlotErr, 0}}},
                  label, /*pdl=*/true);
    };
    launch(bf ? differential_prepare<bf16> : differential_prepare<float>, dim3((unsigned)rows), 128, (unsigned)(d.rot_dims * 4), "differential_prepare");
    const DiffKernel k = bf ? differential_simt<bf16> : differential_simt<float>;
    ensure_max_dynamic_smem((const void*)k, 220 * 1024);
    launch(k, dim3((unsigned)rows, (unsigned)d.heads), kAnyKeys, (unsigned)((d.dim + d.vdim + kAnyKeys) * 8), "differential_simt");
}

}  // namespace oxk
