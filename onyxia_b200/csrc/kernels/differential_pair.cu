// Prompts of differential attention in bf16 on tcgen05, maps of up to 64 dimensions and values of up to 128.
//
// A CTA owns 128 (token, head) rows of one key head and both of their softmax maps, whose scores and sums fill tensor memory; it walks over the keys 128 at a time. Queries come as the
// sum of two bf16, base-2 units included, so scores need no factor: dim / 8 products of 128 × 128 × 16 make those of a map, a thread per row caps, masks and weighs them, and for each 64 keys
// 4 products of 128 × vdim × 16 add the weights' share of the values. While the four warps of one map weigh, the tensor core adds the other map's weighted values and makes its next
// scores. Keys of both maps and values come by TMA, two tiles of either on their way.
#include "differential_tc.cuh"

namespace oxk {

namespace {

constexpr int kKeys = 128, kSoft = 2 * kRows, kCopies = 8, kIssues = 9, kThreads = 11 * 32;  // warps 0-3, 4-7: softmax of a map, 8 copies, 9, 10 issue a map's products
constexpr int kBarriers = 21;
constexpr unsigned kMapK = kKeys * 128, kTileK = 2 * kMapK;

int pair_smem(int vp) { return 1024 + 4 * (int)kPanelQ + 2 * (int)kTileK + 4 * vp * (int)kPanelV + kBarriers * 8 + 24 + kSoft * 4; }

template <bool CAPPED> __global__ void __launch_bounds__(kThreads, 1) differential_pair(const __grid_constant__ PreP pp) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const DiffP& p = pp.kv;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, vp = pp.vp, g = blockIdx.y;
    const unsigned v_stage = vp * kPanelV, sq0 = smem_u32(smem), sk = sq0 + 4 * kPanelQ, sv = sk + 2 * kTileK, bars = sv + 4 * v_stage;  // queries: [map][high, low]
    // barriers: keys there, free (two each), values there, free (four each), scores there, products added (one of each map), weights there (two halves of each map), queries there
    const unsigned k_full = bars, k_free = bars + 16, v_full = bars + 32, v_free = bars + 64, s_full = bars + 96, o_done = bars + 112, w_full = bars + 128, q_full = bars + 160;
    unsigned* tmem_slot = reinterpret_cast<unsigned*>(smem + (bars + kBarriers * 8 - sq0));
    float* squares = reinterpret_cast<float*>(smem + (bars + kBarriers * 8 + 24 - sq0));  // [map][row]
    if (tid == 0) {
        for (int i = 0; i < kBarriers; i++) mbar_init(bars + i * 8, i == 20 ? kSoft : i >= 16 ? kRows / 32 : i == 2 || i == 3 || (i >= 8 && i < 12) ? 2 : 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait();
    const int rep = p.heads / p.kv_heads, tq = kRows / rep;
    int seq, first;
    // long rows first: the last tiles of a sequence see the most keys
    if (!locate_tile(p.seqs, p.n_seqs, (int)gridDim.x - 1 - (int)blockIdx.x, tq, &seq, &first, p.singles ? 1 : 2)) return;
    const SeqRow sq = load_seq(p.seqs, seq);
    const int n_tok = min(tq, sq.len - first), pos0 = sq.past + first, last = pos0 + n_tok - 1, low = first_key(p, pos0);
    // All of tensor memory: scores of both maps, 128 columns each, then sums. Weights take the place of the scores that their thread has read.
    if (warp == kIssues) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    before_sync();
    __syncthreads();
    after_sync();
    pdl_trigger();  // the tensor memory is taken: nothing that starts now can keep it from this CTA
    const unsigned tmem = *tmem_slot;
    const int inv = pp.inv;
    auto token_of = [&](int row) { return row * inv >> 16; };  // row / rep
    const int kt0 = low / kKeys, n = last / kKeys + 1 - kt0;
    bool ok = true;
    // Whether some row of the CTA may see keys of half h of the tile that begins at j0. Halves that nobody sees are neither copied nor multiplied.
    auto seen = [&](int j0, int h) { return j0 + h * kPart <= last && j0 + h * kPart + kPart > low; };

    if (warp == kCopies) {
        // Copies of a page's keys each, where a page holds fewer than a half; those that nobody sees are left out. A tile's keys are asked for before the values of the tile before it.
        const int box0 = max(low, kt0 * kKeys) / pp.box, box1 = last / pp.box;
        auto page = [&](int i) { return i + lane <= box1 ? (int)page_of(p, seq, (i + lane) * pp.box) : 0; };
        PagesAhead keys_pages(box0, page), values_pages(box0, page);
        RingAt keys_at, values_at;
        int halves = 0;
        auto copy = [&](int kv, PagesAhead& pages, int j0, int keys, unsigned full, unsigned to, int panels, unsigned panel, int step) {
            const int b0 = max(j0 / pp.box, box0), b1 = min((j0 + keys) / pp.box - 1, box1);
            if (elect_one() && ok) mbar_expect_tx(full, (unsigned)((b1 - b0 + 1) * pp.box * 128 * panels));
            __syncwarp();
            for (int b = b0; b <= b1; b++) {
                const int j = b * pp.box, row = (int)key_row(p, pages.of(b, page), g, j);
                if (elect_one() && ok)
                    for (int c = 0; c < panels; c++) tma_load_2d(to + c * panel + (j - j0) * 128, pp.maps[kv], c * step, row, full);
                __syncwarp();
            }
        };
        auto copy_keys = [&](int i) {
            if (i >= 2 && ok && !mbar_wait(k_free + keys_at.s * 8, keys_at.parity ^ 1)) ok = false;
            copy(0, keys_pages, (kt0 + i) * kKeys, kKeys, k_full + keys_at.s * 8, sk + keys_at.s * kTileK, 2, kMapK, p.dim);
            keys_at.next(2);
        };
        copy_keys(0);
        for (int i = 0; i < n && ok; i++) {
            if (i + 1 < n) copy_keys(i + 1);
            const int j0 = (kt0 + i) * kKeys;
            for (int h = 0; h < 2; h++) {
                if (!seen(j0, h)) continue;
                if (halves >= 4 && ok && !mbar_wait(v_free + values_at.s * 8, values_at.parity ^ 1)) ok = false;
                copy(1, values_pages, j0 + h * kPart, kPart, v_full + values_at.s * 8, sv + values_at.s * v_stage, vp, kPanelV, 64);
                values_at.next(4);
                halves++;
            }
            ok = __all_sync(0xffffffffu, ok);
        }
    } else if (warp >= kIssues) {
        const int map = warp - kIssues;
        const unsigned base = (1u << 4) | (1u << 7) | (1u << 10) | (8u << 24);  // bf16 × bf16 → f32, M 128
        const unsigned by_keys = base | ((kKeys >> 3) << 17), by_values = base | (1u << 16) | ((unsigned)(vp * 8) << 17);  // the values' wide axis is the result's
        const unsigned long long dq = umma_kmajor_desc(sq0 + map * 2 * kPanelQ), dk = umma_kmajor_desc(sk + map * kMapK), dv = umma_wide_desc(sv);
        const unsigned t_scores = tmem + map * kKeys, t_sum = tmem + 2 * kKeys + map * 128;
        RingAt keys_at, values_at;
        if (!mbar_wait(q_full, 0)) ok = false;
        bool some = false;  // the sums hold something
        for (int i = 0; i < n; i++) {
            if (ok && !mbar_wait(k_full + keys_at.s * 8, keys_at.parity)) ok = false;
            // the products that read the weights in these scores' place have to be done
            if (i > 0 && ok && !mbar_wait(o_done + map * 8, (unsigned)(i - 1) & 1)) ok = false;
            after_sync();
            if (elect_one() && ok) {
                const unsigned long long k = dk + keys_at.s * (kTileK >> 4);
                for (int e = 0; e < p.dim / 16; e++) {
                    umma_bf16(t_scores, dq + e * 2, k + e * 2, by_keys, e > 0);
                    umma_bf16(t_scores, dq + (kPanelQ >> 4) + e * 2, k + e * 2, by_keys, true);
                }
                umma_commit(k_free + keys_at.s * 8);
                umma_commit(s_full + map * 8);
            }
            __syncwarp();
            keys_at.next(2);
            const int j0 = (kt0 + i) * kKeys;
            for (int h = 0; h < 2; h++) {
                if (ok && !mbar_wait(w_full + map * 16 + h * 8, (unsigned)i & 1)) ok = false;
                if (!seen(j0, h)) continue;
                if (ok && !mbar_wait(v_full + values_at.s * 8, values_at.parity)) ok = false;
                after_sync();
                if (elect_one() && ok) {
                    const unsigned long long v = dv + values_at.s * (v_stage >> 4);
#pragma unroll
                    for (int e = 0; e < kPart / 16; e++) umma_weights(t_sum, t_scores + h * (kPart / 2) + e * 8, v + e * 128, by_values, some || e > 0);
                    umma_commit(v_free + values_at.s * 8);
                }
                __syncwarp();
                some = true;
                values_at.next(4);
            }
            if (elect_one() && ok) umma_commit(o_done + map * 8);
            __syncwarp();
        }
    } else {
        const int map = warp >> 2, r = tid & (kRows - 1), tok = token_of(r), head = g * rep + r - tok * rep;
        {
            const int c = r & 15, part = c >> 3, d = c & 7;
            const bf16* src = (const bf16*)p.q + ((((long long)(sq.start + first) * p.heads + g * rep) * 2 + map) * 2 + part) * p.dim + d * 8;
            const unsigned to = sq0 + (map * 2 + part) * kPanelQ;
#pragma unroll 4
            for (int row = r >> 4; row < kRows; row += 8) {
                const int t = token_of(row), h = row - t * rep;
                const bool live = t < n_tok && d * 8 < p.dim;
                cp_async16(to + row * 128 + ((d ^ (row & 7)) << 4), live ? src + ((long long)t * p.heads + h) * 4 * p.dim : (const bf16*)p.q, live);
            }
            cp_async_commit();
            cp_async_wait<0>();
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the tensor core reads them
            asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(q_full) : "memory");
        }
        const unsigned lanes = (unsigned)((warp & 3) * 32) << 16, t_scores = tmem + lanes + map * kKeys, t_sum = tmem + lanes + 2 * kKeys + map * 128;
        const int pos = tok < n_tok ? pos0 + tok : last, mine_low = first_key(p, pos), last_low = first_key(p, last);  // rows without a token compute something harmless
        const float cap2 = p.cap2;
        float m = -1e30f, l = 0.f, l2 = 0.f;  // below every score, and finite: differences stay numbers
        RingAt values_at;
        for (int i = 0; i < n; i++) {
            const int j0 = (kt0 + i) * kKeys;
            // (these scores were issued when the products of the tile before were in the sums)
            if (ok && !mbar_wait(s_full + map * 8, (unsigned)i & 1)) ok = false;
            after_sync();
            float s[kKeys];
#pragma unroll
            for (int c = 0; c < 4; c++) {
                unsigned v[32];
                tmem_ld32(v, t_scores + c * 32);
#pragma unroll
                for (int e = 0; e < 32; e++) s[c * 32 + e] = __uint_as_float(v[e]);
            }
            tmem_ld_wait();
            if (CAPPED) {
#pragma unroll
                for (int e = 0; e < kKeys; e++) s[e] = cap2 - __fdividef(2.f * cap2, 1.f + ex2(s[e]));
            }
            if (j0 + kKeys - 1 > pos0 || j0 < last_low) {
#pragma unroll
                for (int e = 0; e < kKeys; e++)
                    if (j0 + e > pos || j0 + e < mine_low) s[e] = -INFINITY;
            }
            float top = fmaxf(s[0], s[1]), top2 = fmaxf(s[2], s[3]);
#pragma unroll
            for (int e = 4; e < kKeys; e += 4) {
                top = fmaxf(top, fmaxf(s[e], s[e + 1]));
                top2 = fmaxf(top2, fmaxf(s[e + 2], s[e + 3]));
            }
            top = fmaxf(top, top2);
            // Weights are taken against a maximum that may lie up to 2^8 behind: the sums are rarely taken anew, and bf16 holds 2^8 as well as 1.
            if (__any_sync(0xffffffffu, top > m + kLazy)) {
                top = fmaxf(top, m);
                const float keep = ex2(m - top);
                m = top;
                l *= keep;
                l2 *= keep;
                if (i > 0) {
#pragma unroll 1
                    for (int c = 0; c < vp * 64; c += 16) {
                        unsigned o[16];
                        tmem_ld16(o, t_sum + c);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                        tmem_st16(t_sum + c, o);
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int j1 = j0 + h * kPart;
                if (seen(j0, h)) {
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        unsigned w[16];
#pragma unroll
                        for (int e = 0; e < 16; e++) {
                            const int at = h * kPart + c * 32 + 2 * e;
                            w[e] = pack_bf16(ex2(s[at] - m), ex2(s[at + 1] - m));
                            // the sums of the weights as they are multiplied: the rounding of a weight that stands out is in both
                            l += __uint_as_float(w[e] << 16);
                            l2 += __uint_as_float(w[e] & 0xFFFF0000u);
                        }
                        tmem_st16(t_scores + h * (kPart / 2) + c * 16, w);
                    }
                    if (j1 + kPart - 1 > last || j1 < low) {  // what lies behind the last key or in front of the first may be no number, which a weight of 0 would not cancel
                        if (ok && !mbar_wait(v_full + values_at.s * 8, values_at.parity)) ok = false;
                        for (int u = r; u < kPart * vp * 8; u += kRows) {  // (both maps' threads write the same)
                            const int key = u & (kPart - 1), c = u / kPart;
                            const unsigned to = sv + values_at.s * v_stage + (c >> 3) * kPanelV + key * 128 + (c & 7) * 16;
                            if (j1 + key > last || j1 + key < low) asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(to), "r"(0) : "memory");
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    }
                    tmem_st_wait();
                    values_at.next(4);
                }
                before_sync();
                __syncwarp();
                if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(w_full + map * 16 + h * 8) : "memory");
            }
        }
        if (ok && !mbar_wait(o_done + map * 8, (unsigned)(n - 1) & 1)) ok = false;
        after_sync();
        l += l2;
        float f = 1.f / l;
        if (p.sink) {
            const float top = fmaxf(m, 0.f), keep = ex2(m - top);
            f = keep / (l * keep + ex2(-top));
        }
        if (map) f *= p.lambda[head];
        // Map 0 forms the first half of a row's results, map 1 the second: each gives the other half, divided by its sum, to the other through what was queries and keys.
        auto meet = [] { asm volatile("bar.sync 1, %0;" ::"n"(kSoft) : "memory"); };
        const int half = vp * 32, stride = half + 4;
        float *gives = reinterpret_cast<float*>(smem) + (map * kRows + r) * stride, *has = reinterpret_cast<float*>(smem) + ((map ^ 1) * kRows + r) * stride;
        meet();  // both maps' copies and products are done
#pragma unroll 1
        for (int c = 0; c < half; c += 32) {
            unsigned v[32];
            tmem_ld32(v, t_sum + (map ^ 1) * half + c);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; e += 4)
                *reinterpret_cast<float4*>(gives + c + e) =
                    make_float4(__uint_as_float(v[e]) * f, __uint_as_float(v[e + 1]) * f, __uint_as_float(v[e + 2]) * f, __uint_as_float(v[e + 3]) * f);
        }
        meet();
        const float sign = map ? -1.f : 1.f;
        float ss = 0.f;
#pragma unroll 1
        for (int c = 0; c < half; c += 32) {
            unsigned v[32];
            tmem_ld32(v, t_sum + map * half + c);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
                float4 o = *reinterpret_cast<float4*>(has + c + e);
                o.x = (__uint_as_float(v[e]) * f - o.x) * sign;
                o.y = (__uint_as_float(v[e + 1]) * f - o.y) * sign;
                o.z = (__uint_as_float(v[e + 2]) * f - o.z) * sign;
                o.w = (__uint_as_float(v[e + 3]) * f - o.w) * sign;
                ss = fmaf(o.x, o.x, fmaf(o.y, o.y, fmaf(o.z, o.z, fmaf(o.w, o.w, ss))));  // dimensions that are padding are 0
                *reinterpret_cast<float4*>(has + c + e) = o;
            }
        }
        squares[map * kRows + r] = ss;
        meet();
        // a row is written by neighbouring lanes, sixteen bytes each
        const int c = tid & 15;
        if (c * 8 < p.vdim) {
            const int second = c * 8 >= half;  // (which map formed these: they are in the place that the other gave from)
            const float* from = reinterpret_cast<const float*>(smem) + (second ^ 1) * kRows * stride + c * 8 - second * half;
            float gain[8];
#pragma unroll
            for (int e = 0; e < 8; e++) gain[e] = p.gain ? p.gain[c * 8 + e] : 1.f;
#pragma unroll 4
            for (int row = tid >> 4; row < kRows; row += kSoft / 16) {
                const int t = token_of(row);
                const float4 a = *reinterpret_cast<const float4*>(from + row * stride), b = *reinterpret_cast<const float4*>(from + row * stride + 4);
                const float x = p.gain ? 1.f / sqrtf((squares[row] + squares[kRows + row]) / (float)p.vdim + p.head_eps) : 1.f;
                if (t < n_tok && ok)
                    *reinterpret_cast<uint4*>((bf16*)p.out + ((sq.start + first + t) * (long long)p.heads + g * rep + row - t * rep) * p.vdim + c * 8) =
                        make_uint4(pack_bf16(a.x * x * gain[0], a.y * x * gain[1]), pack_bf16(a.z * x * gain[2], a.w * x * gain[3]), pack_bf16(b.x * x * gain[4], b.y * x * gain[5]),
                                   pack_bf16(b.z * x * gain[6], b.w * x * gain[7]));
            }
        }
    }
    if (!ok && lane == 0) report(p.err, ERR_WAIT_TIMEOUT, p.node, (long long)blockIdx.x, (long long)warp);
    before_sync();
    __syncthreads();
    if (warp == kIssues) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

}  // namespace

void emit_differential_pair(Emitter& em, const PreP& p, dim3 grid) {
    void (*const k)(const PreP) = p.kv.cap2 > 0.f ? differential_pair<true> : differential_pair<false>;
    ensure_max_dynamic_smem((const void*)k, 226 * 1024);
    em.launch(k, grid, dim3(kThreads), (unsigned)pair_smem(p.vp), p, {}, "differential_prefill", /*pdl=*/true);
}

}  // namespace oxk
