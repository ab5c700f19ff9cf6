// Prompts of differential attention in bf16 on tcgen05.
//
// A cluster of two CTAs owns 128 (token, head) rows of one key head, each CTA one of the two softmax maps: it walks over that map's keys KEYS (64 or 128) at a time. Queries come as
// the sum of two bf16, base-2 units included, so scores need no factor: dim / 8 products of 128 × KEYS × 16 make them, a thread per row and 64 keys caps, masks and weighs them, and
// 4 products of 128 × vdim × 16 add their weights' share of the values. Keys and values come by TMA.
// From the order to a product to the word that it is done it takes 400 cycles, more than most products themselves (N 64: 47, N 128: 62 each). So nothing waits for two in a row: scores have one
// place, free as soon as they have been read, weights have two of their own, and the next scores are made, and the last weights multiplied, under the exponentials of these.
// In the end each CTA stages the other half of its rows, divided by their sums, copies them into the other's shared memory, and forms difference, norm and results of its own half.
//
// Measured alone, L2 cold: 4096 tokens, 32 heads of 2 × 64 over 16, values of 128 (137 GFLOP) 289–305 us, 450–476 TFLOP/s, twice that with the queries' low part and a product of the values per map;
// 2048, 16 over 4 60 us; 1999 capped and normed behind 1000, 4 heads of 2 × 128 over one, weights in two parts, 73 us (60 in one). A step of 64 keys takes 1 600 cycles with two CTAs per SM, of which both CTAs'
// exponentials take 1 054 of their unit and both CTAs' products, one after the other, 1 280 (the tensor pipe counts as active for 47 % of the whole kernel: products of 64 columns do not fill it, and tiles begin and end);
// what bounds it is their order within a CTA, and a third CTA has no tensor memory. A tile's beginning and end take 16 000 cycles, half of them under the other CTA's steps.
#include <type_traits>

#include "differential.cuh"

namespace oxk {

namespace {

constexpr int kRows = 128, kPart = 64;
constexpr unsigned kPanelQ = kRows * 128, kPanelV = kPart * 128;  // bytes: rows × 64 dimensions
constexpr int kBarriers = 23;
constexpr float kLazy = 8.f;  // how far (base 2) a row's scores may rise above the maximum that its weights are taken against

struct PreP {
    alignas(64) unsigned char maps[2][128];  // keys, values: [rows of the pool, 2 · dim | vdim]
    DiffP kv;
    int kp, vp, box, inv, tiles;  // panels of 64 dimensions, log2 of the keys per copy, 2^16 / heads of a key head, rounded up, tiles of a key head
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two f32 side by side: one instruction adds or multiplies both.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pair_of(float a, float b) {
    f32x2 v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ void apart(f32x2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 v;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}
// Two bf16 side by side onto two sums in f32.
__device__ __forceinline__ void add_bf16(float& a, float& b, unsigned w) {
    asm("{\n .reg .b16 low, high;\n mov.b32 {low, high}, %2;\n add.f32.bf16 %0, low, %0;\n add.f32.bf16 %1, high, %1;\n}\n" : "+f"(a), "+f"(b) : "r"(w));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float v;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(v) : "f"(a), "f"(b), "f"(c));
    return v;
}
__device__ __forceinline__ float max_of(const float (&s)[kPart]) {
    float a = s[0], b = s[1];
#pragma unroll
    for (int e = 2; e + 3 < kPart; e += 4) {
        a = max3(a, s[e], s[e + 1]);
        b = max3(b, s[e + 2], s[e + 3]);
    }
    return max3(a, b, fmaxf(s[kPart - 2], s[kPart - 1]));
}
// s with e^2x = 2^s, x = score / cap, becomes cap2 · tanh x. Caps are there for scores that stand out: while |x| of a warp's scores stays below 1/2, or 1, tanh x / x is a polynomial in x²
// (the best of its degree in relative error, 6e-7), N + 2 instructions for two elements, where an
// exponential and a reciprocal take sixteen cycles of the unit that also makes the weights: 1999 tokens behind 1000, 4 heads of 2 x 128, scores far below the cap, 58 us instead of 74.
template <int N> __device__ __forceinline__ void cap_within(float (&s)[kPart], float cap2, const double (&c)[N + 1]) {
    constexpr double k = 0.34657359027997264;  // x = k · s
    f32x2 q[N + 1];
    double power = k;
#pragma unroll
    for (int j = 0; j <= N; j++, power *= k * k) q[j] = pair_of((float)(c[j] * power) * cap2, (float)(c[j] * power) * cap2);
#pragma unroll
    for (int e = 0; e < kPart; e += 2) {
        const f32x2 x = pair_of(s[e], s[e + 1]), u = mul2(x, x);
        f32x2 y = q[N];
#pragma unroll
        for (int j = N - 1; j >= 0; j--) y = fma2(u, y, q[j]);
        apart(mul2(x, y), s[e], s[e + 1]);
    }
}
__device__ __forceinline__ void cap_scores(float (&s)[kPart], float cap2) {
    float most = 0.f;
#pragma unroll
    for (int e = 0; e < kPart; e += 2) most = max3(most, fabsf(s[e]), fabsf(s[e + 1]));
    if (!__any_sync(0xffffffffu, most > 1.44269504f)) {  // |x| up to 1/2
        constexpr double c[4] = {0.99999946, -0.33326318, 0.13190297, -0.04440223};
        cap_within<3>(s, cap2, c);
    } else if (!__any_sync(0xffffffffu, most > 2.88539008f)) {  // up to 1
        constexpr double c[6] = {0.99999941, -0.33329042, 0.13281434, -0.05160567, 0.01674312, -0.00306706};
        cap_within<5>(s, cap2, c);
    } else {
#pragma unroll
        for (int e = 0; e < kPart; e++) s[e] = cap2 - __fdividef(2.f * cap2, 1.f + ex2(s[e]));
    }
}
// All threads of both CTAs, warps at a time. Every thread of a CTA that has a tile comes here, whatever its waits found.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ unsigned of_cta(unsigned smem_byte_addr, unsigned cta) {
    unsigned to;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_byte_addr), "r"(cta));
    return to;
}

// The pages of the copies to come, 32 at a time and the next 32 on their way: the table's answer to a single question takes as long as a copy.
struct PagesAhead {
    int first, now, next;
    template <class Page> __device__ __forceinline__ PagesAhead(int from, Page&& page) : first(from), now(page(from)), next(page(from + 32)) {}
    // of box i, which does not fall; all lanes ask the same
    template <class Page> __device__ __forceinline__ int of(int i, Page&& page) {
        if (i >= first + 32) {
            first += 32;
            now = next;
            next = page(first + 32);
        }
        return __shfl_sync(0xffffffffu, now, i - first);
    }
};

// LOW: weights are the sum of two bf16 (emit_differential says where). Both are multiplied; their places are those of two turns, so a tile's are written behind the products of the tile before it.
// KEYS 64: 256 columns of tensor memory (values of up to 128), two CTAs per SM, which work under each other's waits. 128: all columns.
template <int KEYS> struct Shape {
    static constexpr int halves = KEYS / kPart, soft = halves * kRows, threads = soft + 64;  // softmax warps, one of copies, one that issues products
    static constexpr int keys = KEYS == 64 ? 3 : 2, values = KEYS == 64 ? 3 : 2;             // tiles of keys and halves of values on their way
};
template <bool CAPPED, int KEYS, bool LOW> __global__ void __launch_bounds__(Shape<KEYS>::threads, KEYS == 64 ? 2 : 1) differential_prefill(const __grid_constant__ PreP pp) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    // (both CTAs of a cluster find the same place: their shared memory begins at the same address)
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const DiffP& p = pp.kv;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, kp = pp.kp, vp = pp.vp, across = 2 * p.kv_heads, map = (int)blockIdx.x & 1, tile = (int)blockIdx.x / across, g = ((int)blockIdx.x - tile * across) >> 1;
    constexpr int kHalves = Shape<KEYS>::halves, kSoft = Shape<KEYS>::soft, kStagesK = Shape<KEYS>::keys, kStagesV = Shape<KEYS>::values;
    constexpr int kCopies = kSoft / 32, kIssues = kCopies + 1;  // warps
    constexpr unsigned kPanelK = KEYS * 128;
    const unsigned k_stage = kp * kPanelK, v_stage = vp * kPanelV;
    const unsigned sq0 = smem_u32(smem), low0 = kp * kPanelQ, sk = sq0 + 2 * low0, sv = sk + kStagesK * k_stage, bars = sv + kStagesV * v_stage;
    // barriers: keys there, free, values there, free (three each), scores there, read, products added (one, one and two), weights there (two halves of two), queries there, rows of the
    // other CTA there (two warps')
    const unsigned k_full = bars, k_free = bars + 24, v_full = bars + 48, v_free = bars + 72, s_full = bars + 96, s_free = bars + 104, o_done = bars + 112, w_full = bars + 128, q_full = bars + 160, r_full = bars + 168;
    unsigned* tmem_slot = reinterpret_cast<unsigned*>(smem + (bars + kBarriers * 8 - sq0));
    float* scales = reinterpret_cast<float*>(smem + (bars + kBarriers * 8 + 8 - sq0));  // [64]: what the norms divide by
    float* shared = scales + 64;  // [turn][half of the keys][row]: what the two threads of a row tell each other
    if (tid == 0) {
        for (int i = 0; i < kBarriers; i++) mbar_init(bars + i * 8, i == 13 ? kSoft / 32 : i == 20 ? kSoft : i >= 16 && i < 20 ? kRows / 32 : 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        for (int i = 0; i < 2; i++) mbar_expect_tx(r_full + i * 8, 32 * 256 * vp);
    }
    if (tid < 2) asm volatile("prefetch.tensormap [%0];" ::"l"(pp.maps[tid]) : "memory");
    pdl_wait();
    const int rep = p.heads / p.kv_heads, tq = kRows / rep;
    int seq, first;
    SeqRow sq;
    // long rows of all heads first: the last tiles of a sequence see the most keys
    if (!locate_rows(p, pp.tiles - 1 - tile, tq, p.singles ? 1 : 2, &seq, &first, &sq)) return;  // both CTAs of the cluster
    const int n_tok = min(tq, sq.len - first), pos0 = sq.past + first, last = pos0 + n_tok - 1, low = first_key(p, pos0);
    // Scores in KEYS columns, weights in two turns of half as many, sums behind them. No more CTAs than have room in tensor memory may be on an SM at a time
    // (differential_prefill_smem), or two clusters could wait for what the other one has.
    constexpr unsigned cols = KEYS * 4;
    if (warp == kIssues) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    const int inv = pp.inv;
    auto token_of = [&](int row) { return row * inv >> 16; };  // row / rep
    before_sync();
    __syncthreads();
    after_sync();
    pdl_trigger();  // the tensor memory is taken: nothing that starts now can keep it from this CTA
    const unsigned tmem = *tmem_slot, t_sum = tmem + 2 * KEYS;
    const int kt0 = low / KEYS, n = last / KEYS + 1 - kt0;
    bool ok = true;
    // Waits until the products of tile i are in the sums. Tiles take turns at two barriers, and who asks has seen the scores of tile i + 1 (or i, the last) and not let the products of
    // tile i + 2 begin. Products are done in the order of their issue, those of tile i − 1 in front of the scores of tile i + 1: the barrier is neither a round behind nor ahead.
    auto added = [&](int i) { return mbar_wait(o_done + (i & 1) * 8, (unsigned)(i >> 1) & 1); };
    // Where the weights of half h of tile i are: two turns, or (LOW) one, whose low parts lie behind them.
    auto weights_of = [&](int i, int h) { return tmem + KEYS + (LOW ? 0 : (i & 1) * (KEYS / 2)) + h * (kPart / 2); };
    // Whether some row of the CTA may see keys of half h of the tile that begins at j0. Halves that nobody sees are neither copied nor multiplied.
    auto seen = [&](int j0, int h) { return j0 + h * kPart <= last && j0 + h * kPart + kPart > low; };

    if (warp == kCopies) {
        // Copies of a page's keys each, where a page holds fewer than a half; those that nobody sees are left out. A tile's keys are asked for before the values of the tile before it.
        const int box = pp.box, box0 = max(low, kt0 * KEYS) >> box, box1 = last >> box;
        auto page = [&](int i) { return i + lane <= box1 ? (int)page_of(p, seq, (i + lane) << box) : 0; };
        PagesAhead keys_pages(box0, page), values_pages(box0, page);
        RingAt keys_at, values_at;
        int halves = 0;
        auto copy = [&](const unsigned char* map_of, PagesAhead& pages, int j0, int keys, unsigned full, unsigned to, int panels, unsigned panel, int x) {
            const int b0 = max(j0 >> box, box0), b1 = min(((j0 + keys) >> box) - 1, box1);
            for (int b = b0; b <= b1; b++) {
                const int j = b << box, row = (int)key_row(p, pages.of(b, page), g, j);
                const unsigned at = to + (j - j0) * 128;
                if (elect_one() && ok) {
                    if (b == b0) mbar_expect_tx(full, (unsigned)(((b1 - b0 + 1) << box) * 128 * panels));
                    tma_load_2d(at, map_of, x, row, full);
                    if (panels > 1) tma_load_2d(at + panel, map_of, x + 64, row, full);
                    if (panels > 2) tma_load_2d(at + 2 * panel, map_of, x + 128, row, full);
                    if (panels > 3) tma_load_2d(at + 3 * panel, map_of, x + 192, row, full);
                }
                __syncwarp();
            }
        };
        auto copy_keys = [&](int i) {
            if (i >= kStagesK && ok && !mbar_wait(k_free + keys_at.s * 8, keys_at.parity ^ 1)) ok = false;
            copy(pp.maps[0], keys_pages, (kt0 + i) * KEYS, KEYS, k_full + keys_at.s * 8, sk + keys_at.s * k_stage, kp, kPanelK, map * p.dim);
            keys_at.next(kStagesK);
        };
        copy_keys(0);
        for (int i = 0; i < n && ok; i++) {
            if (i + 1 < n) copy_keys(i + 1);
            const int j0 = (kt0 + i) * KEYS;
            for (int h = 0; h < kHalves; h++) {
                if (!seen(j0, h)) continue;
                if (halves >= kStagesV && ok && !mbar_wait(v_free + values_at.s * 8, values_at.parity ^ 1)) ok = false;
                copy(pp.maps[1], values_pages, j0 + h * kPart, kPart, v_full + values_at.s * 8, sv + values_at.s * v_stage, vp, kPanelV, 0);
                values_at.next(kStagesV);
                halves++;
            }
            ok = __all_sync(0xffffffffu, ok);
        }
    } else if (warp == kIssues) {
        const unsigned base = (1u << 4) | (1u << 7) | (1u << 10) | (8u << 24);  // bf16 × bf16 → f32, M 128
        const unsigned by_keys = base | ((KEYS >> 3) << 17), by_values = base | (1u << 16) | ((unsigned)(vp * 8) << 17);  // the values' wide axis is the result's
        const unsigned long long dq = umma_kmajor_desc(sq0), dk = umma_kmajor_desc(sk), dv = umma_wide_desc(sv);
        RingAt keys_at, values_at;
        auto scores = [&](int i) {
            if (ok && !mbar_wait(k_full + keys_at.s * 8, keys_at.parity)) ok = false;
            if (i > 0 && ok && !mbar_wait(s_free, (unsigned)(i - 1) & 1)) ok = false;
            after_sync();
            if (elect_one() && ok) {
                const unsigned long long k = dk + keys_at.s * (k_stage >> 4);
                for (int c = 0; c < kp; c++) {
                    const unsigned long long a = dq + c * (kPanelQ >> 4), a2 = a + (low0 >> 4), b = k + c * (kPanelK >> 4);
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (c * 64 + e * 16 < p.dim) {
                            umma_bf16(tmem, a + e * 2, b + e * 2, by_keys, c > 0 || e > 0);
                            umma_bf16(tmem, a2 + e * 2, b + e * 2, by_keys, true);
                        }
                }
                umma_commit(k_free + keys_at.s * 8);
                umma_commit(s_full);
            }
            __syncwarp();
            keys_at.next(kStagesK);
        };
        if (!mbar_wait(q_full, 0)) ok = false;
        scores(0);
        bool some = false;  // the sums hold something
        for (int i = 0; i < n; i++) {
            if (i + 1 < n) scores(i + 1);
            const int j0 = (kt0 + i) * KEYS;
            // The threads of both halves before the products of either: where a row's maximum rises, each of its two threads scales every other sixteen columns of the sums, and products add to all of them.
            for (int h = 0; h < kHalves; h++)
                if (ok && !mbar_wait(w_full + (i & 1) * 16 + h * 8, (unsigned)(i >> 1) & 1)) ok = false;
            for (int h = 0; h < kHalves; h++) {
                if (!seen(j0, h)) continue;
                if (ok && !mbar_wait(v_full + values_at.s * 8, values_at.parity)) ok = false;
                after_sync();
                if (elect_one() && ok) {
                    const unsigned long long v = dv + values_at.s * (v_stage >> 4);
#pragma unroll
                    for (int e = 0; e < kPart / 16; e++) umma_weights(t_sum, weights_of(i, h) + e * 8, v + e * 128, by_values, some || e > 0);
                    if (LOW) {
#pragma unroll
                        for (int e = 0; e < kPart / 16; e++) umma_weights(t_sum, weights_of(i, h) + KEYS / 2 + e * 8, v + e * 128, by_values, true);
                    }
                    umma_commit(v_free + values_at.s * 8);
                }
                __syncwarp();
                some = true;
                values_at.next(kStagesV);
            }
            if (elect_one() && ok) umma_commit(o_done + (i & 1) * 8);
            __syncwarp();
        }
    }
    if (warp < kCopies) {
        const int shift = kp + 2, chunks = 1 << (shift + 1), c = tid & (chunks - 1), part = c >> shift, d = c - (part << shift);  // kp is 1 or 2
        const bf16* src = (const bf16*)p.q + (((g * p.rows + sq.start + first) * rep * 2 + map) * 2 + part) * p.dim + d * 8;
        const unsigned to = sq0 + part * low0 + (d >> 3) * kPanelQ;
#pragma unroll 8
        for (int row = tid / chunks; row < kRows; row += kSoft / chunks) {
            const bool live = row < n_tok * rep && d * 8 < p.dim;
            cp_async16(to + row * 128 + (((d & 7) ^ (row & 7)) << 4), live ? src + row * 4 * p.dim : (const bf16*)p.q, live);
        }
        cp_async_commit();
        cp_async_wait<0>();
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the tensor core reads them
        asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(q_full) : "memory");
    }
    const int r = tid & (kRows - 1), part = tid / kRows, tok = token_of(r), head = g * rep + r - tok * rep;  // thread `part` of a row has its keys of half `part`
    const unsigned lanes = (unsigned)((warp & 3) * 32) << 16;
    // what both threads of a row know: by the two warps that share its rows
    auto both = [&](int turn, float mine) {
        float* at = shared + turn * 2 * kRows + r;
        at[part * kRows] = mine;
        asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 3)) : "memory");
        return at[(part ^ 1) * kRows];
    };
    float f = 0.f;
    if (warp < kCopies) {
        const int pos = tok < n_tok ? pos0 + tok : last, mine_low = first_key(p, pos), last_low = first_key(p, last);  // rows without a token compute something harmless
        const float cap2 = p.cap2;
        float m = -1e30f;  // below every score, and finite: differences stay numbers
        float sums[4] = {};  // of every fourth key's weights each
        int halves = 0;      // of the values, in front of this thread's
        for (int i = 0; i < n; i++) {
            const int j0 = (kt0 + i) * KEYS, j1 = j0 + part * kPart;
            if (ok && !mbar_wait(s_full, (unsigned)i & 1)) ok = false;
            after_sync();
            float s[kPart];
#pragma unroll
            for (int c = 0; c < 2; c++) {
                unsigned v[32];
                tmem_ld32(v, tmem + lanes + part * kPart + c * 32);
#pragma unroll
                for (int e = 0; e < 32; e++) s[c * 32 + e] = __uint_as_float(v[e]);
            }
            tmem_ld_wait();
            before_sync();
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(s_free) : "memory");
            const bool edge = j1 + kPart - 1 > pos0 || j1 < last_low;
            if (CAPPED && edge) {  // how a warp's scores are capped hangs on those that its rows see: the others may be anything
#pragma unroll
                for (int e = 0; e < kPart; e++)
                    if (j1 + e > pos || j1 + e < mine_low) s[e] = 0.f;
            }
            if (CAPPED) cap_scores(s, cap2);
            if (edge) {
#pragma unroll
                for (int e = 0; e < kPart; e++)
                    if (j1 + e > pos || j1 + e < mine_low) s[e] = -INFINITY;
            }
            float top = max_of(s);
            if (kHalves == 2) top = fmaxf(top, both(i & 1, top));
            // Weights are taken against a maximum that may lie up to 2^8 behind, so that the sums are rarely taken anew. The largest weight is then rounded as the others are, where against the maximum itself
            // it is 1; the sums, of the weights as they are multiplied, are off with it, so a key that takes all weight costs nothing either way. Off from 64-bit results, behind → against the maximum
            // itself: 2.31e-3 → 2.12e-3 (1500 keys, scores of a spread of 1.5; of 4: 1.90e-3 → 1.76e-3), 4.07e-3 → 4.16e-3 (scores nearly equal); the rounding of the
            // results alone is 1.66e-3. It would take 22 % of time (4096 tokens, 32 heads of 2 x 64 over 16; 2048, 16 over 4: 14 %; 1999 behind 1000, 4 heads of 2 x 128: 15 %).
            // (LOW: both parts of a weight are there either way.) Both warps of a row see the same tops.
            if (__any_sync(0xffffffffu, top > m + kLazy)) {
                top = fmaxf(top, m);
                const float keep = ex2(m - top);
                m = top;
#pragma unroll
                for (int e = 0; e < 4; e++) sums[e] *= keep;
                if (i > 0) {
                    if (ok && !added(i - 1)) ok = false;
                    after_sync();
#pragma unroll 1
                    for (int c = part * 16; c < vp * 64; c += 16 * kHalves) {
                        unsigned o[16];
                        tmem_ld16(o, t_sum + lanes + c);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                        tmem_st16(t_sum + lanes + c, o);
                    }
                }
            }
            const int before = kHalves == 2 && part == 1 && seen(j0, 0);  // the other half's values come first
            // (these weights' place is free: with the scores of tile i the products of tile i − 2 are done)
            if (seen(j0, part)) {
                const f32x2 behind = pair_of(-m, -m);
                if constexpr (LOW) {
                    unsigned w[32], rest[32];
#pragma unroll
                    for (int e = 0; e < 32; e++) {
                        float a, b;
                        apart(add2(pair_of(s[2 * e], s[2 * e + 1]), behind), a, b);
                        a = ex2(a), b = ex2(b);
                        w[e] = pack_bf16(a, b);
                        rest[e] = pack_bf16(a - __uint_as_float(w[e] << 16), b - __uint_as_float(w[e] & 0xFFFF0000u));
                        sums[(e & 1) * 2] += a, sums[(e & 1) * 2 + 1] += b;
                    }
                    if (i > 0 && ok && !added(i - 1)) ok = false;  // the last tile's weights have been multiplied
                    after_sync();
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        tmem_st16(weights_of(i, part) + lanes + c * 16, *reinterpret_cast<const unsigned(*)[16]>(w + c * 16));
                        tmem_st16(weights_of(i, part) + lanes + KEYS / 2 + c * 16, *reinterpret_cast<const unsigned(*)[16]>(rest + c * 16));
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        unsigned w[16];
#pragma unroll
                        for (int e = 0; e < 16; e++) {
                            float a, b;
                            apart(add2(pair_of(s[c * 32 + 2 * e], s[c * 32 + 2 * e + 1]), behind), a, b);
                            w[e] = pack_bf16(ex2(a), ex2(b));
                            // The sums of the weights as they are multiplied: the rounding of a weight that stands out is in both. Adding bf16 to f32 as they are, four sums at a time, 64 keys of
                            // a row take 660 cycles, of which the exponentials need 512; unpacked, two sums, 900.
                            add_bf16(sums[(e & 1) * 2], sums[(e & 1) * 2 + 1], w[e]);
                        }
                        tmem_st16(weights_of(i, part) + lanes + c * 16, w);
                    }
                }
                if (j1 + kPart - 1 > last || j1 < low) {  // what lies behind the last key or in front of the first may be no number, which a weight of 0 would not cancel
                    const int at = halves + before, stage = at % kStagesV;
                    // The place's values before these have to be there, or the barrier's parity is that of the round before them. With three places they are of tile i − 3, whose products are done; with
                    // two they are of tile i − 1, whose products may still wait for them.
                    if (kHalves == 2 && i > 0 && ok && !added(i - 1)) ok = false;
                    if (ok && !mbar_wait(v_full + stage * 8, (unsigned)(at / kStagesV) & 1)) ok = false;
                    for (int u = r; u < kPart * vp * 8; u += kRows) {
                        const int key = u & (kPart - 1), c = u / kPart;
                        const unsigned to = sv + stage * v_stage + (c >> 3) * kPanelV + key * 128 + (c & 7) * 16;
                        if (j1 + key > last || j1 + key < low) asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(to), "r"(0) : "memory");
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                tmem_st_wait();
            }
            before_sync();
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(w_full + (i & 1) * 16 + part * 8) : "memory");
            halves += seen(j0, 0) + (kHalves == 2 && seen(j0, 1));
        }
        __syncwarp();
        cluster_arrive();  // the last scores are there: nothing reads queries and keys any more
        float l = (sums[0] + sums[1]) + (sums[2] + sums[3]);
        if (kHalves == 2) l += both(n & 1, l);
        if (ok && !added(n - 1)) ok = false;
        after_sync();
        f = 1.f / l;
        if (p.sink) {
            const float top = fmaxf(m, 0.f), keep = ex2(m - top);
            f = keep / (l * keep + ex2(-top));
        }
        if (map) f *= p.lambda[head];
        __syncwarp();
    } else {
        cluster_arrive();
    }
    // A CTA's other 64 rows, [row][vp · 64] in f32, neighbouring rows' sixteen bytes in different banks, go where the other one's queries and keys were: 32 rows a copy, while both still
    // have something to do.
    cluster_wait();
    const unsigned long_row = vp * 256, mine = (r & 63) * long_row;
    auto place = [&](int row, int c) { return (unsigned)(((c >> 2) ^ (row & 7)) << 4); };  // of dimensions c … c + 3
    const bool keeps = (r >> 6) == map;                                                    // CTA 0 has the first 64 rows
    if (warp < kCopies && !keeps) {
#pragma unroll 1
        for (int c = part * 32; c < vp * 64; c += 32 * kHalves) {
            unsigned v[32];
            tmem_ld32(v, t_sum + lanes + c);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; e += 4)
                asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(sv + mine + place(r, c + e)), "f"(__uint_as_float(v[e]) * f), "f"(__uint_as_float(v[e + 1]) * f),
                             "f"(__uint_as_float(v[e + 2]) * f), "f"(__uint_as_float(v[e + 3]) * f)
                             : "memory");
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        if (kHalves == 2)
            asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 3)) : "memory");
        else
            __syncwarp();
        if (part == 0 && lane == 0)
            asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(of_cta(sq0 + mine, map ^ 1)), "r"(sv + mine), "r"(32 * long_row),
                         "r"(of_cta(r_full + (warp & 1) * 8, map ^ 1))
                         : "memory");
        __syncwarp();
    }
    // a row is written by neighbouring lanes, sixteen bytes each
    const int wide = p.vdim > 128 ? 32 : 16, wc = (tid & (wide - 1)) * 8;
    float gain[8];
#pragma unroll
    for (int e = 0; e < 8; e++) gain[e] = p.gain && wc < p.vdim ? p.gain[wc + e] : 1.f;
    if (warp < kCopies && keeps) {
        if (!mbar_wait(r_full + (warp & 1) * 8, 0)) ok = false;
        const float sign = map ? -1.f : 1.f;
        float ss = 0.f;
#pragma unroll 1
        for (int c = part * 32; c < vp * 64; c += 32 * kHalves) {
            unsigned v[32];
            tmem_ld32(v, t_sum + lanes + c);
            float4 theirs[8];
#pragma unroll
            for (int e = 0; e < 32; e += 4) theirs[e / 4] = *reinterpret_cast<const float4*>(smem + mine + place(r, c + e));
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
                float4 o = theirs[e / 4];
                o.x = (__uint_as_float(v[e]) * f - o.x) * sign;
                o.y = (__uint_as_float(v[e + 1]) * f - o.y) * sign;
                o.z = (__uint_as_float(v[e + 2]) * f - o.z) * sign;
                o.w = (__uint_as_float(v[e + 3]) * f - o.w) * sign;
                ss = fmaf(o.x, o.x, fmaf(o.y, o.y, fmaf(o.z, o.z, fmaf(o.w, o.w, ss))));  // dimensions that are padding are 0
                *reinterpret_cast<float4*>(smem + mine + place(r, c + e)) = o;
            }
        }
        if (kHalves == 2) ss += both((n + 1) & 1, ss);
        scales[r & 63] = p.gain ? 1.f / sqrtf(ss / (float)p.vdim + p.head_eps) : 1.f;
    }
    before_sync();
    __syncthreads();
    after_sync();
    cluster_arrive();  // this CTA has what the other one sent
    if (warp < kCopies && wc < p.vdim) {
#pragma unroll 1
        for (int i0 = tid / wide; i0 < 64; i0 += 4 * (kSoft / wide)) {
            float4 a[4], b[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int i = i0 + u * (kSoft / wide);
                a[u] = *reinterpret_cast<const float4*>(smem + i * long_row + place(i, wc));
                b[u] = *reinterpret_cast<const float4*>(smem + i * long_row + place(i, wc + 4));
            }
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int i = i0 + u * (kSoft / wide), at = map * 64 + i, t = token_of(at);
                const float x = scales[i];
                if (t < n_tok && ok)
                    *reinterpret_cast<uint4*>((bf16*)p.out + ((sq.start + first + t) * (long long)p.heads + g * rep + at - t * rep) * p.vdim + wc) =
                        make_uint4(pack_bf16(a[u].x * x * gain[0], a[u].y * x * gain[1]), pack_bf16(a[u].z * x * gain[2], a[u].w * x * gain[3]),
                                   pack_bf16(b[u].x * x * gain[4], b[u].y * x * gain[5]), pack_bf16(b[u].z * x * gain[6], b[u].w * x * gain[7]));
            }
        }
    }
    __syncwarp();
    cluster_wait();  // no CTA leaves while its rows are on their way
    if (!ok && lane == 0) report(p.err, ERR_WAIT_TIMEOUT, p.node, (long long)blockIdx.x, (long long)warp);
    if (warp == kIssues) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
}

// Two CTAs per SM where their shared and tensor memory allow it: 4096 tokens, 32 heads of 2 × 64 over 16 289 us, one CTA of 128 keys 426; 2048, 16 over 4 60 and 80.
int differential_keys(int kp, int vp) { return kp == 1 && vp <= 2 ? 64 : 128; }
}  // namespace

// A CTA that has tensor memory waits for its neighbour, which may be waiting for some: so as many CTAs as share an SM, of either form and whatever their sizes (two sessions run on one
// device), must have room in its tensor memory. Forms of 64 keys take 256 of 512 columns and 85 448 bytes at least: two share an SM (233 472 bytes, 1 024 of them the system's per CTA), three
// do not. Forms of 128 keys take all columns, so they ask for as many bytes as keep the smallest of the others away (120 832 … 198 000 are their own). Kernels of single CTAs that hold tensor
// memory end by themselves, and none of more than 256 columns is small enough to wait beside two CTAs that do not need it.
int differential_prefill_columns(int kp, int vp) { return differential_keys(kp, vp) * 4; }
int differential_prefill_smem(int kp, int vp) {
    const int keys = differential_keys(kp, vp);
    const int kv = keys == 64 ? Shape<64>::keys * 64 * 128 * kp + Shape<64>::values * (int)kPanelV * vp : Shape<128>::keys * 128 * 128 * kp + Shape<128>::values * (int)kPanelV * vp;
    return std::max(1024 + kp * 2 * (int)kPanelQ + kv + kBarriers * 8 + 16 + 256 + 4 * kRows * 4, keys == 64 ? 80 * 1024 : 147 * 1024);
}

bool differential_prefill_fits(const DiffP& p, const TRef& keys, const TRef& values, int64_t out_off) {
    const int64_t rows = (int64_t)p.n_pages * p.kv_heads << p.shift, rep = p.heads / p.kv_heads, tiles = rep <= kRows ? p.rows / (kRows / rep) + 1 + p.n_seqs : 0;
    return 1 << p.shift >= 8 && p.dim % 16 == 0 && p.dim <= 128 && p.vdim % 8 == 0 && p.vdim <= 256 && rep <= kRows && tiles * 2 * p.kv_heads < INT32_MAX && rows < INT32_MAX &&
           keys.buf.off % 16 == 0 && values.buf.off % 16 == 0 && out_off % 16 == 0;
}

void emit_differential_prefill(Emitter& em, const DiffP& kv, const TRef& keys, const TRef& values, std::initializer_list<std::pair<size_t, Buf>> ptrs) {
    PreP p{};
    p.kv = kv;
    p.kp = (kv.dim + 63) / 64;
    p.vp = (kv.vdim + 63) / 64;
    p.box = std::min(6, kv.shift);
    p.inv = (65536 + kv.heads / kv.kv_heads - 1) / (kv.heads / kv.kv_heads);
    const int64_t tq = kRows / (kv.heads / kv.kv_heads), rows = (int64_t)kv.n_pages * kv.kv_heads << kv.shift;
    p.tiles = (int)((kv.rows + tq - 1) / tq + kv.n_seqs);
    auto form = [&](auto capped, auto low) -> void (*)(const PreP) {
        return differential_keys(p.kp, p.vp) == 64 ? differential_prefill<capped.value, 64, low.value> : differential_prefill<capped.value, 128, low.value>;
    };
    const std::true_type yes;
    const std::false_type no;
    void (*const k)(const PreP) = kv.cap2 > 0.f ? (kv.low ? form(yes, yes) : form(yes, no)) : (kv.low ? form(no, yes) : form(no, no));
    const int smem = differential_prefill_smem(p.kp, p.vp);
    ensure_max_dynamic_smem((const void*)k, 226 * 1024);
    LaunchRec& rec = em.launch(k, dim3((unsigned)p.tiles * (unsigned)kv.kv_heads * 2), dim3(differential_keys(p.kp, p.vp) == 64 ? Shape<64>::threads : Shape<128>::threads), (unsigned)smem, p, {}, "differential_prefill", /*pdl=*/true);
    rec.cluster = dim3(2, 1, 1);
    for (auto& pr : ptrs) rec.relocs.push_back(Reloc{(uint32_t)(offsetof(PreP, kv) + pr.first), pr.second});
    rec.tmaps.push_back(TmapReloc{(uint32_t)offsetof(PreP, maps), keys.buf, (uint64_t)kv.dim * 2, (uint64_t)rows, (uint64_t)kv.dim * 4, 64u, 1u << p.box});
    rec.tmaps.push_back(TmapReloc{(uint32_t)offsetof(PreP, maps) + 128, values.buf, (uint64_t)kv.vdim, (uint64_t)rows, (uint64_t)kv.vdim * 2, 64u, 1u << p.box});
}

}  // namespace oxk
