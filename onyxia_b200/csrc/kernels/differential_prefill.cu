// Prompts of differential attention in bf16 on tcgen05.
//
// A cluster of two CTAs owns 128 (token, head) rows of one key head, each CTA one of the two softmax maps: it walks over that map's keys 64 at a time. Queries come as the
// sum of two bf16, base-2 units included, so scores need no factor: 8 · dim / 64 products of 128 × 64 make them, two threads per row cap, mask and weigh them, 4 products of
// 128 × vdim add the weights' share of the values; the scores of the next 64 keys are made under the weights of these. Keys and values come by TMA, three tiles on their way.
// In the end each CTA sends the other half of its rows, divided by their sums, through the cluster's shared memory, and forms difference, norm and results of its own half.
#include "differential.cuh"

namespace oxk {

namespace {

constexpr int kRows = 128, kKeys = 64, kSoft = 256, kThreads = kSoft + 64;  // warps 0-7 softmax, 8 copies, 9 issues products
constexpr int kHalf = kKeys / 2, kStages = 3;
constexpr unsigned kPanelQ = kRows * 128, kPanelKv = kKeys * 128;  // bytes: rows × 64 dimensions
constexpr int kBarriers = 4 * kStages + 6;
constexpr float kLazy = 8.f;  // how far (base 2) a row's scores may rise above the maximum that its weights are taken against

struct PreP {
    alignas(64) unsigned char maps[2][128];  // keys, values: [rows of the pool, 2 · dim | vdim]
    DiffP kv;
    int kp, vp, box;  // panels of 64 dimensions, keys per copy
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Rows of weights in tensor memory (two per column) × values, of which 64 stand side by side for a key.
__device__ __forceinline__ void umma_weights(unsigned d, unsigned a, unsigned long long b, unsigned idesc, bool accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u), "r"(0u)
        : "memory");
}
// Shared-memory matrix descriptor, 128-byte swizzle, 64 elements of the wide axis side by side: groups of eight keys 1 024 bytes apart, the next 64
// elements a panel further.
__device__ __forceinline__ unsigned long long umma_wide_desc(unsigned smem_byte_addr) {
    return (unsigned long long)((smem_byte_addr & 0x3FFFFu) >> 4) | ((unsigned long long)(kPanelKv >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void tmem_ld32(unsigned (&v)[32], unsigned from) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, "
        "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]),
          "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]),
          "=r"(v[30]), "=r"(v[31])
        : "r"(from));
}
__device__ __forceinline__ void tmem_ld16(unsigned (&v)[16], unsigned from) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]),
          "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(from));
}
__device__ __forceinline__ void tmem_st16(unsigned to, const unsigned (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};\n" ::"r"(v[0]), "r"(v[1]), "r"(v[2]),
        "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(to)
        : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// All threads of both CTAs. Every thread of a CTA that has a tile comes here, whatever its waits found.
__device__ __forceinline__ void cluster_meet() {
    asm volatile("barrier.cluster.arrive.release;\n barrier.cluster.wait.acquire;" ::: "memory");
}

template <bool CAPPED> __global__ void __launch_bounds__(kThreads, 2) differential_prefill(const __grid_constant__ PreP pp) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    // (both CTAs of a cluster find the same place: their shared memory begins at the same address)
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const DiffP& p = pp.kv;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, kp = pp.kp, vp = pp.vp, map = blockIdx.y & 1, g = blockIdx.y >> 1;
    const unsigned k_stage = kp * kPanelKv, v_stage = vp * kPanelKv;
    const unsigned sq0 = smem_u32(smem), low0 = kp * kPanelQ, sk = sq0 + 2 * low0, sv = sk + kStages * k_stage, bars = sv + kStages * v_stage;
    const unsigned k_full = bars, k_free = k_full + kStages * 8, v_full = k_free + kStages * 8, v_free = v_full + kStages * 8, s_full = v_free + kStages * 8, w_full = s_full + 16,
                   o_done = w_full + 16;
    unsigned* tmem_slot = reinterpret_cast<unsigned*>(smem + (bars + kBarriers * 8 - sq0));
    float* shared = reinterpret_cast<float*>(smem + (bars + kBarriers * 8 + 16 - sq0));  // [turn][half of the keys][row]: what the two threads of a row tell each other
    if (tid == 0) {
        for (int i = 0; i < kBarriers; i++) mbar_init(bars + i * 8, i == kBarriers - 4 || i == kBarriers - 3 ? kSoft / 32 : 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait();
    const int rep = p.heads / p.kv_heads, tq = kRows / rep;
    int seq, first;
    // long rows first: the last tiles of a sequence see the most keys
    if (!locate_tile(p.seqs, p.n_seqs, (int)gridDim.x - 1 - (int)blockIdx.x, tq, &seq, &first, p.singles ? 1 : 2)) return;  // both CTAs of the cluster
    const SeqRow sq = load_seq(p.seqs, seq);
    const int n_tok = min(tq, sq.len - first), pos0 = sq.past + first, last = pos0 + n_tok - 1, low = first_key(p, pos0);
    // Scores in two turns of 64 columns, weights in two of 32, sums. Up to 128 dimensions weights take their scores' place, so that two CTAs fit an SM. No more of them than have room in
    // tensor memory may be there at a time (differential_smem), or two clusters could wait for what the other one has.
    const bool apart = vp > 2;
    const unsigned cols = apart ? 512 : 256;
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    for (int i = tid; i < kRows * kp * 16; i += kThreads) {
        const int r = i / (kp * 16), c = i % (kp * 16), part = c >= kp * 8, d = c - part * kp * 8, tok = r / rep, h = g * rep + r % rep;
        const bool live = tok < n_tok && d * 8 < p.dim;
        const bf16* src = (const bf16*)p.q;
        cp_async16(sq0 + part * low0 + (d >> 3) * kPanelQ + r * 128 + (((d & 7) ^ (r & 7)) << 4),
                   live ? src + ((((long long)(sq.start + first + tok) * p.heads + h) * 2 + map) * 2 + part) * p.dim + d * 8 : src, live);
    }
    cp_async_commit();
    cp_async_wait<0>();
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the tensor core reads them
    before_sync();
    __syncthreads();
    after_sync();
    pdl_trigger();  // the tensor memory is taken: nothing that starts now can keep it from this CTA
    const unsigned tmem = *tmem_slot, t_weights = apart ? tmem + 128 : tmem, weights_turn = apart ? 32 : kKeys, t_sum = tmem + (apart ? 192 : 128);
    const int kt0 = low / kKeys, n = last / kKeys + 1 - kt0;
    bool ok = true;
    // Waits until the products of tile i are in the sums. Tiles take turns at two barriers. Who has the scores of tile i knows the products of tile i - 2 and of all before it to be
    // done, so the barrier of tile i - 1 or i cannot be a round behind.
    auto added = [&](int i) { return mbar_wait(o_done + (i & 1) * 8, (unsigned)(i >> 1) & 1); };

    if (warp == 8) {
        RingAt at;
        for (int i = 0; i < n && ok; i++) {
            const int j0 = (kt0 + i) * kKeys;
            // copies of a page's keys each, where a page holds fewer than a tile; those that nobody sees are left out
            const int c0 = max(low - j0, 0) / pp.box, c1 = min((last - j0) / pp.box, kKeys / pp.box - 1);
            for (int kv = 0; kv < 2; kv++) {
                const unsigned full = (kv ? v_full : k_full) + at.s * 8, to = kv ? sv + at.s * v_stage : sk + at.s * k_stage;
                const int panels = kv ? vp : kp;
                if (i >= kStages && ok && !mbar_wait((kv ? v_free : k_free) + at.s * 8, at.parity ^ 1)) ok = false;
                if (elect_one() && ok) mbar_expect_tx(full, (unsigned)((c1 - c0 + 1) * pp.box * 128 * panels));
                __syncwarp();
                for (int b = c0; b <= c1; b++) {
                    const int j = j0 + b * pp.box, row = (int)key_row(p, page_of(p, seq, j), g, j);
                    if (elect_one() && ok)
                        for (int c = 0; c < panels; c++) tma_load_2d(to + c * kPanelKv + b * pp.box * 128, pp.maps[kv], (kv ? 0 : map * p.dim) + c * 64, row, full);
                    __syncwarp();
                }
            }
            ok = __all_sync(0xffffffffu, ok);
            at.next(kStages);
        }
    } else if (warp == 9) {
        const unsigned base = (1u << 4) | (1u << 7) | (1u << 10) | (8u << 24);  // bf16 × bf16 → f32, M 128
        const unsigned by_keys = base | ((kKeys >> 3) << 17), by_values = base | (1u << 16) | ((unsigned)(vp * 8) << 17);  // the values' wide axis is the result's
        const unsigned long long dq = umma_kmajor_desc(sq0), dk = umma_kmajor_desc(sk), dv = umma_wide_desc(sv);
        RingAt tile_ahead, ahead, tile, at;  // tiles, and turns of scores and weights
        auto scores = [&] {
            if (ok && !mbar_wait(k_full + tile_ahead.s * 8, tile_ahead.parity)) ok = false;
            after_sync();
            if (elect_one() && ok) {
                const unsigned long long k = dk + tile_ahead.s * (k_stage >> 4);
                for (int e = 0; e < p.dim / 16; e++) {
                    const unsigned long long a = dq + (e >> 2) * (kPanelQ >> 4) + (e & 3) * 2, b = k + (e >> 2) * (kPanelKv >> 4) + (e & 3) * 2;
                    umma_bf16(tmem + ahead.s * kKeys, a, b, by_keys, e > 0);
                    umma_bf16(tmem + ahead.s * kKeys, a + (low0 >> 4), b, by_keys, true);
                }
                umma_commit(k_free + tile_ahead.s * 8);
                umma_commit(s_full + ahead.s * 8);
            }
            __syncwarp();
            tile_ahead.next(kStages);
            ahead.next(2);
        };
        scores();
        for (int i = 0; i < n; i++) {
            if (i + 1 < n) {
                // the other turn's scores were read by the threads that wrote its weights; where these have their place, products have to be done with them
                if (!apart && i > 0 && ok && !added(i - 1)) ok = false;
                scores();
            }
            if (ok && !mbar_wait(w_full + at.s * 8, at.parity)) ok = false;
            if (ok && !mbar_wait(v_full + tile.s * 8, tile.parity)) ok = false;
            after_sync();
            if (elect_one() && ok) {
                const unsigned long long v = dv + tile.s * (v_stage >> 4);
#pragma unroll
                for (int e = 0; e < kKeys / 16; e++) umma_weights(t_sum, t_weights + at.s * weights_turn + e * 8, v + e * 128, by_values, i > 0 || e > 0);
                umma_commit(v_free + tile.s * 8);
                umma_commit(o_done + at.s * 8);
            }
            __syncwarp();
            tile.next(kStages);
            at.next(2);
        }
    }
    // two threads per row, each with half of the keys
    const int r = tid & (kRows - 1), part = tid / kRows, tok = r / rep, head = g * rep + r % rep;
    const unsigned lanes = (unsigned)((warp & 3) * 32) << 16;
    const bool live = tok < n_tok;
    // what both threads of a row know: by the two warps that share its rows
    auto both = [&](int turn, float mine) {
        float* at = shared + turn * 2 * kRows + r;
        at[part * kRows] = mine;
        asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 3)) : "memory");
        return at[(part ^ 1) * kRows];
    };
    float f = 0.f;
    if (warp < 8) {
        const int pos = live ? pos0 + tok : last, mine_low = first_key(p, pos), last_low = first_key(p, last);  // rows without a token compute something harmless
        const float cap2 = p.cap2;
        float m = -1e30f, l = 0.f;  // below every score, and finite: differences stay numbers
        RingAt at, tile;
        for (int i = 0; i < n; i++) {
            const int j0 = (kt0 + i) * kKeys, mine0 = j0 + part * kHalf;
            if (ok && !mbar_wait(s_full + at.s * 8, at.parity)) ok = false;
            after_sync();
            float s[kHalf];
            {
                unsigned v[32];
                tmem_ld32(v, tmem + lanes + at.s * kKeys + part * kHalf);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < kHalf; e++) {
                    const float x = __uint_as_float(v[e]);
                    s[e] = CAPPED ? cap2 - __fdividef(2.f * cap2, 1.f + ex2(x)) : x;
                }
            }
            if (j0 + kKeys - 1 > pos0 || j0 < last_low) {
#pragma unroll
                for (int e = 0; e < kHalf; e++)
                    if (mine0 + e > pos || mine0 + e < mine_low) s[e] = -INFINITY;
            }
            float top = s[0];
#pragma unroll
            for (int e = 1; e < kHalf; e++) top = fmaxf(top, s[e]);
            top = fmaxf(top, both(i & 1, top));
            // Weights are taken against a maximum that may lie up to 2^8 behind: the sums are rarely taken anew, and bf16 holds 2^8 as well as 1. Both warps of a row see the same tops.
            if (__any_sync(0xffffffffu, top > m + kLazy)) {
                top = fmaxf(top, m);
                const float keep = ex2(m - top);
                m = top;
                l *= keep;
                if (i > 0) {
                    if (ok && !added(i - 1)) ok = false;
                    after_sync();
#pragma unroll 1
                    for (int c = part * 16; c < vp * 64; c += 32) {
                        unsigned v[16];
                        tmem_ld16(v, t_sum + lanes + c);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 16; e++) v[e] = __float_as_uint(__uint_as_float(v[e]) * keep);
                        tmem_st16(t_sum + lanes + c, v);
                    }
                }
            }
            unsigned w[kHalf / 2];
#pragma unroll
            for (int e = 0; e < kHalf / 2; e++) {
                const float a = ex2(s[2 * e] - m), b = ex2(s[2 * e + 1] - m);
                l += a + b;
                w[e] = pack_bf16(a, b);
            }
            // Where weights take their scores' place: both threads of the row have read these. Elsewhere: the products that read this turn's last weights were issued
            // before these scores.
            tmem_st16(t_weights + lanes + at.s * weights_turn + part * (kHalf / 2), w);
            if (j0 + kKeys - 1 > last || j0 < low) {  // what lies behind the last key or in front of the first may be no number, which a weight of 0 would not cancel
                if (ok && !mbar_wait(v_full + tile.s * 8, tile.parity)) ok = false;
                for (int u = tid; u < kKeys * vp * 8; u += kSoft) {
                    const int key = u & (kKeys - 1), c = u / kKeys;
                    const unsigned to = sv + tile.s * v_stage + (c >> 3) * kPanelKv + key * 128 + (c & 7) * 16;
                    if (j0 + key > last || j0 + key < low) asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(to), "r"(0) : "memory");
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            }
            tmem_st_wait();
            before_sync();
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(w_full + at.s * 8) : "memory");
            tile.next(kStages);
            at.next(2);
        }
        l += both(n & 1, l);
        if (ok && !added(n - 1)) ok = false;
        after_sync();
        f = 1.f / l;
        if (p.sink) {
            const float top = fmaxf(m, 0.f), keep = ex2(m - top);
            f = keep / (l * keep + ex2(-top));
        }
        if (map) f *= p.lambda[head];
    }
    // Copies and products of both CTAs are done: their places take the other CTA's rows, a quarter of a thread pair's rows [64][vdim + 4] in f32.
    cluster_meet();
    const int stride = vp * 64 + 4;
    const unsigned mine = sq0 + (r & 63) * stride * 4;
    const bool keeps = (r >> 6) == map;  // CTA 0 has the first 64 rows
    if (warp < 8 && !keeps) {
        unsigned to;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(mine), "r"(map ^ 1));
#pragma unroll 1
        for (int c = part * 32; c < vp * 64; c += 64) {
            unsigned v[32];
            tmem_ld32(v, t_sum + lanes + c);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; e += 4)
                asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to + (c + e) * 4), "f"(__uint_as_float(v[e]) * f), "f"(__uint_as_float(v[e + 1]) * f),
                             "f"(__uint_as_float(v[e + 2]) * f), "f"(__uint_as_float(v[e + 3]) * f)
                             : "memory");
        }
    }
    cluster_meet();
    if (warp < 8 && keeps) {
        float* row = reinterpret_cast<float*>(smem + (mine - sq0));
        const float sign = map ? -1.f : 1.f;
        float ss = 0.f;
#pragma unroll 1
        for (int c = part * 32; c < vp * 64; c += 64) {
            unsigned v[32];
            tmem_ld32(v, t_sum + lanes + c);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
                float4 o = *reinterpret_cast<float4*>(row + c + e);
                o.x = (__uint_as_float(v[e]) * f - o.x) * sign;
                o.y = (__uint_as_float(v[e + 1]) * f - o.y) * sign;
                o.z = (__uint_as_float(v[e + 2]) * f - o.z) * sign;
                o.w = (__uint_as_float(v[e + 3]) * f - o.w) * sign;
                ss = fmaf(o.x, o.x, fmaf(o.y, o.y, fmaf(o.z, o.z, fmaf(o.w, o.w, ss))));  // dimensions that are padding are 0
                *reinterpret_cast<float4*>(row + c + e) = o;
            }
        }
        float scale = 1.f;
        if (p.gain) scale = 1.f / sqrtf((ss + both(0, ss)) / (float)p.vdim + p.head_eps);
        if (live && ok) {
            bf16* out = (bf16*)p.out + ((sq.start + first + tok) * (long long)p.heads + head) * p.vdim;
#pragma unroll 1
            for (int c = part * 32; c < vp * 64; c += 64)
#pragma unroll
                for (int e = 0; e < 32; e += 8)
                    if (c + e < p.vdim) {
                        float o[8];
#pragma unroll
                        for (int k = 0; k < 8; k++) o[k] = row[c + e + k] * (p.gain ? scale * p.gain[c + e + k] : 1.f);
                        *reinterpret_cast<uint4*>(out + c + e) = make_uint4(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]), pack_bf16(o[4], o[5]), pack_bf16(o[6], o[7]));
                    }
        }
    }
    if (!ok && lane == 0) report(p.err, ERR_WAIT_TIMEOUT, p.node, (long long)blockIdx.x, (long long)warp);
    before_sync();
    __syncthreads();
    if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
}

// With three tiles on their way no more CTAs share an SM than have room in its tensor memory: 80 KB and more with 256 columns of 512, 128 KB and more with all of them.
int differential_smem(int kp, int vp) { return 1024 + kp * (int)(2 * kPanelQ + kStages * kPanelKv) + vp * kStages * (int)kPanelKv + kBarriers * 8 + 16 + 4 * kRows * 4; }

}  // namespace

bool differential_prefill_fits(const DiffP& p, const TRef& keys, const TRef& values, int64_t out_off) {
    const int64_t rows = (int64_t)p.n_pages * p.kv_heads << p.shift;
    return 1 << p.shift >= 8 && p.dim % 16 == 0 && p.dim <= 128 && p.vdim % 8 == 0 && p.vdim <= 256 && p.heads / p.kv_heads <= kRows && p.kv_heads <= 32767 && rows < INT32_MAX &&
           keys.buf.off % 16 == 0 && values.buf.off % 16 == 0 && out_off % 16 == 0;
}

void emit_differential_prefill(Emitter& em, const DiffP& kv, const TRef& keys, const TRef& values, std::initializer_list<std::pair<size_t, Buf>> ptrs) {
    PreP p{};
    p.kv = kv;
    p.kp = (kv.dim + 63) / 64;
    p.vp = (kv.vdim + 63) / 64;
    p.box = std::min(kKeys, 1 << kv.shift);
    const int64_t tq = kRows / (kv.heads / kv.kv_heads), rows = (int64_t)kv.n_pages * kv.kv_heads << kv.shift;
    void (*const k)(const PreP) = kv.cap2 > 0.f ? differential_prefill<true> : differential_prefill<false>;
    const int smem = differential_smem(p.kp, p.vp);
    ensure_max_dynamic_smem((const void*)k, 226 * 1024);
    LaunchRec& rec = em.launch(k, dim3((unsigned)((kv.rows + tq - 1) / tq + kv.n_seqs), (unsigned)kv.kv_heads * 2), dim3(kThreads), (unsigned)smem, p, {}, "differential_prefill", /*pdl=*/true);
    rec.cluster = dim3(1, 2, 1);
    for (auto& pr : ptrs) rec.relocs.push_back(Reloc{(uint32_t)(offsetof(PreP, kv) + pr.first), pr.second});
    rec.tmaps.push_back(TmapReloc{(uint32_t)offsetof(PreP, maps), keys.buf, (uint64_t)kv.dim * 2, (uint64_t)rows, (uint64_t)kv.dim * 4, 64u, (uint32_t)p.box});
    rec.tmaps.push_back(TmapReloc{(uint32_t)offsetof(PreP, maps) + 128, values.buf, (uint64_t)kv.vdim, (uint64_t)rows, (uint64_t)kv.vdim * 2, 64u, (uint32_t)p.box});
}

}  // namespace oxk
