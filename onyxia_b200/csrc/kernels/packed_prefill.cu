// Prompts over keys and values in 4 bits on tcgen05: scores and sums of values in tensor memory.
//
// A CTA owns one or two tiles of 128 (token, head) rows of one key head and walks over their keys, 64 at a time. One warp copies what the pages hold of them, several steps ahead; four warps turn
// codes into f16 (exactly: packed_cache.cuh), a step ahead of the products; one warp issues these; a thread per row masks and weighs scores. The next 64 keys' scores are made meanwhile: a tile has two turns of them. Two tiles share what is
// unpacked.
//
// A row's softmax is taken in one pass: m, l and the sums of values against a reference below the maximum (kLeast, kMost: packed_cache.cuh). Queries are f16 times a power of two of their own, weights f16,
// all sums f32.
//
// What bounds it: 4096 tokens of 32 heads of 128 over 16 take 187 us, 735 TFLOP/s of 4 · 128 operations per pair (at a plain matrix product's rate 81 us). Of a step's 2430 cycles (two tiles, 64 keys)
// the products take 1900, since a product with 64 keys reads 128 queries from shared memory for half the columns, and the issuing warp waits for weights the other 530. Scores of 128 keys would leave
// tensor memory no place for the next ones beside two tiles' sums. Copies, codes and conversions lie under the products, in 54 % of the issue slots. 1999 tokens behind 1000, capped and normed, of 16
// heads of 128 over 4: 94 us (19): 128 CTAs of 17 to 47 steps, which take as long as the last of them.
#include <type_traits>

#include "packed_cache.cuh"

namespace oxk {

namespace {

constexpr int kRows = 128, kUnpack = 128, kStages = 2, kKeys = 64, kSlots = 8;
constexpr unsigned kPanelQ = kRows * 128, kPanel = kKeys * 128;  // bytes: rows, or keys, × 64 dimensions

__device__ __forceinline__ unsigned ld_shared(unsigned at) {
    unsigned v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}

__device__ __forceinline__ unsigned ld_shared_u8(unsigned at) {
    unsigned v;
    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}

__device__ __forceinline__ void st_shared(unsigned at, unsigned v) { asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(v) : "memory"); }

// CAP: 1, scores are capped; 2, by more than kWideCap
template <int TILES, int CAP> __global__ void __launch_bounds__(TILES * kRows + kUnpack + 64, TILES == 1 ? 2 : 1) packed_prefill(const PackP p) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    constexpr bool CAPPED = CAP != 0;
    constexpr int kSoft = TILES * kRows, kThreads = kSoft + kUnpack + 64, kSoftWarps = kSoft / 32, kIssues = kSoftWarps + kUnpack / 32, kCopies = kIssues + 1;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, kp = (p.dim + 63) / 64, vp = (p.vdim + 63) / 64;
    const unsigned k_stage = kp * kPanel, v_stage = vp * kPanel;
    const unsigned sq0 = smem_u32(smem), sk = sq0 + TILES * kp * kPanelQ, sv = sk + kStages * k_stage, raw = sv + kStages * v_stage, slot = kKeys * max(p.dim, p.vdim) / kPack * 9, bars = raw + p.raw_slots * slot;
    // barriers: keys there, free, values there, free (one per stage), scores there, weights there, sums (two per tile, by turns), copies there, free (one per slot, keys and values by turns)
    const unsigned k_full = bars, k_free = k_full + kStages * 8, v_full = k_free + kStages * 8, v_free = v_full + kStages * 8, s_full = v_free + kStages * 8, w_full = s_full + 32, o_done = w_full + 32, raw_full = o_done + 32, raw_free = raw_full + kSlots * 8;
    unsigned* tmem_slot = reinterpret_cast<unsigned*>(smem + (raw_free + kSlots * 8 - sq0));
    // Which sixteen dimensions are no numbers: of the rows' results, [rows]; of the values of tiles with hidden keys, [stages][1 + keys], behind whether there are any.
    const unsigned row_bad = raw_free + kSlots * 8 + 16, value_bad = row_bad + TILES * kRows * 4;
    if (tid == 0) {
        for (unsigned b = bars; b < raw_free + kSlots * 8; b += 8) mbar_init(b, (b >= k_full && b < k_free) || (b >= v_full && b < v_free) || b >= raw_free ? kUnpack / 32 : b >= w_full && b < o_done ? kRows / 32 : 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait();
    const int rep = p.heads / p.kv_heads, tq = kSoft / rep, g = blockIdx.x % p.kv_heads;
    int seq, first;
    // long rows first, of all heads: the last tiles of a sequence see the most keys
    SeqRow sq;
    if (!locate_rows(p, (int)((gridDim.x - 1 - blockIdx.x) / p.kv_heads), tq, p.singles ? 1 : 2, &seq, &first, &sq)) return;
    const int n_tok = min(tq, sq.len - first), pos0 = sq.past + first, last = pos0 + n_tok - 1;
    const unsigned cols = TILES == 1 && vp <= 2 ? 256 : 512;
    if (warp == kIssues) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // eight lanes a row's 128 bytes
    for (int r = warp * 4 + lane / 8; r < kSoft; r += kThreads / 8) {
        const int tok = over(r, p.by_rep), h = g * rep + r - tok * rep;
        const __half* row = (const __half*)p.q + ((long long)(sq.start + first + tok) * p.heads + h) * p.dim;
        for (int c = 0; c < kp; c++) {
            const int at = c * 64 + lane % 8 * 8;
            const bool live = tok < n_tok && at < p.dim;
            cp_async16(sq0 + (r / kRows * kp + c) * kPanelQ + r % kRows * 128 + ((lane % 8 ^ (r & 7)) << 4), live ? row + at : (const __half*)p.q, live);
        }
    }
    cp_async_commit();
    // dimensions that are padding are 0 in every stage
    auto clear = [&](unsigned base, int panels, int dim) {
        const int from = dim / 8, n = panels * 8 - from;
        for (int i = tid; i < kStages * kKeys * n; i += kThreads) {
            const int c = from + i % n, key = i / n % kKeys, s = i / n / kKeys;
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(base + (s * panels + (c >> 3)) * kPanel + key * 128 + (((c & 7) ^ (key & 7)) << 4)), "r"(0) : "memory");
        }
    };
    if (p.dim % 64) clear(sk, kp, p.dim);
    if (p.vdim % 64) clear(sv, vp, p.vdim);
    cp_async_wait<0>();
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the tensor core reads them
    before_sync();
    __syncthreads();
    after_sync();
    pdl_trigger();  // the tensor memory is taken: nothing that starts now can keep it from this CTA
    const unsigned tmem = *tmem_slot, t_sum = tmem + TILES * 2 * kKeys;  // two turns of scores of each tile; weights take their place
    const int lowest = first_key(p, pos0), kt0 = lowest / kKeys, n = last / kKeys + 1 - kt0;
    bool ok = true;
    const int last_low = first_key(p, last);
    auto hides = [&](int j0) { return j0 + kKeys - 1 > pos0 || j0 < last_low; };  // whether some rows do not see some keys of the tile from j0 on

    if (warp >= kSoftWarps && warp < kIssues) {
        // A thread has sixteen dimensions of a key at a time.
        const int u0 = tid - kSoft;
        auto put = [&](unsigned from, unsigned base, int i, int dim, unsigned by) {
            const int j0 = (kt0 + i) * kKeys, blocks = dim / kPack;
            const bool whole = j0 >= lowest && j0 + kKeys - 1 <= last;
            const unsigned scales = from + kKeys * (dim / 2);
            // Sixteen dimensions of a key. (The first 64 dimensions' lanes begin with the even eighths, the next with the odd ones: eight lanes write 128 bytes in different banks.)
            auto unit = [&](unsigned codes, unsigned scale, unsigned to0, unsigned to1, unsigned first, int key) {
                unsigned x, y, code;
                x = ld_shared(codes + first);
                y = ld_shared(codes + (first ^ 4));
                code = ld_shared_u8(scale);
                // keys that are not there are 0: what was copied in their place, or not, may be no number
                if (!whole && (j0 + key < lowest || j0 + key > last)) code = 0;
                const __half2 s = __low2half2(scales_f16(code));
                __half2 v[4], w[4];
                units8(x, v);
                units8(y, w);
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to0), "r"(bits(__hmul2(v[0], s))), "r"(bits(__hmul2(v[1], s))), "r"(bits(__hmul2(v[2], s))), "r"(bits(__hmul2(v[3], s)))
                             : "memory");
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to1), "r"(bits(__hmul2(w[0], s))), "r"(bits(__hmul2(w[1], s))), "r"(bits(__hmul2(w[2], s))), "r"(bits(__hmul2(w[3], s)))
                             : "memory");
            };
            if ((blocks & blocks - 1) == 0) {  // a thread's units are the same dimensions of keys that lie a multiple of eight apart
                const int b = u0 & blocks - 1, key0 = over(u0, by), keys = over(kUnpack, by);
                const unsigned flip = b >> 2 & 1, c = (b & 3) * 2 + flip, row = base + (b >> 2) * kPanel + key0 * 128, to0 = row + ((c ^ (key0 & 7)) << 4), to1 = row + ((c ^ 1 ^ (key0 & 7)) << 4);
#pragma unroll 4
                for (int k = 0; k + key0 < kKeys; k += keys) unit(from + (u0 + k * blocks) * 8, scales + u0 + k * blocks, to0 + k * 128, to1 + k * 128, flip * 4, k + key0);
            } else {
#pragma unroll 2
                for (int u = u0; u < kKeys * blocks; u += kUnpack) {
                    const int key = over(u, by), b = u - key * blocks;
                    const unsigned flip = b >> 2 & 1, c = (b & 3) * 2 + flip, row = base + (b >> 2) * kPanel + key * 128;
                    unit(from + u * 8, scales + u, row + ((c ^ (key & 7)) << 4), row + ((c ^ 1 ^ (key & 7)) << 4), flip * 4, key);
                }
            }
        };
        // A weight of 0 does not cancel a value that is no number for the rows that do not see it: where there are such, it becomes 0, and the rows that see it are told.
        auto mark = [&](unsigned scales, unsigned bad) {
            if (u0 <= kKeys) st_shared(bad + u0 * 4, 0);
            asm volatile("bar.sync 1, 128;" ::: "memory");
            for (int u = u0; u < kKeys * (p.vdim / kPack); u += kUnpack)
                if ((ld_shared_u8(scales + u) & 127) == 127) {
                    const int key = over(u, p.by_value);
                    asm volatile("red.shared.or.b32 [%0], %1;" ::"r"(bad + 4 + key * 4), "r"(1u << (u - key * (p.vdim / kPack))) : "memory");
                    st_shared(bad, 1);
                    asm volatile("st.shared.u8 [%0], %1;" ::"r"(scales + u), "r"(0) : "memory");
                }
            asm volatile("bar.sync 1, 128;" ::: "memory");
        };
        auto tell = [&](unsigned there, unsigned free) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(there) : "memory");
                asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(free) : "memory");
            }
        };
        RingAt at, in;
        for (int i = 0; i < n; i++) {
            if (ok && !mbar_wait(raw_full + in.s * 8, in.parity)) ok = false;
            if (i >= kStages && ok && !mbar_wait(k_free + at.s * 8, at.parity ^ 1)) ok = false;
            put(raw + in.s * slot, sk + at.s * k_stage, i, p.dim, p.by_key);
            tell(k_full + at.s * 8, raw_free + in.s * 8);
            in.next(p.raw_slots);
            if (ok && !mbar_wait(raw_full + in.s * 8, in.parity)) ok = false;
            if (i >= kStages && ok && !mbar_wait(v_free + at.s * 8, at.parity ^ 1)) ok = false;
            if (hides((kt0 + i) * kKeys)) mark(raw + in.s * slot + kKeys * (p.vdim / 2), value_bad + at.s * (1 + kKeys) * 4);
            put(raw + in.s * slot, sv + at.s * v_stage, i, p.vdim, p.by_value);
            tell(v_full + at.s * 8, raw_free + in.s * 8);
            in.next(p.raw_slots);
            at.next(kStages);
        }
    } else if (warp == kCopies) {
        // What a page holds of 64 keys are two runs of bytes, of smaller pages' two each; pages in front of the window may be anybody's, and behind the last key there may be none.
        const int run = min(kKeys, 1 << p.shift);
        RingAt in;
        for (int i = 0; i < 2 * n; i++) {
            const int j0 = (kt0 + i / 2) * kKeys, d = i & 1 ? p.vdim : p.dim, a = max(j0, lowest) & ~(run - 1), b = min(last + 1, j0 + kKeys);
            unsigned char* pool = i & 1 ? p.values : p.keys;
            if (i >= p.raw_slots && ok && !mbar_wait(raw_free + in.s * 8, in.parity ^ 1)) ok = false;
            const unsigned bar = raw_full + in.s * 8, to = raw + in.s * slot;
            if (elect_one() && ok) {
                const int runs = (b - a + run - 1) >> (p.shift < 6 ? p.shift : 6);
                mbar_expect_tx(bar, runs * run * (d / kPack) * 9);
                for (int j = a; j < b; j += run) {
                    const unsigned char* from = held(p, pool, page_of(p, seq, j), g, d);
                    const int off = j & ((1 << p.shift) - 1);
                    auto copy = [&](unsigned dst, const unsigned char* src, int bytes) {
                        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
                    };
                    copy(to + (j - j0) * (d / 2), from + off * (d / 2), run * (d / 2));
                    copy(to + kKeys * (d / 2) + (j - j0) * (d / kPack), from + (((d / 2) << p.shift) + off * (d / kPack)), run * (d / kPack));
                }
            }
            __syncwarp();
            ok = __all_sync(0xffffffffu, ok);
            in.next(p.raw_slots);
        }
    } else if (warp == kIssues) {
        const unsigned base = (1u << 4) | (8u << 24);  // f16 × f16 → f32, M 128
        const unsigned by_keys = base | ((kKeys >> 3) << 17), by_values = base | (1u << 16) | ((unsigned)(vp * 8) << 17);  // the values' wide axis is the result's
        const unsigned long long dq = umma_kmajor_desc(sq0), dk = umma_kmajor_desc(sk), dv = umma_wide_desc(sv);
        RingAt ahead, at;  // stages of keys, of values
        unsigned turn_ahead = 0, turn = 0, parity = 0;
        auto next_scores = [&] {
            if (ok && !mbar_wait(k_full + ahead.s * 8, ahead.parity)) ok = false;
            after_sync();
            if (elect_one() && ok) {
                const unsigned long long k = dk + ahead.s * (k_stage >> 4);
#pragma unroll
                for (int tile = 0; tile < TILES; tile++) {
                    const unsigned long long q = dq + tile * (kp * kPanelQ >> 4);
                    for (int c = 0; c < kp; c++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            umma_bf16(tmem + (2 * tile + turn_ahead) * kKeys, q + c * (kPanelQ >> 4) + e * 2, k + c * (kPanel >> 4) + e * 2, by_keys, c > 0 || e > 0);
                    if (tile == TILES - 1) umma_commit(k_free + ahead.s * 8);
                    umma_commit(s_full + (2 * tile + turn_ahead) * 8);
                }
            }
            __syncwarp();
            ahead.next(kStages);
            turn_ahead ^= 1;
        };
        next_scores();
        for (int i = 0; i < n; i++) {
            if (i + 1 < n) next_scores();  // the products that read the weights in this place were issued before
            if (ok && !mbar_wait(v_full + at.s * 8, at.parity)) ok = false;
#pragma unroll
            for (int tile = 0; tile < TILES; tile++) {
                if (ok && !mbar_wait(w_full + (2 * tile + turn) * 8, parity)) ok = false;
                after_sync();
                if (elect_one() && ok) {
                    const unsigned long long v = dv + at.s * (v_stage >> 4);
#pragma unroll
                    for (int e = 0; e < kKeys / 16; e++) umma_weights(t_sum + tile * 128, tmem + (2 * tile + turn) * kKeys + e * 8, v + e * 128, by_values, i > 0 || e > 0);
                    if (tile == TILES - 1) umma_commit(v_free + at.s * 8);
                    umma_commit(o_done + (2 * tile + turn) * 8);
                }
                __syncwarp();
            }
            at.next(kStages);
            parity ^= turn;
            turn ^= 1;
        }
    } else {
        const int tile = warp / 4, tok = over(tid, p.by_rep), head = g * rep + tid - tok * rep;
        const bool live = tok < n_tok;
        const int pos = live ? pos0 + tok : last, low = first_key(p, pos);  // rows without a token compute something harmless
        const float mul = live ? p.q_mul[(long long)(sq.start + first + tok) * p.heads + head] : 0.f, cap2 = p.cap2, by_cap = mul * (1.f / kTwiceLog2e);
        const unsigned lanes = (unsigned)((warp & 3) * 32) << 16, sum = t_sum + lanes + tile * 128;
        float m = kNone, l = 0.f, sums[4];
        const float factor = value_factor(p, g);
        st_shared(row_bad + tid * 4, 0);
        RingAt at;
        for (int i = 0; i < n; i++) {
            const int j0 = (kt0 + i) * kKeys;
            if (ok && !mbar_wait(s_full + (2 * tile + at.s) * 8, at.parity)) ok = false;
            after_sync();
            const unsigned place = tmem + lanes + (2 * tile + at.s) * kKeys;
            const bool edge = hides(j0);
            bool near = false;
            // In base 2. Factors are positive (a negative one is in the queries): the largest score is that of the largest product.
            auto score = [&](float d) {
                return CAPPED ? capped_score<CAP == 2>(cap2, d * mul) : __fmul_ru(d, mul);
            };
            auto near_score = [&](float d, auto&& product) {
                const float u = d * by_cap;
                return product(u, cap_series(cap2, u * u));
            };
            auto largest = [&](float d) {
                if (CAP == 2 && near) return near_score(d, [](float u, float s) { return __fmul_ru(u, s); });
                return score(d);
            };
            auto hidden = [&](int j) { return j > pos || j < low; };
            // 32 products at a time, the next ones on their way
            auto each = [&](auto&& take) {
                unsigned v[2][32];
                tmem_ld32(v[0], place);
#pragma unroll
                for (int c = 0; c < kKeys / 32; c++) {
                    tmem_ld_wait();
                    if (c + 1 < kKeys / 32) tmem_ld32(v[(c + 1) & 1], place + (c + 1) * 32);
                    take(c * 32, v[c & 1]);
                }
            };
            float top = -INFINITY, least = INFINITY;
            if (edge) {
                each([&](int c, const unsigned (&v)[32]) {
#pragma unroll
                    for (int e = 0; e < 32; e++) top = fmaxf(top, hidden(j0 + c + e) ? -INFINITY : __uint_as_float(v[e]));
                });
                if (top != -INFINITY) top = largest(top);
            } else {
                each([&](int c, const unsigned (&v)[32]) {
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        top = fmaxf(fmaxf(top, __uint_as_float(v[e])), __uint_as_float(v[e + 1]));
                        if (CAPPED) least = fminf(fminf(least, __uint_as_float(v[e])), __uint_as_float(v[e + 1]));
                    }
                });
                // where no score that the warp's rows see is beyond a quarter of the cap they are a series (capped_score)
                if (CAPPED) near = __all_sync(0xffffffffu, fmaxf(fabsf(top), fabsf(least)) * mul <= 0.25f * kTwiceLog2e);
                top = largest(top);
            }
            if (__any_sync(0xffffffffu, top - m > kMost)) {
                const float now = fmaxf(m, __fsub_ru(top, kLeast)), keep = exp2_fast(m - now);
                m = now;
                l *= keep;
                if (i > 0) {
                    if (ok && !mbar_wait(o_done + (2 * tile + ((i - 1) & 1)) * 8, (unsigned)((i - 1) >> 1) & 1)) ok = false;
                    after_sync();
#pragma unroll 1
                    for (int c = 0; c < vp * 64; c += 16) {
                        unsigned v[16];
                        tmem_ld16(v, sum + c);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 16; e++) v[e] = __float_as_uint(__uint_as_float(v[e]) * keep);
                        tmem_st16(sum + c, v);
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < 4; e++) sums[e] = 0.f;
            auto near_weight = [&](float d) { return near_score(d, [&](float u, float s) { return __fmaf_rn(u, s, -m); }); };
            auto weight = [&](float d) {
                const float a = score(d) - m;
                return CAP == 2 && a > kMost ? kMost : a;  // (far above a quarter of the widest caps a score is off by more than that)
            };
            auto weigh = [&](int c, const unsigned (&v)[32], auto series, auto&& shown) {
                unsigned w[16];
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    float a, b;
                    if constexpr (CAPPED && series) a = near_weight(__uint_as_float(v[e])), b = near_weight(__uint_as_float(v[e + 1]));
                    else if (CAPPED) a = weight(__uint_as_float(v[e])), b = weight(__uint_as_float(v[e + 1]));
                    else a = __fmaf_rn(__uint_as_float(v[e]), mul, -m), b = __fmaf_rn(__uint_as_float(v[e + 1]), mul, -m);
                    a = exp2_fast(shown(a, j0 + c + e));
                    b = exp2_fast(shown(b, j0 + c + e + 1));
                    sums[e / 2 % 2] += a;
                    sums[2 + e / 2 % 2] += b;
                    w[e / 2] = bits(__floats2half2_rn(a, b));
                }
                tmem_st16(place + c / 2, w);  // where scores were that this thread has read twice
            };
            auto plainly = [](float x, int) { return x; };
            if (edge) {
                if (ok && !mbar_wait(v_full + i % kStages * 8, (unsigned)(i / kStages) & 1)) ok = false;
                const unsigned marks = value_bad + i % kStages * (1 + kKeys) * 4;
                if (ld_shared(marks)) {
                    unsigned bad = ld_shared(row_bad + tid * 4);
#pragma unroll 1
                    for (int j = 0; j < kKeys; j++)
                        if (!hidden(j0 + j)) bad |= ld_shared(marks + 4 + j * 4);
                    st_shared(row_bad + tid * 4, bad);
                }
            }
            if (edge) each([&](int c, const unsigned (&v)[32]) { weigh(c, v, std::false_type{}, [&](float x, int j) { return hidden(j) ? -INFINITY : x; }); });
            else if (CAPPED && near) each([&](int c, const unsigned (&v)[32]) { weigh(c, v, std::true_type{}, plainly); });
            else each([&](int c, const unsigned (&v)[32]) { weigh(c, v, std::false_type{}, plainly); });
            l += (sums[0] + sums[1]) + (sums[2] + sums[3]);
            tmem_st_wait();
            before_sync();
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(w_full + (2 * tile + at.s) * 8) : "memory");
            at.next(2);
        }
        if (ok && !mbar_wait(o_done + (2 * tile + ((n - 1) & 1)) * 8, (unsigned)((n - 1) >> 1) & 1)) ok = false;
        after_sync();
        float scale = factor / l;
        if (p.sink) {
            const float top = fmaxf(m, 0.f), keep = exp2_fast(m - top);
            scale = factor * keep / (l * keep + exp2_fast(-top));
        }
        // 64 dimensions of 32 rows at a time by way of shared memory, where the queries were, so that eight lanes write a row's 128 bytes
        unsigned char* mine = smem + tile * kp * kPanelQ + (warp & 3) * 32 * 128;
#pragma unroll 1
        for (int c = 0; c < vp * 64; c += 64) {
            unsigned v[2][32];
            tmem_ld32(v[0], sum + c);
            tmem_ld32(v[1], sum + c + 32);
            tmem_ld_wait();
            const unsigned bad = ld_shared(row_bad + tid * 4) >> c / kPack & 15;
            if (bad)
#pragma unroll
                for (int e = 0; e < 64; e++)
                    if (bad >> e / kPack & 1) v[e / 32][e % 32] = 0x7FFFFFFF;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const unsigned* x = v[e / 4] + e % 4 * 8;
                uint4 q;
                q.x = pack_bf16(__uint_as_float(x[0]) * scale, __uint_as_float(x[1]) * scale);
                q.y = pack_bf16(__uint_as_float(x[2]) * scale, __uint_as_float(x[3]) * scale);
                q.z = pack_bf16(__uint_as_float(x[4]) * scale, __uint_as_float(x[5]) * scale);
                q.w = pack_bf16(__uint_as_float(x[6]) * scale, __uint_as_float(x[7]) * scale);
                *reinterpret_cast<uint4*>(mine + lane * 128 + ((e ^ (lane & 7)) << 4)) = q;
            }
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int row = e * 4 + lane / 8, at = lane % 8, R = tid - lane + row, t = over(R, p.by_rep), h = g * rep + R - t * rep;
                if (t < n_tok && ok && c + at * 8 < p.vdim)
                    *reinterpret_cast<uint4*>((bf16*)p.out + ((long long)(sq.start + first + t) * p.heads + h) * p.vdim + c + at * 8) = *reinterpret_cast<const uint4*>(mine + row * 128 + ((at ^ (row & 7)) << 4));
            }
            __syncwarp();
        }
    }
    if (!ok && lane == 0) report(p.err, ERR_WAIT_TIMEOUT, p.node, (long long)blockIdx.x, (long long)warp);
    before_sync();
    __syncthreads();
    if (warp == kIssues) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
}

// Bytes without the slots of copies
int smem_of(int dim, int vdim, int tiles) {
    const int kp = (dim + 63) / 64, vp = (vdim + 63) / 64;
    return 1024 + tiles * kp * (int)kPanelQ + kStages * (kp + vp) * (int)kPanel + (4 * kStages + 12 + 2 * kSlots) * 8 + 16 + kStages * (1 + kKeys) * 4 + tiles * kRows * 4;
}

}  // namespace

PackedPrefill packed_prefill_of(int64_t dim, int64_t vdim, int64_t rows, int64_t kv_heads, int64_t rep, float cap2) {
    // Two tiles share what is unpacked, one tile has half the rows to wait for. From 96 dimensions of a key on two pay as soon as single tiles would share SMs; below, a tile's products are short, and pairs have
    // to fill the device twice. us a launch with one, two: 4096 tokens of 32 heads over 16 225, 186, of 16 heads over 4 133, 91, of 8 heads of 96 over 4 99, 92; 1999 behind 1000 of 16 heads over 4 81, 71,
    // capped 105, 94; 600 of 32 over 16 (160 single tiles) 24, 26, behind 2000 75, 63, 300 (80) 18, 20; of 80 dimensions and values of 64, 8 heads, 4096 (256) 88, 92, of 64 79, 85, of 12 heads over 2
    // with values of 128 (384) 93, 91, 1999 (188) 46, 51.
    const int64_t pairs = (rows * rep + 2 * kRows - 1) / (2 * kRows) * kv_heads;
    const int tiles = dim <= 128 && vdim <= 128 && (dim >= 96 ? 2 * pairs > sm_count() : pairs >= 2 * sm_count()) ? 2 : 1;
    const PackKernel of[2][3] = {{packed_prefill<1, 0>, packed_prefill<1, 1>, packed_prefill<1, 2>}, {packed_prefill<2, 0>, packed_prefill<2, 1>, packed_prefill<2, 2>}};
    const PackKernel k = of[tiles - 1][cap2 > kWideCap ? 2 : cap2 > 0.f];
    // With 512 columns of tensor memory a CTA has its SM alone, with 256 it shares it with one other.
    const bool alone = tiles == 2 || vdim > 128;
    const int fixed = smem_of((int)dim, (int)vdim, tiles), slot = kKeys * (int)std::max(dim, vdim) / kPack * 9, room = (alone || fixed + 2 * slot > 112 * 1024 ? 226 : 112) * 1024;
    const int slots = std::min(kSlots, (room - fixed) / slot), smem = fixed + slots * slot;
    return {k, alone ? std::max(smem, 120 * 1024) : smem, tiles * kRows, tiles * kRows + kUnpack + 64, slots};
}

}  // namespace oxk
