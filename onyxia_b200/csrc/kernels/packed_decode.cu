// Single tokens over keys and values in 4 bits: sequences with one new token, their keys split over CTAs and warps, rotation, norms, storing and joining in one launch.
//
// A warp copies 32 keys and values at a time for itself (bulk copies: what a page holds of them is four runs of bytes) and takes 16 of them as both products' rows: S^T = K q^T, O^T = V^T P^T
// (`mma.sync`, f16). The order of a contraction is free, so a lane holds for S the whole blocks of 16 dimensions of two keys, whose codes become f16 and are multiplied by their scale (exactly), and
// for O^T the same run of dimensions of four keys: pairs of keys come together by swapping halves of bytes.
//
// What bounds it: 9/16 of a byte per dimension comes from memory, but 16 keys and values of 128 dimensions each cost a warp 313 instructions (70 conversions of codes to f16, 64 products with scales), and
// the four CTAs of an SM issue in 55 % of its slots: 64 sequences behind 8191, 16 heads of keys, 267 us (4.5 TB/s; memory alone 185). Eight query heads of a key at most are multiplied at a time: a wider
// matrix instruction would multiply mostly nothing, and want values as f16 in shared memory first. Loads by registers took 393 us (too few are under way), bulk copies 348, 16 more keys under way while
// the first are weighed 293, even shares of all blocks 267. One sequence behind 519 of a key head of 256: 18 us, a chain of lookups, rotation, keys and joining.
// Of more than eight query heads of a key every eight read and convert the keys again: 64 sequences behind 8191 of one key head of 128 take 36 us with 8 heads, 51 with 9, 53 with 16, 87 with 32.
#include <cmath>
#include <type_traits>

#include "packed_cache.cuh"

namespace oxk {

namespace {

// Weights are those of products that are not rounded before the reference, a rounded one, is subtracted. Where that rounding may come near kLeast, all are rounded alike first.
constexpr float kLarge = 0x1p25f;
constexpr int kWarps = 4, kThreads = kWarps * 32, kPages = 256, kHeads = 8, kKeys = 16, kTile = 2 * kKeys, kStages = 3, kMostParts = 64;

__device__ __forceinline__ void mma_f16(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// KS: blocks of 16 dimensions of a key per lane (64 · KS dimensions at most); VC: bytes of codes of a value per lane (16 · VC dimensions at most)
template <int KS, int VC> struct Smem {
    static constexpr int dk = 64 * KS, dv = 16 * VC;
    static constexpr int q_stride = dk * 2 + 16;
    static constexpr int part = part_size(kHeads, dv);            // floats of one partial result
    static constexpr int stage = kTile * (dk + dv) / kPack * 9;   // codes of keys, scales, codes of values, scales
    static constexpr int rings = kStages * kWarps * stage, parts = kWarps * part * 4;  // [stages][warps][stage]; partial results take their place
    // before the last stage is filled: queries [8 heads] f16, cosines and sines in 64 bits, and in 32, and what comes from the projection: queries of 8 heads, the key, the value
    static constexpr int q = (kStages - 1) * kWarps * stage, angle = q + kHeads * q_stride, raw = angle + dk * 12;
    static constexpr int total = rings > parts ? rings : parts;
    static_assert(raw + (kHeads + 1) * dk * 2 + dv * 2 <= rings && angle % 16 == 0 && raw % 16 == 0, "all of it fits the last stage");
};

// What single tokens have to go through: blocks of 128 keys of every sequence and group of query heads (a cell), cell behind cell.
template <class P> __device__ __forceinline__ int blocks_of(const P& p, const SeqRow& s) {
    return s.len == 1 ? s.past / (kTile * kWarps) + 1 - first_key(p, s.past) / (kTile * kWarps) : 0;
}

// Merged partial results of `heads` heads, a warp each; part k of a head begins at at(k) + head · (DV + 2): maximum, sum, accumulator. n ≤ 64.
template <int DV, class At> __device__ __forceinline__ void join_parts(const PackP& p, At&& at, int n, int heads, int dim, float factor, bf16* out, float* raw) {
    constexpr int C = (DV + 31) / 32;
    const int lane = threadIdx.x & 31;
    for (int r = threadIdx.x >> 5; r < heads; r += kWarps) {
        // lane i weighs parts i and i + 32; a part that saw no key has the maximum kNone, sum and values 0
        float pm[2], pl[2];
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const bool in = k * 32 + lane < n;
            const float* head = at(in ? k * 32 + lane : 0) + r * (DV + 2);
            pm[k] = in ? head[0] : kNone;
            pl[k] = in ? head[1] : 0.f;
        }
        float m = warp_max(fmaxf(pm[0], pm[1]));
        if (!raw && p.sink) m = fmaxf(m, 0.f);  // a score of 0 without a value
        const float f0 = exp2_fast(pm[0] - m), f1 = exp2_fast(pm[1] - m), l = warp_sum(fmaf(pl[0], f0, pl[1] * f1)) + (!raw && p.sink ? exp2_fast(-m) : 0.f);
        float o[C] = {};
#pragma unroll 4
        for (int i = 0; i < n; i++) {
            const float f = __shfl_sync(0xffffffffu, i < 32 ? f0 : f1, i & 31);
            const float* head = at(i) + r * (DV + 2) + 2;
#pragma unroll
            for (int c = 0; c < C; c++)
                if (c * 32 + lane < DV) o[c] = fmaf(head[c * 32 + lane], f, o[c]);
        }
        if (raw) {
            float* to = raw + r * (DV + 2);
            if (lane == 0) to[0] = m, to[1] = l;
#pragma unroll
            for (int c = 0; c < C; c++)
                if (c * 32 + lane < DV) to[2 + c * 32 + lane] = o[c];
        } else {
            const float f = factor / l;
#pragma unroll
            for (int c = 0; c < C; c++)
                if (c * 32 + lane < dim) out[r * dim + c * 32 + lane] = __float2bfloat16_rn(o[c] * f);
        }
    }
}

// CTAs have a piece of a cell each where there is room for all cells at once (emit_packed_attention), otherwise the same share of the blocks of all cells: cells that no CTA has alone are joined by the
// last of those that have a part. WHOLE: keys have 64 · KS dimensions and values 16 · VC.
template <int KS, int VC, bool WHOLE, int RESIDENT> __global__ void __launch_bounds__(kThreads, RESIDENT) packed_decode(const PackP p) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ unsigned arrived;
    __shared__ int page_s[kPages];  // this CTA's pages, checked
    __shared__ float factor_s[kHeads];
    __shared__ __align__(8) unsigned long long full_s[kWarps * kStages];
    using L = Smem<KS, VC>;
    constexpr int step = kTile * kWarps;
    pdl_trigger();
    if (!p.append) pdl_wait();  // another node of the step may have written any of the keys
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g8 = lane >> 2, t4 = lane & 3;
    // no launch of a step writes the batch description or the keys and values of earlier steps (where the module computes the
    // former, this launch does not begin early): they may be read while the launches before this one finish
    const int rep = p.heads / p.kv_heads, groups = (rep + kHeads - 1) / kHeads, n_groups = p.kv_heads * groups, dim = WHOLE ? 64 * KS : p.dim, vdim = WHOLE ? 16 * VC : p.vdim;
    long long each = 0, u0 = 0, left = 0;  // blocks: a CTA's share, where it begins counted over all cells, what it has to do
    int seq = 0, group = 0, begin = 0;     // where it begins: sequence, group, block
    SeqRow sq{0, 0, 0, 0};
    if (p.pieces) {
        const int cell = blockIdx.x / p.pieces, piece = blockIdx.x - cell * p.pieces;
        seq = cell / n_groups;
        group = cell - seq * n_groups;
        sq = checked_seq(p, seq);
        if (p.only && sq.len > 1 && tid == 0) report(p.err, ERR_BATCH_ROWS, p.node, seq, sq.len);
        const int n = blocks_of(p, sq), of = min(n, p.pieces);
        if (piece < of) begin = (int)((long long)n * piece / of), left = (int)((long long)n * (piece + 1) / of) - begin;
    } else {
        long long total = 0;
        int longest = 0;  // cell
#pragma unroll 4
        for (int r0 = 0; r0 < p.n_seqs; r0 += 32) {
            const SeqRow s = r0 + lane < p.n_seqs ? checked_seq(p, r0 + lane) : SeqRow{0, 0, 0, 0};
            if (p.only && s.len > 1 && blockIdx.x == 0 && warp == 0) report(p.err, ERR_BATCH_ROWS, p.node, r0 + lane, s.len);
            const int n = blocks_of(p, s);
            total += (long long)__reduce_add_sync(0xffffffffu, n) * n_groups;
            longest = max(longest, __reduce_max_sync(0xffffffffu, n));
        }
        const long long share = total >> 31 ? (total + gridDim.x - 1) / gridDim.x : ((unsigned)total + gridDim.x - 1) / gridDim.x;
        each = max(share, (long long)((longest + kMostParts - 2) / (kMostParts - 2)));
        u0 = blockIdx.x * each;
        left = min(each, total - u0);
        long long before = 0;
        for (int r0 = 0; left > 0; r0 += 32) {
            const SeqRow s = r0 + lane < p.n_seqs ? checked_seq(p, r0 + lane) : SeqRow{0, 0, 0, 0};
            const int n = blocks_of(p, s);
            const long long chunk = (long long)__reduce_add_sync(0xffffffffu, n) * n_groups;
            if (before + chunk <= u0) {
                before += chunk;
                continue;
            }
            int inc = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += v;
            }
            const int at = __ffs(__ballot_sync(0xffffffffu, before + (long long)inc * n_groups > u0)) - 1, blocks = __shfl_sync(0xffffffffu, n, at);
            const long long in = u0 - before - (long long)(__shfl_sync(0xffffffffu, inc, at) - blocks) * n_groups;
            seq = r0 + at;
            sq = SeqRow{__shfl_sync(0xffffffffu, s.start, at), __shfl_sync(0xffffffffu, s.len, at), __shfl_sync(0xffffffffu, s.past, at), 0};
            group = in >> 31 ? (int)(in / blocks) : (int)((unsigned)in / (unsigned)blocks);
            begin = (int)(in - (long long)group * blocks);
            break;
        }
    }
    if (tid < kWarps * kStages) mbar_init(smem_u32(full_s + tid), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    bool ok = true;
    unsigned rounds = 0;  // parities of the stages' barriers
    long long u = u0;
    if (left <= 0) return pdl_wait();
    // turns per position of two pairs, by the first two warps
    double turns[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int i = tid + k * 64;
        turns[k] = warp < 2 && i < p.half ? (double)p.turns[i] + (double)p.turns[p.half + i] : 0.0;
    }
    while (true) {
        const int g = group / groups, h0 = g * rep + (group % groups) * kHeads, n_heads = min(kHeads, (g + 1) * rep - h0), pos = sq.past, n_blocks = blocks_of(p, sq);
        const int count = (int)min((long long)(n_blocks - begin), left), low = first_key(p, pos), lo = (low / step + begin) * step, hi = min(lo + count * step, pos + 1);
        const int from = max(lo, low), page0 = from >> p.shift, n_pages = ((hi - 1) >> p.shift) - page0 + 1;  // pages in front of the window may be anybody's
        for (int i = tid; i < min(n_pages, kPages); i += kThreads) page_s[i] = (int)page_of(p, seq, (page0 + i) << p.shift);
        const bool newest = begin + count == n_blocks;  // these keys include the new one
        if (u == u0) __syncthreads();
        auto page_at = [&](int j) {
            const int i = (j >> p.shift) - page0;
            return i < kPages ? (long long)page_s[i] : page_of(p, seq, j);
        };
        const int first = lo + warp * kTile, tiles = first < hi ? (hi - first + step - 1) / step : 0;
        const long long key_page = ((long long)p.kv_heads << p.shift) * (dim / kPack) * 9, value_page = ((long long)p.kv_heads << p.shift) * (vdim / kPack) * 9;
        const unsigned char *keys0 = held(p, p.keys, 0, g, dim), *values0 = held(p, p.values, 0, g, vdim);
        // a stage: what a page holds of the tile's keys and values, run behind run
        const int key_scales = kTile * (dim / 2), value_codes = key_scales + kTile * (dim / kPack), value_scales = value_codes + kTile * (vdim / 2);
        const unsigned ring = smem_u32(smem) + warp * L::stage, full = smem_u32(full_s + warp * kStages);
        // Tiles lie in one page, or their halves in one each; what lies beyond the keys of this CTA may be on no page.
        const bool whole_tiles = (1 << p.shift) >= kTile;
        auto copy = [&](int i, unsigned s) {
            if (i >= tiles || !elect_one()) return;
            const int j0 = first + i * step;
            const unsigned to = ring + s * kWarps * L::stage, bar = full + s * 8;
            // keys from j on, which stand `at` keys behind the tile's first
            auto runs = [&](int j, int at, int n) {
                const long long pg = page_at(max(j, from));
                const int off = j & ((1 << p.shift) - 1);
                const unsigned char *k = keys0 + pg * key_page, *v = values0 + pg * value_page;
                auto run = [&](int dst, const unsigned char* src, int bytes) {
                    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to + dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
                };
                run(at * (dim / 2), k + off * (dim / 2), n * (dim / 2));
                run(key_scales + at * (dim / kPack), k + (((dim / 2) << p.shift) + off * (dim / kPack)), n * (dim / kPack));
                run(value_codes + at * (vdim / 2), v + off * (vdim / 2), n * (vdim / 2));
                run(value_scales + at * (vdim / kPack), v + (((vdim / 2) << p.shift) + off * (vdim / kPack)), n * (vdim / kPack));
            };
            const int half_bytes = kKeys * ((dim + vdim) / kPack) * 9;
            if (whole_tiles) {
                if (j0 + kTile > from) {
                    mbar_expect_tx(bar, 2 * half_bytes);
                    runs(j0, 0, kTile);
                } else {
                    mbar_expect_tx(bar, 0);
                }
            } else {
                const bool one = j0 + kKeys > from && j0 < hi, two = j0 + kTile > from && j0 + kKeys < hi;
                mbar_expect_tx(bar, (one + two) * half_bytes);
                if (one) runs(j0, 0, kKeys);
                if (two) runs(j0 + kKeys, kKeys, kKeys);
            }
        };
        // The first tiles are on their way while the launch before this one ends, unless the new key is among them.
        const bool late = newest && p.append && (pos - lo) / step < kStages - 1;
        auto fill = [&](int i, int end) {
#pragma unroll 1
            for (; i < end; i++) copy(i, i);
        };
        if (u == u0 && !late) fill(0, kStages - 1);
        double *cs = reinterpret_cast<double*>(smem + L::angle), *sn = cs + L::dk / 2;
        float *short_cs = reinterpret_cast<float*>(sn + L::dk / 2), *short_sn = short_cs + L::dk / 2;
        const bool stores = newest && p.append;
        if (warp < 2) {
#pragma unroll
            for (int k = 0; k < 2; k++)
                if (tid + k * 64 < p.half) short_angle(pos, turns[k], short_cs + tid + k * 64, short_sn + tid + k * 64);
        } else if (stores) exact_angles(p, pos, cs, sn, tid - 64, 64);
        if (u == u0) pdl_wait();
        // all that comes from the projection at once
        const bf16* x = (const bf16*)p.proj + (long long)sq.start * p.ld;
        bf16 *raw = reinterpret_cast<bf16*>(smem + L::raw), *raw_key = raw + kHeads * L::dk, *raw_value = raw_key + L::dk;
        const bf16 *from_q = x + p.q_off + (long long)h0 * dim, *from_k = x + p.k_off + (long long)g * dim, *from_v = x + p.v_off + (long long)g * vdim;
        if (p.by8) {
            const int chunks = dim / 8;
            for (int c = tid; c < n_heads * chunks; c += kThreads) {
                const int r = over(c, p.by_eighths);
                *reinterpret_cast<uint4*>(raw + r * L::dk + (c - r * chunks) * 8) = *reinterpret_cast<const uint4*>(from_q + c * 8);
            }
            if (stores) {
                for (int c = tid; c < chunks; c += kThreads) *reinterpret_cast<uint4*>(raw_key + c * 8) = *reinterpret_cast<const uint4*>(from_k + c * 8);
                for (int c = kThreads - 1 - tid; c < vdim / 8; c += kThreads) *reinterpret_cast<uint4*>(raw_value + c * 8) = *reinterpret_cast<const uint4*>(from_v + c * 8);
            }
        } else {
            for (int r = warp; r < n_heads; r += kWarps)
                for (int i = lane; i < dim; i += 32) raw[r * L::dk + i] = from_q[r * dim + i];
            for (int i = tid; stores && i < dim; i += kThreads) raw_key[i] = from_k[i];
            for (int i = tid; stores && i < vdim; i += kThreads) raw_value[i] = from_v[i];
        }
        __syncthreads();
        if (u != u0 && !late) fill(0, kStages - 1);
        if (stores) {
            // (where a key head has several groups of queries, each CTA that needs the new key stores it: the same bits)
            const bool key = warp < 2;
            const int d = key ? dim : vdim;
            unsigned char *to = held(p, key ? p.keys : p.values, page_at(pos), g, d), *codes = codes_of(p, to, pos, d), *scales = scales_of(p, to, pos, d);
            const float factor = key ? key_factor(p, g) : value_factor(p, g);
            const double f = key ? norm_factor(p, raw_key) : 1.0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int c = j * 64 + (warp & 1) * 32, i = c + lane;
                if (c >= d) break;
                const float v = i >= d ? 0.f : key ? __bfloat162float(__float2bfloat16_rn((float)(turned(p.half, raw_key, cs, sn, i) * f))) : __bfloat162float(raw_value[i]);
                put_32(codes, scales, c, d, factor, v);
            }
        }
#pragma unroll
        for (int r = warp; r < kHeads; r += kWarps) {
            __half* to = reinterpret_cast<__half*>(smem + L::q + r * L::q_stride);
            if (r >= n_heads) {  // nobody's: nothing
#pragma unroll
                for (int j = 0; j < L::dk / 32; j++) to[j * 32 + lane] = __float2half_rn(0.f);
                if (lane == 0) factor_s[r] = 1.f;
                continue;
            }
            const bf16* from = raw + r * L::dk;
            const float f = (float)norm_factor(p, from);
            float v[L::dk / 32], most = 0.f;
#pragma unroll
            for (int j = 0; j < L::dk / 32; j++) {
                const int i = j * 32 + lane;
                v[j] = 0.f;
                if (i < dim) {
                    const float a = to_f(from[i]);
                    v[j] = i >= 2 * p.half ? a : i < p.half ? a * short_cs[i] - to_f(from[i + p.half]) * short_sn[i] : a * short_cs[i - p.half] + to_f(from[i - p.half]) * short_sn[i - p.half];
                }
                v[j] *= f;
                most = fmaxf(most, fabsf(v[j]));
            }
            const int e = query_exponent(warp_max(most));
            const float down = copysignf(power_down(e), p.mul2);
#pragma unroll
            for (int j = 0; j < L::dk / 32; j++) to[j * 32 + lane] = __float2half_rn(p.mul2 != 0.f ? v[j] * down : 0.f);
            if (lane == 0) factor_s[r] = (p.mul2 != 0.f ? fabsf(p.mul2) : 1.f) * power_up(e) * key_factor(p, g);
        }
        __syncthreads();
        unsigned q[KS][8];
#pragma unroll
        for (int c = 0; c < KS; c++)
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const uint4 v = *reinterpret_cast<const uint4*>(smem + L::q + g8 * L::q_stride + (t4 * KS + c) * 32 + half * 16);
                q[c][4 * half] = v.x;
                q[c][4 * half + 1] = v.y;
                q[c][4 * half + 2] = v.z;
                q[c][4 * half + 3] = v.w;
            }
        // copies read the new key, and take the queries' place
        if (stores) asm volatile("fence.proxy.async;" ::: "memory");
        else asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
        fill(late ? 0 : kStages - 1, kStages);
        // a lane holds scores of keys g8, g8 + 8 and heads 2 · t4, 2 · t4 + 1, and results of dimensions 2 · VC · g8 + 2i, + 1 of these heads
        const float mul[2] = {factor_s[2 * t4], factor_s[2 * t4 + 1]};
        const bool capped = p.cap2 > 0.f;
        const float weigh[2] = {capped ? 1.f : mul[0], capped ? 1.f : mul[1]}, back[2] = {1.f / weigh[0], 1.f / weigh[1]};
        // `top`: what weights are taken against; `most`: what a score may be until that moves, before it is multiplied; `l`: sums of the weights, by a product with ones
        float o[VC][4], l[4] = {0.f, 0.f, 0.f, 0.f}, top[2] = {kNone, kNone}, most[2] = {kNone, kNone};
#pragma unroll
        for (int n = 0; n < VC; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[n][e] = 0.f;
        // Whether it is done: scores beyond kLarge are left to the form for edges.
        auto attend = [&](auto edge, int j0, const unsigned char* stage) {
            // (the two halves in turn, each in two sums: a product does not wait for the one before it)
            uint2 key[2][2][KS];
            unsigned key_scale[2][2];  // KS bytes
#pragma unroll
            for (int half = 0; half < 2; half++)
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    const int row = half * kKeys + g8 + 8 * r;
                    const unsigned char *codes = stage + row * (dim / 2) + t4 * KS * 8, *scales = stage + key_scales + row * (dim / kPack) + t4 * KS;
                    if constexpr (WHOLE && KS == 1) {
                        key[half][r][0] = *reinterpret_cast<const uint2*>(codes);
                        key_scale[half][r] = *scales;
                    } else if constexpr (WHOLE) {
#pragma unroll
                        for (int c = 0; c < KS; c += 2) {
                            const uint4 v = reinterpret_cast<const uint4*>(codes)[c / 2];
                            key[half][r][c] = make_uint2(v.x, v.y);
                            key[half][r][c + 1] = make_uint2(v.z, v.w);
                        }
                        key_scale[half][r] = KS == 2 ? *reinterpret_cast<const unsigned short*>(scales) : *reinterpret_cast<const unsigned*>(scales);
                    } else {
                        key_scale[half][r] = 0;
#pragma unroll
                        for (int c = 0; c < KS; c++) {
                            const bool in = t4 * KS + c < dim / kPack;
                            key[half][r][c] = in ? reinterpret_cast<const uint2*>(codes)[c] : make_uint2(0, 0);
                            key_scale[half][r] |= in ? (unsigned)scales[c] << (8 * c) : 0u;
                        }
                    }
                }
            float s[2][4], more[2][4];
#pragma unroll
            for (int half = 0; half < 2; half++)
#pragma unroll
                for (int e = 0; e < 4; e++) s[half][e] = more[half][e] = 0.f;
#pragma unroll
            for (int c = 0; c < KS; c++)
#pragma unroll
                for (int w = 0; w < 2; w++)
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        const __half2 both = scales_f16(__byte_perm(key_scale[half][0], key_scale[half][1], c | (4 + c) << 4)), s0 = __low2half2(both), s1 = __high2half2(both);
                        __half2 a[4], b[4];
                        units8(w ? key[half][0][c].y : key[half][0][c].x, a);
                        units8(w ? key[half][1][c].y : key[half][1][c].x, b);
                        mma_f16(s[half], bits(__hmul2(a[0], s0)), bits(__hmul2(b[0], s1)), bits(__hmul2(a[1], s0)), bits(__hmul2(b[1], s1)), q[c][4 * w], q[c][4 * w + 1]);
                        mma_f16(more[half], bits(__hmul2(a[2], s0)), bits(__hmul2(b[2], s1)), bits(__hmul2(a[3], s0)), bits(__hmul2(b[3], s1)), q[c][4 * w + 2], q[c][4 * w + 3]);
                    }
#pragma unroll
            for (int half = 0; half < 2; half++)
#pragma unroll
                for (int e = 0; e < 4; e++) s[half][e] += more[half][e];
            bool above = false;
            auto cap = [&](auto wide) {
#pragma unroll
                for (int half = 0; half < 2; half++)
#pragma unroll
                    for (int e = 0; e < 4; e++) s[half][e] = capped_score<decltype(wide)::value>(p.cap2, s[half][e] * mul[e & 1]);
            };
            if (capped) p.cap2 > kWideCap ? cap(std::true_type{}) : cap(std::false_type{});
#pragma unroll
            for (int half = 0; half < 2; half++) {
                if constexpr (edge) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int j = j0 + half * kKeys + g8 + 8 * (e >> 1);
                        if (j >= hi || j < low) s[half][e] = -INFINITY;
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; e++) above |= s[half][e] > most[e & 1];
            }
            if (__any_sync(0xffffffffu, above)) {
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float now = fmaxf(fmaxf(s[0][e], s[0][e + 2]), fmaxf(s[1][e], s[1][e + 2]));
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, d));
                    if (!edge && __any_sync(0xffffffffu, fabsf(now * weigh[e]) > kLarge)) return false;
                    now = now > -INFINITY ? fmaxf(top[e], __fsub_ru(__fmul_ru(now, weigh[e]), kLeast)) : top[e];
                    const float keep = exp2_fast(top[e] - now);
                    top[e] = now;
                    const float beyond = (now + kMost) * back[e];
                    most[e] = now > kNone ? __fmaf_rn(fabsf(beyond), -0x1p-21f, beyond) : kNone;  // (three roundings, 2^-24 of it each)
                    l[e] *= keep;
                    l[e + 2] *= keep;
#pragma unroll
                    for (int n = 0; n < VC; n++) {
                        o[n][e] *= keep;
                        o[n][e + 2] *= keep;
                    }
                }
            }
#pragma unroll
            for (int half = 0; half < 2; half++) {
                unsigned pb[2];
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    auto weight = [&](float x, int e) { return exp2_fast(edge ? __fmul_ru(x, weigh[e]) - top[e] : __fmaf_rn(x, weigh[e], -top[e])); };
                    const float w0 = weight(s[half][2 * r], 0), w1 = weight(s[half][2 * r + 1], 1);
                    pb[r] = transpose8x8(bits(__floats2half2_rn(w0, w1)));
                }
                constexpr unsigned kOnes = 0x3C003C00u;
                mma_f16(l, kOnes, kOnes, kOnes, kOnes, pb[0], pb[1]);
                unsigned value[4][VC / 4], value_scale[4];  // one byte, or two
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int row = half * kKeys + 2 * t4 + (e & 1) + 8 * (e >> 1);
                    const unsigned char *codes = stage + value_codes + row * (vdim / 2) + g8 * VC, *scales = stage + value_scales + row * (vdim / kPack) + (VC == 4 ? g8 / 2 : g8 * (VC / 8));
                    if constexpr (VC < 16) {
                        const bool in = WHOLE || g8 * VC < vdim / 2;
                        if constexpr (VC == 4) {
                            value[e][0] = in ? *reinterpret_cast<const unsigned*>(codes) : 0u;
                        } else {
                            const uint2 w = in ? *reinterpret_cast<const uint2*>(codes) : make_uint2(0, 0);
                            value[e][0] = w.x;
                            value[e][1] = w.y;
                        }
                        value_scale[e] = in ? *scales : 0u;
                    } else if constexpr (WHOLE) {
                        const uint4 w = *reinterpret_cast<const uint4*>(codes);
                        value[e][0] = w.x;
                        value[e][1] = w.y;
                        value[e][2] = w.z;
                        value[e][3] = w.w;
                        value_scale[e] = *reinterpret_cast<const unsigned short*>(scales);
                    } else {
                        value_scale[e] = 0;
#pragma unroll
                        for (int c = 0; c < 2; c++) {
                            const bool in = g8 * VC + c * 8 < vdim / 2;
                            const uint2 w = in ? reinterpret_cast<const uint2*>(codes)[c] : make_uint2(0, 0);
                            value[e][2 * c] = w.x;
                            value[e][2 * c + 1] = w.y;
                            value_scale[e] |= in ? (unsigned)scales[c] << (8 * c) : 0u;
                        }
                    }
                    // what lies beyond the keys may be no number, which a weight of 0 would not cancel: its scale would be none
                    if constexpr (edge)
                        if (j0 + row >= hi || j0 + row < low) value_scale[e] = 0;
                }
#pragma unroll
                for (int b = 0; b < (VC + 7) / 8; b++) {
                    const __half2 s01 = scales_f16(__byte_perm(value_scale[0], value_scale[1], b | (4 + b) << 4)), s23 = scales_f16(__byte_perm(value_scale[2], value_scale[3], b | (4 + b) << 4));
#pragma unroll
                    for (int w = 2 * b; w < 2 * b + (VC < 8 ? 1 : 2); w++) {
                        // pairs of keys in a byte: the earlier dimension of each byte, then the later one
                        constexpr unsigned kLow = 0x0F0F0F0Fu;
                        __half2 a[4], c[4], d[4], f[4];
                        units8((value[0][w] & kLow) | (value[1][w] << 4 & ~kLow), a);
                        units8((value[0][w] >> 4 & kLow) | (value[1][w] & ~kLow), c);
                        units8((value[2][w] & kLow) | (value[3][w] << 4 & ~kLow), d);
                        units8((value[2][w] >> 4 & kLow) | (value[3][w] & ~kLow), f);
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            mma_f16(o[4 * w + e], bits(__hmul2(a[e], s01)), bits(__hmul2(c[e], s01)), bits(__hmul2(d[e], s23)), bits(__hmul2(f[e], s23)), pb[0], pb[1]);
                    }
                }
            }
            return true;
        };
        unsigned at = 0;
        bool large = false;
#pragma unroll 1
        for (int i = 0; i < tiles; i++) {
            if (ok && !mbar_wait(full + at * 8, rounds >> at & 1)) ok = false;
            rounds ^= 1u << at;
            const int j0 = first + i * step;
            const unsigned char* stage = smem + (at * kWarps + warp) * L::stage;
            if (large || j0 + kTile > hi || j0 < low || !attend(std::false_type{}, j0, stage)) {
                attend(std::true_type{}, j0, stage);
                large |= (top[0] > kNone && fabsf(top[0]) > kLarge) || (top[1] > kNone && fabsf(top[1]) > kLarge);
                large = __any_sync(0xffffffffu, large);
            }
            __syncwarp();
            copy(i + kStages, at);
            __syncwarp();
            if (++at == kStages) at = 0;
        }
        __syncthreads();  // the rings become the place of partial results
        float* parts = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int e = 0; e < 2; e++) {
            float* to = parts + warp * L::part + (t4 * 2 + e) * (L::dv + 2);
            if (g8 == 0) {
                to[0] = top[e];
                to[1] = l[e];
            }
#pragma unroll
            for (int n = 0; n < VC; n++) {
                to[2 + g8 * 2 * VC + 2 * n] = o[n][e];
                to[2 + g8 * 2 * VC + 2 * n + 1] = o[n][e + 2];
            }
        }
        __syncthreads();
        bf16* out = (bf16*)p.out + ((long long)sq.start * p.heads + h0) * vdim;
        const float factor = value_factor(p, g);
        auto own = [&](int k) { return parts + k * L::part; };
        if (count == n_blocks) {
            join_parts<L::dv>(p, own, kWarps, n_heads, vdim, factor, out, nullptr);
        } else {
            // Pieces of a cell stand one behind the other. Shares: a CTA's first block has the place 2 · CTA, what it ends with 2 · CTA + 1; a cell's parts are those of the CTAs from the one that has its
            // first block on.
            const long long cell0 = u - begin;
            const int a = p.pieces ? blockIdx.x / p.pieces * p.pieces : (int)(cell0 / each), n = p.pieces ? min(n_blocks, p.pieces) : (int)((cell0 + n_blocks - 1) / each) - a + 1;
            const int step_of = p.pieces ? 1 : 2, late_first = !p.pieces && cell0 != a * each;
            auto place = [&](int k) { return p.part + ((long long)step_of * (a + k) + (k == 0 ? late_first : 0)) * L::part; };
            join_parts<L::dv>(p, own, kWarps, n_heads, vdim, 0.f, nullptr, place((int)blockIdx.x - a));
            __syncthreads();
            unsigned* counter = p.counters + (long long)seq * n_groups + group;
            if (tid == 0) {  // what the others have written is written before this, and read behind it
                __threadfence();
                arrived = atomicAdd(counter, 1u);
                __threadfence();
            }
            __syncthreads();
            if (arrived == (unsigned)n - 1) {
                if (tid == 0) *counter = 0;
                join_parts<L::dv>(p, place, n, n_heads, vdim, factor, out, nullptr);
            }
        }
        u += count;
        left -= count;
        if (left <= 0) break;
        begin = 0;
        if (++group == n_groups) {
            group = 0;
            do sq = checked_seq(p, ++seq);
            while (blocks_of(p, sq) == 0);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();  // the rings, and the pages, are the next cell's
    }
    if (!ok && lane == 0) report(p.err, ERR_WAIT_TIMEOUT, p.node, (long long)blockIdx.x, (long long)warp);
}

template <int KS, int VC> PackedDecode choice(bool whole) {
    constexpr int resident = KS <= 2 && VC <= 8 ? 4 : 2;
    return {whole ? packed_decode<KS, VC, true, resident> : packed_decode<KS, VC, false, resident>, Smem<KS, VC>::total, Smem<KS, VC>::part, resident, kHeads, kTile * kWarps, kMostParts - 2};
}
template <int KS> PackedDecode choice(int64_t dim, int64_t vdim) {
    return vdim <= 64 ? choice<KS, 4>(dim == 64 * KS && vdim == 64) : vdim <= 128 ? choice<KS, 8>(dim == 64 * KS && vdim == 128) : choice<KS, 16>(dim == 64 * KS && vdim == 256);
}

}  // namespace

PackedDecode packed_decode_of(int64_t dim, int64_t vdim) { return dim <= 64 ? choice<1>(dim, vdim) : dim <= 128 ? choice<2>(dim, vdim) : choice<4>(dim, vdim); }

}  // namespace oxk
