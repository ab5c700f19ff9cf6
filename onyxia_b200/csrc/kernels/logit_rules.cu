// What a request's rules make of the logits of its next token, per row:
//
//   t in the row's history (prompt and answer):  l ← l > 0 ? l / repetition : l · repetition
//   t said n > 0 times in the answer:            l ← l − n · frequency − presence
//   biases of t:                                 l ← l + Σ, in the order they are listed
//   t not in the row's mask:                     l ← −∞
//
// in f32, the result too (a half-precision logit times a penalty would be rounded again and could leave its range).
//
// A CTA takes a run of one row's vocabulary: it counts the row's history in shared memory (whole numbers: no order shows), adds up the biases of its tokens there, streams the run and, last, writes
// the few biased tokens again. The history and the biased tokens are read once per run. Bound by the logits' bytes: read once, written once as f32.
// 64 rows of 262144 with 2048 tokens of history, masks and 64 biases each (134 MB): 31.7 us a pass among others (4.3 TB/s), 37.9 cold under the profiler; 41 there while listed tokens searched the list, and ten
// more where the history waits for its length and the mask is asked for token by token. Runs of 8192 (half as many readings of the history, half as many CTAs per SM) took a quarter more.
#include "common.cuh"
#include "kernels.hpp"

namespace oxk {

namespace {

constexpr int kRuleThreads = 256;

struct RulesP {
    const void* x;           // [rows, cols] logits
    float* y;                // [rows, cols]
    const int* history;      // [rows, width], or null
    const int* lengths;      // [rows, 2]: tokens of the prompt, tokens of both
    const float* penalties;  // [rows, 3]: repetition, frequency, presence
    const int* bias_ids;     // [rows, n_bias], or null; negative: none
    const float* bias;       // [rows, n_bias]
    const unsigned* masks;   // [n_masks, words], or null
    const int* mask_of;      // [rows], or null: row r has mask r; negative: none
    ErrWord* err;
    long long rows, cols;
    int width, n_bias, n_masks, words, node;
};

// PER groups of four tokens per thread; VEC: rows begin on 16 bytes.
template <int DT, int PER, bool VEC> __global__ void __launch_bounds__(kRuleThreads) constrain_rows(const RulesP p) {
    constexpr int kRun = kRuleThreads * PER * 4;
    __shared__ __align__(16) unsigned times[kRun];  // how often a token was said, the top bit: it is in the prompt
    extern __shared__ float more[];                 // [kRun], where there are biases: what those of a biased token add up to
    const long long row = blockIdx.y, c0 = (long long)blockIdx.x * kRun, base = row * p.cols;
    const int tid = threadIdx.x, n = (int)min((long long)kRun, p.cols - c0);
    // everything that does not hang on something else is asked for at once
    constexpr int kEarly = 8;
    const int* h = p.history + row * p.width;
    int said[kEarly], prompt = 0, total = 0;
    float repetition = 1.f, frequency = 0.f, presence = 0.f;
    if (p.history) {
        prompt = p.lengths[2 * row], total = p.lengths[2 * row + 1];
        repetition = p.penalties[3 * row], frequency = p.penalties[3 * row + 1], presence = p.penalties[3 * row + 2];
#pragma unroll
        for (int k = 0; k < kEarly; k++) said[k] = k * kRuleThreads + tid < p.width ? h[k * kRuleThreads + tid] : 0;
    }
    const int which = p.masks && p.mask_of ? p.mask_of[row] : (int)row;
    auto token = [&](int i, int e) { return VEC ? (i * kRuleThreads + tid) * 4 + e : (i * 4 + e) * kRuleThreads + tid; };
    float v[PER][4];
#pragma unroll
    for (int i = 0; i < PER; i++) {
        if constexpr (VEC) {
            const int c = token(i, 0);
            if (c < n) {
                if constexpr (DT == DT_F32) {
                    const float4 f = *reinterpret_cast<const float4*>((const float*)p.x + base + c0 + c);
                    v[i][0] = f.x, v[i][1] = f.y, v[i][2] = f.z, v[i][3] = f.w;
                } else {
                    const uint2 u = *reinterpret_cast<const uint2*>((const __half*)p.x + base + c0 + c);
                    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
                    v[i][0] = a.x, v[i][1] = a.y, v[i][2] = b.x, v[i][3] = b.y;
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (token(i, e) < n) v[i][e] = ld<DT>(p.x, base + c0 + token(i, e));
        }
    }
    const unsigned* mask = nullptr;
    if (p.masks) {
        if (which < p.n_masks) mask = which >= 0 ? p.masks + (long long)which * p.words : nullptr;
        else if (blockIdx.x == 0 && tid == 0) report(p.err, ERR_RULES_MASK, p.node, which, p.n_masks);
    }
    unsigned may[PER];  // four tokens' bits of the mask
#pragma unroll
    for (int i = 0; i < PER; i++)
        if (VEC) may[i] = mask && token(i, 0) < n ? mask[(c0 + token(i, 0)) >> 5] >> (token(i, 0) & 31) : ~0u;
    if (p.history) {
        for (int c = tid; c < kRun / 4; c += kRuleThreads) reinterpret_cast<uint4*>(times)[c] = make_uint4(0u, 0u, 0u, 0u);
        if (prompt < 0 || prompt > total || total > p.width) {
            if (blockIdx.x == 0 && tid == 0) report(p.err, ERR_RULES_LENGTH, p.node, row, p.width);
            total = max(0, min(total, p.width));
            prompt = max(0, min(prompt, total));
        }
        __syncthreads();
        auto count = [&](int i, int t) {
            if (i >= total) return;
            const long long c = t - c0;
            if (c >= 0 && c < n) {
                if (i < prompt) atomicOr(&times[c], 0x80000000u);
                else atomicAdd(&times[c], 1u);
            } else if (blockIdx.x == 0 && (t < 0 || t >= p.cols)) {
                report(p.err, ERR_RULES_TOKEN, p.node, t, p.cols);
            }
        };
#pragma unroll
        for (int k = 0; k < kEarly; k++) count(k * kRuleThreads + tid, said[k]);
        for (int i = kEarly * kRuleThreads + tid; i < total; i += kRuleThreads) count(i, h[i]);
        __syncthreads();
    }
    const int* ids = p.bias_ids + row * p.n_bias;
    if (p.bias_ids) {
        // The sums of the biased tokens' biases, each in the order of the list: by one warp, 32 places at a time, those of one token one after the other by its first lane. 64 rows of 262144 with 300, 1000,
        // 4096 biases, one call after the other: 64, 111, 333 us; where each listed token searches the list for its likes 172, 977, 11 907.
        for (int j = tid; j < p.n_bias; j += kRuleThreads) {
            const long long c = ids[j] - c0;
            if (c >= 0 && c < n && ids[j] >= 0) more[c] = 0.f;
        }
        __syncthreads();
        const float* bias = p.bias + row * p.n_bias;
        if (tid < 32)
            for (int j0 = 0; j0 < p.n_bias; j0 += 32) {
                const int t = j0 + tid < p.n_bias ? ids[j0 + tid] : -1;
                if (t >= p.cols && blockIdx.x == 0) report(p.err, ERR_RULES_TOKEN, p.node, t, p.cols);
                const long long c = t - c0;
                const bool mine = t >= 0 && c >= 0 && c < n;
                if (!__any_sync(0xffffffffu, mine)) continue;
                const float b = mine ? bias[j0 + tid] : 0.f;
                const unsigned same = __match_any_sync(0xffffffffu, mine ? t : -1);
                const bool first = mine && __ffs(same) == tid + 1;
                float sum = first ? more[c] : 0.f;
                for (int k = 0; k < 32; k++) {
                    const float theirs = __shfl_sync(0xffffffffu, b, k);
                    if (same >> k & 1u) sum += theirs;
                }
                if (first) more[c] = sum;
                __syncwarp();
            }
    }
    auto penalised = [&](float l, unsigned said) {
        if (said == 0u) return l;
        l = l > 0.f ? l / repetition : l * repetition;
        const unsigned k = said & 0x7FFFFFFFu;
        return k ? l - (float)k * frequency - presence : l;
    };
    auto allowed = [&](long long t) { return !mask || (mask[t >> 5] >> (t & 31) & 1u); };
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const uint4 four = VEC && p.history ? *reinterpret_cast<const uint4*>(times + token(i, 0)) : make_uint4(0u, 0u, 0u, 0u);
        const unsigned found[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int c = token(i, e);
            if (c >= n) continue;
            if (p.history) v[i][e] = penalised(v[i][e], VEC ? found[e] : times[c]);
            if (VEC ? !(may[i] >> e & 1u) : !allowed(c0 + c)) v[i][e] = -INFINITY;
            if (!VEC) p.y[base + c0 + c] = v[i][e];
        }
        if (VEC && token(i, 0) < n) *reinterpret_cast<float4*>(p.y + base + c0 + token(i, 0)) = make_float4(v[i][0], v[i][1], v[i][2], v[i][3]);
    }
    if (!p.bias_ids) return;
    __syncthreads();  // behind the plain results, and the sums
    for (int j = tid; j < p.n_bias; j += kRuleThreads) {
        const int t = ids[j];
        const long long c = t - c0;
        if (t < 0 || c < 0 || c >= n || !allowed(t)) continue;
        float l = ld<DT>(p.x, base + t);
        if (p.history) l = penalised(l, times[c]);
        p.y[base + t] = l + more[c];  // (a token that is listed again gets the same)
    }
}

template <int DT> void emit_rules_of(Emitter& em, const RulesP& p, bool vec, std::initializer_list<std::pair<const void*, Buf>> ptrs) {
    auto go = [&](void (*k)(const RulesP), int per) {
        const long long run = (long long)kRuleThreads * per * 4;
        em.launch(k, dim3((unsigned)((p.cols + run - 1) / run), (unsigned)p.rows), dim3(kRuleThreads), p.n_bias ? (unsigned)(run * 4) : 0u, p, ptrs, "constrain_rows");
    };
    vec ? go(constrain_rows<DT, 4, true>, 4) : go(constrain_rows<DT, 4, false>, 4);
}

}  // namespace

void emit_logit_rules(Emitter& em, const TRef& logits, const TRef& out, const LogitRules& r) {
    RulesP p{};
    p.cols = logits.shape.back();
    p.rows = p.cols ? logits.numel() / p.cols : 0;
    if (p.rows == 0) return;
    p.width = (int)r.width;
    p.n_bias = (int)r.n_bias;
    p.n_masks = (int)r.n_masks;
    p.words = (int)((p.cols + 31) / 32);
    p.node = em.node;
    const std::initializer_list<std::pair<const void*, Buf>> ptrs = {{&p.x, logits.buf}, {&p.y, out.buf}, {&p.history, r.history}, {&p.lengths, r.lengths}, {&p.penalties, r.penalties},
                                                                   {&p.bias_ids, r.bias_ids}, {&p.bias, r.bias}, {&p.masks, r.masks}, {&p.mask_of, r.mask_of}, {&p.err, Buf{kSlotErr, 0}}};
    const bool vec = p.cols % 4 == 0 && r.aligned;
    logits.dtype == DT_F32 ? emit_rules_of<DT_F32>(em, p, vec, ptrs) : emit_rules_of<DT_F16>(em, p, vec, ptrs);
}

}  // namespace oxk
