// What the kernels of differential attention share: their parameters.
#pragma once
#include "paged_util.cuh"

namespace oxk {

struct DiffP {
    const void* proj;            // [rows, ld]
    const float* turns;          // [2, half]
    void *keys, *values;         // [pages, kv_heads, page, 2 · dim | vdim]
    void* q;                     // [rows, heads · 2 · dim]: prepared queries
    void* out;                   // [rows, heads · vdim]
    const int* seqs;             // [R, 4]
    const int* table;            // [R, width]
    const float* lambda;         // [heads]
    const float* gain;           // [vdim], or null: results as they are
    ErrWord* err;
    long long rows, ld, q_off, k_off, v_off;
    int n_seqs, width, n_pages, shift /* log2 of the page */, heads, kv_heads, dim, vdim, half, window, node;
    float scale, cap, eps, head_eps;
    int norm, sink;
    int singles;                 // prepare: also sequences with one new token
};

__device__ __forceinline__ int first_key(const DiffP& p, int pos) { return p.window > 0 ? max(0, pos - p.window + 1) : 0; }
// 1 / root mean square of a map's query or key, by one warp
template <typename T> __device__ __forceinline__ float map_factor(const DiffP& p, const T* x) {
    if (!p.norm) return 1.f;
    float ss = 0.f;
    for (int i = threadIdx.x & 31; i < p.dim; i += 32) {
        const float v = to_f(x[i]);
        ss = fmaf(v, v, ss);
    }
    return 1.f / sqrtf(warp_sum(ss) / (float)p.dim + p.eps);
}

}  // namespace oxk
