// What the kernels of differential prompts share: tiles, tensor memory, copies.
#pragma once
#include "differential.cuh"

namespace oxk {

struct PreP {
    alignas(64) unsigned char maps[2][128];  // keys, values: [rows of the pool, 2 · dim | vdim]
    DiffP kv;
    int kp, vp, box, inv;  // panels of 64 dimensions, keys per copy, 2^16 / heads of a key head, rounded up
};

namespace {

constexpr int kRows = 128, kPart = 64;
constexpr unsigned kPanelQ = kRows * 128, kPanelV = kPart * 128;  // bytes: rows × 64 dimensions
constexpr float kLazy = 8.f;  // how far (base 2) a row's scores may rise above the maximum that its weights are taken against

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
    return (unsigned long long)((smem_byte_addr & 0x3FFFFu) >> 4) | ((unsigned long long)(kPanelV >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
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

}  // namespace

// Records the kernel of both maps in one CTA; the caller adds what is relocated. Grid: (tiles of 128 rows, key heads).
void emit_differential_pair(Emitter&, const PreP&, dim3 grid);

}  // namespace oxk
