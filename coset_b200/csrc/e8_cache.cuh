// Layout of the pages of an E8-coded key/value cache, shared by the kernels that write, read and attend to it.
//
// A row is the D values of one token and one head.  Its blocks of 8 are points of E8 in units of the row's step, f + c / 2 with
// f in [-8, 7] per value and c one bit per block (E8 = D8 u (D8 + 1/2)); the code is the nested pair E8 / 16 Z^8.  A word holds a block:
// f + 8 of value i in bits 4i..4i+3.  A head word holds the step (bf16, high half) and the c of 16 blocks (low half, block b at bit b % 16);
// a row of 256 has two, with the same step.
//
// A record is one page of one head: page_size rows of key codes, of value codes, of key heads, of value heads.  The planes are kept apart so
// that a warp reads each of them as whole aligned lines, and the record together so that a page of a head is one piece of memory.
// (No counterpart in the reference, whose cache is the dense one of the model.)
#pragma once
#include "common.cuh"

namespace coset {
namespace cache {

constexpr float kLevels = 7.0f;       // max|x| / step <= 7 leaves room for the moved coordinate of a block: [-8, 7.5]
constexpr float kGrid = 4096.0f;      // values are rounded to 1/4096 step before the search, which is then exact in small integers
constexpr uint32_t kSmallest = 0x0D800000u;  // 2^-100: a row below it is stored as zeros
constexpr uint32_t kNoNumber = 0x7FC00000u;  // step of a row that holds an infinity or a NaN: it reads back as NaN

__host__ __device__ constexpr int code_words(int dim) { return dim / 8; }
__host__ __device__ constexpr int head_words(int dim) { return (dim + 127) / 128; }
__host__ __device__ constexpr int row_words(int dim) { return 2 * (code_words(dim) + head_words(dim)); }

struct Pages {
    uint32_t* words;
    int64_t n_pages;
    int n_heads, page_log2;
};

// First word of the record of (page, head).
template <int DIM>
__device__ __forceinline__ int64_t record(const Pages& p, int64_t page, int head) { return ((page * p.n_heads + head) << p.page_log2) * row_words(DIM); }

// Two float32 numbers at a time
using Two = unsigned long long;
__device__ __forceinline__ Two two(float x, float y) {
    Two r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 both(Two x) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
    return r;
}
__device__ __forceinline__ Two mul2(Two x, Two y) {
    Two r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}
__device__ __forceinline__ Two add2(Two x, Two y) {
    Two r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}
__device__ __forceinline__ Two fma2(Two x, Two y, Two z) {
    Two r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    return r;
}

inline bool known_dim(int dim) { return dim == 64 || dim == 128 || dim == 256; }

// Checks of what every call is given; 0 or a negative status.
inline int check_pages(const void* pages, int64_t n_pages, int n_heads, int page_size, int head_dim, Pages* out) {
    if (!known_dim(head_dim)) return fail(COSET_E_UNSUPPORTED, "head_dim must be 64, 128 or 256, got %d", head_dim);
    if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1))) return fail(COSET_E_UNSUPPORTED, "page_size must be a power of two from 16 to 1024, got %d", page_size);
    if (n_heads < 1 || n_heads > 32767) return fail(COSET_E_BADARG, "n_heads must lie in [1, 32767], got %d", n_heads);
    if (n_pages < 0 || n_pages > INT32_MAX) return fail(COSET_E_BADARG, "n_pages must lie in [0, 2^31), got %lld", (long long)n_pages);
    if (n_pages > 0 && !pages) return fail(COSET_E_BADARG, "pages is null");
    if (!aligned(pages, 16)) return fail(COSET_E_ALIGN, "pages must be 16-byte aligned");
    out->words = (uint32_t*)const_cast<void*>(pages);
    out->n_pages = n_pages;
    out->n_heads = n_heads;
    out->page_log2 = __builtin_ctz((unsigned)page_size);
    return 0;
}

}  // namespace cache
}  // namespace coset
