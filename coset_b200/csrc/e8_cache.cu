// Writing and reading back an E8-coded key/value cache (layout: e8_cache.cuh).
//
// A row's step s is the smallest bf16 number >= max|x| / 7.  Its values become u = rint(4096 x / s), and each block of 8 the nearest point of
// E8 to u / 4096: the nearer one of the nearest points of D8 and of D8 + 1/2 (Conway and Sloane, Fast quantizing and decoding algorithms for
// lattice quantizers and codes, 1982).  With f = round(x), d = x - f, a = |d|: where the f have an odd sum, the coordinate with the largest a moves
// to its second nearest number, at a cost of 1 - 2 a; the nearest half-odd numbers leave 1/2 - a, the coordinate with the smallest a moves where
// their floors have an odd sum, at 2 a, and the two squared distances differ by (moves apart) 2 - sum a.  In units of 1/4096 all of it is
// exact in integers, so the codes are defined to the bit: the first coordinate moves where several are as far, up where it lies above its
// number and down otherwise, and the whole-number point stands where both are as far.
#include <cuda_bf16.h>

#include "e8_cache.cuh"

using namespace coset;
using namespace coset::cache;

namespace {

constexpr int kThreads = 256;
constexpr float kRound = 12582912.0f;  // 1.5 2^23: added to a small number it rounds it to a whole one, which stands in the low 22 bits

// A thread has two blocks of 8 values, half a row apart (with one, finding the row costs as much as the search), DIM / 16 neighbours a row; a CTA has rows of
// one head, one token after the other, so that codes of tokens that share a page are written and read as whole lines.  Rows of a CTA in one round:
__host__ __device__ constexpr int rows_per_round(int dim) { return kThreads / (dim / 16); }

template <int DT>
struct Block;  // 8 values as they are in memory
template <>
struct Block<COSET_DTYPE_F32> {
    uint4 a, b;
    __device__ __forceinline__ void load(const void* x, int64_t at) {
        const uint4* p = reinterpret_cast<const uint4*>(static_cast<const float*>(x) + at);
        a = __ldcs(p);
        b = __ldcs(p + 1);
    }
    __device__ __forceinline__ void values(float (&v)[8]) const {
        const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
    }
    // bits of the largest |value|: ordered like the numbers, infinities and NaN above all
    __device__ __forceinline__ uint32_t most() const {
        const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, w[i] & 0x7FFFFFFFu);
        return m;
    }
};
template <>
struct Block<COSET_DTYPE_BF16> {
    uint4 a;
    __device__ __forceinline__ void load(const void* x, int64_t at) { a = __ldcs(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(x) + at)); }
    __device__ __forceinline__ void values(float (&v)[8]) const {
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
    __device__ __forceinline__ uint32_t most() const {
        const auto larger = [](uint32_t x, uint32_t y) {
            uint32_t z;
            asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(z) : "r"(x), "r"(y));
            return z;
        };
        const uint32_t m = larger(larger(a.x & 0x7FFF7FFFu, a.y & 0x7FFF7FFFu), larger(a.z & 0x7FFF7FFFu, a.w & 0x7FFF7FFFu));
        return max(m << 16, m & 0xFFFF0000u);
    }
};

// The larger (smaller) one of three
__device__ __forceinline__ float largest(float x, float y, float z) {
    float m;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(x), "f"(y), "f"(z));
    return m;
}
__device__ __forceinline__ float smallest(float x, float y, float z) {
    float m;
    asm("min.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(x), "f"(y), "f"(z));
    return m;
}

// The code word of the nearest point to the scaled values x, and its bit c.  All numbers are whole or have three bits behind the point, in float32 and two at
// a time: u, f (halves up) and the floor h of u / 4096, d = u - 4096 f, and half words of four nibbles, sum 16^i (f + 8).  A number to be rounded is added to
// 1.5 2^23, whose last bit then is the parity.  a goes with the place of its coordinate into one number, a + (7 - i) / 8 or a + i / 8.
__device__ __forceinline__ uint32_t nearest_point(const float (&x)[8], float inv, bool* half) {
    const auto same = [](float v) { return two(v, v); };
    float2 d[4];
    Two f[4], h[4];
    uint32_t odd_f = 0, odd_h = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // values i and i + 4
        const Two u = add2(fma2(mul2(two(x[i], x[i + 4]), same(inv)), same(kGrid), same(kRound)), same(-kRound));  // the product with 4096 is exact
        const Two to_f = fma2(add2(u, same(0.5f)), same(1.0f / kGrid), same(kRound)), to_h = fma2(add2(u, same(0.5f - kGrid / 2)), same(1.0f / kGrid), same(kRound));
        f[i] = add2(to_f, same(-kRound));
        h[i] = add2(to_h, same(-kRound));
        d[i] = both(fma2(f[i], same(-kGrid), u));
        odd_f ^= __float_as_uint(both(to_f).x) ^ __float_as_uint(both(to_f).y);
        odd_h ^= __float_as_uint(both(to_h).x) ^ __float_as_uint(both(to_h).y);
    }
    float top[8], low[8], sum_a = kRound;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float a = fabsf(i < 4 ? d[i & 3].x : d[i & 3].y);
        top[i] = a + (7 - i) * 0.125f;
        low[i] = a + i * 0.125f;
        sum_a += a;
    }
    const float topmost = largest(largest(largest(top[0], top[1], top[2]), top[3], top[4]), top[5], fmaxf(top[6], top[7]));
    const float lowest = smallest(smallest(smallest(low[0], low[1], low[2]), low[3], low[4]), low[5], fminf(low[6], low[7]));
    const int most = __float_as_int(__fmaf_rn(topmost, 8.0f, kRound)) - __float_as_int(kRound), least = __float_as_int(__fmaf_rn(lowest, 8.0f, kRound)) - __float_as_int(kRound);
    odd_f &= 1;
    odd_h &= 1;
    const int far = odd_f ? 4096 - 2 * (most >> 3) : 0, half_far = 8192 - (__float_as_int(sum_a) - __float_as_int(kRound)) + (odd_h ? 2 * (least >> 3) : 0);
    const bool c = half_far < far;
    const auto word_of = [&](const Two (&n)[4]) {
        const float2 w = both(add2(fma2(fma2(fma2(n[3], same(16.0f), n[2]), same(16.0f), n[1]), same(16.0f), n[0]), same(8388608.0f + 0x8888)));
        return __byte_perm(__float_as_uint(w.x), __float_as_uint(w.y), 0x5410);
    };
    const uint32_t word_f = word_of(f), word_h = word_of(h);
    uint32_t word = c ? word_h : word_f;
    // the coordinate that moves: from the whole number towards the value, and from the half-odd one
    const int k = c ? least & 7 : 7 - (most & 7);
    const float d04 = k & 4 ? d[0].y : d[0].x, d15 = k & 4 ? d[1].y : d[1].x, d26 = k & 4 ? d[2].y : d[2].x, d37 = k & 4 ? d[3].y : d[3].x;
    const float even = k & 2 ? d26 : d04, odd = k & 2 ? d37 : d15, its = k & 1 ? odd : even;
    const bool up = c ? its < 0.0f && its > -2048.0f : its > 0.0f;
    if (c ? odd_h : odd_f) word += (up ? 1u : 0xFFFFFFFFu) << (4 * k);
    *half = c;
    return word;
}

// x / 7, correctly rounded: the quotient by the rounded reciprocal, corrected by what it leaves (Markstein, 1990); checked for every significand
__device__ __forceinline__ float seventh(float x) {
    const float r = 1.0f / 7.0f, q = __fmul_rn(x, r);
    return __fmaf_rn(__fmaf_rn(-q, kLevels, x), r, q);
}

struct Write {
    Pages pages;
    const void* x[2];
    int64_t token_stride[2], head_stride[2];
    const int64_t* slots;
    int64_t n_tokens;
};

template <int DIM, int DT, int ROUNDS>
__global__ void __launch_bounds__(kThreads)
k_cache_write(const __grid_constant__ Write w) {
    constexpr int kBlocks = DIM / 8, kLanes = DIM / 16, kRows = rows_per_round(DIM);
    grid_wait();
    grid_trigger();
    const int b = threadIdx.x % kLanes, lane = threadIdx.x & 31, which = blockIdx.y >= w.pages.n_heads, head = blockIdx.y - which * w.pages.n_heads;
    const int64_t token0 = (int64_t)blockIdx.x * (kRows * ROUNDS) + threadIdx.x / kLanes;
    const void* x = (which ? w.x[1] : w.x[0]);
    const int64_t stride = which ? w.token_stride[1] : w.token_stride[0], first = head * (which ? w.head_stride[1] : w.head_stride[0]) + 8 * b;
    int64_t slot[ROUNDS];
    Block<DT> raw[ROUNDS][2];
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) slot[i] = token0 + i * kRows < w.n_tokens ? __ldg(behind_wait(w.slots) + token0 + i * kRows) : -1;
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
        if (slot[i] < 0 || slot[i] >> w.pages.page_log2 >= w.pages.n_pages) slot[i] = -1;
        raw[i][0] = raw[i][1] = {};
        if (slot[i] >= 0) {
            const int64_t at = (token0 + i * kRows) * stride + first;
            raw[i][0].load(x, at);
            raw[i][1].load(x, at + DIM / 2);
        }
    }
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
        uint32_t most = max(raw[i][0].most(), raw[i][1].most());
#pragma unroll
        for (int m = 1; m < kLanes; m *= 2) most = max(most, __shfl_xor_sync(0xFFFFFFFFu, most, m));
        const bool plain = most >= kSmallest && most < 0x7F800000u;
        uint32_t step = 0x3F800000u;
        if (plain) step = (__float_as_uint(seventh(__uint_as_float(most))) + 0xFFFFu) & 0xFFFF0000u;
        const float inv = __frcp_rn(__uint_as_float(step));
        uint32_t word[2], votes[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float v[8];
            raw[i][j].values(v);
            if (!plain) {
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = 0.0f;
            }
            bool half;
            word[j] = nearest_point(v, inv, &half);
            votes[j] = __ballot_sync(0xFFFFFFFFu, half) >> (lane - b) & ((1u << kLanes) - 1u);
        }
        if (slot[i] < 0) continue;
        if (!plain) step = most < kSmallest ? 0u : kNoNumber;
        const int at = (int)slot[i] & ((1 << w.pages.page_log2) - 1);
        uint32_t* rec = w.pages.words + record<DIM>(w.pages, slot[i] >> w.pages.page_log2, head);
        uint32_t* codes = rec + ((which << w.pages.page_log2) + at) * kBlocks + b;
        codes[0] = word[0];
        codes[kLanes] = word[1];
        if (b < head_words(DIM)) {
            const uint32_t bits = DIM == 256 ? (b ? votes[1] : votes[0]) : votes[0] | votes[1] << kLanes % 32;
            rec[((2 * kBlocks + which * head_words(DIM)) << w.pages.page_log2) + at * head_words(DIM) + b] = step | bits;
        }
    }
}

// (x & mask) | bits in one instruction, of which the compiler makes two when it knows both constants
__device__ __forceinline__ uint32_t chosen(uint32_t x, uint32_t mask, uint32_t bits) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(x), "r"(mask), "r"(bits));
    return d;
}

struct Read {
    Pages pages;
    void* out[2];
    const int64_t* slots;
    int64_t n_tokens;
};

template <int DIM, int DT, int ROUNDS>
__global__ void __launch_bounds__(kThreads)
k_cache_read(const __grid_constant__ Read r) {
    constexpr int kBlocks = DIM / 8, kLanes = DIM / 16, kRows = rows_per_round(DIM);
    grid_wait();
    grid_trigger();
    const int b = threadIdx.x % kLanes, which = blockIdx.y >= r.pages.n_heads, head = blockIdx.y - which * r.pages.n_heads;
    const int64_t token0 = (int64_t)blockIdx.x * (kRows * ROUNDS) + threadIdx.x / kLanes;
    int64_t slot[ROUNDS];
    uint32_t word[ROUNDS][2], top[ROUNDS][2];
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) slot[i] = token0 + i * kRows < r.n_tokens ? __ldg(behind_wait(r.slots) + token0 + i * kRows) : -1;
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
        word[i][0] = word[i][1] = 0x88888888u;
        top[i][0] = top[i][1] = 0;
        if (slot[i] >= 0 && slot[i] >> r.pages.page_log2 < r.pages.n_pages) {
            const int at = (int)slot[i] & ((1 << r.pages.page_log2) - 1);
            const uint32_t* rec = r.pages.words + record<DIM>(r.pages, slot[i] >> r.pages.page_log2, head);
            const uint32_t* codes = rec + ((which << r.pages.page_log2) + at) * kBlocks + b;
            word[i][0] = codes[0];
            word[i][1] = codes[kLanes];
            const uint32_t* heads = rec + ((2 * kBlocks + which * head_words(DIM)) << r.pages.page_log2) + at * head_words(DIM);
            top[i][0] = heads[0];
            top[i][1] = DIM == 256 ? heads[1] : top[i][0];
        }
    }
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
        if (token0 + i * kRows >= r.n_tokens) continue;
        void* out = which ? r.out[1] : r.out[0];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int64_t to = ((token0 + i * kRows) * r.pages.n_heads + head) * DIM + 8 * b + j * (DIM / 2);
            const uint32_t c = top[i][j] >> (DIM == 256 ? b : b + j * kLanes) & 1, its = word[i][j];
            if (DT == COSET_DTYPE_F32) {
                // a nibble at bits 1..4 under the exponent of 2^22, and c at bit 0, is the number 2^22 + n + c / 2
                const float step = __uint_as_float(top[i][j] & 0xFFFF0000u);
                float v[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const uint32_t shifted = k == 0 ? its << 1 : its >> (4 * k - 1);
                    v[k] = __fmul_rn(__uint_as_float(chosen(shifted, 0x1Eu, 0x4A800000u | c)) - 4194312.0f, step);
                }
                float4* p = reinterpret_cast<float4*>(static_cast<float*>(out) + to);
                __stcs(p, make_float4(v[0], v[1], v[2], v[3]));
                __stcs(p + 1, make_float4(v[4], v[5], v[6], v[7]));
            } else {
                // the same in bf16, two at a time: 64 + n + c / 2, less 72; the product with the step is rounded once, as the float32 product would be
                const uint32_t exponent = 0x42804280u | c * 0x00010001u, step = __byte_perm(top[i][j], 0, 0x3232);
                uint32_t v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {  // values k and k + 4
                    const uint32_t shifted = k == 0 ? its << 1 : its >> (4 * k - 1);
                    asm("{\n\t.reg .b32 t;\n\tadd.rn.bf16x2 t, %1, %2;\n\tmul.rn.bf16x2 %0, t, %3;\n\t}" : "=r"(v[k]) : "r"(chosen(shifted, 0x001E001Eu, exponent)), "r"(0xC290C290u), "r"(step));
                }
                __stcs(reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(out) + to),
                       make_uint4(__byte_perm(v[0], v[1], 0x5410), __byte_perm(v[2], v[3], 0x5410), __byte_perm(v[0], v[1], 0x7632), __byte_perm(v[2], v[3], 0x7632)));
            }
        }
    }
}

bool known_dtype(int dtype) { return dtype == COSET_DTYPE_F32 || dtype == COSET_DTYPE_BF16; }

// The grid of a call, and whether its CTAs do two rounds: of bf16 tokens from four CTAs per SM on.  us with two rounds and with one, heads of 128: writing 8192
// bf16 tokens of 8 heads 17.6 and 18.1, 32768 61.5 and 63.8, reading 32768 27.1 (96 % of the copy rate) and 28.2; writing 8192 float32 ones 18.8 and 19.7,
// reading them 17.6 and 15.1.  Writes are bound by instructions, 430
// for a thread's two blocks: issue slots 80 %, ALU pipe 71 %, most stalls on a pipe that is taken; reads (135) by memory.
struct Shape {
    dim3 grid;
    bool twice;
};
int shape_of(int64_t n_tokens, int n_heads, int dim, int dtype, Shape* s) {
    const int64_t rows = rows_per_round(dim), once = (n_tokens + rows - 1) / rows;
    s->twice = dtype == COSET_DTYPE_BF16 && once * 2 * n_heads >= 8 * (int64_t)sm_count();
    const int64_t x = s->twice ? (once + 1) / 2 : once;
    if (x > INT32_MAX) return fail(COSET_E_UNSUPPORTED, "too many tokens for one call");
    s->grid = dim3((unsigned)x, 2 * (unsigned)n_heads);
    return 0;
}

template <int DIM, int DT>
int launch_write(const Write& w, const Shape& s, cudaStream_t st) {
    if constexpr (DT == COSET_DTYPE_BF16)
        if (s.twice) return launch_dependent("e8_cache_write", k_cache_write<DIM, DT, 2>, s.grid, kThreads, 0, st, w);
    return launch_dependent("e8_cache_write", k_cache_write<DIM, DT, 1>, s.grid, kThreads, 0, st, w);
}
template <int DIM, int DT>
int launch_read(const Read& r, const Shape& s, cudaStream_t st) {
    if constexpr (DT == COSET_DTYPE_BF16)
        if (s.twice) return launch_dependent("e8_cache_read", k_cache_read<DIM, DT, 2>, s.grid, kThreads, 0, st, r);
    return launch_dependent("e8_cache_read", k_cache_read<DIM, DT, 1>, s.grid, kThreads, 0, st, r);
}
template <int DIM>
int launch_write(const Write& w, int dtype, const Shape& s, cudaStream_t st) {
    return dtype == COSET_DTYPE_F32 ? launch_write<DIM, COSET_DTYPE_F32>(w, s, st) : launch_write<DIM, COSET_DTYPE_BF16>(w, s, st);
}
template <int DIM>
int launch_read(const Read& r, int dtype, const Shape& s, cudaStream_t st) {
    return dtype == COSET_DTYPE_F32 ? launch_read<DIM, COSET_DTYPE_F32>(r, s, st) : launch_read<DIM, COSET_DTYPE_BF16>(r, s, st);
}

}  // namespace

extern "C" {

int coset_e8_cache_row_words(int head_dim) { return known_dim(head_dim) ? row_words(head_dim) : 0; }

int coset_e8_cache_write(void* pages, int64_t n_pages, int n_heads, int page_size, int head_dim, const void* k, int64_t k_token_stride,
                         int64_t k_head_stride, const void* v, int64_t v_token_stride, int64_t v_head_stride, int dtype, const int64_t* slots,
                         int64_t n_tokens, void* stream) {
    Write w;
    if (int e = check_pages(pages, n_pages, n_heads, page_size, head_dim, &w.pages)) return e;
    if (!known_dtype(dtype)) return fail(COSET_E_BADARG, "unknown dtype %d", dtype);
    if (n_tokens < 0) return fail(COSET_E_BADARG, "n_tokens is negative");
    if (n_tokens == 0) return 0;
    if (!k || !v || !slots) return fail(COSET_E_BADARG, "k, v or slots is null");
    const int64_t whole = dtype == COSET_DTYPE_F32 ? 4 : 8;  // elements of 16 bytes
    if (!aligned(k, 16) || !aligned(v, 16) || !aligned(slots, 8) || (k_token_stride | k_head_stride | v_token_stride | v_head_stride) % whole)
        return fail(COSET_E_ALIGN, "rows of k and v must be 16-byte aligned, slots 8-byte aligned");
    w.x[0] = k; w.x[1] = v;
    w.token_stride[0] = k_token_stride; w.token_stride[1] = v_token_stride;
    w.head_stride[0] = k_head_stride; w.head_stride[1] = v_head_stride;
    w.slots = slots;
    w.n_tokens = n_tokens;
    Shape shape;
    if (int e = shape_of(n_tokens, n_heads, head_dim, dtype, &shape)) return e;
    cudaStream_t st = (cudaStream_t)stream;
    return head_dim == 64 ? launch_write<64>(w, dtype, shape, st) : head_dim == 128 ? launch_write<128>(w, dtype, shape, st) : launch_write<256>(w, dtype, shape, st);
}

int coset_e8_cache_read(const void* pages, int64_t n_pages, int n_heads, int page_size, int head_dim, const int64_t* slots, int64_t n_tokens,
                        void* k, void* v, int dtype, void* stream) {
    Read r;
    if (int e = check_pages(pages, n_pages, n_heads, page_size, head_dim, &r.pages)) return e;
    if (!known_dtype(dtype)) return fail(COSET_E_BADARG, "unknown dtype %d", dtype);
    if (n_tokens < 0) return fail(COSET_E_BADARG, "n_tokens is negative");
    if (n_tokens == 0) return 0;
    if (!k || !v || !slots) return fail(COSET_E_BADARG, "k, v or slots is null");
    if (!aligned(k, 16) || !aligned(v, 16) || !aligned(slots, 8)) return fail(COSET_E_ALIGN, "k and v must be 16-byte, slots 8-byte aligned");
    r.out[0] = k; r.out[1] = v;
    r.slots = slots;
    r.n_tokens = n_tokens;
    Shape shape;
    if (int e = shape_of(n_tokens, n_heads, head_dim, dtype, &shape)) return e;
    cudaStream_t st = (cudaStream_t)stream;
    return head_dim == 64 ? launch_read<64>(r, dtype, shape, st) : head_dim == 128 ? launch_read<128>(r, dtype, shape, st) : launch_read<256>(r, dtype, shape, st);
}

}  // extern "C"
