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

template <int DT>
__device__ __forceinline__ void load_block(const void* x, int64_t at, float (&v)[8]);
template <>
__device__ __forceinline__ void load_block<COSET_DTYPE_F32>(const void* x, int64_t at, float (&v)[8]) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(x) + at);
    const float4 a = __ldcs(p), b = __ldcs(p + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <>
__device__ __forceinline__ void load_block<COSET_DTYPE_BF16>(const void* x, int64_t at, float (&v)[8]) {
    const uint4 a = __ldcs(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(x) + at));
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}

// The code word of the nearest point to u / 4096, and its bit c.
__device__ __forceinline__ uint32_t nearest_point(const int (&u)[8], bool* half) {
    int f[8], d[8], sum_f = 0, sum_h = 0, sum_a = 0, top = 0, low = INT32_MAX;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        f[i] = (u[i] + 2048) >> 12;
        d[i] = u[i] - (f[i] << 12);
        const int a = abs(d[i]);
        sum_f += f[i];
        sum_h += f[i] - (d[i] < 0);
        sum_a += a;
        top = max(top, a * 8 + 7 - i);
        low = min(low, a * 8 + i);
    }
    const bool odd_f = sum_f & 1, odd_h = sum_h & 1;
    const int far = odd_f ? 4096 - 2 * (top >> 3) : 0, half_far = 8192 - sum_a + (odd_h ? 2 * (low >> 3) : 0);
    const bool c = half_far < far;
    const int moved = c ? (odd_h ? low & 7 : 8) : (odd_f ? 7 - (top & 7) : 8);
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int whole = f[i] + (i == moved ? (d[i] > 0 ? 1 : -1) : 0);
        const int halved = f[i] - (d[i] < 0) + (i == moved ? (d[i] < 0 && d[i] > -2048 ? 1 : -1) : 0);
        word |= (uint32_t)((c ? halved : whole) + 8) << (4 * i);
    }
    *half = c;
    return word;
}

struct Write {
    Pages pages;
    const void* x[2];
    int64_t token_stride[2], head_stride[2];
    const int64_t* slots;
    int64_t n_rows;  // tokens x 2 x heads
};

// A thread has a block, DIM / 8 neighbours a row.
template <int DIM, int DT>
__global__ void __launch_bounds__(kThreads)
k_cache_write(const __grid_constant__ Write w) {
    constexpr int kBlocks = DIM / 8;
    grid_wait();
    grid_trigger();
    const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    const int64_t row = id / kBlocks;
    const int b = (int)(id % kBlocks), lane = threadIdx.x & 31;
    const int pair = (int)(row % (2 * w.pages.n_heads)), which = pair >= w.pages.n_heads, head = pair - which * w.pages.n_heads;
    const int64_t token = row / (2 * w.pages.n_heads);
    const int64_t slot = row < w.n_rows ? __ldg(behind_wait(w.slots) + token) : -1;
    const bool real = slot >= 0 && slot >> w.pages.page_log2 < w.pages.n_pages;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.0f;
    if (real) load_block<DT>(w.x[which], token * w.token_stride[which] + head * w.head_stride[which] + 8 * b, x);
    uint32_t most = 0;  // of the bits of |x|: ordered like the numbers, infinities and NaN above all
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(x[i]) & 0x7FFFFFFFu);
#pragma unroll
    for (int m = 1; m < kBlocks; m *= 2) most = max(most, __shfl_xor_sync(0xFFFFFFFFu, most, m));
    const bool plain = most >= kSmallest && most < 0x7F800000u;
    uint32_t step = 0x3F800000u;
    if (plain) step = (__float_as_uint(__fdiv_rn(__uint_as_float(most), kLevels)) + 0xFFFFu) & 0xFFFF0000u;
    const float inv = __fdiv_rn(1.0f, __uint_as_float(step));
    int u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = plain ? __float2int_rn(__fmul_rn(__fmul_rn(x[i], inv), kGrid)) : 0;
    bool half;
    const uint32_t word = nearest_point(u, &half);
    const uint32_t votes = __ballot_sync(0xFFFFFFFFu, half);
    if (!real) return;
    if (!plain) step = most < kSmallest ? 0u : kNoNumber;
    const int at = (int)(slot & ((1 << w.pages.page_log2) - 1));
    uint32_t* rec = w.pages.words + record<DIM>(w.pages, slot >> w.pages.page_log2, head);
    rec[(((which << w.pages.page_log2) + at)) * kBlocks + b] = word;
    if (b < head_words(DIM)) {
        const uint32_t mine = votes >> (lane - b + 16 * b);
        rec[((2 * kBlocks + which * head_words(DIM)) << w.pages.page_log2) + at * head_words(DIM) + b] = step | (mine & (kBlocks < 16 ? 0xFFu : 0xFFFFu));
    }
}

struct Read {
    Pages pages;
    void* out[2];
    const int64_t* slots;
    int64_t n_rows;
};

template <int DIM, int DT>
__global__ void __launch_bounds__(kThreads)
k_cache_read(const __grid_constant__ Read r) {
    constexpr int kBlocks = DIM / 8;
    grid_wait();
    grid_trigger();
    const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    const int64_t row = id / kBlocks;
    if (row >= r.n_rows) return;
    const int b = (int)(id % kBlocks);
    const int pair = (int)(row % (2 * r.pages.n_heads)), which = pair >= r.pages.n_heads, head = pair - which * r.pages.n_heads;
    const int64_t token = row / (2 * r.pages.n_heads);
    const int64_t slot = __ldg(behind_wait(r.slots) + token);
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    if (slot >= 0 && slot >> r.pages.page_log2 < r.pages.n_pages) {
        const int at = (int)(slot & ((1 << r.pages.page_log2) - 1));
        const uint32_t* rec = r.pages.words + record<DIM>(r.pages, slot >> r.pages.page_log2, head);
        const uint32_t word = rec[((which << r.pages.page_log2) + at) * kBlocks + b];
        const uint32_t h = rec[((2 * kBlocks + which * head_words(DIM)) << r.pages.page_log2) + at * head_words(DIM) + b / 16];
        const float step = __uint_as_float(h & 0xFFFF0000u), c = (h >> (b % 16)) & 1 ? -7.5f : -8.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __fmul_rn((float)((word >> (4 * i)) & 15u) + c, step);
    }
    const int64_t to = (token * r.pages.n_heads + head) * DIM + 8 * b;
    if (DT == COSET_DTYPE_F32) {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(r.out[which]) + to);
        __stcs(p, make_float4(v[0], v[1], v[2], v[3]));
        __stcs(p + 1, make_float4(v[4], v[5], v[6], v[7]));
    } else {
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h2 = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            o[i] = *reinterpret_cast<const uint32_t*>(&h2);
        }
        __stcs(reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(r.out[which]) + to), make_uint4(o[0], o[1], o[2], o[3]));
    }
}

// Blocks of a launch over n_rows rows of `dim` values; -1: more than a grid holds.
int64_t grid_of(int64_t n_rows, int dim) {
    const int64_t per = kThreads / (dim / 8), need = (n_rows + per - 1) / per;
    return need > INT32_MAX ? -1 : need;
}
bool known_dtype(int dtype) { return dtype == COSET_DTYPE_F32 || dtype == COSET_DTYPE_BF16; }

template <int DIM>
int launch_write(const Write& w, int dtype, unsigned grid, cudaStream_t st) {
    return dtype == COSET_DTYPE_F32 ? launch_dependent("e8_cache_write", k_cache_write<DIM, COSET_DTYPE_F32>, grid, kThreads, 0, st, w)
                                    : launch_dependent("e8_cache_write", k_cache_write<DIM, COSET_DTYPE_BF16>, grid, kThreads, 0, st, w);
}
template <int DIM>
int launch_read(const Read& r, int dtype, unsigned grid, cudaStream_t st) {
    return dtype == COSET_DTYPE_F32 ? launch_dependent("e8_cache_read", k_cache_read<DIM, COSET_DTYPE_F32>, grid, kThreads, 0, st, r)
                                    : launch_dependent("e8_cache_read", k_cache_read<DIM, COSET_DTYPE_BF16>, grid, kThreads, 0, st, r);
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
    if (n_tokens > INT64_MAX / (2 * (int64_t)n_heads)) return fail(COSET_E_UNSUPPORTED, "too many rows for one call");
    w.n_rows = n_tokens * 2 * n_heads;
    const int64_t grid = grid_of(w.n_rows, head_dim);
    if (grid < 0) return fail(COSET_E_UNSUPPORTED, "too many rows for one call");
    cudaStream_t st = (cudaStream_t)stream;
    return head_dim == 64 ? launch_write<64>(w, dtype, (unsigned)grid, st) : head_dim == 128 ? launch_write<128>(w, dtype, (unsigned)grid, st)
                                                                            : launch_write<256>(w, dtype, (unsigned)grid, st);
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
    if (n_tokens > INT64_MAX / (2 * (int64_t)n_heads)) return fail(COSET_E_UNSUPPORTED, "too many rows for one call");
    r.n_rows = n_tokens * 2 * n_heads;
    const int64_t grid = grid_of(r.n_rows, head_dim);
    if (grid < 0) return fail(COSET_E_UNSUPPORTED, "too many rows for one call");
    cudaStream_t st = (cudaStream_t)stream;
    return head_dim == 64 ? launch_read<64>(r, dtype, (unsigned)grid, st) : head_dim == 128 ? launch_read<128>(r, dtype, (unsigned)grid, st)
                                                                           : launch_read<256>(r, dtype, (unsigned)grid, st);
}

}  // extern "C"
