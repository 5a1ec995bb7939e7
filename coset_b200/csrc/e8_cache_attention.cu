// Attention over an E8-coded key/value cache (layout: e8_cache.cuh): out = softmax(scale q K^T + mask) V for the last tokens of every
// sequence, which are one generated token, a chain or a tree of drafted ones.
#include <cuda_bf16.h>

#include "e8_cache.cuh"

using namespace coset;
using namespace coset::cache;

namespace {

struct Attend {
    Pages pages;
    const void* q;
    int64_t q_token_stride, q_head_stride;
    int n_queries, group;
    const int32_t* table;
    int64_t table_stride;
    int max_pages;
    const int32_t* lens;
    const int32_t* starts;
    int n_seqs;
    const int64_t* tree;
    float scale;
    void* out;
    float* lse;
};

constexpr int kWarps = 4;

// One warp for a query and a head; lane l holds values l DIM / 32 and following.
template <int DIM, int DT>
__global__ void __launch_bounds__(32 * kWarps)
k_cache_attend(const __grid_constant__ Attend a) {
    constexpr int kMine = DIM / 32;
    grid_wait();
    grid_trigger();
    const int q_heads = a.group * a.pages.n_heads, lane = threadIdx.x & 31;
    const int64_t id = (int64_t)blockIdx.x * kWarps + threadIdx.x / 32;
    const int query = (int)(id / q_heads), q_head = (int)(id % q_heads), head = q_head / a.group;
    if (query >= a.n_queries) return;
    int seq, first, count;
    if (a.starts) {
        int lo = 0, hi = a.n_seqs;  // the last sequence that starts at or before the query
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (a.starts[mid] <= query) lo = mid;
            else hi = mid;
        }
        seq = lo;
        first = a.starts[seq];
        count = a.starts[seq + 1] - first;
        if (query < first || query >= first + count) return;
    } else {
        count = a.n_queries / a.n_seqs;
        seq = query / count;
        first = seq * count;
    }
    const int page = 1 << a.pages.page_log2;
    const int len = min(a.lens[seq], (int)min((int64_t)a.max_pages << a.pages.page_log2, (int64_t)INT32_MAX));
    const int drafted = len - count, mine = query - first;
    const uint64_t bits = a.tree ? (uint64_t)a.tree[query] : 0;
    const int at = lane * kMine;
    float q[kMine], o[kMine], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        const int64_t e = query * a.q_token_stride + q_head * a.q_head_stride + at + i;
        q[i] = DT == COSET_DTYPE_F32 ? static_cast<const float*>(a.q)[e] : __bfloat162float(static_cast<const __nv_bfloat16*>(a.q)[e]);
        o[i] = 0.0f;
    }
    for (int key = 0; key < len; ++key) {
        const int j = key - drafted;
        if (j >= 0 && !(a.tree ? j < 64 && (bits >> j & 1) : j <= mine)) continue;
        const int p = a.table[seq * a.table_stride + (key >> a.pages.page_log2)];
        if (p < 0 || p >= a.pages.n_pages) continue;
        const uint32_t* rec = a.pages.words + record<DIM>(a.pages, p, head);
        const int row = key & (page - 1), w = row * code_words(DIM) + at / 8, h = row * head_words(DIM) + at / 128, block = at / 8 % 16;
        const uint32_t* heads = rec + 2 * code_words(DIM) * page;
        const uint32_t kw = rec[w], vw = rec[code_words(DIM) * page + w], kh = heads[h], vh = heads[head_words(DIM) * page + h];
        const float kc = (kh >> block & 1) ? -7.5f : -8.0f, vc = (vh >> block & 1) ? -7.5f : -8.0f;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < kMine; ++i) s += q[i] * ((float)(kw >> (4 * ((at + i) % 8)) & 15u) + kc);
#pragma unroll
        for (int d = 1; d < 32; d *= 2) s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
        s *= a.scale * __uint_as_float(kh & 0xFFFF0000u);
        // the running maximum is that of the weight times the size of the value's step (a power of two, zeros counted as 2^-103), so that neither a
        // small weight of a large value nor a large weight of a small one is lost
        const float step = __uint_as_float(vh & 0xFFFF0000u), size = (float)max((int)(vh >> 23 & 255u) - 127, -103) * 0.69314718f;
        const float top = fmaxf(m, s + size), keep = m == -INFINITY ? 0.0f : expf(m - top), e = expf(s - top), ev = e * step;
        l = l * keep + e;
#pragma unroll
        for (int i = 0; i < kMine; ++i) o[i] = o[i] * keep + ev * ((float)(vw >> (4 * ((at + i) % 8)) & 15u) + vc);
        m = top;
    }
    const float r = l == 0.0f ? 0.0f : 1.0f / l;
    const int64_t to = ((int64_t)query * q_heads + q_head) * DIM + at;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        if (DT == COSET_DTYPE_F32) static_cast<float*>(a.out)[to + i] = o[i] * r;
        else static_cast<__nv_bfloat16*>(a.out)[to + i] = __float2bfloat16_rn(o[i] * r);
    }
    if (a.lse && lane == 0) a.lse[(int64_t)query * q_heads + q_head] = m + logf(l);
}

template <int DIM>
int launch(const Attend& a, int dtype, unsigned grid, cudaStream_t st) {
    return dtype == COSET_DTYPE_F32 ? launch_dependent("e8_cache_attention", k_cache_attend<DIM, COSET_DTYPE_F32>, grid, 32 * kWarps, 0, st, a)
                                    : launch_dependent("e8_cache_attention", k_cache_attend<DIM, COSET_DTYPE_BF16>, grid, 32 * kWarps, 0, st, a);
}

}  // namespace

extern "C" {

int64_t coset_e8_cache_attention_scratch_bytes(int head_dim) { return known_dim(head_dim) ? 16 : 0; }

int coset_e8_cache_attention(const void* q, int dtype, int64_t q_token_stride, int64_t q_head_stride, int n_queries, int q_heads, const void* pages,
                             int64_t n_pages, int n_heads, int page_size, int head_dim, const int32_t* table, int64_t table_stride, int max_pages,
                             const int32_t* lens, const int32_t* q_starts, int n_seqs, const int64_t* tree, float scale, void* out, float* lse,
                             void* scratch, int64_t scratch_bytes, void* stream) {
    Attend a;
    if (int e = check_pages(pages, n_pages, n_heads, page_size, head_dim, &a.pages)) return e;
    if (dtype != COSET_DTYPE_F32 && dtype != COSET_DTYPE_BF16) return fail(COSET_E_BADARG, "unknown dtype %d", dtype);
    if (n_queries < 0 || n_seqs < 0 || max_pages < 0 || table_stride < 0) return fail(COSET_E_BADARG, "a size is negative");
    if (q_heads < 1 || q_heads % n_heads) return fail(COSET_E_BADARG, "q_heads (%d) must be a multiple of n_heads (%d)", q_heads, n_heads);
    if (n_queries == 0) return 0;
    if (n_seqs == 0 && !q_starts) return fail(COSET_E_BADARG, "queries without sequences");
    if (!q_starts && n_queries % n_seqs) return fail(COSET_E_BADARG, "%d queries are not shared evenly by %d sequences: q_starts says whose they are", n_queries, n_seqs);
    if (!q || !out || (n_seqs > 0 && (!lens || (max_pages > 0 && !table)))) return fail(COSET_E_BADARG, "q, out, table or lens is null");
    if ((int64_t)max_pages * page_size > INT32_MAX) return fail(COSET_E_UNSUPPORTED, "a sequence of 2^31 or more tokens");
    if (n_seqs == 0) return 0;
    const int64_t whole = dtype == COSET_DTYPE_F32 ? 4 : 8;
    if (!aligned(q, 16) || !aligned(out, 16) || (q_token_stride | q_head_stride) % whole) return fail(COSET_E_ALIGN, "rows of q and out must be 16-byte aligned");
    if (!scratch || scratch_bytes < coset_e8_cache_attention_scratch_bytes(head_dim)) return fail(COSET_E_BADARG, "scratch is null or too small");
    if (!aligned(scratch, 16)) return fail(COSET_E_ALIGN, "scratch must be 16-byte aligned");
    a.q = q; a.q_token_stride = q_token_stride; a.q_head_stride = q_head_stride; a.n_queries = n_queries; a.group = q_heads / n_heads;
    a.table = table; a.table_stride = table_stride; a.max_pages = max_pages; a.lens = lens; a.starts = q_starts; a.n_seqs = n_seqs;
    a.tree = tree; a.scale = scale; a.out = out; a.lse = lse;
    const int64_t grid = ((int64_t)n_queries * q_heads + kWarps - 1) / kWarps;
    if (grid > INT32_MAX) return fail(COSET_E_UNSUPPORTED, "too many rows for one call");
    cudaStream_t st = (cudaStream_t)stream;
    return head_dim == 64 ? launch<64>(a, dtype, (unsigned)grid, st) : head_dim == 128 ? launch<128>(a, dtype, (unsigned)grid, st) : launch<256>(a, dtype, (unsigned)grid, st);
}

}  // extern "C"
