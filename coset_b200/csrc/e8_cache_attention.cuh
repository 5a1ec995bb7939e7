// What the attention kernels over an E8-coded cache share: their arguments, how the work is cut up, and who sees what.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstring>
#include <type_traits>

#include "e8_cache.cuh"

namespace coset {
namespace cache {

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
    uint32_t* counters;  // one per CTA, zero before and after every launch
    float* partials;
};

// One sequence as the kernels see it: whatever lens and starts hold, inside the arrays.
struct Sequence {
    int first, count;  // queries
    int len;           // tokens in the cache
};
__device__ __forceinline__ Sequence sequence(const Attend& a, int b) {
    Sequence s;
    if (a.starts) {
        s.first = min(max(a.starts[b], 0), a.n_queries);
        s.count = max(min(max(a.starts[b + 1], 0), a.n_queries) - s.first, 0);
    } else {
        s.count = a.n_queries / a.n_seqs;
        s.first = b * s.count;
    }
    s.len = min(max(a.lens[b], 0), a.max_pages << a.pages.page_log2);
    return s;
}

// The page of a sequence's token, -1 where the cache has none or the token is none of the sequence's.
__device__ __forceinline__ int page_of(const Attend& a, int b, int token, int len) {
    if (token >= len) return -1;
    const int p = __ldg(a.table + b * a.table_stride + (token >> a.pages.page_log2));
    return p >= 0 && p < a.pages.n_pages ? p : -1;
}

}  // namespace cache
}  // namespace coset
