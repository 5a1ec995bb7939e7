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

constexpr float kNothing = -3.402823466e38f;  // running maximum of a row that has seen nothing
// Exponent of a value's step as far as the running maximum goes: that of the smallest row that is kept.  A weight thus reaches 2^(1 + kSlack + kShift + 103), and sums
// count in units of 2^13 of them: they stay finite for 2^24 tokens whose values are all that small, and for any number of larger ones.  At the other end the
// largest weight is 2^(kShift - e) beside a step of 2^e, and what lies below 2^-126 is lost: 2^-29 of it for e = 103.  (A branch to exponentials with subnormal
// results and other units there kept all, and took 2 to 4 % of every call.)
constexpr int kLeastSize = -103;
constexpr float kSumUnit = 0x1p-13f;
constexpr float kExactly = 12582912.0f;  // 1.5 2^23, to whose last bits small whole numbers are added
// Scratch memory: a counter per CTA, zero between launches, and two parts per CTA of the rows of a tile: maxima, sums, results
constexpr int kMostCtas = 304, kFewRows = 16, kManyRows = 256, kManyCtas = 152;

// The larger one; not a number where one of them is none.
__device__ __forceinline__ float larger(float x, float y) {
    float z;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(z) : "f"(x), "f"(y));
    return z;
}
__device__ __forceinline__ uint32_t half_pair(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float exp2_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^by, by <= 0, for results and for sums whose maximum is -by below another.  Maxima count a value's size, so that sums of weights range over 200 powers of two, and
// tokens whose values are zeros may have a share in one whose maximum is 2^130 above theirs: 2^by may be no number any more where the sum times it is one.
struct Keep {
    float half;
    __device__ __forceinline__ explicit Keep(float by) : half(exp2_of(0.5f * by)) {}
    __device__ __forceinline__ float factor() const { return half * half; }
    __device__ __forceinline__ float of_sum(float sum) const { return sum * half * half; }
};
// (x & mask) | bits in one instruction, of which the compiler makes two when it knows both constants
__device__ __forceinline__ uint32_t chosen(uint32_t x, uint32_t mask, uint32_t bits) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(x), "r"(mask), "r"(bits));
    return d;
}
// The exponent of a value's step, as far as the running maximum goes
__device__ __forceinline__ float size_of(uint32_t head) { return fmaxf(__uint_as_float(0x4B400000u + (head >> 23 & 255u)) - (kExactly + 127.0f), (float)kLeastSize); }

// A place in the CTA's row of units: tile `tile` of `tiles` of (seq, head, query tile).
struct Place {
    Sequence s;
    int seq, head, qtile, qtiles, tile, tiles;
};
// A segment that other CTAs have parts of, to be joined by the last of them
struct Pending {
    Place place;
    int first_cta, parts, slot, is_last;
};
template <int ROWS, int UNIT>
__device__ __forceinline__ void enter(const Attend& a, Place& p) {
    p.s = sequence(a, p.seq);
    p.qtiles = (p.s.count * a.group + ROWS - 1) / ROWS;
    p.tiles = max((p.s.len + UNIT - 1) / UNIT, 1);
}
template <int ROWS, int UNIT>
__device__ __forceinline__ void next_segment(const Attend& a, Place& p) {
    p.tile = 0;
    if (++p.qtile < p.qtiles) return;
    p.qtile = 0;
    if (++p.head < a.pages.n_heads) return;
    p.head = 0;
    do {
        if (++p.seq >= a.n_seqs) return;
        enter<ROWS, UNIT>(a, p);
    } while (p.qtiles == 0);
}

// The cut of all segments, each as long as its units and kSegment: CTA c has base of that, and one more where c < more.
struct Cut {
    int base, more;
    __device__ __forceinline__ int from(int cta) const { return base * cta + min(cta, more); }
    __device__ __forceinline__ int cta_of(int at) const {
        const int longer = more * (base + 1);
        return at < longer ? at / (base + 1) : more + (at - longer) / base;
    }
};

// Row r of a tile of `rows` queries: where its result goes
__device__ __forceinline__ int64_t result_row(const Attend& a, const Place& p, int rows, int r) {
    const int row = p.qtile * rows + r, query = row / a.group;
    return (int64_t)(p.s.first + query) * (a.group * a.pages.n_heads) + p.head * a.group + row - query * a.group;
}
template <bool BF16, int DIM>
__device__ __forceinline__ void put_pair(const Attend& a, const Place& p, int rows, int r, int d, float x, float y) {
    const int64_t at = result_row(a, p, rows, r) * DIM + d;
    if (BF16) *reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(a.out) + at) = __floats2bfloat162_rn(x, y);
    else *reinterpret_cast<float2*>(static_cast<float*>(a.out) + at) = make_float2(x, y);
}
__device__ __forceinline__ void put_lse(const Attend& a, const Place& p, int rows, int r, float highest, float sum) {
    const float size = sum < 1.0f ? log2f(sum * (1.0f / kSumUnit)) : log2f(sum) + 13.0f;
    if (a.lse) a.lse[result_row(a, p, rows, r)] = highest == kNothing ? -INFINITY : (highest + size) * 0.69314718f;
}

// What a CTA does of a launch: segments, each a (sequence, head, tile of ROWS queries) with its units of UNIT tokens and, in the cut, SEGMENT more for
// what it costs beyond them.  Every warp finds it by itself.
template <int ROWS, int UNIT, int SEGMENT>
struct Part {
    Place place;
    Cut cut;
    int from, to;
    __device__ __forceinline__ int64_t length(const Attend& a, int b) {
        place.s.count = 0;
        if (b >= a.n_seqs) return 0;
        place.seq = b;
        enter<ROWS, UNIT>(a, place);
        return (int64_t)place.qtiles * a.pages.n_heads * (place.tiles + SEGMENT);
    }
    static __device__ __forceinline__ int64_t inclusive(int64_t v) {
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int64_t u = __shfl_up_sync(0xFFFFFFFFu, v, d);
            if ((threadIdx.x & 31) >= d) v += u;
        }
        return v;
    }
    // Whether there is anything to do
    __device__ __forceinline__ bool find(const Attend& a, int most_ctas, int least_units) {
        const int lane = threadIdx.x & 31;
        int64_t all = 0;
        for (int b = 32; b < a.n_seqs; b += 32) all += __shfl_sync(0xFFFFFFFFu, inclusive(length(a, b + lane)), 31);
        int64_t its = length(a, lane), upto = inclusive(its);
        all += __shfl_sync(0xFFFFFFFFu, upto, 31);
        if (all < 1 || all > INT32_MAX) return false;  // so many only from starts that overlap: the host refuses as much work
        const int total = (int)all, ctas = min(most_ctas, (total - 1) / (least_units + SEGMENT) + 1);
        if ((int)blockIdx.x >= ctas) return false;
        cut.base = total / ctas;
        cut.more = total - cut.base * ctas;
        from = cut.from(blockIdx.x);
        to = cut.from(blockIdx.x + 1);
        for (int b = 0;;) {
            const uint32_t here = __ballot_sync(0xFFFFFFFFu, upto - its <= from && from < upto);
            if (here || b + 32 >= a.n_seqs) {  // the lane that has this CTA's first unit tells the others
                const int src = here ? __ffs(here) - 1 : 0, rest = from - (int)__shfl_sync(0xFFFFFFFFu, upto - its, src);
                place.s.first = __shfl_sync(0xFFFFFFFFu, place.s.first, src);
                place.s.count = __shfl_sync(0xFFFFFFFFu, place.s.count, src);
                place.s.len = __shfl_sync(0xFFFFFFFFu, place.s.len, src);
                place.qtiles = __shfl_sync(0xFFFFFFFFu, place.qtiles, src);
                place.tiles = __shfl_sync(0xFFFFFFFFu, place.tiles, src);
                place.seq = b + src;
                const int segment = rest / (place.tiles + SEGMENT);
                place.tile = rest - segment * (place.tiles + SEGMENT);
                place.head = segment / place.qtiles;
                place.qtile = segment - place.head * place.qtiles;
                break;
            }
            b += 32;
            const int64_t before = __shfl_sync(0xFFFFFFFFu, upto, 31);
            its = length(a, b + lane);
            upto = before + inclusive(its);
        }
        if (place.tile >= place.tiles) {  // behind the segment's last unit: on to the next one
            from += place.tiles + SEGMENT - place.tile;
            if (from >= to) return false;
            next_segment<ROWS, UNIT>(a, place);
        }
        return true;
    }
};

// The CTAs' parts into one, by the last CTA that has one, in the order of the CTAs; by all `threads` threads of the CTA.  `arrived`, of thread 0: what the
// counters held before.
template <bool BF16, int DIM, int ROWS>
__device__ __forceinline__ void join_ctas(const Attend& a, Pending* pending, int n_pending, const uint32_t* arrived, int threads) {
    constexpr int kPart = ROWS * (DIM + 2);
    if (threadIdx.x == 0) {
        for (int i = 0; i < n_pending; ++i) {
            pending[i].is_last = arrived[i] == (uint32_t)(pending[i].parts - 1);
            if (pending[i].is_last) a.counters[pending[i].first_cta] = 0;
        }
    }
    __syncthreads();
#pragma unroll 1
    for (int i = 0; i < n_pending; ++i) {
        if (!pending[i].is_last) continue;
        const Place& done = pending[i].place;
        const int rows = min(ROWS, done.s.count * a.group - done.qtile * ROWS), first_cta = pending[i].first_cta, parts = pending[i].parts;
#pragma unroll 1
        for (int at = threadIdx.x; at < rows * (DIM / 4); at += threads) {
            const int r = at / (DIM / 4), d = at % (DIM / 4) * 4;
            float highest = kNothing, sum = 0.0f;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            constexpr int kAtOnce = 8;
#pragma unroll 1
            for (int i0 = 0; i0 < parts; i0 += kAtOnce) {
                float m_of[kAtOnce], l_of[kAtOnce];
                float4 x[kAtOnce];
#pragma unroll
                for (int k = 0; k < kAtOnce; ++k) {
                    const float* part = a.partials + ((int64_t)(first_cta + i0 + k) * 2 + (i0 + k == 0 ? 1 : 0)) * kPart;
                    m_of[k] = kNothing;
                    if (i0 + k < parts) {
                        m_of[k] = __ldcg(part + r);
                        l_of[k] = __ldcg(part + ROWS + r);
                        x[k] = __ldcg(reinterpret_cast<const float4*>(part + 2 * ROWS + r * DIM + d));
                    }
                }
                float higher = highest;
#pragma unroll
                for (int k = 0; k < kAtOnce; ++k) higher = larger(higher, m_of[k]);
                const Keep kept(highest - higher);
                const float before = kept.factor();
                v.x *= before; v.y *= before; v.z *= before; v.w *= before;
                sum = kept.of_sum(sum);
                highest = higher;
#pragma unroll
                for (int k = 0; k < kAtOnce; ++k) {
                    if (i0 + k >= parts) continue;
                    const Keep kept(m_of[k] - highest);
                    const float keep = kept.factor();
                    if (keep != 0.0f) {
                        v.x += x[k].x * keep; v.y += x[k].y * keep; v.z += x[k].z * keep; v.w += x[k].w * keep;
                    }
                    sum += kept.of_sum(l_of[k]);
                }
            }
            const float part_of = highest == kNothing ? 0.0f : kSumUnit / sum;
            put_pair<BF16, DIM>(a, done, ROWS, r, d, v.x * part_of, v.y * part_of);
            put_pair<BF16, DIM>(a, done, ROWS, r, d + 2, v.z * part_of, v.w * part_of);
            if (d == 0) put_lse(a, done, ROWS, r, highest, sum);
        }
    }
}

// Counts the CTA's part of a segment as written; the answer, how many were before, takes its time and is looked at in the end.  By one thread, behind a barrier
// of those that wrote.
__device__ __forceinline__ uint32_t count_part(const Attend& a, Pending& own, const Place& done, const Cut& cut, int first) {
    own.place = done;
    own.first_cta = cut.cta_of(first);
    own.parts = cut.cta_of(first + done.tiles - 1) - own.first_cta + 1;
    uint32_t before;
    asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(a.counters + own.first_cta) : "memory");
    return before;
}

int launch_many(const Attend& a, int head_dim, int rows, cudaStream_t stream);  // e8_cache_attention_many.cu

}  // namespace cache
}  // namespace coset
