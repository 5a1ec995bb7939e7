// Attention over an E8-coded key/value cache (layout: e8_cache.cuh): out = softmax(scale q K^T + mask) V for the last tokens of every
// sequence, which are one generated token, a chain or a tree of drafted ones.  Few rows: some queries per cache head.
//
// Nothing dense is made.  A key is step (f + c / 2) with f + 8 a 4-bit number n, so
//     q k / step = sum_i q_i n_i + sum_blocks c_b (sum of q over b) / 2 - 8 sum_i q_i.
// A nibble in a byte of its own IS the 8-bit floating-point number (e4m3) n 2^-9, so an operand of the 8-bit products costs three instructions per
// word of eight; they run at twice the rate of the 16-bit ones and their sums are float32.  A bf16 query is the sum of two e4m3 numbers: exactly, down to 2^-9
// of its row's largest value, and to 2^-17 of that below.  A float32 query is three, and three more for what these leave, 2^12 times as large
// and summed apart.  The bits c go through the 16-bit products, as powers of two made by placing a bit in the exponent's field.
//     sum_j w_j v_j, w_j = p_j step_j, takes 16-bit products: a nibble under the exponent of 1024 (or 64, four bits up) less 1032 (72) is f.  (As the
// subnormal number that its bits are it would need no subtraction, but the tensor cores line up products by their exponents and drop ten bits of such a
// sum: results 1e-3 off.  Without the subtraction the sums' rounding, towards zero, counts 72 times: sum w f is small against sum w.)
//
// Tokens are the rows of mma.sync and eight queries its columns (S^T = K Q^T, O^T = V^T P^T): a cache head's queries are mostly fewer than 16, and this
// way 8 of them cost half of what 16 would.  The order of d inside S and of tokens inside O is free, and is chosen such that a lane reads its part of
// a row as one 8- or 16-byte word: lane (g, t) = (lane / 4, lane % 4) has values t DIM / 4 and following of tokens g and g + 8 for S, and values g DIM / 8
// and following of tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9 for O.  P goes from the one to the other by movmatrix.
//
// Work is cut into units of 32 tokens of one (sequence, head, tile of queries), and the units of all of them in a row are cut evenly among the CTAs, one
// per SM; the lengths are read on the device, so a captured launch follows them.  A warp runs through its units alone, with the running maximum
// and sum of the softmax in registers and the next unit's words on their way (cp.async); the warps of a CTA are joined in shared memory, and where
// several CTAs share a row the last one to arrive joins them in the order of the CTAs.
//
// The running maximum is that of a weight times the size of its value (s + the exponent of the value's step), so that w = p step fits 16 bits: what is
// lost is below 2^-31 of the row's largest.  It follows only when it lags by 2^kSlack.  For float32 queries w is split into two 16-bit numbers.
#include <cuda_fp8.h>

#include "e8_cache_attention.cuh"

using namespace coset;
using namespace coset::cache;

namespace {

constexpr int kUnit = 32;         // tokens of a warp's step
constexpr int kLeastUnits = 4;    // of a CTA
constexpr int kLeastSize = -90;   // exponent of a value's step as far as the running maximum goes: sums of p / 2^kLeastSize stay finite
constexpr int kMostCtas = 192;    // counters in the scratch memory

// The row of a group of 8 that stands in row r of an operand: 0 1 2 3 5 4 7 6.  With the swizzles below no read of codes has a bank conflict.
__device__ __forceinline__ int placed(int r) { return r ^ ((r >> 2) & 1); }

template <int DIM>
struct Shape {
    static constexpr int kRowBytes = DIM / 2, kChunks = kRowBytes / 16, kHeads = head_words(DIM);
    static constexpr int kKeyWords = DIM / 32;    // words of a row that a lane has for S
    static constexpr int kValueWords = DIM / 64;  // for O
    static constexpr int kTiles = DIM / 16;       // of O^T
    static constexpr int kBitTiles = DIM == 256 ? 2 : 1;
    static constexpr int kStage = 2 * kUnit * (kRowBytes + 4 * kHeads);
    // where 16-byte chunk c of row r lies
    static __device__ __forceinline__ int chunk(int r, int c) { return DIM == 64 ? c : DIM == 128 ? c ^ (r & 2) : c ^ (r & 7); }
};

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// f = n - 8 of the nibbles at bits 0..3 (even) or 4..7 (odd) of both halves of x, as 16-bit numbers
__device__ __forceinline__ uint32_t even_values(uint32_t x) {
    uint32_t d;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"((x & 0x000F000Fu) | 0x64006400u), "r"(0xE408E408u));
    return d;
}
__device__ __forceinline__ uint32_t odd_values(uint32_t x) {
    uint32_t d;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"((x & 0x00F000F0u) | 0x54005400u), "r"(0xD480D480u));
    return d;
}
__device__ __forceinline__ uint32_t transposed(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ float exp2_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
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
__device__ __forceinline__ uint32_t rest_pair(float lo, float hi, uint32_t pair) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&pair));
    return half_pair(lo - f.x, hi - f.y);
}
// The e4m3 numbers nearest to x, y, z, w in a word; they become what is left.
__device__ __forceinline__ uint32_t take_bytes(float (&x)[4]) {
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const __nv_fp8x2_storage_t b = __nv_cvt_float2_to_fp8x2(make_float2(x[i], x[i + 1]), __NV_SATFINITE, __NV_E4M3);
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(b, __NV_E4M3);
        const float2 f = __half22float2(__half2(h));
        x[i] -= f.x;
        x[i + 1] -= f.y;
        word |= (uint32_t)b << (8 * i);
    }
    return word;
}
// Where bit b of four stands in the exponent of a 16-bit number, and the number that it is there: bit 10 + b, 2^-14, 2^-13, 2^-11, 2^-7.
__device__ __forceinline__ float of_bit(int b) { return b == 0 ? 0x1p-14f : b == 1 ? 0x1p-13f : b == 2 ? 0x1p-11f : 0x1p-7f; }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory"); }

template <int WORDS>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[WORDS]);
template <>
__device__ __forceinline__ void load_words<1>(const uint8_t* p, uint32_t (&w)[1]) { w[0] = *reinterpret_cast<const uint32_t*>(p); }
template <>
__device__ __forceinline__ void load_words<2>(const uint8_t* p, uint32_t (&w)[2]) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x; w[1] = v.y;
}
template <>
__device__ __forceinline__ void load_words<4>(const uint8_t* p, uint32_t (&w)[4]) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
}

// A tile of queries of one head in shared memory, in the order of the operands.
template <int DIM, int PARTS, int NB>
struct Queries {
    static constexpr int kPairs = PARTS == 2 ? 3 : 1;  // of e4m3 numbers for a query
    uint4 words[NB][kPairs][DIM / 32][32];  // of the operand's word w: values 0, 2, 4, 6 and 1, 3, 5, 7, first the one part, then the other
    uint32_t blocks[NB][DIM / 32][32];      // the sum over block w in two 16-bit parts
    float start[8 * NB];                    // -8 sum of q
    float factor[8 * NB];                   // from a sum to a score in powers of two, but for the key's step
    uint64_t bits[8 * NB];                  // the queried tokens that a query sees
};

template <int DIM, int NB, int WARPS>
struct Joining {
    static constexpr int kStride = DIM * 18 / 16 + 4;  // rows of 16 values lie 18 apart: no bank conflicts between lanes
    float o[WARPS][8][kStride];
    float m[WARPS][8 * NB], l[WARPS][8 * NB];
    static __device__ __forceinline__ int at(int d) { return d + 2 * (d / 16); }
};

template <int DIM, int PARTS, int NB, int WARPS>
struct Layout {
    static constexpr int kStages = 2;
    static constexpr int kRing = 0;
    static constexpr int kQueries = kRing + WARPS * kStages * Shape<DIM>::kStage;
    static constexpr int kJoining = kQueries + (int)sizeof(Queries<DIM, PARTS, NB>);
    static constexpr int kBytes = kJoining + (int)sizeof(Joining<DIM, NB, WARPS>);
};

// A place in the CTA's row of units: tile `tile` of `tiles` of (seq, head, query tile).
struct Place {
    Sequence s;
    int seq, head, qtile, qtiles, tile, tiles;
};
template <int ROWS>
__device__ __forceinline__ void enter(const Attend& a, Place& p) {
    p.s = sequence(a, p.seq);
    p.qtiles = (int)(((int64_t)p.s.count * a.group + ROWS - 1) / ROWS);
    p.tiles = max((p.s.len + kUnit - 1) / kUnit, 1);
}
template <int ROWS>
__device__ __forceinline__ void next_segment(const Attend& a, Place& p) {
    p.tile = 0;
    if (++p.qtile < p.qtiles) return;
    p.qtile = 0;
    if (++p.head < a.pages.n_heads) return;
    p.head = 0;
    do {
        if (++p.seq >= a.n_seqs) return;
        enter<ROWS>(a, p);
    } while (p.qtiles == 0);
}

// What a warp fetches next: the units of its CTA from `place` on, every WARPS-th of a segment.
template <int ROWS, int WARPS>
struct Cursor {
    Place place;
    int64_t left = 0;  // units of the CTA from the segment's first one here on
    int i = 0, n = 0;  // unit in the segment's part that the CTA has, and their number
    int page[2] = {-1, -1};
    __device__ __forceinline__ void look_up(const Attend& a) {
        if (left <= 0) return;
        const int token = (place.tile + i) * kUnit;
        page[0] = page_of(a, place.seq, token, place.s.len);
        page[1] = page_of(a, place.seq, token + 16, place.s.len);
    }
    __device__ __forceinline__ void begin(const Attend& a, const Place& p, int64_t units, int warp) {
        place = p;
        left = units;
        i = warp;
        n = (int)min((int64_t)(place.tiles - place.tile), left);
        settle(a, warp);
    }
    __device__ __forceinline__ void settle(const Attend& a, int warp) {
        while (i >= n) {
            left -= n;
            if (left <= 0) return;
            next_segment<ROWS>(a, place);
            i = warp;
            n = (int)min((int64_t)place.tiles, left);
        }
        look_up(a);
    }
};

template <int DIM, int PARTS, int NB, int WARPS>
__device__ __forceinline__ void load_queries(const Attend& a, const Place& p, Queries<DIM, PARTS, NB>& s, int q_bf16) {
    constexpr int kBlocks = DIM / 8;
    const int rows = min(8 * NB, p.s.count * a.group - p.qtile * 8 * NB);
    for (int at = threadIdx.x; at < 8 * NB * kBlocks; at += 32 * WARPS) {  // whole warps go round together
        const int r = at / kBlocks, b = at % kBlocks, row = p.qtile * 8 * NB + r;
        const int query = row / a.group, q_head = p.head * a.group + row % a.group;
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = 0.0f;
        if (r < rows) {
            const int64_t e = (p.s.first + query) * a.q_token_stride + q_head * a.q_head_stride + 8 * b;
            if (q_bf16) {
                const uint4 v = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.q) + e));
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
            } else {
                const float4 v = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + e)), w = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + e) + 1);
                x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w; x[4] = w.x; x[5] = w.y; x[6] = w.z; x[7] = w.w;
            }
        }
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(x[i]) & 0x7FFFFFFFu);
#pragma unroll
        for (int m = 1; m < kBlocks; m *= 2) most = max(most, __shfl_xor_sync(0xFFFFFFFFu, most, m));
        // a power of two that brings the row's largest into [2^7, 2^8): e4m3 ends at 448, and the sum over a block, 16 times as large, fits 16 bits
        const bool number = most < 0x7F800000u;
        const int exponent = number ? min(7 - ((int)(most >> 23) - 127), 126) : 0;
        const float up = __uint_as_float((uint32_t)(exponent + 127) << 23);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = number ? x[i] * up : 0.0f;
            sum += x[i];
        }
        const int t = b / (DIM / 32), word = b % (DIM / 32), lane = (r % 8) * 4 + t;
        float even[4] = {x[0], x[2], x[4], x[6]}, odd[4] = {x[1], x[3], x[5], x[7]};
        uint32_t part[2 * Queries<DIM, PARTS, NB>::kPairs][2];
#pragma unroll
        for (int i = 0; i < 2 * Queries<DIM, PARTS, NB>::kPairs; ++i) {
            if (i == 3) {
#pragma unroll
                for (int k = 0; k < 4; ++k) { even[k] *= 4096.0f; odd[k] *= 4096.0f; }
            }
            part[i][0] = take_bytes(even);
            part[i][1] = take_bytes(odd);
        }
#pragma unroll
        for (int i = 0; i < Queries<DIM, PARTS, NB>::kPairs; ++i)
            s.words[r / 8][i][word][lane] = make_uint4(part[2 * i][0], part[2 * i][1], part[2 * i + 1][0], part[2 * i + 1][1]);
        float total = 0.0f;  // of what the parts stand for, so that what they leave is not counted eight times
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float unit = PARTS == 2 ? 0x1p-12f : 1.0f;
            total += (x[2 * i] - even[i] * unit) + (x[2 * i + 1] - odd[i] * unit);
        }
#pragma unroll
        for (int m = 1; m < kBlocks; m *= 2) total += __shfl_xor_sync(0xFFFFFFFFu, total, m);
        const float half = sum * (0x1p-10f / of_bit(word & 3));
        const uint32_t first = half_pair(half, 0.0f);
        s.blocks[r / 8][word][lane] = (first & 0xFFFFu) | (rest_pair(half, 0.0f, first) << 16);
        if (b == 0) {
            s.start[r] = -8.0f * 0x1p-9f * total;
            s.factor[r] = number ? 0x1p9f * (a.scale * 1.44269504f) / up : __uint_as_float(0x7FC00000u);
            uint64_t bits = 0;
            if (r < rows) bits = a.tree ? (uint64_t)__ldg(a.tree + p.s.first + query) : 0;
            s.bits[r] = a.tree ? bits : (uint64_t)query;
        }
    }
}

template <int DIM, int PARTS, int NB, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, 1)
k_cache_attend(const __grid_constant__ Attend a, int q_bf16) {
    using S = Shape<DIM>;
    using L = Layout<DIM, PARTS, NB, WARPS>;
    constexpr int kRows = 8 * NB, kThreads = 32 * WARPS;
    constexpr float kSlack = PARTS == 2 ? 2.0f : 8.0f, kShift = PARTS == 2 ? 12.0f : 6.0f;  // weights reach 2^(1 + kSlack + kShift)
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int64_t scan[WARPS + 1];
    __shared__ int64_t found_before;
    __shared__ int found_seq, is_last;
    auto& queries = *reinterpret_cast<Queries<DIM, PARTS, NB>*>(smem + L::kQueries);
    auto& joining = *reinterpret_cast<Joining<DIM, NB, WARPS>*>(smem + L::kJoining);
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    grid_wait();
    grid_trigger();

    // ---- this CTA's units
    int64_t total = 0, before = 0;
    const auto units_of = [&](int b) {
        if (b >= a.n_seqs) return (int64_t)0;
        Place p;
        p.seq = b;
        enter<kRows>(a, p);
        return (int64_t)p.qtiles * a.pages.n_heads * p.tiles;
    };
    // inclusive sum over the threads; *sum: over all of them
    const auto inclusive = [&](int64_t v, int64_t* sum) {
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int64_t u = __shfl_up_sync(0xFFFFFFFFu, v, d);
            if (lane >= d) v += u;
        }
        __syncthreads();
        if (lane == 31) scan[warp] = v;
        __syncthreads();
        int64_t mine = 0, all = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            if (w < warp) mine += scan[w];
            all += scan[w];
        }
        *sum = all;
        return v + mine;
    };
    int64_t units = units_of(threadIdx.x), upto = inclusive(units, &total);
    for (int b = kThreads; b < a.n_seqs; b += kThreads) {
        int64_t more;
        inclusive(units_of(b + threadIdx.x), &more);
        total += more;
    }
    const int64_t ctas = min((int64_t)gridDim.x, (total + kLeastUnits - 1) / kLeastUnits);
    if (blockIdx.x >= ctas) return;
    const int64_t from = total * blockIdx.x / ctas, to = total * (blockIdx.x + 1) / ctas;
    if (threadIdx.x == 0) found_seq = -1;
    for (int b = 0; b < a.n_seqs; b += kThreads) {
        if (b > 0) {
            int64_t sum;
            units = units_of(b + threadIdx.x);
            upto = inclusive(units, &sum) + before;
            if (threadIdx.x == 0) scan[WARPS] = before + sum;
        } else if (threadIdx.x == kThreads - 1) {
            scan[WARPS] = upto;
        }
        __syncthreads();
        before = scan[WARPS];
        if (upto - units <= from && from < upto) {
            found_seq = b + threadIdx.x;
            found_before = upto - units;
        }
        __syncthreads();
        if (found_seq >= 0) break;
    }
    Place place;
    place.seq = found_seq;
    enter<kRows>(a, place);
    {
        const int64_t segment = (from - found_before) / place.tiles;
        place.tile = (int)((from - found_before) % place.tiles);
        place.head = (int)(segment / place.qtiles);
        place.qtile = (int)(segment % place.qtiles);
    }

    // ---- fetching
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + L::kRing + warp * L::kStages * S::kStage;
    const uint8_t* ring_at = smem + L::kRing + warp * L::kStages * S::kStage;
    Cursor<kRows, WARPS> cursor;
    const int page_mask = (1 << a.pages.page_log2) - 1;
    // Fetches the next unit; bit h of the result: its tokens 16 h .. 16 h + 15 have a page.
    const auto fetch = [&](int stage) {
        int there = 0;
        if (cursor.left > 0) {
            const uint32_t dst = ring + stage * S::kStage;
            const int token = (cursor.place.tile + cursor.i) * kUnit;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int page = cursor.page[h];
                if (page < 0) continue;
                there |= 1 << h;
                const uint32_t* rec = a.pages.words + record<DIM>(a.pages, page, cursor.place.head);
                const int row0 = (token + 16 * h) & page_mask;
#pragma unroll
                for (int which = 0; which < 2; ++which) {
                    const uint8_t* src = reinterpret_cast<const uint8_t*>(rec) + ((int64_t)which << a.pages.page_log2) * S::kRowBytes + row0 * S::kRowBytes;
#pragma unroll
                    for (int i = 0; i < 16 * S::kChunks; i += 32) {
                        const int at = i + lane, r = at / S::kChunks, c = at % S::kChunks;
                        copy16(dst + (which * kUnit + 16 * h + r) * S::kRowBytes + 16 * S::chunk(r, c), src + at * 16);
                    }
                }
                // heads: of the keys by the first half of the lanes, of the values by the second
                const int which = lane / 16, r = lane % 16;
                const uint32_t* src = rec + ((2 * code_words(DIM) + which * S::kHeads) << a.pages.page_log2) + (row0 + r) * S::kHeads;
#pragma unroll
                for (int i = 0; i < S::kHeads; ++i)
                    copy4(dst + 2 * kUnit * S::kRowBytes + ((which * kUnit + 16 * h + r) * S::kHeads + i) * 4, src + i);
            }
            cursor.i += WARPS;
            cursor.settle(a, warp);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        return there;
    };
    cursor.begin(a, place, to - from, warp);
    int stage = 0, there = fetch(0);

    // ---- one (sequence, head, tile of queries) after the other
    for (int64_t unit = from; unit < to;) {
        const int n = (int)min((int64_t)(place.tiles - place.tile), to - unit);
        __syncthreads();  // nobody reads the queries before, nor joins any more
        load_queries<DIM, PARTS, NB, WARPS>(a, place, queries, q_bf16);
        __syncthreads();
        float o[NB][S::kTiles][4], bits[NB][S::kBitTiles][4], m[NB][2], l[NB][2];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int k = 0; k < S::kTiles; ++k) o[nb][k][i] = 0.0f;
#pragma unroll
                for (int k = 0; k < S::kBitTiles; ++k) bits[nb][k][i] = 0.0f;
            }
            m[nb][0] = m[nb][1] = -INFINITY;
            l[nb][0] = l[nb][1] = 0.0f;
        }
        const int drafted = place.s.len - place.s.count;
        for (int i = warp; i < n; i += WARPS) {
            __syncwarp();  // every lane has read the stage that is filled next
            const int there_next = fetch(stage ^ 1);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            __syncwarp();
            const uint8_t* at = ring_at + stage * S::kStage;
            const uint32_t* key_heads = reinterpret_cast<const uint32_t*>(at + 2 * kUnit * S::kRowBytes);
            const uint32_t* value_heads = key_heads + kUnit * S::kHeads;
            const int token0 = (place.tile + i) * kUnit;

            // scores: [group of 16 tokens][tile of 8 queries][token g: query 2 t, 2 t + 1; token g + 8: the same]
            float s[2][NB][4], rest[2][NB][4];  // rest: 2^12 times what the first three parts of a float32 query leave
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                const float s0 = queries.start[8 * nb + 2 * t], s1 = queries.start[8 * nb + 2 * t + 1];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    s[h][nb][0] = s[h][nb][2] = s0;
                    s[h][nb][1] = s[h][nb][3] = s1;
                    rest[h][nb][0] = rest[h][nb][1] = rest[h][nb][2] = rest[h][nb][3] = 0.0f;
                }
            }
            uint32_t kw[2][2][S::kKeyWords], kh[2][2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int r = 16 * h + 8 * e + placed(g);
                    const uint8_t* row = at + r * S::kRowBytes;
                    if (DIM == 64) {
                        load_words<S::kKeyWords < 4 ? S::kKeyWords : 1>(row + 8 * t, reinterpret_cast<uint32_t(&)[S::kKeyWords < 4 ? S::kKeyWords : 1]>(kw[h][e]));
                    } else {
#pragma unroll
                        for (int c = 0; c < S::kKeyWords / 4; ++c)
                            load_words<4>(row + 16 * S::chunk(r, t * (S::kKeyWords / 4) + c), reinterpret_cast<uint32_t(&)[4]>(kw[h][e][c * 4]));
                    }
                    kh[h][e] = key_heads[r * S::kHeads + (DIM == 256 ? t / 2 : 0)];
                }
            }
#pragma unroll
            for (int w = 0; w < S::kKeyWords; ++w) {
                uint32_t x[2][4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    x[h][0] = kw[h][0][w] & 0x0F0F0F0Fu;
                    x[h][1] = kw[h][1][w] & 0x0F0F0F0Fu;
                    x[h][2] = kw[h][0][w] >> 4 & 0x0F0F0F0Fu;
                    x[h][3] = kw[h][1][w] >> 4 & 0x0F0F0F0Fu;
                }
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int pair = 0; pair < (PARTS == 2 ? 3 : 1); ++pair) {
                        const uint4 q = queries.words[nb][pair][w][lane];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            mma8(2 * pair < 3 ? s[h][nb] : rest[h][nb], x[h][0], x[h][1], x[h][2], x[h][3], q.x, q.y);
                            mma8(2 * pair + 1 < 3 ? s[h][nb] : rest[h][nb], x[h][0], x[h][1], x[h][2], x[h][3], q.z, q.w);
                        }
                    }
            }
#pragma unroll
            for (int w = 0; w < S::kKeyWords; w += 2) {
                uint32_t x[2][2];  // the lane's bits of this and the next blocks at bit 10 and following of both halves
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        x[h][e] = __byte_perm(kh[h][e], 0, 0x1010) >> ((DIM == 64 ? 2 * t : DIM == 128 ? 4 * t : 8 * (t & 1)) + (w & ~3)) << 10;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    const uint32_t q0 = queries.blocks[nb][w][lane], q1 = queries.blocks[nb][w + 1][lane];
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        mma(s[h][nb], x[h][0] & (0x04000400u << (w & 3)), x[h][1] & (0x04000400u << (w & 3)), x[h][0] & (0x08000800u << (w & 3)),
                            x[h][1] & (0x08000800u << (w & 3)), q0, q1);
                }
            }

            // softmax
            const bool all = token0 + kUnit <= drafted && there == 3;
            float step[2][2], value_step[2][2], size[2][2];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    step[h][e] = __uint_as_float(kh[h][e] & 0xFFFF0000u);
                    const uint32_t v = value_heads[(16 * h + 8 * e + placed(g)) * S::kHeads];
                    value_step[h][e] = __uint_as_float(v & 0xFFFF0000u);
                    size[h][e] = (float)max((int)(v >> 23 & 255u) - 127, kLeastSize);
                }
            uint32_t seen[NB] = {};  // bit 4 h + 2 e + c: token 16 h + 8 e + g is seen by query 2 t + c
            if (!all) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const uint64_t who = queries.bits[8 * nb + 2 * t + c];
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const int token = token0 + 16 * h + 8 * e + placed(g), j = token - drafted;
                                const bool yes = token < place.s.len && (there >> h & 1) &&
                                                 (j < 0 || (a.tree ? j < 64 && (who >> j & 1) : j <= (int)who));
                                seen[nb] |= (uint32_t)yes << (4 * h + 2 * e + c);
                            }
                    }
            }
            uint32_t p[2][NB][2][PARTS];  // weights as 16-bit pairs of queries, [group][tile][token g, g + 8][part]
            float lag = -INFINITY, top[NB][2];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const float f = queries.factor[8 * nb + 2 * t + c];
                    top[nb][c] = -INFINITY;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float& x = s[h][nb][2 * e + c];
                            if (PARTS == 2) x += rest[h][nb][2 * e + c] * 0x1p-12f;
                            x *= step[h][e];
                            if (all || (seen[nb] >> (4 * h + 2 * e + c) & 1)) top[nb][c] = larger(top[nb][c], __fmaf_rn(x, f, size[h][e]));
                        }
                    if (top[nb][c] != -INFINITY) lag = larger(lag, top[nb][c] - kShift - m[nb][c]);
                }
            if (__any_sync(0xFFFFFFFFu, !(lag <= kSlack))) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float x = top[nb][c];
#pragma unroll
                        for (int d = 4; d < 32; d *= 2) x = larger(x, __shfl_xor_sync(0xFFFFFFFFu, x, d));
                        x = larger(m[nb][c], x - kShift);
                        const float keep = x == -INFINITY ? 1.0f : exp2_of(m[nb][c] - x);
                        m[nb][c] = x;
                        l[nb][c] *= keep;
#pragma unroll
                        for (int k = 0; k < S::kTiles; ++k) { o[nb][k][c] *= keep; o[nb][k][c + 2] *= keep; }
#pragma unroll
                        for (int k = 0; k < S::kBitTiles; ++k) { bits[nb][k][c] *= keep; bits[nb][k][c + 2] *= keep; }
                    }
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                const float f[2] = {queries.factor[8 * nb + 2 * t], queries.factor[8 * nb + 2 * t + 1]};
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float w[2];
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            float x = exp2_of(__fmaf_rn(s[h][nb][2 * e + c], f[c], -m[nb][c]));
                            w[c] = x * value_step[h][e];
                            if (!all && !(seen[nb] >> (4 * h + 2 * e + c) & 1)) x = w[c] = 0.0f;
                            l[nb][c] += x;
                        }
                        const uint32_t pair = half_pair(w[0], w[1]);
                        p[h][nb][e][0] = transposed(pair);
                        if (PARTS == 2) p[h][nb][e][PARTS - 1] = transposed(rest_pair(w[0], w[1], pair));
                    }
            }

            // values
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t vw[4][S::kValueWords], vh[4];  // tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int r = 16 * h + 8 * (k >> 1) + placed(2 * t + (k & 1));
                    const uint8_t* row = at + (kUnit + r) * S::kRowBytes;
                    const int byte = g * (DIM / 16);
                    load_words<S::kValueWords>(row + 16 * S::chunk(r, byte / 16) + byte % 16, vw[k]);
                    vh[k] = value_heads[r * S::kHeads + (DIM == 256 ? g / 4 : 0)];
                }
                const auto add = [&](float (&acc)[NB][S::kTiles][4], int tile, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int part = 0; part < PARTS; ++part) mma(acc[nb][tile], a0, a1, a2, a3, p[h][nb][0][part], p[h][nb][1][part]);
                };
#pragma unroll
                for (int w = 0; w < S::kValueWords; ++w)
#pragma unroll
                    for (int high = 0; high < 2; ++high) {
                        const uint32_t x = __byte_perm(vw[0][w], vw[1][w], high ? 0x7632 : 0x5410), y = __byte_perm(vw[2][w], vw[3][w], high ? 0x7632 : 0x5410);
                        add(o, 4 * w + 2 * high, even_values(x), odd_values(x), even_values(y), odd_values(y));
                        add(o, 4 * w + 2 * high + 1, even_values(x >> 8), odd_values(x >> 8), even_values(y >> 8), odd_values(y >> 8));
                    }
                const int shift = DIM == 64 ? g : DIM == 128 ? 2 * g : 4 * (g & 3);
                const uint32_t x = __byte_perm(vh[0], vh[1], 0x5410) >> shift << 10, y = __byte_perm(vh[2], vh[3], 0x5410) >> shift << 10;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int part = 0; part < PARTS; ++part)
#pragma unroll
                        for (int k = 0; k < S::kBitTiles; ++k)
                            mma(bits[nb][k], x & (0x04000400u << (2 * k)), x & (0x08000800u << (2 * k)), y & (0x04000400u << (2 * k)), y & (0x08000800u << (2 * k)),
                                p[h][nb][0][part], p[h][nb][1][part]);
            }
            stage ^= 1;
            there = there_next;
        }

        // ---- the warps' parts into one, tile of 8 queries by tile
        const int64_t first_unit = unit - place.tile, end_unit = first_unit + place.tiles;  // of the segment, whoever has them
        const bool whole = place.tile == 0 && n == place.tiles;
        const int rows = min(kRows, place.s.count * a.group - place.qtile * kRows);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float x = l[nb][c];
#pragma unroll
                for (int d = 4; d < 32; d *= 2) x += __shfl_xor_sync(0xFFFFFFFFu, x, d);
                if (g == 0) {
                    joining.m[warp][8 * nb + 2 * t + c] = m[nb][c];
                    joining.l[warp][8 * nb + 2 * t + c] = x;
                }
            }
        __syncthreads();
        const int slot = place.tile > 0 ? 0 : 1;  // a segment that began before this CTA, or one that goes on behind it
        float* partial = a.partials + ((int64_t)blockIdx.x * 2 + slot) * kRows * (DIM + 2);
        const int q_heads = a.group * a.pages.n_heads;
        // row r of the tile: where its result goes
        const auto row_of = [&](int r) {
            const int row = place.qtile * kRows + r;
            return (int64_t)(place.s.first + row / a.group) * q_heads + place.head * a.group + row % a.group;
        };
        const auto put = [&](int r, int d, float v) {
            if (q_bf16) static_cast<__nv_bfloat16*>(a.out)[row_of(r) * DIM + d] = __float2bfloat16_rn(v);
            else static_cast<float*>(a.out)[row_of(r) * DIM + d] = v;
        };
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            float scale[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float x = -INFINITY;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) x = larger(x, joining.m[w][8 * nb + 2 * t + c]);
                scale[c] = m[nb][c] == -INFINITY ? 0.0f : exp2_of(m[nb][c] - x);
            }
            if (nb > 0) __syncthreads();  // the tile before is read
#pragma unroll
            for (int k = 0; k < S::kTiles; ++k) {
                const int d = g * (DIM / 8) + 2 * k, block = k / 4;  // of the lane's blocks
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const float half = bits[nb][block / 2][c + 2 * (block & 1)] * (0.5f / of_bit(block));
                    float2 v = make_float2((o[nb][k][c] + half) * scale[c], (o[nb][k][c + 2] + half) * scale[c]);
                    if (scale[c] == 0.0f) v = make_float2(0.0f, 0.0f);
                    *reinterpret_cast<float2*>(&joining.o[warp][2 * t + c][joining.at(d)]) = v;
                }
            }
            __syncthreads();
            for (int at = threadIdx.x; at < 8 * DIM; at += kThreads) {
                const int r = 8 * nb + at / DIM, d = at % DIM;
                if (r >= rows) continue;
                float v = 0.0f, top = -INFINITY, sum = 0.0f;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) {
                    v += joining.o[w][at / DIM][joining.at(d)];
                    top = larger(top, joining.m[w][r]);
                }
#pragma unroll
                for (int w = 0; w < WARPS; ++w) sum += joining.m[w][r] == -INFINITY ? 0.0f : joining.l[w][r] * exp2_of(joining.m[w][r] - top);
                if (whole) {
                    put(r, d, top == -INFINITY ? 0.0f : v / sum);
                    if (d == 0 && a.lse) a.lse[row_of(r)] = top == -INFINITY ? -INFINITY : (top + log2f(sum)) * 0.69314718f;
                } else {
                    partial[r * (DIM + 2) + d] = v;
                    if (d == 0) { partial[r * (DIM + 2) + DIM] = top; partial[r * (DIM + 2) + DIM + 1] = sum; }
                }
            }
        }
        if (!whole) {
            // the CTAs that share the segment: the one with its first unit to the one with its last
            const int64_t first_cta = ((first_unit + 1) * ctas - 1) / total, last_cta = (end_unit * ctas - 1) / total;
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) is_last = atomicAdd(a.counters + first_cta, 1u) == (uint32_t)(last_cta - first_cta);
            __syncthreads();
            if (is_last) {
                __threadfence();
                const auto part = [&](int64_t cta) { return a.partials + (cta * 2 + (cta == first_cta ? 1 : 0)) * kRows * (DIM + 2); };
                for (int at = threadIdx.x; at < rows * DIM; at += kThreads) {
                    const int r = at / DIM, d = at % DIM;
                    float top = -INFINITY, v = 0.0f, sum = 0.0f;
                    for (int64_t cta = first_cta; cta <= last_cta; ++cta) top = larger(top, __ldcg(part(cta) + r * (DIM + 2) + DIM));
                    for (int64_t cta = first_cta; cta <= last_cta; ++cta) {
                        const float* x = part(cta) + r * (DIM + 2);
                        const float its = __ldcg(x + DIM), keep = its == -INFINITY ? 0.0f : exp2_of(its - top);
                        if (its != -INFINITY) {
                            v += __ldcg(x + d) * keep;
                            sum += __ldcg(x + DIM + 1) * keep;
                        }
                    }
                    put(r, d, top == -INFINITY ? 0.0f : v / sum);
                    if (d == 0 && a.lse) a.lse[row_of(r)] = top == -INFINITY ? -INFINITY : (top + log2f(sum)) * 0.69314718f;
                }
                if (threadIdx.x == 0) a.counters[first_cta] = 0;
            }
        }
        unit += n;
        next_segment<kRows>(a, place);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

constexpr int kMostRows = 16;
int64_t scratch_bytes_of(int head_dim) { return 4 * kMostCtas + (int64_t)kMostCtas * 2 * kMostRows * (head_dim + 2) * 4; }

template <int DIM, int PARTS, int NB, int WARPS>
int launch_as(const Attend& a, int q_bf16, cudaStream_t st) {
    using L = Layout<DIM, PARTS, NB, WARPS>;
    static_assert(L::kBytes <= 227 * 1024 - 1024, "shared memory");
    static_assert(8 * NB <= kMostRows, "scratch memory");
    const auto kernel = k_cache_attend<DIM, PARTS, NB, WARPS>;
    if (int e = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes), "cudaFuncSetAttribute")) return e;
    const int sms = sm_count(), grid = sms < kMostCtas ? sms : kMostCtas;
    return launch_dependent("e8_cache_attention", kernel, (unsigned)grid, 32 * WARPS, L::kBytes, st, a, q_bf16);
}

template <int DIM, int PARTS>
int launch(const Attend& a, int q_bf16, cudaStream_t st) {
    const int64_t rows = ((int64_t)a.n_queries + a.n_seqs - 1) / a.n_seqs * a.group;  // of a cache head, on average
    if (rows <= 8) return launch_as<DIM, PARTS, 1, DIM == 256 ? 8 : 16>(a, q_bf16, st);
    return launch_as<DIM, PARTS, 2, DIM == 256 && PARTS == 2 ? 6 : 8>(a, q_bf16, st);
}

}  // namespace

extern "C" {

int64_t coset_e8_cache_attention_scratch_bytes(int head_dim) { return known_dim(head_dim) ? scratch_bytes_of(head_dim) : 0; }

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
    if ((int64_t)max_pages * page_size > INT32_MAX - 64) return fail(COSET_E_UNSUPPORTED, "a sequence of 2^31 or more tokens");
    if ((int64_t)n_queries * q_heads > INT32_MAX - 64) return fail(COSET_E_UNSUPPORTED, "too many rows for one call");
    if (n_seqs == 0) return 0;
    const int64_t whole = dtype == COSET_DTYPE_F32 ? 4 : 8;
    if (!aligned(q, 16) || !aligned(out, 16) || (q_token_stride | q_head_stride) % whole) return fail(COSET_E_ALIGN, "rows of q and out must be 16-byte aligned");
    if (!scratch || scratch_bytes < coset_e8_cache_attention_scratch_bytes(head_dim)) return fail(COSET_E_BADARG, "scratch is null or too small");
    if (!aligned(scratch, 16)) return fail(COSET_E_ALIGN, "scratch must be 16-byte aligned");
    a.q = q; a.q_token_stride = q_token_stride; a.q_head_stride = q_head_stride; a.n_queries = n_queries; a.group = q_heads / n_heads;
    a.table = table; a.table_stride = table_stride; a.max_pages = max_pages; a.lens = lens; a.starts = q_starts; a.n_seqs = n_seqs;
    a.tree = tree; a.scale = scale; a.out = out; a.lse = lse;
    a.counters = (uint32_t*)scratch;
    a.partials = (float*)scratch + kMostCtas;
    cudaStream_t st = (cudaStream_t)stream;
    const int bf16 = dtype == COSET_DTYPE_BF16;
    if (head_dim == 64) return bf16 ? launch<64, 1>(a, 1, st) : launch<64, 2>(a, 0, st);
    if (head_dim == 128) return bf16 ? launch<128, 1>(a, 1, st) : launch<128, 2>(a, 0, st);
    return bf16 ? launch<256, 1>(a, 1, st) : launch<256, 2>(a, 0, st);
}

}  // extern "C"
