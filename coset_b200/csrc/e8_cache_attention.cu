// Attention over an E8-coded key/value cache (layout: e8_cache.cuh): out = softmax(scale q K^T + mask) V for the last tokens of every
// sequence, which are one generated token, a chain or a tree of drafted ones.  Few rows: some queries per cache head.
//
// Nothing dense is made.  A key is step (f + c / 2) with f + 8 a 4-bit number n, so
//     q k / step = sum_i q_i n_i + sum_blocks c_b (sum of q over b) / 2 - 8 sum_i q_i,
// and with q in fixed point (24 bits from the row's largest on, a power of two per row) all of it is a sum of products of
// bytes: three instructions make eight operands of a word of codes, the sums are exact in 32 bits, and start from the bits of 1.5 2^23, so that they are read
// as floating-point numbers.  What a query loses is 2^-24 of its row's largest value; bf16 loses nothing down to 2^-16 of it.  (Two bytes instead of three
// take 5 % less time, but what they lose of small bf16 values shows in the logarithms of the sums: 1e-5.  As 8-bit floating-point numbers, which a nibble
// is too, the products are no instruction of this chip but fourteen.)
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
// or two per SM; the lengths are read on the device, so a captured launch follows them.  A warp runs through its units alone, with the running maximum
// and sum of the softmax in registers and the next units' codes on their way to shared memory (its lanes look up the pages of 32 units at a time, so that
// addresses cost little); the warps of a CTA are joined in shared memory, and where several CTAs share a row the last one to arrive joins them in the
// order of the CTAs.
//
// The running maximum is that of a weight times the size of its value (s + the exponent of the value's step), so that w = p step fits 16 bits: what is
// lost is below 2^-31 of the row's largest (and, in a run of tokens that the tensor cores sum up, 2^-23 of the sum per token: they cut off what lies behind its 24
// bits).  It follows only when it lags by 2^kSlack.  For float32 queries w is split into two 16-bit numbers.
//
// Measured, 8 heads of 128, 4 bf16 rows each: 32 sequences of 6144 tokens 64 us, of 12,288 115, of 24,576 215, so 4.2 TB/s of codes (64 % of the copy rate)
// beyond 13 us that a launch, the cut, the first loads and two joins cost.  A unit takes 700 instructions (values 250, keys 160, softmax 125, fetching 60): issue slots
// 52 %, ALU pipe 44 %, tensor cores 29 %; twelve warps per SM instead of eight are not faster (67 and 70 us against 63 for lengths of 4000 to 8192).
#include "e8_cache_attention.cuh"

using namespace coset;
using namespace coset::cache;

namespace {

constexpr int kUnit = 32;         // tokens of a warp's step
// With kSegment, the least of the cut that a CTA has, counted in units and the segments' cost: one sequence of 1000 tokens and 8 heads, 8 times 32 units and 16 more, is
// cut among 20 CTAs, of 3 to 20 units.
constexpr int kLeastUnits = 4;
constexpr int kQueryBytes = 3;         // of a query in fixed point
constexpr int kExact = 0x4B400000;  // the bits of kExactly = 1.5 2^23; a whole number of up to 22 bits added to them is added to it
// What a segment costs a CTA beyond its units, in units: its queries, its first loads' latency, its joining.  The cut counts it once per segment, behind its last
// unit, though each of several CTAs that share one pays for it.  (32 sequences of 4000 to 8192 tokens: 63 us, with 24 64, with 32 66; one sequence of 131,071
// 55, 53, 53.)
constexpr int kSegment = 16;

// The row of a group of 8 that stands in row r of an operand: 0 1 2 3 5 4 7 6.  With the swizzle below no read of codes has a bank conflict.
__device__ __forceinline__ int placed(int r) { return r ^ ((r >> 2) & 1); }

// A unit in shared memory: keys, values, heads of keys, heads of values
template <int DIM>
struct Shape {
    static constexpr int kRowBytes = DIM / 2, kChunks = kRowBytes / 16, kHeads = head_words(DIM);
    static constexpr int kKeyWords = DIM / 32;    // words of a row that a lane has for S
    static constexpr int kValueWords = DIM / 64;  // for O
    static constexpr int kTiles = DIM / 16;       // of O^T
    static constexpr int kBitTiles = DIM == 256 ? 2 : 1;  // of the blocks' bits, for S and for O
    static constexpr int kPlane = kUnit * kRowBytes, kHeadsAt = 2 * kPlane, kStage = kHeadsAt + 2 * kUnit * kHeads * 4;
    // Where byte b of row r lies in a plane: 16-byte chunks of rows of 64 (128) bytes are turned by bits of the row, the same ones in every group of 8
    static __device__ __forceinline__ int place(int r, int b) {
        const int turn = DIM == 64 ? 0 : DIM == 128 ? r & 2 : r & 7;
        return r * kRowBytes + ((b / 16 ^ turn) * 16 | b % 16);
    }
};

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// bytes without a sign by bytes with one (the top part of a query) or without
template <bool SIGNED>
__device__ __forceinline__ void mma_bytes(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (SIGNED)
        asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.u8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// f = n - 8 of the nibbles at bits 0..3 (even) or 4..7 (odd) of both halves of x, as 16-bit numbers.  The compiler makes two instructions of masking and
// setting the exponent when it knows both constants (120 of them in a unit), hence the registers whose contents it does not know, and the instruction by its name.
struct Exponents {
    uint32_t even, odd;  // of 1024 and of 64
    __device__ __forceinline__ Exponents() {
        asm volatile("mov.b32 %0, 0x64006400;" : "=r"(even));
        asm volatile("mov.b32 %0, 0x54005400;" : "=r"(odd));
    }
    __device__ __forceinline__ uint32_t even_values(uint32_t x) const {
        uint32_t d;
        asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(chosen(x, 0x000F000Fu, even)), "r"(0xE408E408u));
        return d;
    }
    __device__ __forceinline__ uint32_t odd_values(uint32_t x) const {
        uint32_t d;
        asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(chosen(x, 0x00F000F0u, odd)), "r"(0xD480D480u));
        return d;
    }
};
__device__ __forceinline__ uint32_t transposed(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ uint32_t rest_pair(float lo, float hi, uint32_t pair) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&pair));
    return half_pair(lo - f.x, hi - f.y);
}
// Where bit b of four stands in the exponent of a 16-bit number, and the number that it is there: bit 10 + b, 2^-14, 2^-13, 2^-11, 2^-7.
__device__ __forceinline__ float of_bit(int b) { return b == 0 ? 0x1p-14f : b == 1 ? 0x1p-13f : b == 2 ? 0x1p-11f : 0x1p-7f; }
// Bits 0..3 of x as the bytes of a word
__device__ __forceinline__ uint32_t bytes_of_bits(uint32_t x) { return (x & 15u) * 0x00204081u & 0x01010101u; }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory"); }

template <int WORDS>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t* w) {
    if (WORDS == 1) {
        w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else if (WORDS == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x; w[1] = v.y;
    } else {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    }
}

// A tile of queries of one head in shared memory, in the order of the operands.  Part 0 of a number is its top byte, with the sign.
template <int DIM, int NB>
struct Queries {
    uint2 words[NB][DIM / 32][32][kQueryBytes];                 // of word w: values 0, 2, 4, 6 and 1, 3, 5, 7 of its block
    uint2 blocks[NB][kQueryBytes][Shape<DIM>::kBitTiles][32];   // half the sums of four blocks: the part's bytes, and 64ths of what the top part is too small for
    int start[kQueryBytes][8 * NB];                             // kExact - 8 sum of the part
    float factor[8 * NB];                                 // from a sum to a score in powers of two, but for the key's step
    uint64_t bits[8 * NB];                                // the queried tokens that a query sees
};

template <int DIM, int NB, int WARPS>
struct Joining {
    static constexpr int kStride = DIM * 18 / 16 + 4;  // rows of 16 values lie 18 apart: no bank conflicts between lanes
    float o[WARPS][8 * NB][kStride];      // the warps' sums of w f,
    float bits[WARPS][8 * NB][DIM / 8];   // of w c by block,
    float m[8 * NB][WARPS], l[8 * NB][WARPS];  // their maxima and sums of p
    static __device__ __forceinline__ int at(int d) { return d + 2 * (d / 16); }
};

template <int DIM, int NB, int WARPS>
struct Layout {
    static constexpr int kStages = DIM == 256 ? 2 : 3;
    static constexpr int kQueries = WARPS * kStages * Shape<DIM>::kStage;
    static constexpr int kJoining = kQueries + 2 * (int)sizeof(Queries<DIM, NB>);
    static constexpr int kPending = kJoining + (int)sizeof(Joining<DIM, NB, WARPS>);
    static constexpr int kBytes = kPending + 2 * (int)sizeof(Pending);
};

// A thread's part of a tile of queries on its way to shared memory: blocks of 8 values of rows, whole warps at a time.
template <int DIM, bool BF16, int NB, int WARPS>
struct QueryBlocks {
    static constexpr int kQuads = BF16 ? 1 : 2;  // 16-byte words of a block
    static constexpr int kBlocks = DIM / 8, kAll = 8 * NB * kBlocks, kRounds = (kAll + 32 * WARPS - 1) / (32 * WARPS);
    uint4 x[kRounds][kQuads];
    uint64_t bits[kRounds];
    __device__ __forceinline__ void load(const Attend& a, const Place& p) {
        const int rows = min(8 * NB, p.s.count * a.group - p.qtile * 8 * NB);
#pragma unroll
        for (int i = 0; i < kRounds; ++i) {
            const int at = threadIdx.x + i * 32 * WARPS, r = at / kBlocks, b = at % kBlocks;
#pragma unroll
            for (int k = 0; k < kQuads; ++k) x[i][k] = make_uint4(0, 0, 0, 0);
            bits[i] = 0;
            if (r < rows) {
                const int row = p.qtile * 8 * NB + r, query = row / a.group;
                const int64_t e = (p.s.first + query) * a.q_token_stride + (p.head * a.group + row - query * a.group) * a.q_head_stride + 8 * b;
                const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.q) + e * (BF16 ? 2 : 4));
#pragma unroll
                for (int k = 0; k < kQuads; ++k) x[i][k] = __ldg(src + k);
                if (b == 0) bits[i] = a.tree ? (uint64_t)__ldg(a.tree + p.s.first + query) : (uint64_t)query;
            }
        }
    }
    __device__ __forceinline__ void put(const Attend& a, Queries<DIM, NB>& s) const {
#pragma unroll
        for (int i = 0; i < kRounds; ++i) {
            if (threadIdx.x / 32 * 32 + i * 32 * WARPS < kAll) put_one(a, s, threadIdx.x + i * 32 * WARPS, x[i], bits[i]);
        }
    }
    static __device__ __forceinline__ void put_one(const Attend& a, Queries<DIM, NB>& s, int at, const uint4 (&raw)[kQuads], uint64_t bits) {
        const int r = at / kBlocks, b = at % kBlocks;
        float x[8];
        const uint32_t w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[kQuads - 1].x, raw[kQuads - 1].y, raw[kQuads - 1].z, raw[kQuads - 1].w};
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(!BF16 ? w[i] : i & 1 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(x[i]) & 0x7FFFFFFFu);
#pragma unroll
        for (int m = 1; m < kBlocks; m *= 2) most = max(most, __shfl_xor_sync(0xFFFFFFFFu, most, m));
        // fixed point: a power of two brings the row's largest into [2^(8 kQueryBytes - 2), 2^(8 kQueryBytes - 1))
        constexpr int kTop = 8 * kQueryBytes - 1;
        const bool number = most < 0x7F800000u;
        const int exponent = number ? min(kTop - 1 - ((int)(most >> 23) - 127), 126) : 0;
        const float up = number ? __uint_as_float((uint32_t)(exponent + 127) << 23) : 0.0f;
        uint32_t q[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = number ? (uint32_t)min(__float2int_rn(x[i] * up), (1 << kTop) - 1) : 0u;
        const int lane = (r % 8) * 4 + b / (DIM / 32), word = b % (DIM / 32);
        int part_sum[kQueryBytes], sum = 0;
#pragma unroll
        for (int j = 0; j < kQueryBytes; ++j) {
            const int byte = kQueryBytes - 1 - j;  // of q
            const uint32_t pick = byte * 0x11 + 0x40;
            const uint32_t even = __byte_perm(__byte_perm(q[0], q[2], pick), __byte_perm(q[4], q[6], pick), 0x5410);
            const uint32_t odd = __byte_perm(__byte_perm(q[1], q[3], pick), __byte_perm(q[5], q[7], pick), 0x5410);
            s.words[r / 8][word][lane][j] = make_uint2(even, odd);
            part_sum[j] = j == 0 ? __dp4a((int)even, 0x01010101, __dp4a((int)odd, 0x01010101, 0)) : (int)__dp4a(even, 0x01010101u, __dp4a(odd, 0x01010101u, 0u));
            sum = sum * 256 + part_sum[j];
        }
        // bytes of half the block's sum, four blocks to a word
        const int half = (sum + 1) >> 1;
#pragma unroll
        for (int j = 0; j < kQueryBytes; ++j) {
            const int part = half >> (8 * (kQueryBytes - 1 - j));
            uint8_t* at_block = reinterpret_cast<uint8_t*>(&s.blocks[r / 8][j][word / 4][lane]) + (word & 3);
            at_block[0] = (uint8_t)(j == 0 ? part & 63 : part);
            at_block[4] = (uint8_t)(j == 0 ? part >> 6 : 0);
            if (DIM == 64) at_block[2] = at_block[6] = 0;  // a lane has two blocks of 64 values
        }
        int total = part_sum[0] * 65536 + part_sum[kQueryBytes - 1];  // both fit 16 bits when summed: |q| < 2^7 and 2^8 in 256 values
        int middle = part_sum[1];
#pragma unroll
        for (int m = 1; m < kBlocks; m *= 2) {
            total += __shfl_xor_sync(0xFFFFFFFFu, total, m);
            middle += __shfl_xor_sync(0xFFFFFFFFu, middle, m);
        }
        if (b == 0) {
            s.start[kQueryBytes - 1][r] = kExact - 8 * (total & 0xFFFF);
            s.start[0][r] = kExact - 8 * (total >> 16);
            s.start[1][r] = kExact - 8 * middle;
            s.factor[r] = number ? a.scale * 1.44269504f * __uint_as_float((uint32_t)(127 - exponent) << 23) : __uint_as_float(0x7FC00000u);
            s.bits[r] = bits;
        }
    }
};

// Half a block's bit, from the sum over what the bit stands for as a 16-bit number
template <int DIM>
__device__ __forceinline__ float half_of_bit(int block) { return 0.5f / of_bit(block % (DIM / 64)); }
template <int DIM, bool BF16, int NB, int WARPS, int CTAS>
__global__ void __launch_bounds__(32 * WARPS, CTAS)
k_cache_attend(const __grid_constant__ Attend a) {
    using S = Shape<DIM>;
    using L = Layout<DIM, NB, WARPS>;
    constexpr int kRows = 8 * NB, kThreads = 32 * WARPS, kWeights = BF16 ? 1 : 2;  // 16-bit parts of a weight
    constexpr int kPart = kRows * (DIM + 2);  // floats of a CTA's part: maxima, sums, rows; it has one for a segment that began before it and one for one that goes on behind it
    // Units after which a warp's sums are added to float32 ones in shared memory.  The tensor cores round their sums towards zero: each of a unit's two (float32
    // queries: four) products takes some 2^-24.6 of a sum of one sign with it, so that float32 results of 131,072 tokens which one warp had were 2.7e-4 too
    // small.  Now that is 2^-19.6 (bf16: 2^-17.6) at any length; it takes 1 us per run of a warp, 5 % of long float32 calls and 2 % of bf16 ones (all 16 units: 5 %).
    constexpr int kRun = BF16 ? 64 : 8;
    constexpr float kSlack = BF16 ? 8.0f : 2.0f, kShift = BF16 ? 6.0f : 12.0f;  // weights reach 2^(1 + kSlack + kShift)
    extern __shared__ __align__(128) uint8_t smem[];
    auto* const all_queries = reinterpret_cast<Queries<DIM, NB>*>(smem + L::kQueries);
    auto& joining = *reinterpret_cast<Joining<DIM, NB, WARPS>*>(smem + L::kJoining);
    auto* const pending = reinterpret_cast<Pending*>(smem + L::kPending);
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    grid_wait();
    grid_trigger();

    Part<kRows, kUnit, kSegment> part;
    if (!part.find(a, gridDim.x, kLeastUnits)) return;
    Place place = part.place;
    const Cut cut = part.cut;
    int at_unit = part.from;  // place in the cut
    const int to = part.to;
    QueryBlocks<DIM, BF16, NB, WARPS> raw;
    raw.load(a, place);

    // ---- fetching: the units of a segment's part, every WARPS-th for this warp.  Lane j knows where the rows of the j-th unit ahead are: the first and
    // the last 16 tokens' keys, as bytes from the pages' begin, negative where the cache has no such page.
    const int page_log2 = a.pages.page_log2, page_mask = (1 << page_log2) - 1;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * L::kStages * S::kStage;
    const uint8_t* codes = reinterpret_cast<const uint8_t*>(a.pages.words) + lane * 16;
    const uint32_t value_bytes = (uint32_t)S::kRowBytes << page_log2;
    const uint32_t to_chunk = ring + S::place(lane / S::kChunks, lane % S::kChunks * 16);
    const uint32_t to_odd_chunk = ring + S::place(lane / S::kChunks + 4, lane % S::kChunks * 16) - 4 * S::kRowBytes;  // four rows of 256 values further
    const uint32_t to_head = ring + S::kHeadsAt + ((lane / 16) * kUnit + lane % 16) * S::kHeads * 4;
    const int64_t from_head = ((int64_t)(2 * S::kRowBytes + (lane / 16) * S::kHeads * 4) << page_log2) + lane % 16 * S::kHeads * 4 - lane * 16;  // from a page's first key
    int64_t keys_of[2];
    uint32_t there = 0;  // bits 2 s and 2 s + 1: the tokens of the unit in stage s have a page
    int stage = 0;
    const auto look_up = [&](int k0, int n) {  // from the warp's unit k0 on
        const int i = warp + (k0 + lane) * WARPS;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int token = (place.tile + i) * kUnit + 16 * h, page = i < n ? page_of(a, place.seq, token, place.s.len) : -1;
            keys_of[h] = page < 0 ? -1 : (((int64_t)page * a.pages.n_heads + place.head) * (row_words(DIM) * 4) << page_log2) + (token & page_mask) * S::kRowBytes;
        }
    };
    // Fetches the warp's unit k into the stage `to`; its group of copies is empty where there is none.
    const auto fetch = [&](int k, int units, int to) {
        if (k < units) {
            uint32_t got = 0;
            const int row = (place.tile + warp + k * WARPS) * kUnit;
            const uint32_t stage_at = to * S::kStage;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int64_t at = __shfl_sync(0xFFFFFFFFu, keys_of[h], k & 31);
                if (at < 0) continue;
                got |= 1u << h;
                const uint8_t* key = codes + at;
                const uint8_t* value = key + value_bytes;
                const uint8_t* head = key + (from_head - ((row + 16 * h) & page_mask) * (S::kRowBytes - S::kHeads * 4));
#pragma unroll
                for (int i = 0; i < S::kRowBytes / 32; ++i) {  // 32 chunks at a time
                    const uint32_t to_at = (DIM == 256 && (i & 1) ? to_odd_chunk : to_chunk) + stage_at + (16 * h * S::kRowBytes + i * 512);
                    copy16(to_at, key + i * 512);
                    copy16(to_at + S::kPlane, value + i * 512);
                }
#pragma unroll
                for (int i = 0; i < S::kHeads; ++i) copy4(to_head + stage_at + (16 * h * S::kHeads + i) * 4, head + 4 * i);
            }
            there = (there & ~(3u << 2 * to)) | got << 2 * to;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // The first units of a segment's part; returns how many the warp has.
    const auto begin = [&](int n) {
        const int units = n > warp ? (n - warp - 1) / WARPS + 1 : 0;
        look_up(0, n);
#pragma unroll 1
        for (int k = 0; k < L::kStages - 1; ++k) fetch(k, units, (stage + k) % L::kStages);
        return units;
    };
    int n = min(place.tiles - place.tile, to - at_unit), my_units = begin(n), buffer = 0, n_pending = 0;
    uint32_t arrived[2] = {0, 0};  // of thread 0
    raw.put(a, all_queries[0]);
    __syncthreads();
    // where a lane reads in a stage: keys of token g, values of tokens 2 t and 2 t + 1, and their heads
    const int key_at = S::place(placed(g), t * (DIM / 8)), key_at_1 = S::place(placed(g), t * (DIM / 8) + 16);  // of 256 values, the second half
    const int value_at = S::kPlane + S::place(placed(2 * t), g * (DIM / 16)), value_at_1 = S::kPlane + S::place(placed(2 * t + 1), g * (DIM / 16));
    const int head_at = S::kHeadsAt + placed(g) * S::kHeads * 4;
    const int pair_at = S::kHeadsAt + (kUnit + placed(2 * t)) * S::kHeads * 4 + (DIM == 256 ? g / 4 * 4 : 0);
    const int pair_at_1 = S::kHeadsAt + (kUnit + placed(2 * t + 1)) * S::kHeads * 4 + (DIM == 256 ? g / 4 * 4 : 0);
    const Exponents exponents;

    // ---- one (sequence, head, tile of queries) after the other
    while (true) {
        const auto& queries = all_queries[buffer];
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
            m[nb][0] = m[nb][1] = kNothing;
            l[nb][0] = l[nb][1] = 0.0f;
        }
        // The warp's sums so far to its place in shared memory.  ADD: onto those of the segment's earlier runs, if there are any; what the addition rounds off stays in
        // the registers.
        const auto deposit = [&](auto adds, bool any) {
            constexpr bool ADD = decltype(adds)::value;
            float by[NB][2] = {};
            if (ADD) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int c = 0; c < 2; ++c) by[nb][c] = any ? joining.m[8 * nb + 2 * t + c][warp] - m[nb][c] : 0.0f;
                __syncwarp();  // the maxima are read
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int r = 8 * nb + 2 * t + c;
                    const Keep keep(by[nb][c]);
                    const auto sum_of = [&](float kept, float& x) {
                        const float sum = kept + x;
                        x -= sum - kept;
                        return sum;
                    };
                    const auto put = [&](float& at, float& x) { at = ADD ? sum_of(any ? at * keep.factor() : 0.0f, x) : x; };
                    float x = l[nb][c];
#pragma unroll
                    for (int d = 4; d < 32; d *= 2) x += __shfl_xor_sync(0xFFFFFFFFu, x, d);
                    if (g == 0) {
                        joining.m[r][warp] = m[nb][c];
                        joining.l[r][warp] = ADD ? sum_of(any ? keep.of_sum(joining.l[r][warp]) : 0.0f, x) : x;
                    }
                    l[nb][c] = g == 0 ? x : 0.0f;
#pragma unroll
                    for (int k = 0; k < S::kTiles; ++k) {
                        float2& at = *reinterpret_cast<float2*>(&joining.o[warp][r][joining.at(g * (DIM / 8) + 2 * k)]);
                        float2 its = ADD ? at : make_float2(0.0f, 0.0f);
                        put(its.x, o[nb][k][c]);
                        put(its.y, o[nb][k][c + 2]);
                        at = its;
                    }
#pragma unroll
                    for (int k = 0; k < S::kBitTiles; ++k) {
                        float* const at = &joining.bits[warp][r][g * (DIM / 64) + 2 * k];
                        put(at[0], bits[nb][k][c]);
                        if (DIM > 64) put(at[1], bits[nb][k][c + 2]);
                    }
                }
        };
        const int drafted = place.s.len - place.s.count;
        for (int k = 0; k < my_units;) {
            if (k > 0) deposit(std::true_type(), k > kRun);
            for (const int end = min(k + kRun, my_units); k < end; ++k) {
                __syncwarp();  // every lane has read the stage that is filled next
                if ((k + L::kStages - 1) % 32 == 0) look_up(k + L::kStages - 1, n);
                fetch(k + L::kStages - 1, my_units, stage == 0 ? L::kStages - 1 : stage - 1);
                asm volatile("cp.async.wait_group %0;" ::"n"(L::kStages - 1) : "memory");
                __syncwarp();
                const uint8_t* at = smem + (warp * L::kStages + stage) * S::kStage;
                const auto head_word = [&](int byte) { return *reinterpret_cast<const uint32_t*>(at + byte); };
                const int token0 = (place.tile + warp + k * WARPS) * kUnit;

                // scores: [group of 16 tokens][tile of 8 queries][token g: query 2 t, 2 t + 1; token g + 8: the same]
                float s[2][NB][4], step[2][2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    int sum[kQueryBytes][NB][4];
#pragma unroll
                    for (int j = 0; j < kQueryBytes; ++j)
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            const int2 s0 = *reinterpret_cast<const int2*>(&queries.start[j][8 * nb + 2 * t]);
                            sum[j][nb][0] = sum[j][nb][2] = s0.x;
                            sum[j][nb][1] = sum[j][nb][3] = s0.y;
                        }
                    uint32_t kw[2][S::kKeyWords], kh[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int rows = (16 * h + 8 * e) * S::kRowBytes;
                        if (DIM == 64) load_words<2>(at + key_at + rows, kw[e]);
                        else load_words<4>(at + key_at + rows, kw[e]);
                        if (DIM == 256) load_words<4>(at + key_at_1 + rows, kw[e] + S::kKeyWords / 2);
                        kh[e] = head_word(head_at + (16 * h + 8 * e) * S::kHeads * 4 + (DIM == 256 ? t / 2 * 4 : 0));
                        step[h][e] = __uint_as_float(kh[e] & 0xFFFF0000u);
                    }
#pragma unroll
                    for (int w = 0; w < S::kKeyWords; ++w) {
                        const uint32_t x0 = kw[0][w] & 0x0F0F0F0Fu, x1 = kw[1][w] & 0x0F0F0F0Fu, x2 = kw[0][w] >> 4 & 0x0F0F0F0Fu, x3 = kw[1][w] >> 4 & 0x0F0F0F0Fu;
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            const auto& q = queries.words[nb][w][lane];
                            mma_bytes<true>(sum[0][nb], x0, x1, x2, x3, q[0].x, q[0].y);
#pragma unroll
                            for (int j = 1; j < kQueryBytes; ++j) mma_bytes<false>(sum[j][nb], x0, x1, x2, x3, q[j].x, q[j].y);
                        }
                    }
#pragma unroll
                    for (int k = 0; k < S::kBitTiles; ++k) {
                        const int shift = (DIM == 64 ? 2 * t : DIM == 128 ? 4 * t : 8 * (t & 1)) + 4 * k;
                        const uint32_t x0 = bytes_of_bits(kh[0] >> shift), x1 = bytes_of_bits(kh[1] >> shift);
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                            for (int j = 0; j < kQueryBytes; ++j) {
                                const uint2 q = queries.blocks[nb][j][k][lane];
                                if (j == 0) mma_bytes<true>(sum[j][nb], x0, x1, x0 * 64, x1 * 64, q.x, q.y);
                                else mma_bytes<false>(sum[j][nb], x0, x1, x0, x1, q.x, 0);
                            }
                    }
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int i4 = 0; i4 < 4; ++i4) {
                            float x = __int_as_float(sum[0][nb][i4]) - kExactly;
#pragma unroll
                            for (int j = 1; j < kQueryBytes; ++j) x = __fmaf_rn(x, 256.0f, __int_as_float(sum[j][nb][i4]) - kExactly);
                            s[h][nb][i4] = x;
                        }
                }

                // softmax
                const bool all_seen = token0 + kUnit <= drafted && (there >> 2 * stage & 3) == 3;
                float value_step[2][2], size[2][2], lag = -INFINITY, top[NB][2];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const uint32_t v = head_word(head_at + (kUnit + 16 * h + 8 * e) * S::kHeads * 4);
                        value_step[h][e] = __uint_as_float(v & 0xFFFF0000u);
                        size[h][e] = size_of(v);
                    }
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    const float2 factor = *reinterpret_cast<const float2*>(&queries.factor[8 * nb + 2 * t]);
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            s[h][nb][2 * e] *= step[h][e] * factor.x;
                            s[h][nb][2 * e + 1] *= step[h][e] * factor.y;
                        }
                }
                if (!all_seen) {
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
                                    const bool seen = token < place.s.len && (there >> (2 * stage + h) & 1) && (j < 0 || (a.tree ? j < 64 && (who >> j & 1) : j <= (int)who));
                                    if (!seen) s[h][nb][2 * e + c] = -INFINITY;
                                }
                        }
                }
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        top[nb][c] = s[0][nb][c] + size[0][0];
                        top[nb][c] = larger(top[nb][c], s[0][nb][2 + c] + size[0][1]);
                        top[nb][c] = larger(top[nb][c], s[1][nb][c] + size[1][0]);
                        top[nb][c] = larger(top[nb][c], s[1][nb][2 + c] + size[1][1]);
                        lag = larger(lag, top[nb][c] - m[nb][c]);
                    }
                if (__any_sync(0xFFFFFFFFu, !(lag <= kSlack + kShift))) {
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            float x = top[nb][c];
#pragma unroll
                            for (int d = 4; d < 32; d *= 2) x = larger(x, __shfl_xor_sync(0xFFFFFFFFu, x, d));
                            x = larger(m[nb][c], x - kShift);
                            const Keep kept(m[nb][c] - x);
                            const float keep = kept.factor();
                            m[nb][c] = x;
                            l[nb][c] = kept.of_sum(l[nb][c]);
#pragma unroll
                            for (int k = 0; k < S::kTiles; ++k) { o[nb][k][c] *= keep; o[nb][k][c + 2] *= keep; }
#pragma unroll
                            for (int k = 0; k < S::kBitTiles; ++k) { bits[nb][k][c] *= keep; bits[nb][k][c + 2] *= keep; }
                        }
                }
                uint32_t p[2][NB][2][kWeights];  // weights as 16-bit pairs of queries, [group][tile][token g, g + 8][part]
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float sum[2][2];
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                float& its = s[h][nb][2 * e + c];
                                const float x = exp2_of(its - m[nb][c]);
                                sum[h][e] = x;
                                its = x * value_step[h][e];
                                if (!all_seen && x == 0.0f) its = 0.0f;  // whatever stands in a place that is not seen
                            }
                        l[nb][c] = __fmaf_rn((sum[0][0] + sum[0][1]) + (sum[1][0] + sum[1][1]), kSumUnit, l[nb][c]);
                    }
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float w0 = s[h][nb][2 * e], w1 = s[h][nb][2 * e + 1];
                            const uint32_t pair = half_pair(w0, w1);
                            p[h][nb][e][0] = transposed(pair);
                            if (kWeights == 2) p[h][nb][e][kWeights - 1] = transposed(rest_pair(w0, w1, pair));
                        }

                // values
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t vw[4][S::kValueWords], vh[4];  // tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int rows = 16 * h + 8 * (k >> 1);
                        load_words<S::kValueWords>(at + (k & 1 ? value_at_1 : value_at) + rows * S::kRowBytes, vw[k]);
                        vh[k] = head_word((k & 1 ? pair_at_1 : pair_at) + rows * S::kHeads * 4);
                    }
                    const auto add = [&](float (&acc)[NB][S::kTiles][4], int tile, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                            for (int part = 0; part < kWeights; ++part) mma(acc[nb][tile], a0, a1, a2, a3, p[h][nb][0][part], p[h][nb][1][part]);
                    };
#pragma unroll
                    for (int w = 0; w < S::kValueWords; ++w)
#pragma unroll
                        for (int high = 0; high < 2; ++high) {
                            const uint32_t x = __byte_perm(vw[0][w], vw[1][w], high ? 0x7632 : 0x5410), y = __byte_perm(vw[2][w], vw[3][w], high ? 0x7632 : 0x5410);
                            add(o, 4 * w + 2 * high, exponents.even_values(x), exponents.odd_values(x), exponents.even_values(y), exponents.odd_values(y));
                            add(o, 4 * w + 2 * high + 1, exponents.even_values(x >> 8), exponents.odd_values(x >> 8), exponents.even_values(y >> 8), exponents.odd_values(y >> 8));
                        }
                    const int shift = DIM == 64 ? g : DIM == 128 ? 2 * g : 4 * (g & 3);
                    const uint32_t x = __byte_perm(vh[0], vh[1], 0x5410) >> shift << 10, y = __byte_perm(vh[2], vh[3], 0x5410) >> shift << 10;
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int part = 0; part < kWeights; ++part)
#pragma unroll
                            for (int k = 0; k < S::kBitTiles; ++k)
                                mma(bits[nb][k], x & (0x04000400u << (2 * k)), x & (0x08000800u << (2 * k)), y & (0x04000400u << (2 * k)), y & (0x08000800u << (2 * k)),
                                    p[h][nb][0][part], p[h][nb][1][part]);
                }
                if (++stage == L::kStages) stage = 0;
            }
        }

        // ---- the warps' parts into one
        const Place done = place;
        const int done_units = n, live = min(n, WARPS);  // the first `live` warps had units
        const bool deposited = my_units > kRun;
        const bool whole = done.tile == 0 && n == done.tiles;
        at_unit += n;
        if (done.tile + n == done.tiles) at_unit += kSegment;
        const bool more = at_unit < to;
        if (more) {  // the next segment's queries and first units, on their way meanwhile
            next_segment<kRows, kUnit>(a, place);
            raw.load(a, place);
            n = min(place.tiles, to - at_unit);
            my_units = begin(n);
        }
        if (warp < live) {
            if (deposited) deposit(std::true_type(), true);
            else deposit(std::false_type(), false);
        }
        if (more) raw.put(a, all_queries[buffer ^ 1]);
        __syncthreads();
        const int rows = min(kRows, done.s.count * a.group - done.qtile * kRows);
        float* partial = a.partials + ((int64_t)blockIdx.x * 2 + (done.tile > 0 ? 0 : 1)) * kPart;
#pragma unroll 1
        for (int at = threadIdx.x; at < rows * (DIM / 2); at += kThreads) {
            const int r = at / (DIM / 2), d = at % (DIM / 2) * 2;
            float highest = kNothing, sum = 0.0f;
            for (int w = 0; w < live; ++w) highest = larger(highest, joining.m[r][w]);
            float2 v = make_float2(0.0f, 0.0f);
#pragma unroll 1
            for (int w = 0; w < live; ++w) {
                const Keep kept(joining.m[r][w] - highest);
                const float keep = kept.factor();
                if (keep != 0.0f) {  // a warp that saw nothing has nothing to add, whatever the row's maximum is
                    const float2 x = *reinterpret_cast<const float2*>(&joining.o[w][r][joining.at(d)]);
                    const float half = joining.bits[w][r][d / 8] * half_of_bit<DIM>(d / 8);
                    v.x += (x.x + half) * keep;
                    v.y += (x.y + half) * keep;
                }
                sum += kept.of_sum(joining.l[r][w]);
            }
            if (whole) {
                const float part_of = highest == kNothing ? 0.0f : kSumUnit / sum;
                put_pair<BF16, DIM>(a, done, kRows, r, d, v.x * part_of, v.y * part_of);
                if (d == 0) put_lse(a, done, kRows, r, highest, sum);
            } else {
                *reinterpret_cast<float2*>(partial + 2 * kRows + r * DIM + d) = v;
                if (d == 0) {
                    partial[r] = highest;
                    partial[kRows + r] = sum;
                }
            }
        }
        __syncthreads();  // joined, and the parts written
        if (!whole) {  // the parts are those of the CTA with the segment's first unit to the one with its last
            if (threadIdx.x == 0)
                arrived[n_pending] = count_part(a, pending[n_pending], done, cut, at_unit - (done.tile + done_units == done.tiles ? kSegment : 0) - done_units - done.tile);
            ++n_pending;
        }
        if (!more) break;
        buffer ^= 1;
    }

    if (n_pending > 0) join_ctas<BF16, DIM, kRows>(a, pending, n_pending, arrived, kThreads);
    asm volatile("cp.async.wait_all;" ::: "memory");
}


template <int DIM, bool BF16, int NB, int WARPS, int CTAS>
int launch_as(const Attend& a, cudaStream_t st) {
    using L = Layout<DIM, NB, WARPS>;
    static_assert(CTAS * (L::kBytes + 1024) <= 228 * 1024, "shared memory");
    static_assert(8 * NB <= kFewRows, "scratch memory");
    const auto kernel = k_cache_attend<DIM, BF16, NB, WARPS, CTAS>;
    if (int e = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes), "cudaFuncSetAttribute")) return e;
    const int most = CTAS * sm_count(), grid = most < kMostCtas ? most : kMostCtas;
    return launch_dependent("e8_cache_attention", kernel, (unsigned)grid, 32 * WARPS, L::kBytes, st, a);
}

// Up to so many rows of a cache head, on average over the sequences, stay here; bf16 queries with more go to the kernel for many.  8 cache heads, us here and
// there: of 128 values, 8 sequences of 500 to 3000 tokens with 16, 24, 32 rows 26 and 27, 32 and 27, 36 and 28; 4 of 8000 to 16384 45 and 53, 61 and 53, 64 and
// 55; 32 of 3000 to 6000 84 and 138, 146 and 139, 153 and 140; of 64 values, 8 of 500 to 3000 with 24, 32, 64 rows 22 and 24, 24 and 24, 35 and 25; 32 of 3000 to
// 6000 with 24, 32 rows 97 and 114, 100 and 115.  A batch goes to one kernel as a whole: 63 single tokens and a chain of 16, 64, 512 over 3000 tokens each take 77, 100 and
// 240 us in one call, 66 and 26, 55, 77 in a call each.
constexpr int few_rows_at_most(int head_dim) { return head_dim == 64 ? 32 : 16; }

template <int DIM, bool BF16>
int launch(const Attend& a, cudaStream_t st) {
    const int64_t rows = ((int64_t)a.n_queries + a.n_seqs - 1) / a.n_seqs * a.group;  // of a cache head, on average
    // 16 queries of 128 values take all registers of a thread and 60 to 72 bytes more; 256 values of 16 do not fit at all: 8 sequences of 500 to 3000 tokens with
    // 16 rows 49 us in one tile, 36 in two of 8; 128 rows 166, 147
    if constexpr (DIM == 256) return launch_as<DIM, BF16, 1, 6, 1>(a, st);
    // Fewer parts to join where few heads' tokens are shared by all CTAs, more overlap of one CTA's joining with the other's units elsewhere.  us with one CTA of 8
    // warps and with two of 4: 8 heads of 131,071 tokens 49 and 55, of 32,000 19.7 and 20.5, 2 heads of 32,000 16.5 and 19.1; 64 of 4000 to 8000 24.2 and 22.8,
    // 512 of 300 to 600 28.6 and 24.1.
    else if (rows <= 8 && (int64_t)a.n_seqs * a.pages.n_heads < 16) return launch_as<DIM, BF16, 1, 8, 1>(a, st);
    else if (rows <= 8) return launch_as<DIM, BF16, 1, 4, 2>(a, st);
    else return launch_as<DIM, BF16, 2, 4, 2>(a, st);
}

}  // namespace

extern "C" {

int64_t coset_e8_cache_attention_scratch_bytes(int head_dim) {
    if (!known_dim(head_dim)) return 0;
    const int64_t few = (int64_t)kMostCtas * kFewRows, many = head_dim == 256 ? 0 : (int64_t)kManyCtas * kManyRows;
    static_assert(4 * kMostCtas <= COSET_E8_CACHE_SCRATCH_ZEROS, "the counters");
    return COSET_E8_CACHE_SCRATCH_ZEROS + (few > many ? few : many) * 2 * (head_dim + 2) * 4;
}

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
    // no more than this many units are cut among the CTAs, however the queries are shared among the sequences
    const int64_t tiles = ((int64_t)n_queries * (q_heads / n_heads) + 7) / 8 + n_seqs, longest = ((int64_t)max_pages * page_size + kUnit - 1) / kUnit + 1 + kSegment;
    if (n_pages * n_heads >= UINT32_MAX) return fail(COSET_E_UNSUPPORTED, "2^32 or more records");
    if ((double)tiles * n_heads * longest > 2e9) return fail(COSET_E_UNSUPPORTED, "too much work for one call: queries x pages of the table");
    const int64_t whole = dtype == COSET_DTYPE_F32 ? 4 : 8;
    if (!aligned(q, 16) || !aligned(out, 16) || (q_token_stride | q_head_stride) % whole) return fail(COSET_E_ALIGN, "rows of q and out must be 16-byte aligned");
    if (!scratch || scratch_bytes < coset_e8_cache_attention_scratch_bytes(head_dim)) return fail(COSET_E_BADARG, "scratch is null or too small");
    if (!aligned(scratch, 16)) return fail(COSET_E_ALIGN, "scratch must be 16-byte aligned");
    a.q = q; a.q_token_stride = q_token_stride; a.q_head_stride = q_head_stride; a.n_queries = n_queries; a.group = q_heads / n_heads;
    a.table = table; a.table_stride = table_stride; a.max_pages = max_pages; a.lens = lens; a.starts = q_starts; a.n_seqs = n_seqs;
    a.tree = tree; a.scale = scale; a.out = out; a.lse = lse;
    a.counters = (uint32_t*)scratch;
    a.partials = (float*)scratch + COSET_E8_CACHE_SCRATCH_ZEROS / 4;
    cudaStream_t st = (cudaStream_t)stream;
    const int bf16 = dtype == COSET_DTYPE_BF16;
    const int64_t rows = ((int64_t)n_queries + n_seqs - 1) / n_seqs * a.group;  // of a cache head, on average over the sequences
    if (bf16 && head_dim != 256 && rows > few_rows_at_most(head_dim)) return launch_many(a, head_dim, (int)rows, st);
    if (head_dim == 64) return bf16 ? launch<64, true>(a, st) : launch<64, false>(a, st);
    if (head_dim == 128) return bf16 ? launch<128, true>(a, st) : launch<128, false>(a, st);
    return bf16 ? launch<256, true>(a, st) : launch<256, false>(a, st);
}

}  // extern "C"
