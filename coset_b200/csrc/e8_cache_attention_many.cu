// Attention over an E8-coded key/value cache for many bf16 rows: tiles of 128 queries (of one sequence and cache head) by 128 tokens on tcgen05.
//
// The codes are decoded once for a tile's 128 queries, to 16-bit numbers f + c / 2 in shared memory (a nibble and its block's bit under the exponent of 512,
// less 520): they and the queries, scaled by a power of two per row, are exact, so S = Q K^T is rounded in its float32 sums alone.  The steps are applied to
// S (keys) and to the weights (values).  Both operands lie as rows of tokens of 64 values, 128-byte swizzle: for S the K-major second operand, for
// O += P V the MN-major one, without a transposition.  Inside a block of 8 the values stand as 0 4 1 5 2 6 3 7, which is how they come out of a word, in
// the queries as in the results' columns.
//
// A CTA has 13 warps: two groups of four do the softmax, a thread a row (no shuffles), four decode, one issues the products.  The groups go their own ways,
// each with its S, which its weights P overwrite as the products' operand in tensor memory, its running maxima and its O: while one waits for products
// the other computes.  They take the tiles of tokens in turn and are joined at the end; or, with more than 128 queries, each takes half of 256 and the
// codes are decoded once for both (PAIR).  The running maximum follows only when it lags by 2^kSlack, so O is seldom scaled.  Work is cut among the CTAs
// as for few rows.
//
// Measured: 4 sequences of 8000 to 16384 tokens, 64 queries of 8 heads per cache head, 8 cache heads of 128: 195 us, 0.59 PFLOP/s of S and O.  A group's turn of
// 128 queries by 128 tokens takes some 6300 cycles: 1450 for the maxima, 2700 for the weights, 1900 until the next S.  No unit is full (issue slots 42 %,
// shared memory's pipe 55 %, tensor cores 28 %): what bounds it is the softmax's chain of dependent instructions in two warps per scheduler.  Without any one
// of decoding, maxima, weights, loads of steps it would be 3 to 15 % faster.  Tried: one group with halves of rows 232 us; eight decoding warps and registers
// moved to the softmax 197; loops over tokens unrolled by two or with tensor memory's loads ahead 196 and 235, by 16 instead of 32 tokens 205.
//
// With up to 128 queries (32 sequences of 3000 to 6000 tokens, 32 rows: 140 us) a tile takes some 3800 cycles and the decoding warps bound it: keys and values 850 each with
// the fence behind them, addresses and loads 1500, waits 700.  Two tiles' codes ahead in registers of eight warps 138 us, asynchronous copies to shared memory 137, their
// loops not unrolled 152; the smaller cases were slower by as much.
// Every wait is bounded; when one gives up, the CTA's results are not numbers.
#include "e8_cache_attention.cuh"
#include "umma.cuh"

using namespace coset;
using namespace coset::cache;
using namespace coset::umma;

namespace {

constexpr int kTileRows = 128, kTile = 128;  // queries and tokens of a tile
constexpr int kLeastPage = 16;           // tokens of a page
// A segment's cost beyond its tiles, in tiles, and, with it, the least of the cut that a CTA has.  4 sequences of 8000 to 16384 tokens with 512 rows 194 us (2 tiles: 200, 8: 197), 32 of 3000 to
// 6000 with 32 rows 140 (139, 145); 2 of 300 to 600 with 28 rows 17.9 us (at least 1 tile: 18.4, 4: 23.4).
constexpr int kSegment = 4, kLeastTiles = 2;
constexpr int kSoftmaxWarps = 8, kDecodeWarps = 4, kProductWarp = kSoftmaxWarps + kDecodeWarps, kThreads = 32 * (kProductWarp + 1);
constexpr float kSlack = 8.0f, kShift = 6.0f;  // weights reach 2^(1 + kSlack + kShift)
// Tiles after which a group's sums are added to float32 ones in scratch memory and begin anew.  The tensor cores round their sums towards zero: each of a tile's
// eight products takes some 2^-23.8 of a sum of one sign with it, so that results of 131,072 tokens in one CTA were 2^-10.8 too small.  Now that is 2^-14.8 at any
// length; it takes 2 % of such calls (4 sequences of 100,000 to 120,000 tokens with 128 rows 390 us, without 383), and nothing of those with fewer tiles.
constexpr int kRun = 64;

template <int DIM, bool PAIR>
struct Layout {
    static constexpr int kRows = PAIR ? 256 : 128, kPanels = DIM / 64, kPanel = 128 * 128;  // a panel: 128 rows of 64 16-bit numbers
    static constexpr int kOperand = kPanels * kPanel;
    static constexpr int kQueries = 0, kKeys = kRows / kTileRows * kOperand, kValues = kKeys + 2 * kOperand;
    static constexpr int kUsed = kValues + 2 * kOperand, kWeights = kManyCtas * kRows * 4;  // of parts that are joined, in the same room
    static constexpr int kSteps = kUsed > kWeights ? kUsed : kWeights;                       // [2 stages] of key steps, value steps, sizes
    static constexpr int kJoined = kSteps + 2 * 3 * kTile * 4;  // [2][128] maxima and sums of the groups
    static constexpr int kBars = kJoined + 2 * kTileRows * 8;
    static constexpr int kPendings = kBars + 8 * 18;
    static constexpr int kBytes = kPendings + 2 * (int)sizeof(Pending) + 16 + 1024;
    static constexpr uint32_t kColumns = 512, kResult = 256;  // of tensor memory: two S, then two O
};
// barriers
enum { kKeysFull = 0, kKeysEmpty = 2, kValuesFull = 4, kValuesEmpty = 6, kScoresFull = 8, kWeightsFull = 10, kResultDone = 12, kQueriesFull = 14 };

__device__ __forceinline__ uint32_t element(int row, int chunk) { return (uint32_t)(row * 128 + ((chunk ^ (row & 7)) << 4)); }
__device__ __forceinline__ void store16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void seen_by_products() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ uint32_t half_sum(uint32_t x, uint32_t y) {
    uint32_t z;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(z) : "r"(x), "r"(y));
    return z;
}
// 16 columns of tensor memory, to be waited for
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t at, float* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
          "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
        : "r"(at) : "memory");
}
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// The product with its first operand in tensor memory: a row per lane, two 16-bit numbers per column
__device__ __forceinline__ void umma_f16_from_tmem(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}

// Which of 32 tokens a query sees, the first of them `at` behind the first drafted one: as a chain (who: its place) or as a tree (who: its mask).
__device__ __forceinline__ uint32_t seen_of(bool tree, uint64_t who, int at) {
    if (at <= -32) return 0xFFFFFFFFu;
    if (tree) {
        if (at < 0) return (uint32_t)(who << -at) | ((1u << -at) - 1u);
        return at < 64 ? (uint32_t)(who >> at) : 0u;
    }
    const int n = (int)who + 1 - at;
    return n >= 32 ? 0xFFFFFFFFu : n <= 0 ? 0u : (1u << n) - 1u;
}

// r += kept * keep, of 32 columns; neighbouring rows' results are neighbours, the next four columns lie `rows` further
__device__ __forceinline__ void add_kept(uint32_t (&r)[32], const float4* kept, int rows, float keep, bool any) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float4 old = any ? kept[j * rows] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        r[4 * j] = __float_as_uint(__fmaf_rn(old.x, keep, __uint_as_float(r[4 * j])));
        r[4 * j + 1] = __float_as_uint(__fmaf_rn(old.y, keep, __uint_as_float(r[4 * j + 1])));
        r[4 * j + 2] = __float_as_uint(__fmaf_rn(old.z, keep, __uint_as_float(r[4 * j + 2])));
        r[4 * j + 3] = __float_as_uint(__fmaf_rn(old.w, keep, __uint_as_float(r[4 * j + 3])));
    }
}

// join_ctas for parts of many rows: first the rows' maxima and sums, which give each part's weight (`weights`: room for ROWS floats per CTA of the launch),
// then the weighted sums of the results, each thread with eight of its 16-byte loads under way.  Three parts of 256 rows of 128 in 13 us, with join_ctas 28.
template <int DIM, int ROWS>
__device__ __forceinline__ void join_many(const Attend& a, Pending* pending, int n_pending, const uint32_t* arrived, float* weights) {
    constexpr int kPart = ROWS * (DIM + 2);
    constexpr int kItems = 2, kParts = 4;  // of a thread, under way
    const auto part_at = [&](int first_cta, int k) { return a.partials + ((int64_t)(first_cta + k) * 2 + (k == 0 ? 1 : 0)) * kPart; };
    if (threadIdx.x == 0) {
        for (int i = 0; i < n_pending; ++i) {
            pending[i].is_last = arrived[i] == (uint32_t)(pending[i].parts - 1);
            if (pending[i].is_last) a.counters[pending[i].first_cta] = 0;
        }
    }
#pragma unroll 1
    for (int i = 0; i < n_pending; ++i) {
        __syncthreads();  // who joins is known; the weights before are used
        if (!pending[i].is_last) continue;
        const Place done = pending[i].place;
        const int rows = min(ROWS, done.s.count * a.group - done.qtile * ROWS), first_cta = pending[i].first_cta, parts = pending[i].parts;
#pragma unroll 1
        for (int r = threadIdx.x; r < rows; r += kThreads) {
            float highest = kNothing, sum = 0.0f;
#pragma unroll 4
            for (int k = 0; k < parts; ++k) {
                const float* part = part_at(first_cta, k);
                const float m = __ldcg(part + r), l = __ldcg(part + ROWS + r), higher = larger(highest, m);
                sum = Keep(highest - higher).of_sum(sum) + Keep(m - higher).of_sum(l);
                highest = higher;
                weights[k * ROWS + r] = m;
            }
            const float part_of = highest == kNothing ? 0.0f : kSumUnit / sum;
            for (int k = 0; k < parts; ++k) weights[k * ROWS + r] = exp2_of(weights[k * ROWS + r] - highest) * part_of;
            put_lse(a, done, ROWS, r, highest, sum);
        }
        __syncthreads();
#pragma unroll 1
        for (int at0 = threadIdx.x; at0 < rows * (DIM / 4); at0 += kItems * kThreads) {
            float4 v[kItems];
#pragma unroll
            for (int n = 0; n < kItems; ++n) v[n] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
            for (int k0 = 0; k0 < parts; k0 += kParts) {
                float4 x[kItems][kParts];
#pragma unroll
                for (int k = 0; k < kParts; ++k) {
                    const float* part = part_at(first_cta, min(k0 + k, parts - 1)) + 2 * ROWS;
#pragma unroll
                    for (int n = 0; n < kItems; ++n)
                        x[n][k] = __ldcg(reinterpret_cast<const float4*>(part) + min(at0 + n * kThreads, rows * (DIM / 4) - 1));
                }
#pragma unroll
                for (int k = 0; k < kParts; ++k) {
#pragma unroll
                    for (int n = 0; n < kItems; ++n) {
                        const int r = min((at0 + n * kThreads) / (DIM / 4), rows - 1);
                        const float w = k0 + k < parts ? weights[(k0 + k) * ROWS + r] : 0.0f;
                        if (w != 0.0f) {
                            v[n].x += x[n][k].x * w; v[n].y += x[n][k].y * w; v[n].z += x[n][k].z * w; v[n].w += x[n][k].w * w;
                        }
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < kItems; ++n) {
                const int at = at0 + n * kThreads, r = at / (DIM / 4), d = at % (DIM / 4) * 4;
                if (r >= rows) continue;
                put_pair<true, DIM>(a, done, ROWS, r, d, v[n].x, v[n].y);
                put_pair<true, DIM>(a, done, ROWS, r, d + 2, v[n].z, v[n].w);
            }
        }
    }
}

template <int DIM, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
k_cache_attend_many(const __grid_constant__ Attend a) {
    using L = Layout<DIM, PAIR>;
    constexpr int kRows = L::kRows;
    constexpr int kPart = kRows * (DIM + 2), kChunks = DIM / 32;  // 16-byte chunks of a row of codes
    static_assert(PAIR || 2 * kPart + 2 * kTileRows * (DIM + 2) <= 2 * kManyRows * (DIM + 2), "scratch memory");
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_base = smem_u32(smem_raw), base = (raw_base + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (base - raw_base);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    grid_wait();
    grid_trigger();
    Part<kRows, kTile, kSegment> part;
    if (!part.find(a, gridDim.x, kLeastTiles)) return;
    Place place = part.place;
    int at_unit = part.from;
    const int to = part.to;

    const auto bar = [&](int i) { return base + L::kBars + 8 * i; };
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kPendings + 2 * sizeof(Pending));
    volatile uint32_t* lost = tmem_slot + 1;  // a wait gave up
    auto* const pending = reinterpret_cast<Pending*>(smem + L::kPendings);
    if (warp == kProductWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(L::kColumns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        for (int s = 0; s < 2; ++s) {
            mbar_init(bar(kKeysFull + s), kDecodeWarps);
            mbar_init(bar(kKeysEmpty + s), 1);
            mbar_init(bar(kValuesFull + s), kDecodeWarps);
            mbar_init(bar(kValuesEmpty + s), 1 + kSoftmaxWarps / (PAIR ? 1 : 2));
            mbar_init(bar(kScoresFull + s), 1);
            mbar_init(bar(kWeightsFull + s), kSoftmaxWarps / 2);
            mbar_init(bar(kResultDone + s), 1);
        }
        mbar_init(bar(kQueriesFull), kSoftmaxWarps);
        *lost = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    // Waits of a whole warp, which gives up once at most
    bool gave_up = false;
    const auto await = [&](int i, uint32_t parity) {
        if (!gave_up && !mbar_wait_warp(bar(i), parity)) {
            gave_up = true;
            *lost = 1;
        }
    };
    const auto arrive = [&](int i) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(i));
    };
    int n_pending = 0;
    uint32_t arrived[2] = {0, 0};

    if (warp < kSoftmaxWarps) {
        // ---- a row per thread
        const int group = warp / 4, mine = warp % 4 * 32 + lane, tile_row = PAIR ? group * kTileRows + mine : mine;
        const uint32_t lanes = tmem + ((uint32_t)(warp % 4 * 32) << 16), scores = lanes + group * kTile;
        const auto sync_softmax = [&]() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kSoftmaxWarps) : "memory"); };
        int tile_count = 0, turn = 0;  // tiles of the CTA, over all segments; of the group
        while (true) {
            const int n = min(place.tiles - place.tile, to - at_unit), row = place.qtile * kRows + tile_row, query = row / a.group;
            const bool real = row < place.s.count * a.group;
            // queries: those before are used, for all scores have come
            float factor;
            {
                const int64_t e = (int64_t)(place.s.first + query) * a.q_token_stride + (place.head * a.group + row - query * a.group) * a.q_head_stride;
                const uint4* src = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.q) + e);
                uint32_t most = 0;
#pragma unroll
                for (int b = 0; b < DIM / 8; ++b) {
                    const uint4 x = real ? __ldg(src + b) : make_uint4(0, 0, 0, 0);
                    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) most = max(most, max(w[i] << 16 & 0x7FFFFFFFu, w[i] & 0x7FFF0000u));
                }
                // a power of two brings the row's largest into [2^10, 2^11)
                const bool number = most < 0x7F800000u;
                const int exponent = number ? min(10 - ((int)(most >> 23) - 127), 126) : 0;
                const float up = number ? __uint_as_float((uint32_t)(exponent + 127) << 23) : 0.0f;
                factor = number ? a.scale * 1.44269504f * __uint_as_float((uint32_t)(127 - exponent) << 23) : __uint_as_float(0x7FC00000u);
                const uint32_t to_operand = base + L::kQueries + (PAIR ? group * L::kOperand : 0);
                constexpr int kBlocks = PAIR ? DIM / 8 : DIM / 16;  // the groups share 128 rows
#pragma unroll 4
                for (int i = 0; i < kBlocks; ++i) {
                    const int b = PAIR ? i : group * kBlocks + i;
                    const uint4 x = real ? __ldg(src + b) : make_uint4(0, 0, 0, 0);
                    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
                    uint32_t o[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {  // values k and k + 4
                        const uint32_t lo = k & 1 ? w[k / 2] & 0xFFFF0000u : w[k / 2] << 16, hi = k & 1 ? w[2 + k / 2] & 0xFFFF0000u : w[2 + k / 2] << 16;
                        o[k] = number ? half_pair(__uint_as_float(lo) * up, __uint_as_float(hi) * up) : 0u;
                    }
                    store16(to_operand + b / 8 * L::kPanel + element(mine, b % 8), o[0], o[1], o[2], o[3]);
                }
            }
            uint64_t who = 0;
            if (real) who = a.tree ? (uint64_t)__ldg(a.tree + place.s.first + query) : (uint64_t)query;
            seen_by_products();
            arrive(kQueriesFull);
            const int drafted = place.s.len - place.s.count;
            const Two factors = two(factor, factor);
            float m = kNothing;
            Two l = two(0.0f, 0.0f);
            bool first = true;  // no results of this segment in tensor memory
            // The row's maximum, sum and results of earlier runs of tiles: with two groups of rows in the segment's part, which is written in the end only, else
            // behind all the parts
            float* const run = PAIR ? a.partials + ((int64_t)blockIdx.x * 2 + (place.tile > 0 ? 0 : 1)) * kPart
                                    : a.partials + (int64_t)gridDim.x * 2 * kPart + (blockIdx.x * 2 + group) * (kTileRows * (DIM + 2));
            float4* const results = reinterpret_cast<float4*>(run + 2 * kRows) + tile_row;
            bool any_kept = false;
            for (int i = PAIR ? 0 : (tile_count ^ group) & 1; i < n; i += PAIR ? 1 : 2, ++turn) {
                const int stage = (tile_count + i) & 1;
                await(kValuesFull + stage, (uint32_t)((tile_count + i) >> 1) & 1u);  // the steps
                await(kScoresFull + group, (uint32_t)turn & 1u);                     // and the products of this group before
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (const int before = PAIR ? i : i / 2; before > 0 && before % kRun == 0) {
                    const Keep kept(any_kept ? run[tile_row] - m : 0.0f);
#pragma unroll 1
                    for (int c = 0; c < DIM / 32; ++c) {
                        uint32_t r[32];
                        tmem_ld32(lanes + L::kResult + group * DIM + c * 32, r);
                        add_kept(r, results + c * 8 * kRows, kRows, kept.factor(), any_kept);
#pragma unroll
                        for (int j = 0; j < 32; j += 4)
                            results[(c * 8 + j / 4) * kRows] = make_float4(__uint_as_float(r[j]), __uint_as_float(r[j + 1]), __uint_as_float(r[j + 2]), __uint_as_float(r[j + 3]));
                    }
                    const float2 sums = both(l);
                    run[kRows + tile_row] = (any_kept ? kept.of_sum(run[kRows + tile_row]) : 0.0f) + (sums.x + sums.y);
                    run[tile_row] = m;
                    l = two(0.0f, 0.0f);
                    any_kept = first = true;
                }
                const float* key_step = reinterpret_cast<const float*>(smem + L::kSteps) + stage * 3 * kTile;
                const float *value_step = key_step + kTile, *size = value_step + kTile;
                const int at0 = (place.tile + i) * kTile - drafted;
                // sizes of tokens that are not there are minus infinity
                bool gap = at0 + kTile > 0;
#pragma unroll
                for (int c = 0; c < kTile / 32; ++c) gap |= size[c * 32 + lane] == -INFINITY;
                const auto softmax = [&](auto every) {
                    constexpr bool kAll = decltype(every)::value;
                    const auto seen_in = [&](int c) { return kAll ? 0xFFFFFFFFu : seen_of(a.tree != nullptr, who, at0 + c * 32) & __ballot_sync(0xFFFFFFFFu, size[c * 32 + lane] != -INFINITY); };
                    float top = -INFINITY, top2 = -INFINITY;
#pragma unroll 1
                    for (int c = 0; c < kTile / 32; ++c) {
                        const uint32_t seen = seen_in(c);
                        uint32_t s[32];
                        tmem_ld32(scores + c * 32, s);
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            const float4 k = *reinterpret_cast<const float4*>(key_step + c * 32 + j), z = *reinterpret_cast<const float4*>(size + c * 32 + j);
#pragma unroll
                            for (int e = 0; e < 4; e += 2) {
                                const Two y = mul2(two(__uint_as_float(s[j + e]), __uint_as_float(s[j + e + 1])), e ? two(k.z, k.w) : two(k.x, k.y));
                                float2 t = both(fma2(y, factors, e ? two(z.z, z.w) : two(z.x, z.y)));
                                if (!kAll) {
                                    if (!(seen >> (j + e) & 1)) t.x = -INFINITY;
                                    if (!(seen >> (j + e + 1) & 1)) t.y = -INFINITY;
                                }
                                top = larger(top, t.x);
                                top2 = larger(top2, t.y);
                            }
                        }
                    }
                    top = larger(top, top2);
                    if (__any_sync(0xFFFFFFFFu, !(top - m <= kSlack + kShift))) {
                        const float higher = larger(m, top - kShift), keep_half = Keep(m - higher).half, keep = keep_half * keep_half;
                        m = higher;
                        l = mul2(mul2(l, two(keep_half, keep_half)), two(keep_half, keep_half));
                        if (!first) {
#pragma unroll 1
                            for (int c = 0; c < DIM / 32; ++c) {
                                uint32_t r[32];
                                const uint32_t at = lanes + L::kResult + group * DIM + c * 32;
                                tmem_ld32(at, r);
#pragma unroll
                                for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * keep);
                                tmem_st16(at, r);
                                tmem_st16(at + 16, r + 16);
                            }
                        }
                    }
                    const Two less = two(-m, -m);
                    Two sum = two(0.0f, 0.0f);
#pragma unroll 1
                    for (int c = 0; c < kTile / 32; ++c) {
                        const uint32_t seen = seen_in(c);
                        uint32_t s[32], w[16];
                        tmem_ld32(scores + c * 32, s);
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            const float4 k = *reinterpret_cast<const float4*>(key_step + c * 32 + j), z = *reinterpret_cast<const float4*>(value_step + c * 32 + j);
#pragma unroll
                            for (int e = 0; e < 4; e += 2) {
                                const Two y = mul2(two(__uint_as_float(s[j + e]), __uint_as_float(s[j + e + 1])), e ? two(k.z, k.w) : two(k.x, k.y));
                                float2 t = both(fma2(y, factors, less));
                                if (!kAll) {
                                    if (!(seen >> (j + e) & 1)) t.x = -INFINITY;
                                    if (!(seen >> (j + e + 1) & 1)) t.y = -INFINITY;
                                }
                                const Two x = two(exp2_of(t.x), exp2_of(t.y));
                                sum = add2(sum, x);
                                float2 v = both(mul2(x, e ? two(z.z, z.w) : two(z.x, z.y)));
                                if (!kAll) {  // whatever stands in a place that is not seen
                                    if (!(seen >> (j + e) & 1)) v.x = 0.0f;
                                    if (!(seen >> (j + e + 1) & 1)) v.y = 0.0f;
                                }
                                w[(j + e) / 2] = half_pair(v.x, v.y);
                            }
                        }
                        tmem_st16(scores + c * 16, w);  // over scores that are read
                    }
                    l = fma2(sum, two(kSumUnit, kSumUnit), l);
                };
                if (__any_sync(0xFFFFFFFFu, gap)) softmax(std::false_type());
                else softmax(std::true_type());
                first = false;
                tmem_stored();
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                arrive(kWeightsFull + group);
                if (lane == 0) mbar_arrive(bar(kValuesEmpty + stage));
            }
            // the row's sum, and the results
            const float2 sums = both(l);
            float sum = sums.x + sums.y;
            if (!first) await(kResultDone + group, (uint32_t)(turn - 1) & 1u);
            if (any_kept) {
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const Keep kept(run[tile_row] - m);
                sum += kept.of_sum(run[kRows + tile_row]);
#pragma unroll 1
                for (int c = 0; c < DIM / 32; ++c) {
                    uint32_t r[32];
                    const uint32_t at = lanes + L::kResult + group * DIM + c * 32;
                    tmem_ld32(at, r);
                    add_kept(r, results + c * 8 * kRows, kRows, kept.factor(), true);
                    tmem_st16(at, r);
                    tmem_st16(at + 16, r + 16);
                }
                tmem_stored();
                if (PAIR) sync_softmax();  // all of it is read before the part is written: the groups have the same tiles
            }
            float keeps[2] = {1.0f, 1.0f};
            if (!PAIR) {
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                float2* const joined = reinterpret_cast<float2*>(smem + L::kJoined) + mine;
                joined[group * kTileRows] = make_float2(m, sum);
                sync_softmax();
                const float2 x0 = joined[0], x1 = joined[kTileRows];
                m = larger(x0.x, x1.x);
                const Keep kept0(x0.x - m), kept1(x1.x - m);
                keeps[0] = kept0.factor();
                keeps[1] = kept1.factor();
                sum = kept0.of_sum(x0.y) + kept1.of_sum(x1.y);
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const bool whole = place.tile == 0 && n == place.tiles, failed = *lost != 0;
            if (failed) sum = __uint_as_float(0x7FC00000u);
            const float part_of = m == kNothing && !failed ? 0.0f : kSumUnit / sum;
            float* partial = a.partials + ((int64_t)blockIdx.x * 2 + (place.tile > 0 ? 0 : 1)) * kPart;
            const int64_t result = real ? result_row(a, place, kRows, tile_row) * DIM : 0;
            const int only = PAIR ? group : n == 1 ? tile_count & 1 : -1;  // the group with all results
            constexpr int kColumnsEach = PAIR ? DIM : DIM / 2;
#pragma unroll 1
            for (int c = PAIR ? 0 : group * kColumnsEach; c < (PAIR ? DIM : (group + 1) * kColumnsEach); c += 16) {
                float r[16];
                tmem_ld16(lanes + L::kResult + (only >= 0 ? only * DIM : 0) + c, r);
                if (only < 0) {
                    float o[16];
                    tmem_ld16(lanes + L::kResult + DIM + c, o);
#pragma unroll
                    for (int k = 0; k < 16; ++k) r[k] = r[k] * keeps[0] + o[k] * keeps[1];
                }
                if (real) {
#pragma unroll
                    for (int b = 0; b < 16; b += 8) {  // columns of a block: values 0 4 1 5 2 6 3 7
                        float v[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) v[(k & 1) * 4 + k / 2] = r[b + k];
                        if (whole) {
                            uint32_t o[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k) o[k] = pack_bf16x2(v[2 * k] * part_of, v[2 * k + 1] * part_of);
                            *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + result + c + b) = make_uint4(o[0], o[1], o[2], o[3]);
                        } else {
                            float4* dst = reinterpret_cast<float4*>(partial + 2 * kRows + tile_row * DIM + c + b);
                            dst[0] = make_float4(v[0], v[1], v[2], v[3]);
                            dst[1] = make_float4(v[4], v[5], v[6], v[7]);
                        }
                    }
                }
                __syncwarp();
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            if (real && (PAIR || group == 0)) {
                if (whole) {
                    put_lse(a, place, kRows, tile_row, failed ? sum : m, sum);
                } else {
                    partial[tile_row] = failed ? sum : m;
                    partial[kRows + tile_row] = sum;
                }
            }
            tile_count += n;
            const Place done = place;
            at_unit += n;
            if (done.tile + n == done.tiles) at_unit += kSegment;
            const bool more = at_unit < to;
            if (more) next_segment<kRows, kTile>(a, place);
            sync_softmax();  // what the groups share is read, the part is written
            if (!whole) {
                if (tid == 0)
                    arrived[n_pending] = count_part(a, pending[n_pending], done, part.cut, at_unit - (done.tile + n == done.tiles ? kSegment : 0) - n - done.tile);
                ++n_pending;
            }
            if (!more) break;
        }
    } else if (warp < kProductWarp) {
        // ---- decoding: a thread has a 16-byte chunk of kMine rows that are four apart and in one page.  Eight neighbours have two chunks of four rows:
        // their 16 bytes of an operand lie in different banks.
        constexpr int kMine = kTile * kChunks / (32 * kDecodeWarps);
        static_assert(4 * kMine <= kLeastPage, "a thread's rows are in one page");
        const int t = tid - 32 * kSoftmaxWarps, chunk = (t & 1) | (kChunks == 4 ? t >> 2 & 2 : 0), row0 = t / (4 * kChunks) * (4 * kMine) + (t >> 1 & 3);
        const int page_log2 = a.pages.page_log2, page_mask = (1 << page_log2) - 1;
        int tile_count = 0;
        uint4 codes[2][kMine];
        uint32_t head[2][kMine];
        int page = -1, there = 0, there_next = 0;  // of the tile that is loaded next: the page as the table has it; which rows are there
        const uint32_t* rec = nullptr;
        int at = 0;
        const auto look_up = [&](const Place& p, int tile) {
            const int token = tile * kTile + row0;
            page = -1;
            if (token < p.s.len) page = __ldg(a.table + p.seq * a.table_stride + (token >> page_log2));
        };
        const auto load = [&](const Place& p, int tile, int which) {
            if (which == 0) {
                const int token = tile * kTile + row0;
                at = token & page_mask;
                there_next = 0;
                if (page >= 0 && page < a.pages.n_pages) {
                    rec = a.pages.words + record<DIM>(a.pages, page, p.head);
#pragma unroll
                    for (int i = 0; i < kMine; ++i) there_next |= (token + 4 * i < p.s.len) << i;
                }
            }
            const uint32_t* const its_codes = rec + ((which << page_log2) + at) * code_words(DIM) + chunk * 4;
            const uint32_t* const its_head = rec + ((2 * code_words(DIM) + which) << page_log2) + at;
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                codes[which][i] = make_uint4(0, 0, 0, 0);
                head[which][i] = 0;
                if (there_next >> i & 1) {
                    codes[which][i] = __ldg(reinterpret_cast<const uint4*>(its_codes + 4 * i * code_words(DIM)));
                    head[which][i] = __ldg(its_head + 4 * i);
                }
            }
        };
        const auto put = [&](uint32_t to_operand, const uint4 (&x)[kMine], const uint32_t (&its)[kMine]) {
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
                const int row = row0 + 4 * i;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    // two nibbles of a half word under the exponents of 512 (in units of 1 / 2) and of 32 (1 / 32), less 520 and 40
                    const int word = chunk * 4 + k;
                    const uint32_t coset = its[i] >> word & 1, of_low = coset * 0x00010001u + 0x60006000u, of_high = coset * 0x00100010u + 0x50005000u;
                    const uint32_t w01 = w[k] << 1, w23 = w[k] >> 7;
                    uint32_t o[4];
                    o[0] = half_sum(chosen(w01, 0x001E001Eu, of_low), 0xE010E010u);
                    o[1] = half_sum(chosen(w01, 0x01E001E0u, of_high), 0xD100D100u);
                    o[2] = half_sum(chosen(w23, 0x001E001Eu, of_low), 0xE010E010u);
                    o[3] = half_sum(chosen(w23, 0x01E001E0u, of_high), 0xD100D100u);
                    store16(to_operand + word / 8 * L::kPanel + element(row, word % 8), o[0], o[1], o[2], o[3]);
                }
            }
            seen_by_products();
        };
        // the tile behind the one of (p, tile), if the CTA has it
        Place ahead = place;
        int ahead_unit = at_unit, ahead_tile = place.tile;
        const auto step = [&]() {
            ++ahead_unit;
            if (++ahead_tile < ahead.tiles) return;
            ahead_unit += kSegment;
            if (ahead_unit < to) next_segment<kRows, kTile>(a, ahead);
            ahead_tile = 0;
        };
        bool have = true;
        look_up(ahead, ahead_tile);
        load(ahead, ahead_tile, 0);
        load(ahead, ahead_tile, 1);
        while (have) {
            const int stage = tile_count & 1;
            const uint32_t parity = (uint32_t)((tile_count >> 1) - 1) & 1u;
            there = there_next;
            step();
            have = ahead_unit < to;
            if (have) look_up(ahead, ahead_tile);
            uint32_t key_heads[kMine];
#pragma unroll
            for (int i = 0; i < kMine; ++i) key_heads[i] = head[0][i];
            if (tile_count >= 2) await(kKeysEmpty + stage, parity);
            put(base + L::kKeys + stage * L::kOperand, codes[0], head[0]);
            arrive(kKeysFull + stage);
            if (have) load(ahead, ahead_tile, 0);
            if (tile_count >= 2) await(kValuesEmpty + stage, parity);
            if (chunk == 0) {
                float* steps = reinterpret_cast<float*>(smem + L::kSteps) + stage * 3 * kTile;
#pragma unroll
                for (int i = 0; i < kMine; ++i) {
                    const int row = row0 + 4 * i;
                    steps[row] = __uint_as_float(key_heads[i] & 0xFFFF0000u);
                    steps[kTile + row] = __uint_as_float(head[1][i] & 0xFFFF0000u);
                    steps[2 * kTile + row] = there >> i & 1 ? size_of(head[1][i]) : -INFINITY;
                }
            }
            put(base + L::kValues + stage * L::kOperand, codes[1], head[1]);
            arrive(kValuesFull + stage);
            if (have) load(ahead, ahead_tile, 1);
            ++tile_count;
        }
    } else {
        // ---- products: S of a group's tile, then O of the other group's tile before
        constexpr uint32_t kScoresDesc = (1u << 4) | ((uint32_t)(kTile >> 3) << 17) | ((uint32_t)(kTileRows >> 4) << 24);
        constexpr uint32_t kResultDesc = (1u << 4) | (1u << 16) | ((uint32_t)(DIM >> 3) << 17) | ((uint32_t)(kTileRows >> 4) << 24);
        const uint64_t k_major = umma_desc(base);
        // MN-major: blocks of 64 values lie a panel apart
        const uint32_t high = (uint32_t)(k_major >> 32), queries = (uint32_t)k_major + (L::kQueries >> 4), keys = (uint32_t)k_major + (L::kKeys >> 4);
        const uint32_t values = (((uint32_t)k_major & 0xFFFFu) | ((uint32_t)(L::kPanel >> 4) << 16)) + (L::kValues >> 4);
        constexpr int kEach = PAIR ? 2 : 1;  // groups that take a tile
        int tile_count = 0, segment = 0;
        uint32_t phases = 0;
        while (true) {
            const int n = min(place.tiles - place.tile, to - at_unit);
            await(kQueriesFull, (uint32_t)segment & 1u);
            for (int i = 0; i <= n * kEach; ++i) {
                if (i < n * kEach) {
                    // the scores of the group before are read and their weights used: those products came before these
                    const int count = tile_count + i / kEach, stage = count & 1, group = PAIR ? i & 1 : stage;
                    if (!PAIR || group == 0) await(kKeysFull + stage, (uint32_t)(count >> 1) & 1u);
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < DIM / 16; ++k)
                            umma_f16(tmem + group * kTile, make_desc(queries + (PAIR ? group * (L::kOperand >> 4) : 0) + k / 4 * (L::kPanel >> 4) + k % 4 * 2, high),
                                     make_desc(keys + stage * (L::kOperand >> 4) + k / 4 * (L::kPanel >> 4) + k % 4 * 2, high), kScoresDesc, k > 0);
                        umma_commit(bar(kScoresFull + group));
                        if (!PAIR || group == 1) umma_commit(bar(kKeysEmpty + stage));
                    }
                    __syncwarp();
                }
                if (i > 0) {
                    const int count = tile_count + (i - 1) / kEach, stage = count & 1, group = PAIR ? (i - 1) & 1 : stage;
                    if (!PAIR || group == 0) await(kValuesFull + stage, (uint32_t)(count >> 1) & 1u);
                    await(kWeightsFull + group, phases >> group & 1u);
                    phases ^= 1u << group;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < kTile / 16; ++k)  // 16 tokens: two groups of eight lines of a panel
                            umma_f16_from_tmem(tmem + L::kResult + group * DIM, tmem + group * kTile + k * 8, make_desc(values + stage * (L::kOperand >> 4) + k * 128, high),
                                               kResultDesc, (i - 1) / 2 % kRun > 0 || k > 0);
                        umma_commit(bar(kResultDone + group));
                        if (!PAIR || group == 1) umma_commit(bar(kValuesEmpty + stage));
                    }
                    __syncwarp();
                }
            }
            tile_count += n;
            ++segment;
            const bool done = place.tile + n == place.tiles;
            at_unit += n + (done ? kSegment : 0);
            if (at_unit >= to) break;
            next_segment<kRows, kTile>(a, place);
        }
    }
    if (*lost)
        for (int i = 0; i < 64; ++i) __nanosleep(1000);  // a wait gave up: products still under way get time to end
    n_pending = __shfl_sync(0xFFFFFFFFu, n_pending, 0);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    int* const shared_pending = reinterpret_cast<int*>(tmem_slot + 2);
    if (tid == 0) *shared_pending = n_pending;
    __syncthreads();
    if (warp == kProductWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::kColumns) : "memory");
    n_pending = *shared_pending;
    if (n_pending > 0) join_many<DIM, kRows>(a, pending, n_pending, arrived, reinterpret_cast<float*>(smem));
}

template <int DIM, bool PAIR>
int launch_as(const Attend& a, cudaStream_t st) {
    static_assert(Layout<DIM, PAIR>::kBytes <= 227 * 1024, "shared memory");
    const auto kernel = k_cache_attend_many<DIM, PAIR>;
    if (int e = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<DIM, PAIR>::kBytes), "cudaFuncSetAttribute")) return e;
    const int sms = sm_count(), grid = sms < kManyCtas ? sms : kManyCtas;
    return launch_dependent("e8_cache_attention", kernel, (unsigned)grid, kThreads, Layout<DIM, PAIR>::kBytes, st, a);
}

}  // namespace

namespace coset {
namespace cache {

int launch_many(const Attend& a, int head_dim, int rows, cudaStream_t stream) {
    if (rows > kTileRows) return head_dim == 64 ? launch_as<64, true>(a, stream) : launch_as<128, true>(a, stream);
    return head_dim == 64 ? launch_as<64, false>(a, stream) : launch_as<128, false>(a, stream);
}

}  // namespace cache
}  // namespace coset
