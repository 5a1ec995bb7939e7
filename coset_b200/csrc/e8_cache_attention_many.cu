// Attention over an E8-coded key/value cache for many bf16 rows: tiles of 128 queries (of one sequence and cache head) by 128 tokens on tcgen05.
//
// The codes are decoded once for a tile's 128 queries, to 16-bit numbers f + c / 2 in shared memory (a nibble and its block's bit under the exponent of 512,
// less 520): they and the queries, scaled by a power of two per row, are exact, so S = Q K^T is rounded in its float32 sums alone.  The steps are applied to
// S (keys) and to the weights (values).  Both operands lie as rows of tokens of 64 values, 128-byte swizzle: for S the K-major second operand, for
// O += P V the MN-major one, without a transposition.  Inside a block of 8 the values stand as 0 4 1 5 2 6 3 7, which is how they come out of a word, in
// the queries as in the results' columns.
//
// A CTA has 13 warps: four have a row of the tile per thread (softmax, no shuffles: the row's maximum and sum are a thread's own), eight decode, one issues the
// products.  S has two buffers in tensor memory, so that S of the next tile runs under the softmax of this one; keys and values have two each.  The running
// maximum follows only when it lags by 2^kSlack, so the results in tensor memory are seldom scaled.  Work is cut among the CTAs as for few rows.
// Every wait is bounded; when one gives up, the CTA's results are not numbers.
#include "e8_cache_attention.cuh"
#include "umma.cuh"

using namespace coset;
using namespace coset::cache;
using namespace coset::umma;

namespace {

constexpr int kRows = 128, kTile = 128;  // queries and tokens of a tile
constexpr int kSegment = 4, kLeastTiles = 2;
constexpr int kSoftmaxWarps = 4, kDecodeWarps = 8, kProductWarp = kSoftmaxWarps + kDecodeWarps, kThreads = 32 * (kProductWarp + 1);
constexpr float kSlack = 8.0f, kShift = 6.0f;  // weights reach 2^(1 + kSlack + kShift)

template <int DIM>
struct Layout {
    static constexpr int kPanels = DIM / 64, kPanel = 128 * 128;  // a panel: 128 rows of 64 16-bit numbers
    static constexpr int kOperand = kPanels * kPanel;
    static constexpr int kKeys = kOperand, kValues = kKeys + 2 * kOperand, kWeights = kValues + 2 * kOperand;  // behind the queries
    static constexpr int kSteps = kWeights + 2 * kPanel;  // [2 stages] of key steps, value steps, sizes
    static constexpr int kBars = kSteps + 2 * 3 * kTile * 4;
    static constexpr int kPendings = kBars + 8 * 16;
    static constexpr int kBytes = kPendings + 2 * (int)sizeof(Pending) + 16 + 1024;
    static constexpr uint32_t kColumns = 512, kResult = 256;  // of tensor memory: two S, then O
};
// barriers
enum { kKeysFull = 0, kKeysEmpty = 2, kValuesFull = 4, kValuesEmpty = 6, kScoresFull = 8, kScoresEmpty = 10, kWeightsFull = 12, kResultDone = 13, kQueriesFull = 14 };

__device__ __forceinline__ uint32_t element(int row, int chunk) { return (uint32_t)(row * 128 + ((chunk ^ (row & 7)) << 4)); }
__device__ __forceinline__ void store16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void seen_by_products() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tmem_st32(uint32_t at, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
          "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
          "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

template <int DIM>
__global__ void __launch_bounds__(kThreads, 1)
k_cache_attend_many(const __grid_constant__ Attend a) {
    using L = Layout<DIM>;
    constexpr int kPart = kRows * (DIM + 2), kChunks = DIM / 32;  // 16-byte chunks of a row of codes
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
            mbar_init(bar(kValuesEmpty + s), 1 + kSoftmaxWarps);
            mbar_init(bar(kScoresFull + s), 1);
            mbar_init(bar(kScoresEmpty + s), kSoftmaxWarps);
        }
        mbar_init(bar(kWeightsFull), kSoftmaxWarps);
        mbar_init(bar(kResultDone), 1);
        mbar_init(bar(kQueriesFull), kSoftmaxWarps);
        *lost = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    // Waits of a whole warp
    const auto await = [&](int i, uint32_t parity) {
        if (*lost) return;
        if (!mbar_wait_warp(bar(i), parity)) *lost = 1;
    };
    const auto arrive = [&](int i) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(i));
    };
    int n_pending = 0;
    uint32_t arrived[2] = {0, 0};

    if (warp < kSoftmaxWarps) {
        // ---- a row per thread
        const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
        int tile_count = 0;  // of the CTA, over all segments
        while (true) {
            const int n = min(place.tiles - place.tile, to - at_unit), row = place.qtile * kRows + tid, query = row / a.group;
            const bool real = row < place.s.count * a.group;
            // queries: the product warp is through with those before, for all scores have come
            float factor;
            {
                const int64_t e = (int64_t)(place.s.first + query) * a.q_token_stride + (place.head * a.group + row - query * a.group) * a.q_head_stride;
                const uint4* src = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.q) + e);
                uint32_t most = 0;
                uint4 x[DIM / 8];
#pragma unroll
                for (int b = 0; b < DIM / 8; ++b) {
                    x[b] = real ? __ldg(src + b) : make_uint4(0, 0, 0, 0);
                    const uint32_t w[4] = {x[b].x, x[b].y, x[b].z, x[b].w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) most = max(most, max(w[i] << 16 & 0x7FFFFFFFu, w[i] & 0x7FFF0000u));
                }
                // a power of two brings the row's largest into [2^10, 2^11)
                const bool number = most < 0x7F800000u;
                const int exponent = number ? min(10 - ((int)(most >> 23) - 127), 126) : 0;
                const float up = number ? __uint_as_float((uint32_t)(exponent + 127) << 23) : 0.0f;
                factor = number ? a.scale * 1.44269504f * __uint_as_float((uint32_t)(127 - exponent) << 23) : __uint_as_float(0x7FC00000u);
#pragma unroll
                for (int b = 0; b < DIM / 8; ++b) {
                    const uint32_t w[4] = {x[b].x, x[b].y, x[b].z, x[b].w};
                    uint32_t o[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {  // values i and i + 4
                        const uint32_t lo = i & 1 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16, hi = i & 1 ? w[2 + i / 2] & 0xFFFF0000u : w[2 + i / 2] << 16;
                        o[i] = number ? half_pair(__uint_as_float(lo) * up, __uint_as_float(hi) * up) : 0u;
                    }
                    store16(base + b / 8 * L::kPanel + element(tid, b % 8), o[0], o[1], o[2], o[3]);
                }
            }
            uint64_t who = 0;
            if (real) who = a.tree ? (uint64_t)__ldg(a.tree + place.s.first + query) : (uint64_t)query;
            seen_by_products();
            arrive(kQueriesFull);
            const int drafted = place.s.len - place.s.count;
            float m = kNothing, l = 0.0f;
            for (int i = 0; i < n; ++i, ++tile_count) {
                const int stage = tile_count & 1;
                const uint32_t parity = (uint32_t)(tile_count >> 1) & 1u;
                await(kValuesFull + stage, parity);  // the steps
                await(kScoresFull + stage, parity);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const float* key_step = reinterpret_cast<const float*>(smem + L::kSteps) + stage * 3 * kTile;
                const float *value_step = key_step + kTile, *size = value_step + kTile;
                const int token0 = (place.tile + i) * kTile;
                bool bad = false;  // sizes of tokens that are not there are minus infinity
#pragma unroll
                for (int k = 0; k < 4; ++k) bad |= size[lane + 32 * k] == -INFINITY;
                const bool all_seen = token0 + kTile <= drafted && !__any_sync(0xFFFFFFFFu, bad);
                const auto seen = [&](int j) {  // token j of the tile
                    const int at = token0 + j - drafted;
                    return size[j] != -INFINITY && (at < 0 || (a.tree ? at < 64 && (who >> at & 1) : at <= (int)who));
                };
                // scores in powers of two, 32 columns at a time
                const auto scores = [&](int chunk, uint32_t (&s)[32]) {
                    tmem_ld32(lanes + stage * kTile + chunk * 32, s);
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        const float4 k = *reinterpret_cast<const float4*>(key_step + chunk * 32 + j);
                        s[j] = __float_as_uint(__uint_as_float(s[j]) * (k.x * factor));
                        s[j + 1] = __float_as_uint(__uint_as_float(s[j + 1]) * (k.y * factor));
                        s[j + 2] = __float_as_uint(__uint_as_float(s[j + 2]) * (k.z * factor));
                        s[j + 3] = __float_as_uint(__uint_as_float(s[j + 3]) * (k.w * factor));
                    }
                    if (!all_seen) {
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (!seen(chunk * 32 + j)) s[j] = 0xFF800000u;
                    }
                };
                float top = -INFINITY;
#pragma unroll 1
                for (int chunk = 0; chunk < 4; ++chunk) {
                    uint32_t s[32];
                    scores(chunk, s);
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        const float4 z = *reinterpret_cast<const float4*>(size + chunk * 32 + j);
                        top = larger(top, larger(larger(__uint_as_float(s[j]) + z.x, __uint_as_float(s[j + 1]) + z.y),
                                                 larger(__uint_as_float(s[j + 2]) + z.z, __uint_as_float(s[j + 3]) + z.w)));
                    }
                }
                if (tile_count > 0) await(kResultDone, (uint32_t)(tile_count - 1) & 1u);  // the weights are free, and the results the warp's
                if (__any_sync(0xFFFFFFFFu, !(top - m <= kSlack + kShift))) {
                    const float higher = larger(m, top - kShift), keep = exp2_of(m - higher);
                    m = higher;
                    l *= keep;
                    if (i > 0) {
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
                        for (int chunk = 0; chunk < DIM / 32; ++chunk) {
                            uint32_t r[32];
                            tmem_ld32(lanes + L::kResult + chunk * 32, r);
#pragma unroll
                            for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * keep);
                            tmem_st32(lanes + L::kResult + chunk * 32, r);
                        }
                    }
                }
#pragma unroll 1
                for (int chunk = 0; chunk < 4; ++chunk) {
                    uint32_t s[32], w[16];
                    scores(chunk, s);
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        const float4 z = *reinterpret_cast<const float4*>(value_step + chunk * 32 + j);
                        float x[4], v[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            x[k] = exp2_of(__uint_as_float(s[j + k]) - m);
                            l += x[k];
                        }
                        v[0] = x[0] * z.x; v[1] = x[1] * z.y; v[2] = x[2] * z.z; v[3] = x[3] * z.w;
                        if (!all_seen) {
#pragma unroll
                            for (int k = 0; k < 4; ++k) v[k] = x[k] == 0.0f ? 0.0f : v[k];  // whatever stands in a place that is not seen
                        }
                        w[j / 2] = half_pair(v[0], v[1]);
                        w[j / 2 + 1] = half_pair(v[2], v[3]);
                    }
                    const uint32_t panel = base + L::kWeights + chunk / 2 * L::kPanel;
#pragma unroll
                    for (int k = 0; k < 4; ++k) store16(panel + element(tid, chunk % 2 * 4 + k), w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                seen_by_products();
                arrive(kWeightsFull);
                if (lane == 0) {
                    mbar_arrive(bar(kScoresEmpty + stage));
                    mbar_arrive(bar(kValuesEmpty + stage));
                }
            }
            // the row's result
            await(kResultDone, (uint32_t)(tile_count - 1) & 1u);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const bool whole = place.tile == 0 && n == place.tiles, failed = *lost != 0;
            if (failed) l = __uint_as_float(0x7FC00000u);
            const float part_of = m == kNothing && !failed ? 0.0f : 1.0f / l;
            float* partial = a.partials + ((int64_t)blockIdx.x * 2 + (place.tile > 0 ? 0 : 1)) * kPart;
            const int64_t result = real ? result_row(a, place, kRows, tid) * DIM : 0;
#pragma unroll 1
            for (int chunk = 0; chunk < DIM / 32; ++chunk) {
                uint32_t r[32];
                tmem_ld32(lanes + L::kResult + chunk * 32, r);
                if (real) {
#pragma unroll
                    for (int b = 0; b < 32; b += 8) {  // columns of a block: values 0 4 1 5 2 6 3 7
                        float v[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) v[(k & 1) * 4 + k / 2] = __uint_as_float(r[b + k]);
                        if (whole) {
                            uint32_t o[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k) o[k] = pack_bf16x2(v[2 * k] * part_of, v[2 * k + 1] * part_of);
                            *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + result + chunk * 32 + b) = make_uint4(o[0], o[1], o[2], o[3]);
                        } else {
                            float4* dst = reinterpret_cast<float4*>(partial + 2 * kRows + tid * DIM + chunk * 32 + b);
                            dst[0] = make_float4(v[0], v[1], v[2], v[3]);
                            dst[1] = make_float4(v[4], v[5], v[6], v[7]);
                        }
                    }
                }
                __syncwarp();
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            if (real) {
                if (whole) {
                    put_lse(a, place, kRows, tid, failed ? l : m, l);
                } else {
                    partial[tid] = failed ? l : m;
                    partial[kRows + tid] = l;
                }
            }
            const Place done = place;
            at_unit += n;
            if (done.tile + n == done.tiles) at_unit += kSegment;
            const bool more = at_unit < to;
            if (more) next_segment<kRows, kTile>(a, place);
            if (!whole) {
                asm volatile("bar.sync 1, %0;" ::"n"(32 * kSoftmaxWarps) : "memory");  // the part is written
                if (tid == 0)
                    arrived[n_pending] = count_part(a, pending[n_pending], done, part.cut, at_unit - (done.tile + n == done.tiles ? kSegment : 0) - n - done.tile);
                ++n_pending;
            }
            if (!more) break;
        }
    } else if (warp < kProductWarp) {
        // ---- decoding: thread t has 16-byte chunk t % kChunks of rows t / kChunks and, of 128 values, that and 64
        constexpr int kMine = kTile * kChunks / (32 * kDecodeWarps);
        const int t = tid - 32 * kSoftmaxWarps, chunk = t % kChunks;
        const int page_log2 = a.pages.page_log2, page_mask = (1 << page_log2) - 1;
        int tile_count = 0;
        struct Codes {
            uint4 x[2][kMine];
            uint32_t head[2][kMine];
        };
        // pages of a tile's rows; -1 behind the end
        int page[kMine];
        const auto look_up = [&](const Place& p, int tile) {
#pragma unroll
            for (int i = 0; i < kMine; ++i) page[i] = page_of(a, p.seq, tile * kTile + t / kChunks + i * (kTile / kMine), p.s.len);
        };
        const auto load = [&](const Place& p, int tile, Codes& c) {
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                const int at = (tile * kTile + t / kChunks + i * (kTile / kMine)) & page_mask;
                const uint32_t* rec = a.pages.words + record<DIM>(a.pages, max(page[i], 0), p.head);
#pragma unroll
                for (int which = 0; which < 2; ++which) {
                    c.x[which][i] = make_uint4(0, 0, 0, 0);
                    c.head[which][i] = 0;
                    if (page[i] >= 0) {
                        c.x[which][i] = __ldg(reinterpret_cast<const uint4*>(rec + ((which << page_log2) + at) * code_words(DIM)) + chunk);
                        c.head[which][i] = __ldg(rec + ((2 * code_words(DIM) + which) << page_log2) + at);
                    }
                }
            }
        };
        const auto put = [&](uint32_t to_operand, const uint4 (&x)[kMine], const uint32_t (&head)[kMine]) {
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
                const int row = t / kChunks + i * (kTile / kMine);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int word = chunk * 4 + k;
                    const uint32_t exponent = 0x60006000u | (head[i] >> word & 1) * 0x00010001u;
                    uint32_t o[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        asm("add.rn.f16x2 %0, %1, %2;" : "=r"(o[j]) : "r"(chosen(j == 0 ? w[k] << 1 : w[k] >> (4 * j - 1), 0x001E001Eu, exponent)), "r"(0xE010E010u));
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
        Codes codes;
        bool have = true;
        look_up(ahead, ahead_tile);
        load(ahead, ahead_tile, codes);
        while (have) {
            const int stage = tile_count & 1;
            const uint32_t parity = (uint32_t)((tile_count >> 1) - 1) & 1u;
            bool there[kMine];
#pragma unroll
            for (int i = 0; i < kMine; ++i) there[i] = page[i] >= 0;
            step();
            have = ahead_unit < to;
            if (have) look_up(ahead, ahead_tile);
            if (tile_count >= 2) await(kKeysEmpty + stage, parity);
            put(base + L::kKeys + stage * L::kOperand, codes.x[0], codes.head[0]);
            arrive(kKeysFull + stage);
            if (tile_count >= 2) await(kValuesEmpty + stage, parity);
            if (chunk == 0) {
                float* steps = reinterpret_cast<float*>(smem + L::kSteps) + stage * 3 * kTile;
#pragma unroll
                for (int i = 0; i < kMine; ++i) {
                    const int row = t / kChunks + i * (kTile / kMine);
                    steps[row] = __uint_as_float(codes.head[0][i] & 0xFFFF0000u);
                    steps[kTile + row] = __uint_as_float(codes.head[1][i] & 0xFFFF0000u);
                    steps[2 * kTile + row] = there[i] ? size_of(codes.head[1][i]) : -INFINITY;
                }
            }
            put(base + L::kValues + stage * L::kOperand, codes.x[1], codes.head[1]);
            arrive(kValuesFull + stage);
            if (have) load(ahead, ahead_tile, codes);
            ++tile_count;
        }
    } else {
        // ---- products: S of a tile, then O of the one before
        constexpr uint32_t kScoresDesc = (1u << 4) | ((uint32_t)(kTile >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
        constexpr uint32_t kResultDesc = (1u << 4) | (1u << 16) | ((uint32_t)(DIM >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
        const uint64_t k_major = umma_desc(base);
        // MN-major: blocks of 64 values lie a panel apart
        const uint32_t high = (uint32_t)(k_major >> 32), queries = (uint32_t)k_major, weights = queries + (L::kWeights >> 4);
        const uint32_t keys = queries + (L::kKeys >> 4), values = ((queries & 0xFFFFu) | ((uint32_t)(L::kPanel >> 4) << 16)) + (L::kValues >> 4);
        int tile_count = 0, segment = 0;
        while (true) {
            const int n = min(place.tiles - place.tile, to - at_unit);
            await(kQueriesFull, (uint32_t)segment & 1u);
            for (int i = 0; i <= n; ++i) {
                if (i < n) {
                    const int count = tile_count + i, stage = count & 1;
                    await(kKeysFull + stage, (uint32_t)(count >> 1) & 1u);
                    if (count >= 2) await(kScoresEmpty + stage, (uint32_t)((count >> 1) - 1) & 1u);
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < DIM / 16; ++k)
                            umma_f16(tmem + stage * kTile, make_desc(queries + k / 4 * (L::kPanel >> 4) + k % 4 * 2, high),
                                     make_desc(keys + stage * (L::kOperand >> 4) + k / 4 * (L::kPanel >> 4) + k % 4 * 2, high), kScoresDesc, k > 0);
                        umma_commit(bar(kScoresFull + stage));
                        umma_commit(bar(kKeysEmpty + stage));
                    }
                    __syncwarp();
                }
                if (i > 0) {
                    const int count = tile_count + i - 1, stage = count & 1;
                    await(kValuesFull + stage, (uint32_t)(count >> 1) & 1u);
                    await(kWeightsFull, (uint32_t)count & 1u);
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < kTile / 16; ++k)  // 16 tokens: two groups of eight lines of a panel
                            umma_f16(tmem + L::kResult, make_desc(weights + k / 4 * (L::kPanel >> 4) + k % 4 * 2, high),
                                     make_desc(values + stage * (L::kOperand >> 4) + k * 128, high), kResultDesc, i > 1 || k > 0);
                        umma_commit(bar(kResultDone));
                        umma_commit(bar(kValuesEmpty + stage));
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
    if (n_pending > 0) join_ctas<true, DIM, kRows>(a, pending, n_pending, arrived, kThreads);
}

template <int DIM>
int launch_as(const Attend& a, cudaStream_t st) {
    static_assert(Layout<DIM>::kBytes <= 227 * 1024, "shared memory");
    const auto kernel = k_cache_attend_many<DIM>;
    if (int e = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<DIM>::kBytes), "cudaFuncSetAttribute")) return e;
    const int sms = sm_count(), grid = sms < kManyCtas ? sms : kManyCtas;
    return launch_dependent("e8_cache_attention", kernel, (unsigned)grid, kThreads, Layout<DIM>::kBytes, st, a);
}

}  // namespace

namespace coset {
namespace cache {

int launch_many(const Attend& a, int head_dim, cudaStream_t stream) { return head_dim == 64 ? launch_as<64>(a, stream) : launch_as<128>(a, stream); }

}  // namespace cache
}  // namespace coset
