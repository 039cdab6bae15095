// Products of microscaled rows (see microscaled.cuh) on the fifth-generation tensor cores:
//     Y[token, n] = sum_k X[token, k] W[n, k]      X: [tokens, K] in 8 bits (e4m3) or 4 (e2m1), W: [N, K] in 4 bits (e2m1)
// both with a power of two per 32 columns, which the instruction multiplies in (tcgen05.mma with block scales: kind::mxf8f6f4 for rows of 8 bits,
// kind::mxf4, twice its rate, for rows of 4).  Sums are of 32 bits.  As in the bfloat16 products D = W X^T: rows of W are the accumulator's 128 lanes,
// tokens its columns.
//
// A stage of the ring holds 128 bytes of every row: 128 columns of X in 8 bits, or 256 in 4.  Beside rows of 8 bits the 4-bit elements of W are
// spread by the copy itself to 16 of them in 16 bytes (8 with elements, 8 empty), the form that products of mixed types read, so that W crosses L2
// in 4 bits.  Scales come as they lie: a tile of 512 bytes for 128 rows and 128 columns, copied on to four columns of tensor memory (tcgen05.cp),
// which the products behind it read; all three are issued by one thread and keep their order.
//
// Gated: 64 rows of `up` and the same 64 of `gate` are the lanes of one accumulator, and the epilogue brings up * act(gate) into 8 bits again.  The
// scales of half a tile of each are put together by a warp of their own (what the bulk copy moves is 16 bytes at least, half a row's scales are 8).
#include "microscaled.cuh"
#include "tcgen05.cuh"

namespace lb {

constexpr int kMsRows = 128;   // lanes of an accumulator
constexpr int kMsMostRows = 0x7fffff00;   // of either operand: places are counted in whole tiles

struct MsParams {
    const unsigned char *w_scales, *gate_scales, *x_scales;
    void* out;                  // [tokens, n] bfloat16 or float32; gated: codes [tokens, out_chunks * 128]
    unsigned char* out_scales;  // gated
    int tokens, n;              // n: rows of W (gated: of each of the two)
    int chunks;                 // K in 128s
    int out_chunks;             // gated: the output's width in 128s
    int out_is_float, bulk_store;
    int activation;
    float limit;
    int row_tiles, token_tiles, wide_tiles;   // of the tokens' tiles the first wide_tiles have kMsWide, the others kMsNarrow
    int* status;
};

__device__ __forceinline__ void bulk_load(void* destination, const void* source, uint32_t bytes, uint64_t* barrier) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_address(destination)), "l"(source), "r"(bytes),
                 "r"(smem_address(barrier))
                 : "memory");
}

// True in one lane of the warp.  The copying and the issuing warp walk their loops as a whole, and an elected lane issues: inside a branch on the
// lane's number the same instructions took 55 cycles each, which bounded a stage of the ring at 500.
// (The same lane is elected every time, so that products keep their order and a commit counts them.)
__device__ __forceinline__ bool elect_lane() {
    uint32_t elected;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(elected));
    return elected != 0u;
}

// A whole warp waits, and its lanes go on together or not at all.  (Where one lane waited for the others, what the warp issues afterwards took twice as long.)
// CLUSTER: sees what another CTA did before it arrived.
template <bool CLUSTER = false>
__device__ __forceinline__ bool barrier_wait_warp(uint64_t* barrier, uint32_t parity) {
    if constexpr (!CLUSTER) return __all_sync(0xffffffffu, barrier_wait_parked(barrier, parity));
    bool waited = false;
    const unsigned long long start = nanoseconds_now();
    for (;;) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(smem_address(barrier)), "r"(parity), "r"(100000u)
            : "memory");
        waited = done != 0u;
        if (waited || nanoseconds_now() - start > kTcWaitNanoseconds) break;
    }
    return __all_sync(0xffffffffu, waited);
}

// A tile of scales, 32 rows of 16 bytes one behind the other (groups of 8 rows 128 bytes apart, no swizzle), for tcgen05.cp.
__device__ __forceinline__ uint64_t scale_descriptor(const void* tile) {
    const uint64_t address = smem_address(tile);
    return ((address & 0x3FFFFull) >> 4) | (static_cast<uint64_t>(128 >> 4) << 32) | (1ull << 46);
}
// To four columns of tensor memory, the same in each quarter of the lanes.  PAIR: each CTA of the pair from its own shared memory, at the same place.
template <bool PAIR>
__device__ __forceinline__ void copy_scales(uint32_t tmem, const void* tile) {
    if constexpr (PAIR) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(scale_descriptor(tile)) : "memory");
    else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(scale_descriptor(tile)) : "memory");
}

// D float32 [128, N] (+)= A [128, 32] e2m1 (spread) B [N, 32] e4m3, or A [128, 64] e2m1 B [N, 64] e2m1, each block of 32 times its two scales.  PAIR: [256, N] over two
// CTAs, each with 128 rows of A and of D, half of the rows of B, its rows' scales and all of the tokens'.
#define LB_MMA_MICROSCALED(group, kind, scales)                                                                                                    \
    asm volatile(                                                                                                                                  \
        "{\n\t.reg .pred p;\n\t"                                                                                                                  \
        "setp.ne.b32 p, %4, 0;\n\t"                                                                                                               \
        "tcgen05.mma.cta_group::" group ".kind::" kind ".block_scale.scale_vec::" scales " [%0], %1, %2, %3, [%5], [%6], p;\n\t}"                 \
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate ? 1u : 0u), "r"(scales_a), "r"(scales_b)                                \
        : "memory")
template <int BITS, bool PAIR>
__device__ __forceinline__ void mma_microscaled(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t scales_a, uint32_t scales_b, bool accumulate) {
    static_assert(!PAIR || BITS == 8, "what pairs take");
    if constexpr (PAIR) LB_MMA_MICROSCALED("2", "mxf8f6f4", "1X");
    else if constexpr (BITS == 8) LB_MMA_MICROSCALED("1", "mxf8f6f4", "1X");
    else LB_MMA_MICROSCALED("1", "mxf4", "2X");
}
#undef LB_MMA_MICROSCALED

// The instruction's description: A (W) e2m1, B (X) e4m3 or e2m1, scales e8m0, N columns, 128 lanes (a pair's 256); the bytes of the scales' words follow per product.
template <int BITS>
__device__ __forceinline__ uint32_t microscaled_descriptor(int columns, int lanes = kMsRows) {
    const uint32_t types = BITS == 8 ? (5u << 7) | (0u << 10) : (1u << 7) | (1u << 10);
    return types | (static_cast<uint32_t>(columns >> 3) << 17) | (1u << 23) | (static_cast<uint32_t>(lanes >> 4) << 24);
}
// Product `k` of the four of a stage takes the scales from this chunk of the stage, and from this byte on of its words.
template <int BITS>
__device__ __forceinline__ int product_chunk(int k) { return BITS == 8 ? 0 : k >> 1; }
template <int BITS>
__device__ __forceinline__ uint32_t product_scales(int k) {
    const uint32_t byte = BITS == 8 ? static_cast<uint32_t>(k) : static_cast<uint32_t>(k & 1) * 2u;
    return (byte << 4) | (byte << 29);
}

// BN: tokens of a tile, of which a CTA loads OWN.  A tile of more than 128 begins at a multiple of 64, so that two tiles of scales cover it.
template <int BITS, int BN, int OWN = BN>
struct MsShape {
    static constexpr int kChunks = BITS == 8 ? 1 : 2;             // of 128 columns, a stage
    static constexpr int kScaleTiles = BN > 128 ? 2 : 1;          // of 128 tokens, that a tile's tokens lie in
    static constexpr int kWBytes = kMsRows * 128;
    static constexpr int kXBytes = OWN * 128;
    static constexpr int kWScaleBytes = kChunks * kScaleTileBytes;
    static constexpr int kXScaleBytes = kScaleTiles * kChunks * kScaleTileBytes;
    static constexpr int kStageBytes = (kWBytes + kXBytes + kWScaleBytes + kXScaleBytes + 1023) / 1024 * 1024;   // tiles start on 1024 bytes
    // what the copy of a tile of W counts on its barrier: the bytes it has read
    static constexpr uint32_t kWCounted = BITS == 8 ? kWBytes / 2 : kWBytes;
};

// A landed stage's scales to a set of columns of tensor memory.  The whole warp comes here, and a lane is elected for every instruction (gated 8192 x 2048 from L2, 8 tokens:
// 6.5 us, and 7.1 with one lane for all of a stage, both before the clusters' last meeting ordered the reads); for a pair one lane comes, elected for all of them (4,096 tokens, 2048 x 8192: 61 us, and 96 with one each).
template <typename Shape, bool PAIR>
__device__ __forceinline__ void copy_stage_scales(const unsigned char* stage, uint32_t columns, int chunks) {
    const unsigned char* scales = stage + Shape::kWBytes + Shape::kXBytes;
#pragma unroll
    for (int c = 0; c < Shape::kChunks; ++c) {
        if (c >= chunks) break;
        if (PAIR || elect_lane()) copy_scales<PAIR>(columns + 4 * c, scales + c * kScaleTileBytes);
#pragma unroll
        for (int t = 0; t < Shape::kScaleTiles; ++t)
            if (PAIR || elect_lane())
                copy_scales<PAIR>(columns + 4 * (Shape::kChunks + c * Shape::kScaleTiles + t), scales + Shape::kWScaleBytes + (t * Shape::kChunks + c) * kScaleTileBytes);
    }
}
// Its four products under them, and the stage's return to the producer(s), likewise.
template <int BITS, typename Shape, bool PAIR>
__device__ __forceinline__ void issue_stage(uint32_t tmem_d, const unsigned char* stage, uint32_t columns, uint32_t token_column, uint32_t idesc, int chunks, bool accumulate,
                                            uint64_t* empty) {
    const uint64_t desc_w = tile_descriptor(stage), desc_x = tile_descriptor(stage + Shape::kWBytes);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int c = product_chunk<BITS>(k);
        if (c >= chunks) break;
        if (PAIR || elect_lane())
            mma_microscaled<BITS, PAIR>(tmem_d, desc_w + 2 * k, desc_x + 2 * k, idesc | product_scales<BITS>(k), columns + 4 * c,
                                        columns + 4 * (Shape::kChunks + c * Shape::kScaleTiles) + token_column, accumulate || k > 0);
    }
    if (PAIR || elect_lane()) {
        if constexpr (PAIR) mma_commit_pair(empty);
        else mma_commit(empty);
    }
}

constexpr int kMsWide = 192, kMsNarrow = 128;   // tokens of the walking kernel's tiles, which begin at multiples of 64
constexpr int kMsThreads = 20 * 32;             // producer, issuer, scales of a gated product, one idle; sixteen warps of the epilogue
constexpr int kMsGroup = 16;                    // tokens that four warps of the epilogue take at a time
constexpr int kMsTurnedPitch = kMsRows + 4;     // floats: the 16 bytes of eight lanes and of the next token's lie in different banks
constexpr int kMsTurnedBytes = kMsGroup * kMsTurnedPitch * 4;
constexpr int kMsRegionBytes = 11 * 1024;       // per four warps: gated, 16 tokens turned over and two output buffers; else two output buffers of bfloat16, or one of float32
static_assert(kMsRegionBytes >= kMsTurnedBytes + 2 * kMsGroup * 64 && kMsRegionBytes >= kMsGroup * kMsRows * 4, "room for either");
constexpr int kMsSharedLimit = 227 * 1024;

template <int BITS, bool PAIR>
struct MsWalk {
    static constexpr int BN = kMsWide;
    using Shape = MsShape<BITS, BN, PAIR ? BN / 2 : BN>;
    static constexpr int kStages = (kMsSharedLimit - 4 * kMsRegionBytes - 1024 - 256) / Shape::kStageBytes;
    static constexpr int kBytes = kStages * Shape::kStageBytes + 4 * kMsRegionBytes + 1024 + 256;
    static constexpr int kScaleSet = 4 * Shape::kChunks * (1 + Shape::kScaleTiles);
    static constexpr int kScaleColumns = (PAIR ? 2 : 1) * kScaleSet;
    static constexpr int kColumns = 512;
    static_assert(kStages >= 3 && kStages <= 12 && 2 * BN + kScaleColumns <= kColumns, "a ring, its barriers, two accumulators and the scales");
};

// One CTA per multiprocessor walks the tiles of 128 lanes x 192 or 128 tokens, rows fastest, with two accumulators: the epilogue of a tile runs while the
// products of the next are issued.  PAIR: the walkers are pairs of CTAs that share a tile of 256 lanes; each loads its rows of W, half of the tokens and all
// of their scales, all bytes count on the even CTA's barriers, and that one issues products over both CTAs' shared and tensor memory.  (Not for gated products,
// whose scales would have to be announced across the pair, nor rows of 4 bits: 4096 x 8192 x 2048 40.3 us and 38.0 without.)
template <int BITS, bool GATED, bool PAIR>
__global__ void __launch_bounds__(kMsThreads)
gemm_microscaled_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_gate, const __grid_constant__ CUtensorMap map_x,
                        const __grid_constant__ CUtensorMap map_x_narrow, const __grid_constant__ CUtensorMap map_w_scales, const __grid_constant__ CUtensorMap map_x_scales, const __grid_constant__ CUtensorMap map_out,
                        const MsParams p) {
    static_assert(!PAIR || (BITS == 8 && !GATED), "what pairs take");
    using Walk = MsWalk<BITS, PAIR>;
    using Shape = typename Walk::Shape;
    constexpr int STAGES = Walk::kStages, BN = Walk::BN;
    constexpr int kPairs = PAIR ? 2 : 1;   // CTAs of a walker
    const int rank = PAIR ? static_cast<int>(cluster_rank()) : 0;
    const int walker = static_cast<int>(blockIdx.x) / kPairs, walkers = static_cast<int>(gridDim.x) / kPairs;
    extern __shared__ unsigned char raw_shared[];
    unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw_shared) + 1023) & ~static_cast<uintptr_t>(1023));
    unsigned char* regions = ring + STAGES * Shape::kStageBytes;
    uint64_t* barriers = reinterpret_cast<uint64_t*>(regions + 4 * kMsRegionBytes);
    uint64_t* full = barriers;
    uint64_t* empty = barriers + STAGES;
    uint64_t* tmem_full = barriers + 2 * STAGES;
    uint64_t* tmem_empty = barriers + 2 * STAGES + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(barriers + 2 * STAGES + 4);
    __shared__ int failed;

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    constexpr int kRowsPerCta = GATED ? kMsRows / 2 : kMsRows;
    const int num_stages = (p.chunks + Shape::kChunks - 1) / Shape::kChunks;
    const int num_tiles = p.row_tiles * p.token_tiles;
    auto chunks_of = [&](int stage) { return min(Shape::kChunks, p.chunks - stage * Shape::kChunks); };
    auto row_of = [&](int tile) { return ((tile % p.row_tiles) * kPairs + rank) * kRowsPerCta; };   // this CTA's first
    auto is_wide = [&](int tile) { return tile / p.row_tiles < p.wide_tiles; };
    auto token_of = [&](int tile) {
        const int index = tile / p.row_tiles;
        return index * kMsNarrow + min(index, p.wide_tiles) * (kMsWide - kMsNarrow);
    };
    // The tokens that a tile's products take: the last tile's only as many as there are, in whole 16s of each CTA.
    auto columns_of = [&](int tile) { return min(is_wide(tile) ? kMsWide : kMsNarrow, (p.tokens - token_of(tile) + 16 * kPairs - 1) / (16 * kPairs) * (16 * kPairs)); };

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            barrier_init(&full[s], GATED ? 2 : 1);   // the producer, and the warp that puts the scales together
            barrier_init(&empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            barrier_init(&tmem_full[a], 1);
            barrier_init(&tmem_empty[a], 16 * kPairs);
        }
        failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_address(tmem_slot)), "r"(Walk::kColumns) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_address(tmem_slot)), "r"(Walk::kColumns) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if constexpr (PAIR) cluster_sync();   // the partner's barriers exist before anything arrives on them
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = *tmem_slot;
    const uint32_t tmem_scales = tmem_base + 2 * BN;
    // Everything that is read may come from the kernel before this one, the weights too (quantised just now).
    wait_for_previous_kernel();
    allow_next_kernel();

    if (warp == 0) {
        int s = 0, round = 0;
        bool ok = true;
        for (int tile = walker; tile < num_tiles && ok; tile += walkers) {
            const int row0 = row_of(tile), token0 = token_of(tile), own_token0 = token0 + rank * (columns_of(tile) / 2);
            const bool wide = is_wide(tile);
            const uint32_t x_bytes = static_cast<uint32_t>((wide ? kMsWide : kMsNarrow) / kPairs * 128);
            for (int stage = 0; stage < num_stages; ++stage) {
                ok = round == 0 || barrier_wait_warp<PAIR>(&empty[s], (round - 1) & 1);
                if (!ok) {
                    atomicExch(&failed, 1);
                    break;
                }
                if (elect_lane()) {
                    unsigned char* at = ring + s * Shape::kStageBytes;
                    const int column = stage * 128;   // of the map: elements of W where they are spread and of X in 8 bits, bytes of rows in 4
                    const int word = stage * Shape::kChunks * (kScaleTileBytes / 4);
                    if (rank == 0) barrier_expect(&full[s], kPairs * (Shape::kWCounted + x_bytes + (GATED ? 0 : Shape::kWScaleBytes) + Shape::kXScaleBytes));
                    auto load = [&](void* to, const CUtensorMap* map, int x, int y) {
                        if constexpr (PAIR) tma_load_2d_pair(to, map, x, y, cluster_address(&full[s], 0));
                        else tma_load_2d(to, map, x, y, &full[s]);
                    };
                    load(at, &map_w, column, row0);
                    if constexpr (GATED) load(at + Shape::kWBytes / 2, &map_gate, column, row0);
                    load(at + Shape::kWBytes, wide ? &map_x : &map_x_narrow, column, own_token0);
                    at += Shape::kWBytes + Shape::kXBytes;
                    if constexpr (!GATED) load(at, &map_w_scales, word, row0 / 128);
                    load(at + Shape::kWScaleBytes, &map_x_scales, word, token0 / 128);
                }
                if (++s == STAGES) s = 0, ++round;
            }
        }
    } else if (warp == 1) {
        int s = 0, round = 0, local = 0, left = (num_tiles - walker + walkers - 1) / walkers * num_stages;
        uint32_t set = 0u;
        bool ok = rank == 0, copied = false;
        for (int tile = walker; tile < num_tiles && ok; tile += walkers, ++local) {
            const int accumulator = local & 1, use = local >> 1;
            ok = use == 0 || barrier_wait_warp<PAIR>(&tmem_empty[accumulator], (use - 1) & 1);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t tmem_d = tmem_base + static_cast<uint32_t>(accumulator * BN);
            const uint32_t idesc = microscaled_descriptor<BITS>(columns_of(tile), kPairs * kMsRows);
            const uint32_t token_column = static_cast<uint32_t>((token_of(tile) & 127) >> 5);   // of the scales: 32 tokens a column
            for (int stage = 0; stage < num_stages && ok; ++stage) {
                const unsigned char* at = ring + s * Shape::kStageBytes;
                if constexpr (!PAIR) {
                    ok = barrier_wait_warp(&full[s], round & 1);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    copy_stage_scales<Shape, false>(at, tmem_scales, chunks_of(stage));
                    issue_stage<BITS, Shape, false>(tmem_d, at, tmem_scales, token_column, idesc, chunks_of(stage), stage > 0, &empty[s]);
                    if (++s == STAGES) s = 0, ++round;
                } else {
                    // A pair's scales of the stage after go out before this stage's products if that stage is there (4096 tokens x 2048 x 8192: 60.8 us, and 65.4 with
                    // copies just before their products; a CTA by itself does not gain by it, 69.1 and 68.4).
                    const uint32_t columns = tmem_scales + set * Walk::kScaleSet;
                    if (!copied) {
                        ok = barrier_wait_warp<true>(&full[s], round & 1);
                        if (!ok) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        if (elect_lane()) copy_stage_scales<Shape, true>(at, columns, chunks_of(stage));
                    }
                    const int next = s + 1 == STAGES ? 0 : s + 1, next_round = s + 1 == STAGES ? round + 1 : round;
                    copied = --left > 0 && __all_sync(0xffffffffu, barrier_test(&full[next], next_round & 1));
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    if (elect_lane()) {
                        if (copied)
                            copy_stage_scales<Shape, true>(ring + next * Shape::kStageBytes, tmem_scales + (set ^ 1u) * Walk::kScaleSet, chunks_of(stage + 1 == num_stages ? 0 : stage + 1));
                        issue_stage<BITS, Shape, true>(tmem_d, at, columns, token_column, idesc, chunks_of(stage), stage > 0, &empty[s]);
                    }
                    s = next, round = next_round, set ^= 1u;
                }
            }
            if (!ok) {
                atomicExch(&failed, 1);
            } else if (elect_lane()) {
                if constexpr (PAIR) mma_commit_pair(&tmem_full[accumulator]);
                else mma_commit(&tmem_full[accumulator]);
            }
        }
    } else if (GATED && warp == 2) {
        // Lane l puts together the 16 bytes of the rows l, l + 32 of `up` and of `gate` in the accumulator's order.  Four stages are read at once: a
        // read from L2 takes about as long as the products of two.
        int s = 0, round = 0;
        bool ok = true;
        for (int tile = walker; tile < num_tiles && ok; tile += walkers) {
            const int row0 = row_of(tile);
            const size_t offset = static_cast<size_t>(row0 / 128) * p.chunks * kScaleTileBytes + lane * 16 + ((row0 & 64) >> 3);
            for (int first = 0; first < num_stages && ok; first += 4) {
                uint2 up[4][Shape::kChunks], gate[4][Shape::kChunks];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
#pragma unroll
                    for (int c = 0; c < Shape::kChunks; ++c) {
                        const int chunk = (first + i) * Shape::kChunks + c;
                        up[i][c] = gate[i][c] = make_uint2(0u, 0u);
                        if (chunk < p.chunks) {
                            up[i][c] = *reinterpret_cast<const uint2*>(p.w_scales + offset + static_cast<size_t>(chunk) * kScaleTileBytes);
                            gate[i][c] = *reinterpret_cast<const uint2*>(p.gate_scales + offset + static_cast<size_t>(chunk) * kScaleTileBytes);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (first + i >= num_stages) break;
                    ok = round == 0 || barrier_wait_warp(&empty[s], (round - 1) & 1);
                    if (!ok) {
                        atomicExch(&failed, 1);
                        break;
                    }
                    unsigned char* at = ring + s * Shape::kStageBytes + Shape::kWBytes + Shape::kXBytes + lane * 16;
#pragma unroll
                    for (int c = 0; c < Shape::kChunks; ++c)
                        *reinterpret_cast<uint4*>(at + c * kScaleTileBytes) = make_uint4(up[i][c].x, up[i][c].y, gate[i][c].x, gate[i][c].y);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) barrier_arrive(&full[s]);
                    if (++s == STAGES) s = 0, ++round;
                }
            }
        }
    } else if (warp >= 4) {
        // Sixteen warps in four sets: warp & 3 is the quarter of the lanes that a warp may read, and the sets take 16 tokens at a time in turn.
        const int quarter = warp & 3, set = (warp - 4) >> 2, set_barrier = 1 + set;
        const bool issuer = quarter == 0 && lane == 0;
        unsigned char* region = regions + set * kMsRegionBytes;
        int local = 0, groups = 0;
        for (int tile = walker; tile < num_tiles; tile += walkers, ++local) {
            const int accumulator = local & 1, use = local >> 1;
            const int row0 = row_of(tile), token0 = token_of(tile);
            uint32_t arrived = barrier_wait_warp<PAIR>(&tmem_full[accumulator], use & 1) ? 1u : 0u;
            {
                // Warps that meet at named barriers below go on together or not at all.
                uint32_t all;
                asm volatile(
                    "{\n"
                    ".reg .pred mine, all;\n"
                    "setp.ne.u32 mine, %1, 0;\n"
                    "bar.red.and.pred all, %2, 128, mine;\n"
                    "selp.u32 %0, 1, 0, all;\n"
                    "}\n"
                    : "=r"(all)
                    : "r"(arrived), "r"(set_barrier)
                    : "memory");
                arrived = all;
            }
            if (!arrived) {
                atomicExch(&failed, 1);
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t tmem_d = tmem_base + static_cast<uint32_t>(accumulator * BN) + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll 1
            for (int column = set * kMsGroup; column < (is_wide(tile) ? kMsWide : kMsNarrow); column += 4 * kMsGroup, ++groups) {
                const int first_token = token0 + column;
                if (first_token >= p.tokens) break;   // the same for the whole set
                uint32_t v[kMsGroup];
                tmem_load_16(tmem_d + static_cast<uint32_t>(column), v);
                if constexpr (GATED) {
                    // Lanes 0 to 63 hold `up` and lanes 64 to 127 the same rows of `gate`: turned over in shared memory, so that a thread has eight
                    // channels of a token (four of every 32) and eight threads its 64.
                    float* turned = reinterpret_cast<float*>(region);
                    unsigned char* out_buffer = region + kMsTurnedBytes + (groups & 1) * (kMsGroup * 64);
#pragma unroll
                    for (int i = 0; i < kMsGroup; ++i) turned[i * kMsTurnedPitch + quarter * 32 + lane] = __uint_as_float(v[i]);
                    if (issuer) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");   // the store before last has read this buffer
                    named_barrier(set_barrier, 128);
                    const int token_here = quarter * 4 + (lane >> 3), part = lane & 7;
                    float up[8], gate[8], h[8];   // four of each of the two blocks
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const float* from = turned + token_here * kMsTurnedPitch + b * 32 + part * 4;
                        const float4 u = *reinterpret_cast<const float4*>(from), g = *reinterpret_cast<const float4*>(from + kMsRows / 2);
                        up[4 * b] = u.x, up[4 * b + 1] = u.y, up[4 * b + 2] = u.z, up[4 * b + 3] = u.w;
                        gate[4 * b] = g.x, gate[4 * b + 1] = g.y, gate[4 * b + 2] = g.z, gate[4 * b + 3] = g.w;
                    }
                    gated_values(up, gate, p.activation, p.limit, h);
                    if (row0 + kMsRows / 2 > p.n) {   // past the last row: zeros, whatever the scales there
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (row0 + (i >> 2) * 32 + part * 4 + (i & 3) >= p.n) h[i] = 0.0f;
                    }
                    float largest[2];
                    int byte[2];
#pragma unroll
                    for (int b = 0; b < 2; ++b) largest[b] = larger_size(larger_size(h[4 * b], h[4 * b + 1]), larger_size(h[4 * b + 2], h[4 * b + 3]));
#pragma unroll
                    for (int offset = 1; offset < 8; offset <<= 1) {
#pragma unroll
                        for (int b = 0; b < 2; ++b) largest[b] = larger_size(largest[b], __shfl_xor_sync(0xffffffffu, largest[b], offset));
                    }
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        byte[b] = scale_byte<8>(__float_as_uint(largest[b]) & 0x7fffffffu);
                        const float inverse = scale_inverse(byte[b]);
                        *reinterpret_cast<uint32_t*>(out_buffer + token_here * 64 + b * 32 + part * 4) =
                            pack_e4m3(h[4 * b] * inverse, h[4 * b + 1] * inverse, h[4 * b + 2] * inverse, h[4 * b + 3] * inverse);
                    }
                    const int token = first_token + token_here, block = row0 / 32;   // an even one
                    if (part == 0 && token < p.tokens)
                        *reinterpret_cast<uint16_t*>(p.out_scales + scale_word(token, block >> 2, p.out_chunks) + (block & 3)) = static_cast<uint16_t>(byte[0] | byte[1] << 8);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    named_barrier(set_barrier, 128);
                    if (issuer) bulk_store_2d(&map_out, out_buffer, row0, first_token, false);
                } else if (p.bulk_store) {
                    // Stores issued by the threads themselves queue behind the loads of the stages.  One buffer of float32, or two of bfloat16.
                    unsigned char* out_buffer = region + (p.out_is_float ? 0 : (groups & 1) * (kMsGroup * kMsRows * 2));
                    if (issuer) {
                        if (p.out_is_float) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                        else asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
                    }
                    named_barrier(set_barrier, 128);
                    if (p.out_is_float) {
                        float* to = reinterpret_cast<float*>(out_buffer) + quarter * 32 + lane;
#pragma unroll
                        for (int i = 0; i < kMsGroup; ++i) to[i * kMsRows] = __uint_as_float(v[i]);
                    } else {
                        __nv_bfloat16* to = reinterpret_cast<__nv_bfloat16*>(out_buffer) + quarter * 32 + lane;
#pragma unroll
                        for (int i = 0; i < kMsGroup; ++i) to[i * kMsRows] = __float2bfloat16_rn(__uint_as_float(v[i]));
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    named_barrier(set_barrier, 128);
                    if (issuer) bulk_store_2d(&map_out, out_buffer, row0, first_token, false);
                } else {
                    const int row = row0 + quarter * 32 + lane, tokens_here = min(kMsGroup, p.tokens - first_token);
                    if (row < p.n) {
                        const size_t first = static_cast<size_t>(first_token) * p.n + row;
#pragma unroll
                        for (int i = 0; i < kMsGroup; ++i) {
                            if (i >= tokens_here) break;
                            if (p.out_is_float) static_cast<float*>(p.out)[first + static_cast<size_t>(i) * p.n] = __uint_as_float(v[i]);
                            else static_cast<__nv_bfloat16*>(p.out)[first + static_cast<size_t>(i) * p.n] = __float2bfloat16_rn(__uint_as_float(v[i]));
                        }
                    }
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                if constexpr (PAIR) barrier_arrive_cluster(cluster_address(&tmem_empty[accumulator], 0));
                else barrier_arrive(&tmem_empty[accumulator]);
            }
        }
        if (issuer) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (failed) {
        // Let whatever copies are still in flight land before the shared memory goes away.
        if (threadIdx.x == 0) report_error(p.status, kWaitTimeout);
        for (int spin = 0; spin < 2000; ++spin) __nanosleep(1000);
        __syncthreads();
    }
    // PAIR: neither CTA leaves, or gives its tensor memory back, while the other may still touch them.
    if constexpr (PAIR) cluster_sync();
    if (warp == 1) {
        if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(Walk::kColumns) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(Walk::kColumns) : "memory");
    }
}

// ---------------------------------------------------------------------------------------------
// The same where the tiles alone would leave most multiprocessors idle (few tokens, or few of both): the CTAs of a cluster share a tile's K, and the sums of
// their parts meet in shared memory.  Every CTA then adds up the tokens rank, rank + S, ... of the tile, part after part in the parts' order, and sends
// them off; a second launch and a trip of the parts through memory are saved.
// ---------------------------------------------------------------------------------------------
constexpr int kMsSplitThreads = 256;   // producer, issuer, scales of a gated product, one idle, four that read tensor memory; all of them add up
constexpr int kMsLargestSplit = 8;     // CTAs of a cluster
constexpr int kMsSplitStages = 8;      // of the ring, at most
constexpr int kMsSplitShared = 112 * 1024;   // beside the variables: half a multiprocessor's

template <int BITS, int BN>
struct MsSplit {
    static constexpr int kScaleColumns = 4 * MsShape<BITS, BN>::kChunks * (1 + MsShape<BITS, BN>::kScaleTiles);
    static constexpr int kColumns = BN + kScaleColumns <= 32 ? 32 : BN + kScaleColumns <= 64 ? 64 : BN + kScaleColumns <= 128 ? 128 : 256;
    static constexpr int kPartBytes = BN * kMsRows * 4;   // the parts' sums, where the ring was
    static constexpr int kSlack = 1024 + 256;             // alignment and barriers
    static constexpr int kRoom = (kMsSplitShared - kSlack) / MsShape<BITS, BN>::kStageBytes;
    static constexpr int kMostStages = kRoom < kMsSplitStages ? kRoom : kMsSplitStages;
    static int bytes(int stages) {
        const int ring = stages * MsShape<BITS, BN>::kStageBytes;
        return (ring > kPartBytes ? ring : kPartBytes) + kSlack;
    }
};

__device__ __forceinline__ float4 load_cluster(uint32_t address) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(address));
    return v;
}

template <int BITS, int BN, bool GATED>
__global__ void __launch_bounds__(kMsSplitThreads)
gemm_microscaled_split_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_gate, const __grid_constant__ CUtensorMap map_x, const MsParams p,
                              int splits, int stages_per_split, int ring_stages) {
    using Shape = MsShape<BITS, BN>;
    using Split = MsSplit<BITS, BN>;
    static_assert(BN <= 128, "one tile of scales for the tokens");
    extern __shared__ unsigned char raw_shared[];
    __shared__ uint64_t barriers[2 * kMsSplitStages + 1];
    __shared__ uint32_t tmem_slot;
    __shared__ int failed;
    unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw_shared) + 1023) & ~static_cast<uintptr_t>(1023));
    uint64_t* full = barriers;
    uint64_t* empty = barriers + kMsSplitStages;
    uint64_t* accumulated = barriers + 2 * kMsSplitStages;

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    constexpr int kRowsPerTile = GATED ? kMsRows / 2 : kMsRows;
    const int rank = static_cast<int>(blockIdx.x) % splits;   // the cluster's CTAs are neighbours
    const int row0 = static_cast<int>(blockIdx.x) / splits * kRowsPerTile, token0 = blockIdx.y * BN;
    const int num_stages = (p.chunks + Shape::kChunks - 1) / Shape::kChunks;
    const int first_stage = rank * stages_per_split, count = min(stages_per_split, num_stages - first_stage);   // at least one: the launcher sees to it
    auto chunks_of = [&](int stage) { return min(Shape::kChunks, p.chunks - stage * Shape::kChunks); };

    if (threadIdx.x == 0) {
        for (int s = 0; s < ring_stages; ++s) {
            barrier_init(&full[s], GATED ? 2 : 1);
            barrier_init(&empty[s], 1);
        }
        barrier_init(accumulated, 1);
        failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_address(&tmem_slot)), "r"(Split::kColumns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = tmem_slot;
    wait_for_previous_kernel();   // the weights may be what it has made
    allow_next_kernel();

    if (warp == 0) {
        const unsigned char* w_scales = p.w_scales + static_cast<size_t>(row0 / 128) * p.chunks * kScaleTileBytes;
        const unsigned char* x_scales = p.x_scales + static_cast<size_t>(token0 / 128) * p.chunks * kScaleTileBytes;
        for (int i = 0, s = 0, round = 0; i < count; ++i) {
            if (round > 0 && !barrier_wait_warp(&empty[s], (round - 1) & 1)) {
                atomicExch(&failed, 1);
                break;
            }
            if (elect_lane()) {
                const int stage = first_stage + i, column = stage * 128, chunk = stage * Shape::kChunks;
                unsigned char* at = ring + s * Shape::kStageBytes;
                const uint32_t scale_bytes = static_cast<uint32_t>(chunks_of(stage) * kScaleTileBytes);
                barrier_expect(&full[s], Shape::kWCounted + Shape::kXBytes + (GATED ? 1u : 2u) * scale_bytes);
                tma_load_2d(at, &map_w, column, row0, &full[s]);
                if constexpr (GATED) tma_load_2d(at + Shape::kWBytes / 2, &map_gate, column, row0, &full[s]);
                tma_load_2d(at + Shape::kWBytes, &map_x, column, token0, &full[s]);
                at += Shape::kWBytes + Shape::kXBytes;
                if constexpr (!GATED) bulk_load(at, w_scales + static_cast<size_t>(chunk) * kScaleTileBytes, scale_bytes, &full[s]);
                bulk_load(at + Shape::kWScaleBytes, x_scales + static_cast<size_t>(chunk) * kScaleTileBytes, scale_bytes, &full[s]);
            }
            if (++s == ring_stages) s = 0, ++round;
        }
    } else if (warp == 1) {
        const uint32_t idesc = microscaled_descriptor<BITS>(BN);
        bool ok = true;
        for (int i = 0, s = 0, round = 0; i < count; ++i) {
            ok = barrier_wait_warp(&full[s], round & 1);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const unsigned char* at = ring + s * Shape::kStageBytes;
            copy_stage_scales<Shape, false>(at, tmem_base + BN, chunks_of(first_stage + i));
            issue_stage<BITS, Shape, false>(tmem_base, at, tmem_base + BN, static_cast<uint32_t>((token0 & 127) >> 5), idesc, chunks_of(first_stage + i), i > 0, &empty[s]);
            if (++s == ring_stages) s = 0, ++round;
        }
        if (!ok) atomicExch(&failed, 1);
        else if (elect_lane()) mma_commit(accumulated);
    } else if (GATED && warp == 2) {
        // as in the walking kernel
        const size_t offset = static_cast<size_t>(row0 / 128) * p.chunks * kScaleTileBytes + lane * 16 + ((row0 & 64) >> 3);
        bool ok = true;
        for (int first = 0, s = 0, round = 0; first < count && ok; first += 4) {
            uint2 up[4][Shape::kChunks], gate[4][Shape::kChunks];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int c = 0; c < Shape::kChunks; ++c) {
                    const int chunk = (first_stage + first + i) * Shape::kChunks + c;
                    up[i][c] = gate[i][c] = make_uint2(0u, 0u);
                    if (chunk < p.chunks) {
                        up[i][c] = *reinterpret_cast<const uint2*>(p.w_scales + offset + static_cast<size_t>(chunk) * kScaleTileBytes);
                        gate[i][c] = *reinterpret_cast<const uint2*>(p.gate_scales + offset + static_cast<size_t>(chunk) * kScaleTileBytes);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (first + i >= count) break;
                ok = round == 0 || barrier_wait_warp(&empty[s], (round - 1) & 1);
                if (!ok) {
                    atomicExch(&failed, 1);
                    break;
                }
                unsigned char* at = ring + s * Shape::kStageBytes + Shape::kWBytes + Shape::kXBytes + lane * 16;
#pragma unroll
                for (int c = 0; c < Shape::kChunks; ++c) *reinterpret_cast<uint4*>(at + c * kScaleTileBytes) = make_uint4(up[i][c].x, up[i][c].y, gate[i][c].x, gate[i][c].y);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) barrier_arrive(&full[s]);
                if (++s == ring_stages) s = 0, ++round;
            }
        }
    } else if (warp >= 4) {
        const int quarter = warp & 3;
        if (barrier_wait_warp(accumulated, 0)) {
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            float* part = reinterpret_cast<float*>(ring) + quarter * 32 + lane;
#pragma unroll 1
            for (int column = 0; column < BN; column += 16) {
                if (token0 + column >= p.tokens) break;
                uint32_t v[16];
                tmem_load_16(tmem_base + static_cast<uint32_t>(column) + (static_cast<uint32_t>(quarter * 32) << 16), v);
#pragma unroll
                for (int i = 0; i < 16; ++i) part[(column + i) * kMsRows] = __uint_as_float(v[i]);
            }
        } else if (lane == 0) {
            atomicExch(&failed, 1);
        }
    }
    // Tensor memory goes back before the CTAs wait for one another: one that waits to get some, without a limit, never waits for a CTA that waits for it.
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (failed) {
        // Let whatever copies and products are still in flight land before their memories go away.
        if (threadIdx.x == 0) report_error(p.status, kWaitTimeout);
        for (int spin = 0; spin < 2000; ++spin) __nanosleep(1000);
        __syncthreads();
    }
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(Split::kColumns) : "memory");
    if (splits > 1) cluster_sync();   // all parts are there, or some CTA has failed and said so
    const int tokens_here = min(BN, p.tokens - token0);
    const uint32_t part = smem_address(ring);
    // Four rows (of a token) at each of one or two places, part after part; all parts are read before the first is added.
    auto add_up = [&](int first, int second, bool both, float4 (&sums)[2]) {
        float4 v[kMsLargestSplit], w[kMsLargestSplit];
#pragma unroll
        for (int q = 0; q < kMsLargestSplit; ++q) {
            if (q < splits) {
                uint32_t at;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(part), "r"(q));
                v[q] = load_cluster(at + first * 4);
                w[q] = both ? load_cluster(at + second * 4) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
        }
        sums[0] = v[0], sums[1] = w[0];
#pragma unroll
        for (int q = 1; q < kMsLargestSplit; ++q) {
            if (q < splits) {
                sums[0].x += v[q].x, sums[0].y += v[q].y, sums[0].z += v[q].z, sums[0].w += v[q].w;
                sums[1].x += w[q].x, sums[1].y += w[q].y, sums[1].z += w[q].z, sums[1].w += w[q].w;
            }
        }
    };
    // No CTA leaves while another still reads its part: a warp arrives when it has read all that it reads, before it writes what it read last.  The arrival orders the
    // reads before it (a relaxed one would not, and a CTA could leave, its shared memory go to another, under a read), and the writes of the passes before, if any.
    // (One warp that hears from the others and arrives for all: gated 8192 x 2048, 8 tokens 7.5 us and 7.7 this way, but 2048 x 8192 5.8 and 5.6.)
    bool arrived = splits == 1;
    const auto has_read = [&]() {
        if (arrived) return;
        arrived = true;
        __syncwarp();   // the lanes may have parted where the pass before wrote
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    };
    if constexpr (!GATED) {
        // A warp takes two tokens at a time, a lane four rows of each.
        const int row = row0 + lane * 4;
        for (int t = rank + 2 * warp * splits; t < tokens_here; t += 16 * splits) {
            float4 sums[2];
            add_up(t * kMsRows + lane * 4, (t + splits) * kMsRows + lane * 4, t + splits < tokens_here, sums);
            if (t + 16 * splits >= tokens_here) has_read();
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int token = t + i * splits;
                if (token >= tokens_here) break;
                const size_t at = static_cast<size_t>(token0 + token) * p.n + row;
                if (p.bulk_store && row < p.n) {   // four rows are 16 (8) aligned bytes
                    if (p.out_is_float) {
                        *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = sums[i];
                    } else {
                        uint2 packed;
                        __nv_bfloat162* halves = reinterpret_cast<__nv_bfloat162*>(&packed);
                        halves[0] = __floats2bfloat162_rn(sums[i].x, sums[i].y);
                        halves[1] = __floats2bfloat162_rn(sums[i].z, sums[i].w);
                        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + at) = packed;
                    }
                } else {
                    const float values[4] = {sums[i].x, sums[i].y, sums[i].z, sums[i].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (row + e >= p.n) break;
                        if (p.out_is_float) static_cast<float*>(p.out)[at + e] = values[e];
                        else static_cast<__nv_bfloat16*>(p.out)[at + e] = __float2bfloat16_rn(values[e]);
                    }
                }
            }
        }
    } else {
        // Half a warp takes a token, eight lanes a block of 32 channels.
        const int channel = (lane & 15) * 4;
        for (int first = rank + 2 * warp * splits; first < tokens_here; first += 16 * splits) {   // the same for the whole warp
            const int t = first + (lane >> 4) * splits;
            const bool valid = t < tokens_here;
            const int at = (valid ? t : first) * kMsRows + channel;
            float4 sums[2];
            add_up(at, at + kMsRows / 2, true, sums);
            if (first + 16 * splits >= tokens_here) has_read();
            const float up[4] = {sums[0].x, sums[0].y, sums[0].z, sums[0].w}, gate[4] = {sums[1].x, sums[1].y, sums[1].z, sums[1].w};
            float h[4];
            gated_values(up, gate, p.activation, p.limit, h);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (row0 + channel + e >= p.n) h[e] = 0.0f;
            float largest = larger_size(larger_size(h[0], h[1]), larger_size(h[2], h[3]));
#pragma unroll
            for (int offset = 1; offset < 8; offset <<= 1) largest = larger_size(largest, __shfl_xor_sync(0xffffffffu, largest, offset));
            const int byte = scale_byte<8>(__float_as_uint(largest) & 0x7fffffffu);
            const float inverse = scale_inverse(byte);
            const int token = token0 + t, block = (row0 + channel) / 32;
            if (valid) {
                *reinterpret_cast<uint32_t*>(static_cast<unsigned char*>(p.out) + static_cast<size_t>(token) * p.out_chunks * 128 + row0 + channel) =
                    pack_e4m3(h[0] * inverse, h[1] * inverse, h[2] * inverse, h[3] * inverse);
                if ((lane & 7) == 0) p.out_scales[scale_word(token, block >> 2, p.out_chunks) + (block & 3)] = static_cast<unsigned char>(byte);
            }
        }
    }
    has_read();   // a warp that had no tokens
    __syncwarp();
    if (splits > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Codes as boxes of [box_rows, 128 bytes of shared memory] with 128-byte swizzle; `spread`: 4-bit elements to 16 in 16 bytes (boxes of 128 elements),
// else the bytes as they are.  What lies outside reads as zero.
static bool make_codes_map(CUtensorMap* map, const void* codes, int rows, int row_bytes, int box_rows, bool spread) {
    EncodeTiled encode = encode_tiled();
    if (encode == nullptr) return false;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(spread ? row_bytes * 2 : row_bytes), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(row_bytes)};
    const cuuint32_t box[2] = {128, static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t element_strides[2] = {1, 1};
    return encode(map, spread ? CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B : CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), dims, strides, box, element_strides,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The output [tokens, width] as boxes of [box_tokens, box_width], laid down in shared memory row after row.
static bool make_ms_out_map(CUtensorMap* map, void* base, int tokens, int width, CUtensorMapDataType type, int size, int box_width, int box_tokens) {
    EncodeTiled encode = encode_tiled();
    if (encode == nullptr) return false;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(width), static_cast<cuuint64_t>(tokens)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(width) * size};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_width), static_cast<cuuint32_t>(box_tokens)};
    const cuuint32_t element_strides[2] = {1, 1};
    return encode(map, type, 2, base, dims, strides, box, element_strides, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Scales as boxes of [tiles, chunks] of them, in words.
static bool make_scales_map(CUtensorMap* map, const void* scales, int row_tiles, int chunks, int box_tiles, int box_chunks) {
    EncodeTiled encode = encode_tiled();
    if (encode == nullptr) return false;
    constexpr cuuint32_t words = kScaleTileBytes / 4;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(chunks) * words, static_cast<cuuint64_t>(row_tiles)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(chunks) * kScaleTileBytes};
    const cuuint32_t box[2] = {box_chunks * words, static_cast<cuuint32_t>(box_tiles)};
    const cuuint32_t element_strides[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(scales), dims, strides, box, element_strides, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int BITS, bool GATED, bool PAIR>
int launch_microscaled(const void* x, const void* w, const void* gate, MsParams p, int token_tiles, int wide_tiles, cudaStream_t stream) {
    using Walk = MsWalk<BITS, PAIR>;
    using Shape = typename Walk::Shape;
    constexpr int kCtas = PAIR ? 2 : 1;
    CUtensorMap map_w, map_gate, map_x, map_x_narrow, map_w_scales, map_x_scales, map_out;
    const int w_bytes = p.chunks * 64, x_bytes = p.chunks * 16 * BITS;
    if (!make_codes_map(&map_w, w, p.n, w_bytes, GATED ? kMsRows / 2 : kMsRows, BITS == 8) || !make_codes_map(&map_x, x, p.tokens, x_bytes, kMsWide / kCtas, false) ||
        !make_codes_map(&map_x_narrow, x, p.tokens, x_bytes, kMsNarrow / kCtas, false) ||
        !make_scales_map(&map_w_scales, p.w_scales, (p.n + 127) / 128, p.chunks, 1, Shape::kChunks) ||
        !make_scales_map(&map_x_scales, p.x_scales, (p.tokens + 127) / 128, p.chunks, Shape::kScaleTiles, Shape::kChunks))
        return -5;
    map_gate = map_w, map_out = map_x;
    int row_tiles;
    if constexpr (GATED) {
        if (!make_codes_map(&map_gate, gate, p.n, w_bytes, kMsRows / 2, BITS == 8) ||
            !make_ms_out_map(&map_out, p.out, p.tokens, p.out_chunks * 128, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, kMsRows / 2, kMsGroup))
            return -5;
        row_tiles = p.out_chunks * 2;
    } else {
        const int size = p.out_is_float ? 4 : 2;
        p.bulk_store = (static_cast<size_t>(p.n) * size) % 16 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0 ? 1 : 0;
        if (p.bulk_store && !make_ms_out_map(&map_out, p.out, p.tokens, p.n, p.out_is_float ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, size,
                                             kMsRows, kMsGroup))
            return -5;
        row_tiles = (p.n + kMsRows - 1) / kMsRows;
    }
    p.row_tiles = (row_tiles + kCtas - 1) / kCtas;
    p.token_tiles = token_tiles;
    p.wide_tiles = wide_tiles;
    auto kernel = gemm_microscaled_kernel<BITS, GATED, PAIR>;
    static OncePerDevice configured;
    if (allow_shared_memory(configured, kernel, Walk::kBytes) != cudaSuccess) return static_cast<int>(cudaGetLastError());
    const int tiles = p.row_tiles * p.token_tiles, walkers = multiprocessor_count() / kCtas;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((tiles < walkers ? tiles : walkers) * kCtas);
    config.blockDim = dim3(kMsThreads);
    config.dynamicSmemBytes = Walk::kBytes;
    config.stream = stream;
    cudaLaunchAttribute attributes[2];
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = overlap_launches() ? 1 : 0;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = 2;
    attributes[1].val.clusterDim.y = 1;
    attributes[1].val.clusterDim.z = 1;
    config.attrs = attributes;
    config.numAttrs = PAIR ? 2 : 1;
    return static_cast<int>(cudaLaunchKernelEx(&config, kernel, map_w, map_gate, map_x, map_x_narrow, map_w_scales, map_x_scales, map_out, p));
}

template <int BITS, int BN, bool GATED>
int launch_microscaled_split(const void* x, const void* w, const void* gate, MsParams p, cudaStream_t stream) {
    CUtensorMap map_w, map_gate, map_x;
    const int w_bytes = p.chunks * 64, x_bytes = p.chunks * 16 * BITS;
    if (!make_codes_map(&map_w, w, p.n, w_bytes, GATED ? kMsRows / 2 : kMsRows, BITS == 8) || !make_codes_map(&map_x, x, p.tokens, x_bytes, BN, false)) return -5;
    map_gate = map_w;
    if (GATED && !make_codes_map(&map_gate, gate, p.n, w_bytes, kMsRows / 2, BITS == 8)) return -5;
    // four rows of an output's row are whole 16 (of bfloat16 8) bytes
    p.bulk_store = p.n % 4 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0 ? 1 : 0;
    const int row_tiles = GATED ? p.out_chunks * 2 : (p.n + kMsRows - 1) / kMsRows, token_tiles = (p.tokens + BN - 1) / BN, sms = multiprocessor_count();
    const int stages = (p.chunks + MsShape<BITS, BN>::kChunks - 1) / MsShape<BITS, BN>::kChunks;
    // Two CTAs fit a multiprocessor: clusters of eight that have one each do not all find room at once (2048 x 8192 and a token: 9.1 us, and 5.2 with room for two),
    // and a deeper ring gains nothing.  A stage takes 0.18 us, the meetings of up to four CTAs 1.0 us and of eight 1.6, more with more tokens: beyond four where each still has
    // three stages (8 tokens, rows of 4 bits, 2048 x 2048: 3.2 us by four, 3.8 by eight; of 8 bits, 1024 x 4608 4.8 and 4.2), and of more than 32 tokens six at most (128 tokens,
    // 2048 x 8192: 11.4 us by four, 10.6 by six, 12.9 by eight).
    int wanted = max(1, min(min(sms / (row_tiles * token_tiles), stages), min(max(4, stages / 3), BN > 32 ? 6 : kMsLargestSplit)));
    // Gated tiles that nearly fill the multiprocessors are cut in two all the same, two CTAs to each, where that saves each more than four stages or there are many tokens: 8192 x
    // 8192, 16 tokens 17.5 us and 21.5, 8192 x 1024, 128 tokens 10.1 and 10.9; with few of both the meetings cost more: 8192 x 1024, 8 tokens 5.0 us and 4.5, rows of 4 bits, 2048
    // columns, 6.2 and 5.2.  (Other products lose by it, 6.4 us and 7.3.)
    if (GATED && wanted == 1 && stages > (BN > 64 ? 1 : 8) && row_tiles * token_tiles <= sms) wanted = 2;
    const int per_split = (stages + wanted - 1) / wanted, splits = (stages + per_split - 1) / per_split;   // each has a stage at least
    const int ring = min(per_split, MsSplit<BITS, BN>::kMostStages);
    auto kernel = gemm_microscaled_split_kernel<BITS, BN, GATED>;
    static OncePerDevice configured;
    if (allow_shared_memory(configured, kernel, kMsSplitShared) != cudaSuccess) return static_cast<int>(cudaGetLastError());
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(row_tiles * splits, token_tiles);
    config.blockDim = dim3(kMsSplitThreads);
    config.dynamicSmemBytes = MsSplit<BITS, BN>::bytes(ring);
    config.stream = stream;
    cudaLaunchAttribute attributes[2];
    attributes[0].id = cudaLaunchAttributeClusterDimension;
    attributes[0].val.clusterDim.x = splits;
    attributes[0].val.clusterDim.y = 1;
    attributes[0].val.clusterDim.z = 1;
    attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[1].val.programmaticStreamSerializationAllowed = overlap_launches() ? 1 : 0;
    config.attrs = attributes;
    config.numAttrs = 2;
    return static_cast<int>(cudaLaunchKernelEx(&config, kernel, map_w, map_gate, map_x, p, splits, per_split, ring));
}

// How the tokens are cut into tiles: of all numbers of tiles, the first as many of them wide as it takes, or one more, which leaves fewer tokens to the last, the cut whose first
// walker, which has the most and the widest tiles, is done first.  What a stage of K costs (hundredths of a microsecond, measured at 4,096 tokens, 2048 x 8192, under
// sustained load): 29 with 128 tokens and 36 with 192; of a pair 27 and 32; with rows of 4 bits 30 and 36.
struct TokenTiles {
    int count, wide;
    long long cost;   // of the walk
};
inline TokenTiles cut_tokens(int tokens, long long row_tiles, int walkers, long long stages, int narrow_cost, int wide_cost) {
    constexpr int kStep = kMsWide - kMsNarrow;
    TokenTiles best = {0, 0, -1};
    const auto rounds = [&](int tiles) { return (row_tiles * tiles + walkers - 1) / walkers; };   // of the first walker that begin before so many of the tokens' tiles end
    for (int count = (tokens + kMsWide - 1) / kMsWide; count <= (tokens + kMsNarrow - 1) / kMsNarrow; ++count) {
        const int more = tokens - count * kMsNarrow, least = more > 0 ? (more + kStep - 1) / kStep : 0;
        for (int wide = least; wide <= min(least + 1, count); ++wide) {
            const int last = tokens - ((count - 1) * kMsNarrow + min(wide, count - 1) * kStep);   // tokens of the last tile
            if (last < 1) break;
            const long long before = rounds(count - 1), wides = min(rounds(min(wide, count - 1)), before);
            const long long cost = wides * wide_cost + (before - wides) * narrow_cost + (rounds(count) - before) * (narrow_cost + (last - kMsNarrow) * (wide_cost - narrow_cost) / kStep);
            if (best.cost < 0 || cost * stages < best.cost) best = {count, wide, cost * stages};
        }
    }
    return best;
}

// Which kernel.  Few tiles are cut along K: up to 128 tokens, and up to half of the multiprocessors in tiles of 128 x 128.  Else the tiles are walked, by pairs of CTAs where
// those are sooner done although they start some 2.5 us later.
enum MsKernel { kMsShared, kMsWalked, kMsPairs };
struct MsChoice {
    MsKernel kernel;
    TokenTiles cut;   // of the walked ones
};
template <int BITS, bool GATED>
MsChoice choose_microscaled(int tokens, int n, int chunks) {
    const long long row_tiles = GATED ? (n + 127) / 128 * 2 : (n + kMsRows - 1) / kMsRows;
    const int sms = multiprocessor_count();
    if (tokens <= 128 || row_tiles * ((tokens + 127) / 128) <= sms / 2) return {kMsShared, {}};
    const long long stages = (chunks + MsShape<BITS, 128>::kChunks - 1) / MsShape<BITS, 128>::kChunks;
    const TokenTiles alone = cut_tokens(tokens, row_tiles, sms, stages, BITS == 8 ? 29 : 30, 36);
    if constexpr (BITS == 8 && !GATED) {
        const TokenTiles pairs = cut_tokens(tokens, (row_tiles + 1) / 2, max(1, sms / 2), stages, 27, 32);
        if (sms > 1 && pairs.cost + 250 < alone.cost) return {kMsPairs, pairs};
    }
    return {kMsWalked, alone};
}

template <int BITS, bool GATED>
int launch_microscaled_tiles(const void* x, const void* w, const void* gate, const MsParams& p, cudaStream_t stream) {
    const MsChoice choice = choose_microscaled<BITS, GATED>(p.tokens, p.n, p.chunks);
    if (choice.kernel == kMsShared) {
        if (p.tokens <= 16) return launch_microscaled_split<BITS, 16, GATED>(x, w, gate, p, stream);
        if (p.tokens <= 32) return launch_microscaled_split<BITS, 32, GATED>(x, w, gate, p, stream);
        if (p.tokens <= 64) return launch_microscaled_split<BITS, 64, GATED>(x, w, gate, p, stream);
        return launch_microscaled_split<BITS, 128, GATED>(x, w, gate, p, stream);
    }
    if constexpr (BITS == 8 && !GATED) {
        if (choice.kernel == kMsPairs) return launch_microscaled<BITS, GATED, true>(x, w, gate, p, choice.cut.count, choice.cut.wide, stream);
    }
    return launch_microscaled<BITS, GATED, false>(x, w, gate, p, choice.cut.count, choice.cut.wide, stream);
}

}  // namespace lb

extern "C" {

// Which kernel runs a product of these sizes on the current device: 0 tiles whose K is shared out, 1 walked tiles, 2 by pairs of CTAs; -2 for sizes that none takes,
// -3 without a device.
int lb_microscaled_kernel(int tokens, int n, int chunks, int bits, int gated) {
    if (tokens < 1 || tokens > lb::kMsMostRows || n < 1 || n > lb::kMsMostRows || chunks < 1 || chunks > (1 << 22) || (bits != 4 && bits != 8)) return -2;
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return -3;
    if (gated) return bits == 8 ? lb::choose_microscaled<8, true>(tokens, n, chunks).kernel : lb::choose_microscaled<4, true>(tokens, n, chunks).kernel;
    return bits == 8 ? lb::choose_microscaled<8, false>(tokens, n, chunks).kernel : lb::choose_microscaled<4, false>(tokens, n, chunks).kernel;
}

// out [tokens, n] = x w^T, bfloat16 or float32.  x [tokens, 128 * chunks] in `bits` bits, w [n, 128 * chunks] in 4.
// Returns 0, a CUDA error, -2 for sizes or addresses that the kernel does not take, -5 if no tensor map could be made.
int lb_gemm_microscaled(const void* x, const void* x_scales, const void* w, const void* w_scales, void* out, int tokens, int n, int chunks, int bits, int out_is_float,
                        int* status, cudaStream_t stream) {
    if (tokens < 1 || tokens > lb::kMsMostRows || n < 1 || n > lb::kMsMostRows || chunks < 1 || chunks > (1 << 22) || (bits != 4 && bits != 8)) return -2;
    if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(x_scales) | reinterpret_cast<uintptr_t>(w_scales)) & 15 || reinterpret_cast<uintptr_t>(w) & 31) return -2;
    lb::MsParams p = {};
    p.w_scales = static_cast<const unsigned char*>(w_scales);
    p.x_scales = static_cast<const unsigned char*>(x_scales);
    p.out = out;
    p.tokens = tokens;
    p.n = n;
    p.chunks = chunks;
    p.out_is_float = out_is_float;
    p.status = status;
    return bits == 8 ? lb::launch_microscaled_tiles<8, false>(x, w, nullptr, p, stream) : lb::launch_microscaled_tiles<4, false>(x, w, nullptr, p, stream);
}

// codes and scales of (x up^T) * act(x gate^T) in 8 bits: [tokens, n made up to whole 128s].
int lb_gated_microscaled(const void* x, const void* x_scales, const void* up, const void* up_scales, const void* gate, const void* gate_scales, void* out, void* out_scales,
                         int tokens, int n, int chunks, int bits, int activation, float limit, int* status, cudaStream_t stream) {
    if (tokens < 1 || tokens > lb::kMsMostRows || n < 1 || n > lb::kMsMostRows || chunks < 1 || chunks > (1 << 22) || (bits != 4 && bits != 8) || activation < 0 || activation > 3) return -2;
    if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(x_scales) | reinterpret_cast<uintptr_t>(up_scales) | reinterpret_cast<uintptr_t>(gate_scales) |
         reinterpret_cast<uintptr_t>(out)) & 15 || (reinterpret_cast<uintptr_t>(up) | reinterpret_cast<uintptr_t>(gate)) & 31)
        return -2;
    lb::MsParams p = {};
    p.w_scales = static_cast<const unsigned char*>(up_scales);
    p.gate_scales = static_cast<const unsigned char*>(gate_scales);
    p.x_scales = static_cast<const unsigned char*>(x_scales);
    p.out = out;
    p.out_scales = static_cast<unsigned char*>(out_scales);
    p.tokens = tokens;
    p.n = n;
    p.chunks = chunks;
    p.out_chunks = (n + 127) / 128;
    p.activation = activation;
    p.limit = limit;
    p.status = status;
    return bits == 8 ? lb::launch_microscaled_tiles<8, true>(x, up, gate, p, stream) : lb::launch_microscaled_tiles<4, true>(x, up, gate, p, stream);
}

}  // extern "C"
