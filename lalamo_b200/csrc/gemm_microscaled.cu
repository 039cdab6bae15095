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
    int row_tiles, token_tiles;
    int* status;
};

__device__ __forceinline__ void bulk_load(void* destination, const void* source, uint32_t bytes, uint64_t* barrier) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_address(destination)), "l"(source), "r"(bytes),
                 "r"(smem_address(barrier))
                 : "memory");
}

// A tile of scales, 32 rows of 16 bytes one behind the other (groups of 8 rows 128 bytes apart, no swizzle), for tcgen05.cp.
__device__ __forceinline__ uint64_t scale_descriptor(const void* tile) {
    const uint64_t address = smem_address(tile);
    return ((address & 0x3FFFFull) >> 4) | (static_cast<uint64_t>(128 >> 4) << 32) | (1ull << 46);
}
// To four columns of tensor memory, the same in each quarter of the lanes.
__device__ __forceinline__ void copy_scales(uint32_t tmem, const void* tile) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(scale_descriptor(tile)) : "memory");
}

// D float32 [128, N] (+)= A [128, 32] e2m1 (spread) B [N, 32] e4m3, or A [128, 64] e2m1 B [N, 64] e2m1, each block of 32 times its two scales.
template <int BITS>
__device__ __forceinline__ void mma_microscaled(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t scales_a, uint32_t scales_b, bool accumulate) {
    if constexpr (BITS == 8) {
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
            ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate ? 1u : 0u), "r"(scales_a), "r"(scales_b)
            : "memory");
    } else {
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
            ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate ? 1u : 0u), "r"(scales_a), "r"(scales_b)
            : "memory");
    }
}

// The instruction's description: A (W) e2m1, B (X) e4m3 or e2m1, scales e8m0, N columns, 128 lanes; the bytes of the scales' words follow per product.
template <int BITS>
__device__ __forceinline__ uint32_t microscaled_descriptor(int columns) {
    const uint32_t types = BITS == 8 ? (5u << 7) | (0u << 10) : (1u << 7) | (1u << 10);
    return types | (static_cast<uint32_t>(columns >> 3) << 17) | (1u << 23) | (static_cast<uint32_t>(kMsRows >> 4) << 24);
}
// Product `k` of the four of a stage takes the scales from this chunk of the stage, and from this byte on of its words.
template <int BITS>
__device__ __forceinline__ int product_chunk(int k) { return BITS == 8 ? 0 : k >> 1; }
template <int BITS>
__device__ __forceinline__ uint32_t product_scales(int k) {
    const uint32_t byte = BITS == 8 ? static_cast<uint32_t>(k) : static_cast<uint32_t>(k & 1) * 2u;
    return (byte << 4) | (byte << 29);
}

// What the gate side of a gated product multiplies with, and the up side.
__device__ __forceinline__ float ms_gate_side(float g, int activation, float limit) {
    if (activation == kSigmoidLimit) {
        const float c = fminf(g, limit);
        return __fdividef(c, 1.0f + __expf(-kSigmoidLimitSlope * c));
    }
    if (activation == 0) return __fdividef(g, 1.0f + __expf(-g));
    if (activation == 1) return 0.5f * g * (1.0f + erff(g * 0.70710678118654752440f));
    return g;
}
__device__ __forceinline__ float ms_up_side(float u, int activation, float limit) {
    return activation == kSigmoidLimit ? fminf(fmaxf(u, -limit), limit) + 1.0f : u;
}

// BN: tokens of a tile.  A tile of more than 128 begins at a multiple of 64, so that two tiles of scales cover it.
template <int BITS, int BN>
struct MsShape {
    static constexpr int kChunks = BITS == 8 ? 1 : 2;             // of 128 columns, a stage
    static constexpr int kScaleTiles = BN > 128 ? 2 : 1;          // of 128 tokens, that a tile's tokens lie in
    static constexpr int kWBytes = kMsRows * 128;
    static constexpr int kXBytes = BN * 128;
    static constexpr int kWScaleBytes = kChunks * kScaleTileBytes;
    static constexpr int kXScaleBytes = kScaleTiles * kChunks * kScaleTileBytes;
    static constexpr int kStageBytes = (kWBytes + kXBytes + kWScaleBytes + kXScaleBytes + 1023) / 1024 * 1024;   // tiles start on 1024 bytes
    // what the copy of a tile of W counts on its barrier: the bytes it has read
    static constexpr uint32_t kWCounted = BITS == 8 ? kWBytes / 2 : kWBytes;
};

constexpr int kMsThreads = 12 * 32;             // producer, issuer, scales of a gated product, one idle; eight warps of the epilogue
constexpr int kMsRegionBytes = 20 * 1024;       // per half of the epilogue: two output buffers of 8 KB; gated: two of 2 KB and four handovers of 4 KB
constexpr int kMsSharedLimit = 227 * 1024;

template <int BITS, int BN>
struct MsWalk {
    static constexpr int kStages = (kMsSharedLimit - 2 * kMsRegionBytes - 1024 - 256) / MsShape<BITS, BN>::kStageBytes;
    static constexpr int kBytes = kStages * MsShape<BITS, BN>::kStageBytes + 2 * kMsRegionBytes + 1024 + 256;
    static constexpr int kScaleColumns = 4 * MsShape<BITS, BN>::kChunks * (1 + MsShape<BITS, BN>::kScaleTiles);
    static constexpr int kColumns = 2 * BN + kScaleColumns <= 256 ? 256 : 512;
    static_assert(kStages >= 3 && kStages <= 12 && 2 * BN + kScaleColumns <= 512, "a ring, its barriers, two accumulators and the scales");
};

// One CTA per multiprocessor walks the tiles of 128 lanes x BN tokens, rows fastest, with two accumulators: the epilogue of a tile runs while the
// products of the next are issued.
template <int BITS, int BN, bool GATED>
__global__ void __launch_bounds__(kMsThreads)
gemm_microscaled_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_gate, const __grid_constant__ CUtensorMap map_x,
                        const __grid_constant__ CUtensorMap map_out, const MsParams p) {
    using Shape = MsShape<BITS, BN>;
    using Walk = MsWalk<BITS, BN>;
    constexpr int STAGES = Walk::kStages;
    extern __shared__ unsigned char raw_shared[];
    unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw_shared) + 1023) & ~static_cast<uintptr_t>(1023));
    unsigned char* regions = ring + STAGES * Shape::kStageBytes;
    uint64_t* barriers = reinterpret_cast<uint64_t*>(regions + 2 * kMsRegionBytes);
    uint64_t* full = barriers;
    uint64_t* empty = barriers + STAGES;
    uint64_t* tmem_full = barriers + 2 * STAGES;
    uint64_t* tmem_empty = barriers + 2 * STAGES + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(barriers + 2 * STAGES + 4);
    __shared__ int failed;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int kRowsPerTile = GATED ? kMsRows / 2 : kMsRows;
    const int num_stages = (p.chunks + Shape::kChunks - 1) / Shape::kChunks;
    const int num_tiles = p.row_tiles * p.token_tiles;
    auto chunks_of = [&](int stage) { return min(Shape::kChunks, p.chunks - stage * Shape::kChunks); };

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            barrier_init(&full[s], GATED ? 2 : 1);   // the producer, and the warp that puts the scales together
            barrier_init(&empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            barrier_init(&tmem_full[a], 1);
            barrier_init(&tmem_empty[a], 8);
        }
        failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_address(tmem_slot)), "r"(Walk::kColumns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = *tmem_slot;
    const uint32_t tmem_w_scales = tmem_base + 2 * BN, tmem_x_scales = tmem_w_scales + 4 * Shape::kChunks;
    // Everything that is read may come from the kernel before this one, the weights too (quantised just now).
    wait_for_previous_kernel();
    allow_next_kernel();

    if (warp == 0 && lane == 0) {
        int issued = 0;
        bool ok = true;
        for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x) {
            const int row0 = (tile % p.row_tiles) * kRowsPerTile, token0 = (tile / p.row_tiles) * BN;
            const int scale_tiles = min(Shape::kScaleTiles, (p.tokens + 127) / 128 - token0 / 128);
            const unsigned char* w_scales = p.w_scales + static_cast<size_t>(row0 / 128) * p.chunks * kScaleTileBytes;
            const unsigned char* x_scales = p.x_scales + static_cast<size_t>(token0 / 128) * p.chunks * kScaleTileBytes;
            for (int stage = 0; stage < num_stages; ++stage, ++issued) {
                const int s = issued % STAGES, round = issued / STAGES;
                if (round > 0 && !barrier_wait(&empty[s], (round - 1) & 1)) {
                    atomicExch(&failed, 1);
                    ok = false;
                    break;
                }
                unsigned char* at = ring + s * Shape::kStageBytes;
                const int column = stage * 128;   // of the map: elements of W where they are spread and of X in 8 bits, bytes of rows in 4
                const int chunk = stage * Shape::kChunks;
                const uint32_t scale_bytes = static_cast<uint32_t>(chunks_of(stage) * kScaleTileBytes);
                barrier_expect(&full[s], Shape::kWCounted + Shape::kXBytes + (GATED ? 0u : scale_bytes) + scale_tiles * scale_bytes);
                tma_load_2d(at, &map_w, column, row0, &full[s]);
                if constexpr (GATED) tma_load_2d(at + Shape::kWBytes / 2, &map_gate, column, row0, &full[s]);
                tma_load_2d(at + Shape::kWBytes, &map_x, column, token0, &full[s]);
                at += Shape::kWBytes + Shape::kXBytes;
                if constexpr (!GATED) bulk_load(at, w_scales + static_cast<size_t>(chunk) * kScaleTileBytes, scale_bytes, &full[s]);
                at += Shape::kWScaleBytes;
                for (int t = 0; t < scale_tiles; ++t)
                    bulk_load(at + t * Shape::kWScaleBytes, x_scales + (static_cast<size_t>(t) * p.chunks + chunk) * kScaleTileBytes, scale_bytes, &full[s]);
            }
        }
    } else if (warp == 1 && lane == 0) {
        const uint32_t idesc = microscaled_descriptor<BITS>(BN);
        int consumed = 0, local = 0;
        bool ok = true;
        for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x, ++local) {
            const int accumulator = local & 1, use = local >> 1;
            if (use > 0 && !barrier_wait(&tmem_empty[accumulator], (use - 1) & 1)) {
                atomicExch(&failed, 1);
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t tmem_d = tmem_base + static_cast<uint32_t>(accumulator * BN);
            const int token0 = (tile / p.row_tiles) * BN;
            const uint32_t x_scales = tmem_x_scales + static_cast<uint32_t>((token0 & 127) >> 5);   // 32 tokens a column
            for (int stage = 0; stage < num_stages; ++stage, ++consumed) {
                const int s = consumed % STAGES, round = consumed / STAGES;
                if (!barrier_wait(&full[s], round & 1)) {
                    atomicExch(&failed, 1);
                    ok = false;
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                unsigned char* at = ring + s * Shape::kStageBytes;
                const unsigned char* scales = at + Shape::kWBytes + Shape::kXBytes;
                const int here = chunks_of(stage);
#pragma unroll
                for (int c = 0; c < Shape::kChunks; ++c) {
                    if (c >= here) break;
                    copy_scales(tmem_w_scales + 4 * c, scales + c * kScaleTileBytes);
#pragma unroll
                    for (int t = 0; t < Shape::kScaleTiles; ++t)
                        copy_scales(tmem_x_scales + 4 * (c * Shape::kScaleTiles + t), scales + Shape::kWScaleBytes + (t * Shape::kChunks + c) * kScaleTileBytes);
                }
                const uint64_t desc_w = tile_descriptor(at), desc_x = tile_descriptor(at + Shape::kWBytes);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int c = product_chunk<BITS>(k);
                    if (c >= here) break;
                    mma_microscaled<BITS>(tmem_d, desc_w + 2 * k, desc_x + 2 * k, idesc | product_scales<BITS>(k), tmem_w_scales + 4 * c,
                                          x_scales + 4 * Shape::kScaleTiles * c, stage > 0 || k > 0);
                }
                mma_commit(&empty[s]);
            }
            if (ok) mma_commit(&tmem_full[accumulator]);
        }
    } else if (GATED && warp == 2) {
        // Lane l puts together the 16 bytes of the rows l, l + 32 of `up` and of `gate` in the accumulator's order.  Four stages are read at once: a
        // read from L2 takes about as long as the products of two.
        int issued = 0;
        bool ok = true;
        for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x) {
            const int row0 = (tile % p.row_tiles) * kRowsPerTile;
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
                    const int s = issued % STAGES, round = issued / STAGES;
                    // the lanes go on together or not at all
                    ok = __all_sync(0xffffffffu, round == 0 || barrier_wait(&empty[s], (round - 1) & 1));
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
                    ++issued;
                }
            }
        }
    } else if (warp >= 4) {
        // Eight warps: warp & 3 is the quarter of the lanes that a warp may read, and each half of the tokens has four warps.
        const int quarter = warp & 3, half = (warp - 4) >> 2;
        constexpr int kLowerPart = (BN / 2 + 31) / 32 * 32;   // whole 32s
        const int part_begin = half ? kLowerPart : 0, part_tokens = half ? BN - kLowerPart : kLowerPart;
        const int half_barrier = 5 + half;   // 1 to 4 belong to the pairs of warps of the gated epilogue
        const bool issuer = quarter == 0 && lane == 0;
        unsigned char* region = regions + half * kMsRegionBytes;
        int local = 0, groups = 0;
        for (int tile = blockIdx.x; tile < num_tiles; tile += gridDim.x, ++local) {
            const int accumulator = local & 1, use = local >> 1;
            const int row0 = (tile % p.row_tiles) * kRowsPerTile, token0 = (tile / p.row_tiles) * BN + part_begin;
            uint32_t arrived = barrier_wait(&tmem_full[accumulator], use & 1) ? 1u : 0u;
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
                    : "r"(arrived), "r"(half_barrier)
                    : "memory");
                arrived = all;
            }
            if (!arrived) {
                atomicExch(&failed, 1);
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t tmem_d = tmem_base + static_cast<uint32_t>(accumulator * BN + part_begin) + (static_cast<uint32_t>(quarter * 32) << 16);
            const int step = !GATED && p.out_is_float && p.bulk_store ? 16 : 32;
#pragma unroll 1
            for (int column = 0; column < part_tokens; column += step, ++groups) {
                if (token0 + column >= p.tokens) break;   // the same for the whole half
                if constexpr (GATED) {
                    unsigned char* out_buffer = region + (groups & 1) * 2048;
                    if (issuer) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");   // the store before last has read this buffer
                    named_barrier(half_barrier, 128);
                    uint32_t v[32];
                    tmem_load_32(tmem_d + static_cast<uint32_t>(column), v);
                    // Lanes 64 to 127 hold `gate`, lanes 0 to 63 the same rows of `up`: handed over in 32 bits.
                    float* handover = reinterpret_cast<float*>(region + 4096 + ((quarter & 1) * 2 + (groups & 1)) * 4096) + lane;
                    const int pair_barrier = 1 + half * 2 + (quarter & 1);
                    if (quarter >= 2) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) handover[i * 32] = ms_gate_side(__uint_as_float(v[i]), p.activation, p.limit);
                        named_barrier(pair_barrier, 64);
                    } else {
                        named_barrier(pair_barrier, 64);
                        const bool exists = row0 + quarter * 32 + lane < p.n;   // past the last row: zeros, whatever the scales there
                        int kept = 0;
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            // A token's 32 lanes of this warp are one block of the output.
                            const float h = exists ? ms_up_side(__uint_as_float(v[i]), p.activation, p.limit) * handover[i * 32] : 0.0f;
                            const uint32_t largest = __reduce_max_sync(0xffffffffu, __float_as_uint(h) & 0x7fffffffu);
                            const int byte = scale_byte<8>(largest);
                            const float scaled = byte == kNoNumber ? 0.0f : h * scale_inverse(byte);
                            out_buffer[i * 64 + quarter * 32 + lane] = static_cast<unsigned char>(pack_e4m3(scaled, 0.0f, 0.0f, 0.0f));
                            if (lane == i) kept = byte;
                        }
                        const int token = token0 + column + lane, block = row0 / 32 + quarter;
                        if (token < p.tokens) p.out_scales[scale_word(token, block >> 2, p.out_chunks) + (block & 3)] = static_cast<unsigned char>(kept);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    named_barrier(half_barrier, 128);
                    if (issuer) bulk_store_2d(&map_out, out_buffer, row0, token0 + column, false);
                } else if (p.bulk_store) {
                    unsigned char* out_buffer = region + (groups & 1) * 8192;
                    if (issuer) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
                    named_barrier(half_barrier, 128);
                    if (p.out_is_float) {
                        uint32_t v[16];
                        tmem_load_16(tmem_d + static_cast<uint32_t>(column), v);
                        float* stage = reinterpret_cast<float*>(out_buffer) + quarter * 32 + lane;
#pragma unroll
                        for (int i = 0; i < 16; ++i) stage[i * kMsRows] = __uint_as_float(v[i]);
                    } else {
                        uint32_t v[32];
                        tmem_load_32(tmem_d + static_cast<uint32_t>(column), v);
                        __nv_bfloat16* stage = reinterpret_cast<__nv_bfloat16*>(out_buffer) + quarter * 32 + lane;
#pragma unroll
                        for (int i = 0; i < 32; ++i) stage[i * kMsRows] = __float2bfloat16_rn(__uint_as_float(v[i]));
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    named_barrier(half_barrier, 128);
                    if (issuer) bulk_store_2d(&map_out, out_buffer, row0, token0 + column, false);
                } else {
                    uint32_t v[32];
                    tmem_load_32(tmem_d + static_cast<uint32_t>(column), v);
                    const int row = row0 + quarter * 32 + lane, tokens_here = min(32, p.tokens - token0 - column);
                    if (row < p.n) {
                        const size_t first = static_cast<size_t>(token0 + column) * p.n + row;
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            if (i >= tokens_here) break;
                            if (p.out_is_float) static_cast<float*>(p.out)[first + static_cast<size_t>(i) * p.n] = __uint_as_float(v[i]);
                            else static_cast<__nv_bfloat16*>(p.out)[first + static_cast<size_t>(i) * p.n] = __float2bfloat16_rn(__uint_as_float(v[i]));
                        }
                    }
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) barrier_arrive(&tmem_empty[accumulator]);
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
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(Walk::kColumns) : "memory");
}

// ---------------------------------------------------------------------------------------------
// The same where the tiles alone would leave most multiprocessors idle (few tokens, or few of both): the CTAs of a cluster share a tile's K, and the sums of
// their parts meet in shared memory.  Every CTA then adds up the tokens rank, rank + S, ... of the tile, part after part in the parts' order, and sends
// them off; a second launch and a trip of the parts through memory are saved.
// ---------------------------------------------------------------------------------------------
constexpr int kMsSplitThreads = 256;   // producer, issuer, scales of a gated product, one idle, four that read tensor memory; all of them add up
constexpr int kMsLargestSplit = 8;     // CTAs of a cluster
constexpr int kMsSplitStages = 11;     // of the ring, at most
constexpr int kMsSplitShared = kMsSharedLimit - 1024;   // beside the variables

template <int BITS, int BN>
struct MsSplit {
    static constexpr int kScaleColumns = 4 * MsShape<BITS, BN>::kChunks * 2;
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

__device__ __forceinline__ float load_cluster(uint32_t address) {
    float value;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(value) : "r"(address) : "memory");
    return value;
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

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
    const uint32_t tmem_w_scales = tmem_base + BN, tmem_x_scales = tmem_w_scales + 4 * Shape::kChunks;
    wait_for_previous_kernel();   // the weights may be what it has made
    allow_next_kernel();

    if (warp == 0 && lane == 0) {
        const unsigned char* w_scales = p.w_scales + static_cast<size_t>(row0 / 128) * p.chunks * kScaleTileBytes;
        const unsigned char* x_scales = p.x_scales + static_cast<size_t>(token0 / 128) * p.chunks * kScaleTileBytes;
        for (int i = 0, s = 0, round = 0; i < count; ++i) {
            if (round > 0 && !barrier_wait(&empty[s], (round - 1) & 1)) {
                atomicExch(&failed, 1);
                break;
            }
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
            if (++s == ring_stages) s = 0, ++round;
        }
    } else if (warp == 1 && lane == 0) {
        const uint32_t idesc = microscaled_descriptor<BITS>(BN);
        const uint32_t x_column = tmem_x_scales + static_cast<uint32_t>((token0 & 127) >> 5);
        bool ok = true;
        for (int i = 0, s = 0, round = 0; i < count; ++i) {
            if (!barrier_wait(&full[s], round & 1)) {
                atomicExch(&failed, 1);
                ok = false;
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            unsigned char* at = ring + s * Shape::kStageBytes;
            const unsigned char* scales = at + Shape::kWBytes + Shape::kXBytes;
            const int here = chunks_of(first_stage + i);
#pragma unroll
            for (int c = 0; c < Shape::kChunks; ++c) {
                if (c >= here) break;
                copy_scales(tmem_w_scales + 4 * c, scales + c * kScaleTileBytes);
                copy_scales(tmem_x_scales + 4 * c, scales + Shape::kWScaleBytes + c * kScaleTileBytes);
            }
            const uint64_t desc_w = tile_descriptor(at), desc_x = tile_descriptor(at + Shape::kWBytes);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int c = product_chunk<BITS>(k);
                if (c >= here) break;
                mma_microscaled<BITS>(tmem_base, desc_w + 2 * k, desc_x + 2 * k, idesc | product_scales<BITS>(k), tmem_w_scales + 4 * c, x_column + 4 * c, i > 0 || k > 0);
            }
            mma_commit(&empty[s]);
            if (++s == ring_stages) s = 0, ++round;
        }
        if (ok) mma_commit(accumulated);
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
                ok = __all_sync(0xffffffffu, round == 0 || barrier_wait(&empty[s], (round - 1) & 1));
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
        const bool ok = __all_sync(0xffffffffu, barrier_wait(accumulated, 0));
        if (ok) {
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
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncwarp();
    cluster_sync();   // all parts are there, or some CTA has failed and says so below
    const int tokens_here = min(BN, p.tokens - token0);
    const uint32_t part = smem_address(ring);
    uint32_t parts[kMsLargestSplit];
#pragma unroll
    for (int q = 0; q < kMsLargestSplit; ++q) {
        parts[q] = part;
        if (q < splits) asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(parts[q]) : "r"(part), "r"(q));
    }
    auto sum_of = [&](int token, int row) {
        const uint32_t offset = static_cast<uint32_t>(token * kMsRows + row) * 4u;
        float v[kMsLargestSplit], sum = 0.0f;
#pragma unroll
        for (int q = 0; q < kMsLargestSplit; ++q) v[q] = q < splits ? load_cluster(parts[q] + offset) : 0.0f;
#pragma unroll
        for (int q = 0; q < kMsLargestSplit; ++q) sum = q == 0 ? v[0] : q < splits ? sum + v[q] : sum;
        return sum;
    };
    if constexpr (!GATED) {
        const int row = threadIdx.x & 127;
        if (row0 + row < p.n) {
#pragma unroll 2
            for (int t = rank + (threadIdx.x >> 7) * splits; t < tokens_here; t += 2 * splits) {
                const float sum = sum_of(t, row);
                const size_t at = static_cast<size_t>(token0 + t) * p.n + row0 + row;
                if (p.out_is_float) static_cast<float*>(p.out)[at] = sum;
                else static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(sum);
            }
        }
    } else {
        // A warp takes a block of 32 channels of a token at a time.
        const int half = warp & 1, channel = half * 32 + lane;
        const bool exists = row0 + channel < p.n;
        for (int t = rank + (warp >> 1) * splits; t < tokens_here; t += 4 * splits) {
            const float u = sum_of(t, channel), g = sum_of(t, kMsRows / 2 + channel);
            const float h = exists ? ms_up_side(u, p.activation, p.limit) * ms_gate_side(g, p.activation, p.limit) : 0.0f;
            const int byte = scale_byte<8>(__reduce_max_sync(0xffffffffu, __float_as_uint(h) & 0x7fffffffu));
            const float scaled = byte == kNoNumber ? 0.0f : h * scale_inverse(byte);
            const int token = token0 + t, block = row0 / 32 + half;
            static_cast<unsigned char*>(p.out)[static_cast<size_t>(token) * p.out_chunks * 128 + row0 + channel] = static_cast<unsigned char>(pack_e4m3(scaled, 0.0f, 0.0f, 0.0f));
            if (lane == 0) p.out_scales[scale_word(token, block >> 2, p.out_chunks) + (block & 3)] = static_cast<unsigned char>(byte);
        }
    }
    __syncthreads();
    if (failed) {
        if (threadIdx.x == 0) report_error(p.status, kWaitTimeout);
        for (int spin = 0; spin < 2000; ++spin) __nanosleep(1000);
        __syncthreads();
    }
    cluster_sync();   // nobody leaves while another still reads its part
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(Split::kColumns) : "memory");
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

template <int BITS, int BN, bool GATED>
int launch_microscaled(const void* x, const void* w, const void* gate, MsParams p, cudaStream_t stream) {
    CUtensorMap map_w, map_gate, map_x, map_out;
    const int w_bytes = p.chunks * 64, x_bytes = p.chunks * 16 * BITS;
    if (!make_codes_map(&map_w, w, p.n, w_bytes, GATED ? kMsRows / 2 : kMsRows, BITS == 8) || !make_codes_map(&map_x, x, p.tokens, x_bytes, BN, false)) return -5;
    map_gate = map_w, map_out = map_x;
    if constexpr (GATED) {
        if (!make_codes_map(&map_gate, gate, p.n, w_bytes, kMsRows / 2, BITS == 8) ||
            !make_ms_out_map(&map_out, p.out, p.tokens, p.out_chunks * 128, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, kMsRows / 2, 32))
            return -5;
        p.row_tiles = p.out_chunks * 2;
    } else {
        const int size = p.out_is_float ? 4 : 2;
        p.bulk_store = (static_cast<size_t>(p.n) * size) % 16 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0 ? 1 : 0;
        if (p.bulk_store && !make_ms_out_map(&map_out, p.out, p.tokens, p.n, p.out_is_float ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, size,
                                             kMsRows, p.out_is_float ? 16 : 32))
            return -5;
        p.row_tiles = (p.n + kMsRows - 1) / kMsRows;
    }
    p.token_tiles = (p.tokens + BN - 1) / BN;
    auto kernel = gemm_microscaled_kernel<BITS, BN, GATED>;
    static OncePerDevice configured;
    if (allow_shared_memory(configured, kernel, MsWalk<BITS, BN>::kBytes) != cudaSuccess) return static_cast<int>(cudaGetLastError());
    const int tiles = p.row_tiles * p.token_tiles, sms = multiprocessor_count();
    return static_cast<int>(launch_overlapped(kernel, dim3(tiles < sms ? tiles : sms), dim3(kMsThreads), MsWalk<BITS, BN>::kBytes, stream, map_w, map_gate, map_x, map_out, p));
}

template <int BITS, int BN, bool GATED>
int launch_microscaled_split(const void* x, const void* w, const void* gate, MsParams p, cudaStream_t stream) {
    CUtensorMap map_w, map_gate, map_x;
    const int w_bytes = p.chunks * 64, x_bytes = p.chunks * 16 * BITS;
    if (!make_codes_map(&map_w, w, p.n, w_bytes, GATED ? kMsRows / 2 : kMsRows, BITS == 8) || !make_codes_map(&map_x, x, p.tokens, x_bytes, BN, false)) return -5;
    map_gate = map_w;
    if (GATED && !make_codes_map(&map_gate, gate, p.n, w_bytes, kMsRows / 2, BITS == 8)) return -5;
    const int row_tiles = GATED ? p.out_chunks * 2 : (p.n + kMsRows - 1) / kMsRows, token_tiles = (p.tokens + BN - 1) / BN, sms = multiprocessor_count();
    const int stages = (p.chunks + MsShape<BITS, BN>::kChunks - 1) / MsShape<BITS, BN>::kChunks;
    const int wanted = max(1, min(min(sms / (row_tiles * token_tiles), kMsLargestSplit), stages));
    const int per_split = (stages + wanted - 1) / wanted, splits = (stages + per_split - 1) / per_split;   // each has a stage at least
    int ring = min(per_split, MsSplit<BITS, BN>::kMostStages);
    // more CTAs than multiprocessors: half the ring, so that two share one
    if (row_tiles * token_tiles * splits > sms) ring = min(ring, (kMsSplitShared / 2 - 1024 - MsSplit<BITS, BN>::kSlack) / MsShape<BITS, BN>::kStageBytes);
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

// Which kernel: tiles of 128 rows x 192 tokens that fill the multiprocessors are walked; fewer are cut along K.
template <int BITS, bool GATED>
int launch_microscaled_tiles(const void* x, const void* w, const void* gate, const MsParams& p, cudaStream_t stream) {
    const int row_tiles = GATED ? p.out_chunks * 2 : (p.n + kMsRows - 1) / kMsRows, sms = multiprocessor_count();
    if (p.tokens <= 16) return launch_microscaled_split<BITS, 16, GATED>(x, w, gate, p, stream);
    if (p.tokens <= 32) return launch_microscaled_split<BITS, 32, GATED>(x, w, gate, p, stream);
    if (p.tokens <= 64) return launch_microscaled_split<BITS, 64, GATED>(x, w, gate, p, stream);
    if (p.tokens <= 128 || row_tiles * ((p.tokens + 127) / 128) <= sms / 2) return launch_microscaled_split<BITS, 128, GATED>(x, w, gate, p, stream);
    if (row_tiles * ((p.tokens + 127) / 128) <= sms) return launch_microscaled<BITS, 128, GATED>(x, w, gate, p, stream);
    return launch_microscaled<BITS, 192, GATED>(x, w, gate, p, stream);
}

}  // namespace lb

extern "C" {

// out [tokens, n] = x w^T, bfloat16 or float32.  x [tokens, 128 * chunks] in `bits` bits, w [n, 128 * chunks] in 4.
// Returns 0, a CUDA error, -2 for sizes or addresses that the kernel does not take, -5 if no tensor map could be made.
int lb_gemm_microscaled(const void* x, const void* x_scales, const void* w, const void* w_scales, void* out, int tokens, int n, int chunks, int bits, int out_is_float,
                        int* status, cudaStream_t stream) {
    if (tokens < 1 || n < 1 || chunks < 1 || chunks > (1 << 22) || (bits != 4 && bits != 8)) return -2;
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
    if (tokens < 1 || n < 1 || chunks < 1 || chunks > (1 << 22) || (bits != 4 && bits != 8) || activation < 0 || activation > 3) return -2;
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
