// Products of e4m3 operands with a power-of-two scale per block of 128:  out[M][N] = (A o SA) (B o SB)^T (+ bias).
//
// tcgen05.mma.kind::mxf8f6f4 multiplies a UE8M0 scale into every 32 elements of the contraction; the packings give the four
// 32-blocks of a 128-block the same byte, so the tensor cores apply the block scale themselves and accumulate in FP32 tensor
// memory, emptied into registers only where a long contraction would lose bits there (CHUNK below), without a pass of multiply-adds
// per block on the CUDA cores.
//
// Two kernels.
//   fp8_gemm_kernel        persistent clusters of two CTAs on 256 x 256 tiles (cta_group::2, M256 x N256 x K32 instructions), for
//                          problems that fill the GPU with such tiles.  A stage is 33.5 KB per SM for 512 cycles of tensor
//                          work, 65 bytes a cycle, which is what an SM takes in from L2 (measured: 64): tensor issue and
//                          operand delivery bound it together, and under the power cap the clock.  8192 x 4096 x 4096:
//                          95 us, 2.9 PFLOP/s, 0.87 of twice the measured BF16 rate.
//   fp8_gemm_split_kernel  one tile of up to 128 rows of A and 128 of B per cluster of 1 to 8 CTAs, each with a share of the
//                          contraction; the FP32 partial tiles are added through distributed shared memory in rank order.  B's
//                          rows are the 128 of the instruction and A's its columns, so that few rows of A cost what they are
//                          (sixteens).  For few rows (the weight is read once, HBM or latency is the bound) and few tiles.
//                          1 x 4096 x 4096: 8.0 us, of which launch, clusters and pipeline ends are 5.
// The host picks by the estimated time of each (split_for below).
// Operands are unpadded in M and N: tile loads beyond the tensor arrive as zeros, stores are cropped.
// Every wait is bounded as in the NVFP4 GEMM: on expiry the status word is raised, all roles leave, and the kernel returns.
#include "async.cuh"
#include "tcgen05.cuh"
#include "vec.cuh"

#include <algorithm>
#include <type_traits>

namespace nvfp4 {

constexpr int G8_BK = 128;                  // elements (and bytes) of the contraction per stage: one scale block
constexpr int G8_SF = 512;                  // bytes of a scale block: 128 rows x 4
constexpr int G8_OPERAND = 128 * 128;       // bytes of 128 rows of an operand per stage

// The tensor cores drop bits towards zero when they add to an accumulator, so a sum of terms of one sign falls behind steadily,
// and faster the longer it is (measured relative error of the paired kernel, positive operands: 5e-7 after 2048 elements, 1.4e-6
// after 4096, 9.9e-6 after 16384, 1.05e-4 after 66000; signs that cancel: 1.1e-7, 2.2e-7, 1.2e-6 after 16384).  So a contraction
// goes in chunks of CHUNK k-tiles, between which the accumulator is emptied into FP32 registers, and the error is that of one chunk
// whatever the length.  FP32 results: 2048 elements, 5e-7 (1.2e-7).  The tensor cores wait about 0.6 us for the epilogue between
// chunks: 14336 x 4096 x 8192 341 -> 364 us, 8192 x 4096 x 4096 100 -> 106; chunks of 1024 bring 1.9e-7 and cost 14 to 20 %; of
// 4096, 1.4e-6 and 4 to 5 %.  16-bit results are rounded by half a step of 3.9e-3 (BF16) or 4.9e-4 (FP16) and take 4096 elements,
// 1.4e-6; up to there they keep the one accumulator and packed registers of a kernel without chunks.  Against no chunks,
// 14336 x 4096 x 16384 BF16 comes to the other neighbour of the exact sum in 0.035 % of the elements instead of 0.12 % (a sum in
// FP32: 0.02 %), and 16384 x 4096 x 14336 takes 705 instead of 682 us; chunks of 8192: 0.07 % and 698 us.
template <typename TO> constexpr int CHUNK = sizeof(TO) == 4 ? 16 : 32;

struct Gemm8Args {
    const void* bias;
    void* out;
    int* status;
    int64_t ldo;
    int bias_dtype, M, N, k_tiles, tiles_m, tiles_n, tma_store, a_rows;      // a_rows: rows of A per tile of the split kernel
};

__device__ __forceinline__ uint32_t instr_desc8(int n, int m) {    // e4m3 x e4m3, UE8M0 scales, K-major A and B
    return (1u << 23) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
template <bool PAIR>
__device__ __forceinline__ void mma8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate, uint32_t tmem_sfa,
                                     uint32_t tmem_sfb) {
    if constexpr (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.block32 [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
            ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(tmem_sfa), "r"(tmem_sfb) : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.block32 [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
            ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(tmem_sfa), "r"(tmem_sfb) : "memory");
}
// Tile t in an order that keeps the tiles in flight near one another: eight row tiles high, so that 74 pairs of CTAs read about
// 8 + 9 operand panels at a time instead of all the rows and one column (the panels then come from L2).
__device__ __forceinline__ int2 tile_at(int t, int tiles_m, int tiles_n) {
    const int band = t / (8 * tiles_n), first = band * 8, high = min(8, tiles_m - first), in = t - band * 8 * tiles_n;
    return make_int2(first + in % high, in / high);
}
__device__ __forceinline__ float bias_at(const Gemm8Args& g, int64_t col) {
    float b[1];
    load_param<1>(g.bias, g.bias_dtype, col, b);
    return b[0];
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    const T lo = from_float<T>(a), hi = from_float<T>(b);
    return static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(&lo)) | static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(&hi)) << 16;
}

// ====================================================================================================================
// clusters of two on 256 x 256 tiles
// ====================================================================================================================
namespace pair8 {
constexpr int THREADS = 320, EPI_WARPS = 8, FIRST_EPI_WARP = 2;
constexpr int STAGES = 6;
constexpr int OPERANDS = 2 * G8_OPERAND;             // this CTA's 128 rows of A and its 128 of the tile's 256 rows of B
constexpr int SCALES = 3 * G8_SF;                    // this CTA's rows of A; all 256 rows of B
constexpr int STAGE_BYTES = OPERANDS + SCALES;
// Tensor memory: two accumulators of 256 columns that share 32 ([0, 256) and [224, 480)), so that two scale buffers of
// 4 + 8 columns fit behind them.  The epilogue reads the shared columns first, and only that read gates the next tile.
constexpr int ACC_STRIDE = 224, SF_BASE = 480, SF_COLS = 12, TMEM_COLS = 512;
// Staging of an epilogue warp: units of 32 rows x 16 columns, two of 16-bit results or one of FP32.  (FP32 as two boxes 32 bytes
// wide was slower, 4096 x 4096 x 1024 30.7 against 26.7 us; five load stages and two or three units were no faster.)
constexpr int STAGING = 2048;
constexpr int BARS = 2 * STAGES + 4;
constexpr int SMEM = STAGES * STAGE_BYTES + EPI_WARPS * STAGING + 1024 + 256;
static_assert(SF_BASE + 2 * SF_COLS <= TMEM_COLS && BARS * 8 + 16 <= 256 && SMEM <= 232448, "budgets");
}  // namespace pair8

template <typename TO, bool CHUNKS>
__global__ void __launch_bounds__(pair8::THREADS, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_sfa,
                const __grid_constant__ CUtensorMap map_sfb, const __grid_constant__ CUtensorMap map_out, const Gemm8Args g) {
    using namespace pair8;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* epi_smem = smem + STAGES * OPERANDS;
    uint8_t* sf_smem = epi_smem + EPI_WARPS * STAGING;
    uint64_t* full = reinterpret_cast<uint64_t*>(sf_smem + STAGES * SCALES);
    uint64_t* empty = full + STAGES;
    uint64_t* acc_full = empty + STAGES;
    uint64_t* shared_drained = acc_full + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(shared_drained + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int rank = static_cast<int>(cluster_rank());
    const bool leader = rank == 0;
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int a = 0; a < 2; ++a) mbar_init(&acc_full[a], 1);
        mbar_init(shared_drained, EPI_WARPS * 2);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "n"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int total_tiles = g.tiles_m * g.tiles_n;
    const int first_tile = static_cast<int>(blockIdx.x >> 1), tile_step = static_cast<int>(gridDim.x >> 1);

    if (warp == 0) {
        // ---- loads: the whole warp runs the loop, one elected lane issues; both CTAs' bytes count on the leader's barrier ----
        int stage = 0, issued = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int t = first_tile; t < total_tiles && ok; t += tile_step) {
            const int2 tile = tile_at(t, g.tiles_m, g.tiles_n);
            const int tm = tile.x * 2 + rank, tn = tile.y;
            for (int kt = 0; kt < g.k_tiles; ++kt) {
                if (!mbar_wait_warp(&empty[stage], phase ^ 1, abort_flag)) { ok = false; break; }
                if (elect_one()) {
                    uint8_t* st = smem + stage * OPERANDS;
                    uint8_t* sf = sf_smem + stage * SCALES;
                    if (leader) mbar_expect_tx(&full[stage], 2 * STAGE_BYTES);
                    tma_load_2d_pair(st, &map_a, kt * G8_BK, tm * 128, &full[stage]);
                    tma_load_2d_pair(st + G8_OPERAND, &map_b, kt * G8_BK, tn * 256 + rank * 128, &full[stage]);
                    tma_load_2d_pair(sf, &map_sfa, 0, tm * g.k_tiles + kt, &full[stage]);
                    tma_load_2d_pair(sf + G8_SF, &map_sfb, 0, tn * 2 * g.k_tiles + kt, &full[stage]);
                    tma_load_2d_pair(sf + 2 * G8_SF, &map_sfb, 0, (tn * 2 + 1) * g.k_tiles + kt, &full[stage]);
                }
                __syncwarp();
                ++issued;
                if (++stage == STAGES) { stage = 0; phase ^= 1; }
            }
        }
        if (!ok && lane == 0) {
            // loads in flight still write into this CTA's shared memory: a bounded chance to land
            const int pending = min(issued, STAGES);
            for (int i = 0; i < pending; ++i) {
                if (--stage < 0) { stage = STAGES - 1; phase ^= 1; }
                const long long t0 = clock64();
                if (leader) while (!mbar_try(&full[stage], phase) && clock64() - t0 < WAIT_CYCLES / 8) {}
            }
            const long long t0 = clock64();
            while (clock64() - t0 < 400000) {}
        }
    } else if (warp == 1) {
        // ---- MMA issue, by the leader for both CTAs; scale copies and MMAs execute in issue order ----
        if (leader) {
            const uint32_t idesc = instr_desc8(256, 256);
            int stage = 0, local = 0, sf_buf = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int t = first_tile; t < total_tiles && ok; t += tile_step) {
                for (int k0 = 0, k1; k0 < g.k_tiles && ok; k0 = k1, ++local) {       // a chunk, or the whole contraction
                    k1 = CHUNKS ? min(k0 + CHUNK<TO>, g.k_tiles) : g.k_tiles;
                    const int acc = local & 1;
                    const uint32_t tmem_acc = tmem_base + acc * ACC_STRIDE;
                    if (local > 0) {       // the shared columns of the one before are read, and with them everything of the one before that
                        if (!mbar_wait_warp(shared_drained, (local - 1) & 1, abort_flag)) { ok = false; break; }
                        tc_fence_after();
                    }
                    for (int kt = k0; kt < k1; ++kt) {
                        if (!mbar_wait_warp(&full[stage], phase, abort_flag)) { ok = false; break; }
                        tc_fence_after();
                        if (elect_one()) {
                            const uint32_t sa = smem_u32(smem + stage * OPERANDS), sb = sa + G8_OPERAND, sf = smem_u32(sf_smem + stage * SCALES);
                            const uint32_t tsfa = tmem_base + SF_BASE + sf_buf * SF_COLS, tsfb = tsfa + 4;
                            tc_cp_sf_pair(tsfa, scale_desc(sf));
                            tc_cp_sf_pair(tsfb, scale_desc(sf + G8_SF));
                            tc_cp_sf_pair(tsfb + 4, scale_desc(sf + 2 * G8_SF));
#pragma unroll
                            for (int kb = 0; kb < 4; ++kb)
                                mma8<true>(tmem_acc, operand_desc(sa + kb * 32), operand_desc(sb + kb * 32), idesc, (kt > k0 || kb) ? 1u : 0u, tsfa, tsfb);
                            tc_commit_pair(&empty[stage]);
                        }
                        __syncwarp();
                        sf_buf ^= 1;
                        if (++stage == STAGES) { stage = 0; phase ^= 1; }
                    }
                    if (ok && elect_one()) tc_commit_pair(&acc_full[acc]);
                    __syncwarp();
                }
            }
        }
    } else {
        // ---- epilogue: two warps per TMEM sub-partition, eight 16-column units of the tile each ----
        constexpr int ESZ = sizeof(TO), SLAB = 32 * 16 * ESZ, SLABS = STAGING / SLAB;
        const int sub = warp & 3, half = (warp - FIRST_EPI_WARP) >> 2;
        uint8_t* slabs = epi_smem + (warp - FIRST_EPI_WARP) * STAGING;
        int local = 0, turn = 0;
        // A unit: 32 rows x 16 columns, a row per lane, through a staging slab and a TMA store (which crops), or directly.
        // (Each lane storing its row's 32 bytes itself was slower wherever tiles end together: 4304 x 1152 x 1000 17.5 against 13.8 us.)
        auto emit = [&](const uint32_t (&w)[4 * ESZ], int64_t row, int64_t col0, int tile_row0) {
            if (g.tma_store) {
                uint8_t* slab = slabs + turn * SLAB;
                turn = turn + 1 == SLABS ? 0 : turn + 1;
                if (lane == 0) bulk_wait_read<SLABS - 1>();      // the store that last used this slab has read it
                __syncwarp();
                const int sw = (lane >> (ESZ == 2 ? 2 : 1)) & (ESZ - 1);      // the map's swizzle: 16-byte pieces by row, free of bank conflicts
#pragma unroll
                for (int c = 0; c < ESZ; ++c)
                    *reinterpret_cast<uint4*>(slab + lane * 16 * ESZ + ((c ^ sw) << 4)) = make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
                fence_async_shared();
                __syncwarp();
                if (lane == 0) { tma_store_2d(&map_out, static_cast<int>(col0), tile_row0, slab); bulk_commit(); }
            } else if (row < g.M) {
                TO* dst = static_cast<TO*>(g.out) + row * g.ldo + col0;
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (col0 + j < g.N) {
                        if constexpr (ESZ == 4) reinterpret_cast<uint32_t*>(dst)[j] = w[j];
                        else reinterpret_cast<uint16_t*>(dst)[j] = static_cast<uint16_t>(w[j >> 1] >> ((j & 1) * 16));
                    }
            }
        };
        auto release = [&] {               // this warp has read what it reads of the shared columns
            tc_fence_before();
            __syncwarp();
            if (lane == 0) { if (leader) mbar_arrive(shared_drained); else mbar_arrive_leader(shared_drained); }
        };
        auto add_bias = [&](float (&v)[16], int64_t c0) {
            if (!g.bias) return;
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (c0 + j < g.N) v[j] += bias_at(g, c0 + j);
        };
        bool ok = true;
        for (int t = first_tile; t < total_tiles && ok; t += tile_step) {
            const int2 tile = tile_at(t, g.tiles_m, g.tiles_n);
            const int tm = tile.x * 2 + rank, tn = tile.y;
            const int tile_row0 = tm * 128 + sub * 32;
            const int64_t row = tile_row0 + lane, colbase = static_cast<int64_t>(tn) * 256;
            const uint32_t lane_at = tmem_base + (static_cast<uint32_t>(sub * 32) << 16);
            if constexpr (!CHUNKS) {       // drain to packed registers, then store
                const int acc = local & 1;
                if (!mbar_wait_warp(&acc_full[acc], (local >> 1) & 1, abort_flag)) { ok = false; break; }
                tc_fence_after();
                // unit i of this warp: the shared one first (the last two of stage 0, the first two of stage 1), then seven of its own
                auto unit_of = [&](int i) { return i == 0 ? (acc == 0 ? 14 + half : half) : (acc == 0 ? 0 : 2) + half * 7 + (i - 1); };
                uint32_t packed[8][8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    uint32_t r[16];
                    tc_ld16(lane_at + acc * ACC_STRIDE + unit_of(i) * 16, r);
                    tc_wait_ld();
                    if (i == 0) release();
                    float v[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r[j]);
                    add_bias(v, colbase + unit_of(i) * 16);
#pragma unroll
                    for (int j = 0; j < 8; ++j) packed[i][j] = pack2<TO>(v[2 * j], v[2 * j + 1]);
                }
                if (tile_row0 < g.M) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int64_t col0 = colbase + unit_of(i) * 16;
                        if (col0 < g.N) emit(packed[i], row, col0, tile_row0);
                    }
                }
                ++local;
            } else {                       // eight units of its own throughout, summed over the chunks in registers, rounded once
                float sum[8][16];
                for (int k0 = 0; k0 < g.k_tiles; k0 += CHUNK<TO>, ++local) {
                    const int acc = local & 1;
                    if (!mbar_wait_warp(&acc_full[acc], (local >> 1) & 1, abort_flag)) { ok = false; break; }
                    tc_fence_after();
                    // the shared columns are the last two units of stage 0 (the upper half's) and the first two of stage 1 (the lower's)
                    const bool holds_shared = half != acc;
                    if (!holds_shared) release();
                    auto drain = [&](auto rotated) {
#pragma unroll
                        for (int o = 0; o < 8; ++o) {
                            const int u = decltype(rotated)::value ? (o + 6) & 7 : o;
                            uint32_t r[16];
                            tc_ld16(lane_at + acc * ACC_STRIDE + (half * 8 + u) * 16, r);
                            tc_wait_ld();
                            if (o == 1 && holds_shared) release();
#pragma unroll
                            for (int j = 0; j < 16; ++j) sum[u][j] = k0 ? sum[u][j] + __uint_as_float(r[j]) : __uint_as_float(r[j]);
                        }
                    };
                    if (half == 1 && acc == 0) drain(std::true_type{}); else drain(std::false_type{});
                }
                if (!ok) break;
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const int64_t col0 = colbase + (half * 8 + u) * 16;
                    if (tile_row0 >= g.M || col0 >= g.N) continue;
                    add_bias(sum[u], col0);
                    uint32_t w[4 * ESZ];
#pragma unroll
                    for (int j = 0; j < 4 * ESZ; ++j) {
                        if constexpr (ESZ == 2) w[j] = pack2<TO>(sum[u][2 * j], sum[u][2 * j + 1]);
                        else w[j] = __float_as_uint(sum[u][j]);
                    }
                    emit(w, row, col0, tile_row0);
                }
            }
        }
        if (lane == 0) bulk_wait_all();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();      // neither CTA leaves while the other may still touch its memory or barriers
    if (threadIdx.x == 0 && *abort_flag && g.status) atomicExch(g.status, NVFP4_ERR_TIMEOUT);
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "n"(TMEM_COLS) : "memory");
    }
}

// ====================================================================================================================
// one 128 x 128 tile per cluster, the contraction split over its CTAs
// ====================================================================================================================
namespace split8 {
constexpr int THREADS = 192, MAX_STAGES = 12;
constexpr int SCALES = 2 * G8_SF;
constexpr int SF_COLS = 8;
constexpr int PITCH = 132;                           // floats per row of the partial tile: lanes of a quarter warp hit different banks
constexpr int BARS = 2 * MAX_STAGES + 4;
constexpr int FIXED = 1024 + 256;
constexpr int SMEM = 6 * (2 * G8_OPERAND + SCALES) + FIXED;
// Bytes in flight are what a few rows need (their k-tiles come from HBM at its latency): fewer rows of A, more stages.
__host__ __device__ constexpr int operands(int a_rows) { return (a_rows + 128) * 128; }
__host__ __device__ constexpr int stages(int a_rows) {
    const int n = (SMEM - FIXED) / (operands(a_rows) + SCALES);
    return n < MAX_STAGES ? n : MAX_STAGES;
}
static_assert(128 * PITCH * 4 <= stages(128) * operands(128) && 16 * PITCH * 4 <= stages(16) * operands(16) && BARS * 8 + 16 <= 256 && SMEM <= 232448, "budgets");
}  // namespace split8

__device__ __forceinline__ float4 cluster_load4(uint32_t addr, int rank) {     // 16 bytes at this shared-memory offset of CTA `rank`
    uint32_t there;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(there) : "memory");
    return v;
}

template <typename TO, bool CHUNKS>
__global__ void __launch_bounds__(split8::THREADS, 1)
fp8_gemm_split_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_sfa,
                      const __grid_constant__ CUtensorMap map_sfb, const Gemm8Args g, const int splits) {
    using namespace split8;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int depth = stages(g.a_rows), stage_operands = operands(g.a_rows);
    uint8_t* sf_smem = smem + depth * stage_operands;
    uint64_t* full = reinterpret_cast<uint64_t*>(sf_smem + depth * SCALES);
    uint64_t* empty = full + depth;
    uint64_t* acc_full = empty + depth;           // two accumulators of 128 columns where the contraction goes in chunks, else one
    uint64_t* acc_free = acc_full + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_free + 2);
    constexpr int SF_BASE = CHUNKS ? 256 : 128, TMEM_COLS = 2 * SF_BASE;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int rank = splits > 1 ? static_cast<int>(cluster_rank()) : 0;
    const int tile = static_cast<int>(blockIdx.x) / splits;
    const int tm = tile % g.tiles_m, tn = tile / g.tiles_m;
    const int k0 = static_cast<int>(static_cast<int64_t>(g.k_tiles) * rank / splits), k1 = static_cast<int>(static_cast<int64_t>(g.k_tiles) * (rank + 1) / splits);
    if (threadIdx.x == 0) {
        for (int s = 0; s < depth; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int a = 0; a < 2; ++a) { mbar_init(&acc_full[a], 1); mbar_init(&acc_free[a], 4); }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "n"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0) {
        // a stage holds 128 rows of B, then a_rows of A
        bool ok = true;
        int kt = k0, stage = 0, filled = 0;
        uint32_t phase = 1;
        for (; kt < k1; ++kt) {
            if (!mbar_wait_warp(&empty[stage], phase, abort_flag)) { ok = false; break; }
            if (elect_one()) {
                uint8_t* st = smem + stage * stage_operands;
                uint8_t* sf = sf_smem + stage * SCALES;
                mbar_expect_tx(&full[stage], stage_operands + SCALES);
                tma_load_2d(st, &map_b, kt * G8_BK, tn * 128, &full[stage]);
                tma_load_2d(st + G8_OPERAND, &map_a, kt * G8_BK, tm * 128, &full[stage]);
                tma_load_2d(sf, &map_sfa, 0, tm * g.k_tiles + kt, &full[stage]);
                tma_load_2d(sf + G8_SF, &map_sfb, 0, tn * g.k_tiles + kt, &full[stage]);
            }
            __syncwarp();
            filled = min(filled + 1, depth);
            if (++stage == depth) { stage = 0; phase ^= 1; }
        }
        if (!ok && lane == 0) {      // a bounded chance for the loads in flight to land
            for (int i = 0; i < filled; ++i) {
                if (--stage < 0) { stage = depth - 1; phase ^= 1; }
                const long long t0 = clock64();
                while (!mbar_try(&full[stage], phase ^ 1) && clock64() - t0 < WAIT_CYCLES / 8) {}
            }
        }
    } else if (warp == 1) {
        const uint32_t idesc = instr_desc8(g.a_rows, 128);      // B's rows are the instruction's 128, A's its columns
        bool ok = true;
        int stage = 0;
        uint32_t phase = 0;
        for (int i0 = 0, i1, part = 0; i0 < k1 - k0 && ok; i0 = i1, ++part) {
            i1 = CHUNKS ? min(i0 + CHUNK<TO>, k1 - k0) : k1 - k0;
            const int acc = part & 1;
            if (part > 1) {                     // this accumulator's last chunk has been read
                if (!mbar_wait_warp(&acc_free[acc], ((part >> 1) - 1) & 1, abort_flag)) { ok = false; break; }
                tc_fence_after();
            }
            for (int i = i0; i < i1; ++i) {
                if (!mbar_wait_warp(&full[stage], phase, abort_flag)) { ok = false; break; }
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t sb = smem_u32(smem + stage * stage_operands), sa = sb + G8_OPERAND, sf = smem_u32(sf_smem + stage * SCALES);
                    const uint32_t tsfa = tmem_base + SF_BASE + (i & 1) * SF_COLS, tsfb = tsfa + 4;
                    tc_cp_sf(tsfa, scale_desc(sf + G8_SF));
                    tc_cp_sf(tsfb, scale_desc(sf));
#pragma unroll
                    for (int kb = 0; kb < 4; ++kb)
                        mma8<false>(tmem_base + acc * 128, operand_desc(sb + kb * 32), operand_desc(sa + kb * 32), idesc, (i > i0 || kb) ? 1u : 0u, tsfa, tsfb);
                    tc_commit(&empty[stage]);
                }
                __syncwarp();
                if (++stage == depth) { stage = 0; phase ^= 1; }
            }
            if (ok && elect_one()) tc_commit(&acc_full[acc]);
            __syncwarp();
        }
    } else {
        // Behind the last MMA every operand has been read: their shared memory takes the FP32 partial tile [rows of A][128]; a lane
        // holds a column of it.
        const uint32_t lane_at = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        float* mine = reinterpret_cast<float*>(smem) + (warp & 3) * 32 + lane;
        if constexpr (CHUNKS) {
            float sum[8][16];
            bool ok = true;
            for (int i0 = 0, part = 0; i0 < k1 - k0; i0 += CHUNK<TO>, ++part) {
                const int acc = part & 1;
                if (!mbar_wait_warp(&acc_full[acc], (part >> 1) & 1, abort_flag)) { ok = false; break; }
                tc_fence_after();
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    if (u * 16 >= g.a_rows) continue;
                    uint32_t r[16];
                    tc_ld16(lane_at + acc * 128 + u * 16, r);
                    tc_wait_ld();
#pragma unroll
                    for (int j = 0; j < 16; ++j) sum[u][j] = part ? sum[u][j] + __uint_as_float(r[j]) : __uint_as_float(r[j]);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&acc_free[acc]);
            }
            if (ok) {
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    if (u * 16 >= g.a_rows) continue;
#pragma unroll
                    for (int j = 0; j < 16; ++j) mine[(u * 16 + j) * PITCH] = sum[u][j];
                }
            }
        } else if (mbar_wait_warp(acc_full, 0, abort_flag)) {
            tc_fence_after();
            for (int u = 0; u < g.a_rows; u += 16) {
                uint32_t r[16];
                tc_ld16(lane_at + u, r);
                tc_wait_ld();
#pragma unroll
                for (int j = 0; j < 16; ++j) mine[(u + j) * PITCH] = __uint_as_float(r[j]);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (splits > 1) cluster_sync();
    if (!*abort_flag) {
        // groups of four columns of the live rows, shared out over the cluster; the partial sums are added in rank order
        const int rows = min(128, g.M - tm * 128);
        const int64_t col_tile = static_cast<int64_t>(tn) * 128;
        const uint32_t base = smem_u32(smem);
        for (int e = rank * THREADS + threadIdx.x; e < rows * 32; e += splits * THREADS) {
            const int r = e >> 5, c = (e & 31) * 4;
            const uint32_t at = base + (r * PITCH + c) * 4;
            const int64_t col = col_tile + c;
            if (col >= g.N) continue;
            float f[4];
            if (splits > 1) {
                float4 v = cluster_load4(at, 0);
                for (int s = 1; s < splits; ++s) {
                    const float4 w = cluster_load4(at, s);
                    v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
                }
                f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
            } else {
                const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem) + r * PITCH + c);
                f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
            }
            TO* dst = static_cast<TO*>(g.out) + (static_cast<int64_t>(tm) * 128 + r) * g.ldo + col;
            if (g.bias) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (col + j < g.N) f[j] += bias_at(g, col + j);
            }
            if (col + 4 <= g.N && (reinterpret_cast<uintptr_t>(dst) & (4 * sizeof(TO) - 1)) == 0) {
                store_pack(dst, pack<TO, 4>(f));
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (col + j < g.N) dst[j] = from_float<TO>(f[j]);
            }
        }
    }
    __syncthreads();
    if (splits > 1) cluster_sync();      // a CTA's partial tile stays until the others have read it
    if (threadIdx.x == 0 && *abort_flag && g.status) atomicExch(g.status, NVFP4_ERR_TIMEOUT);
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "n"(TMEM_COLS) : "memory");
    }
}

// ---- host side -------------------------------------------------------------------------------------------------------
static bool map_2d(CUtensorMap* map, CUtensorMapDataType type, const void* base, int64_t inner, int64_t outer, int64_t pitch_bytes, int box_inner,
                   int box_outer, CUtensorMapSwizzle swizzle) {
    aop::EncodeTiledFn fn = aop::encode_fn();
    if (!fn) return false;
    cuuint64_t dims[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer)};
    cuuint64_t strides[1] = {static_cast<cuuint64_t>(pitch_bytes)};
    cuuint32_t box[2] = {static_cast<cuuint32_t>(box_inner), static_cast<cuuint32_t>(box_outer)};
    cuuint32_t one[2] = {1, 1};
    return fn(map, type, 2, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
static bool operand_map(CUtensorMap* map, const uint8_t* base, int64_t rows, int64_t k, int box_rows) {
    return map_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, k, rows, k, G8_BK, box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}
static bool scale_map(CUtensorMap* map, const uint8_t* base, int64_t rows, int64_t k) {      // one 512-byte block per row
    return map_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, base, G8_SF / 4, (rows + 127) / 128 * (k / 128), G8_SF, G8_SF / 4, 1, CU_TENSOR_MAP_SWIZZLE_NONE);
}

// 0: paired CTAs on 256 x 256 tiles; else the number of CTAs that share a tile's contraction.  The smallest of the times that a
// fit to measurements gives, in ns (16 shapes from 1 x 4096 x 128 to 16384 x 4096 x 14336; within 20 %, and the fastest way
// picked for each): paired, 8 us and 360 ns per k-tile of every wave (its tensor time at 1.4 GHz); split, 1.5 us and per wave
// a start and end of 2 to 4.5 us (3.2 to 6.5 in a cluster) and 240 to 390 ns per k-tile by the rows of A, which is the
// operands' way from L2 rather than their products.  For example 1 x 4096 x 4096: paired 17.0 us, one CTA a tile 10.7, two 8.8,
// four 8.0, eight (three waves of clusters) 17.3; 1000 x 1152 x 4304: 18.0, 15.8, 13.6, 31.1; 2048 x 2048 x 2048: 13.8, 22.2.
struct Slots { int clusters[4]; int pairs; };        // tiles in flight: split clusters of 1, 2, 4, 8 CTAs; paired CTAs
static int split_for(const Gemm8Args& g, const Slots& slots) {
    auto waves = [](int64_t work, int64_t slots) { return (work + slots - 1) / slots; };
    const int64_t pair_waves = waves(static_cast<int64_t>((g.M + 255) / 256) * ((g.N + 255) / 256), slots.pairs);
    int64_t best = 8000 + pair_waves * g.k_tiles * 360 + (pair_waves - 1) * 600;
    int pick = 0;
    const int64_t tiles = static_cast<int64_t>((g.M + 127) / 128) * ((g.N + 127) / 128);
    for (int s = 1, i = 0; s <= 8 && s <= g.k_tiles && slots.clusters[i]; s *= 2, ++i) {
        const int64_t ends = s > 1 ? 3200 + 26 * g.a_rows : 2000 + 20 * g.a_rows;
        const int64_t cost = 1500 + waves(tiles, slots.clusters[i]) * (ends + waves(g.k_tiles, s) * (240 + g.a_rows * 6 / 5));
        if (cost < best) { best = cost; pick = s; }
    }
    return pick;
}

template <typename TO, bool CHUNKS>
static int launch_gemm8(Gemm8Args& g, const uint8_t* a, const CUtensorMap& mb, const CUtensorMap& msa, const CUtensorMap& msb, cudaStream_t st) {
    int dev = 0;
    cudaGetDevice(&dev);
    static bool configured[64] = {};
    static Slots slots[64] = {};
    NVFP4_REQUIRE(dev >= 0 && dev < 64, NVFP4_ERR_UNSUPPORTED, "nvfp4_fp8_gemm: device index above 63");
    if (!configured[dev]) {
        cudaError_t e = cudaFuncSetAttribute(fp8_gemm_kernel<TO, CHUNKS>, cudaFuncAttributeMaxDynamicSharedMemorySize, pair8::SMEM);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(fp8_gemm_split_kernel<TO, CHUNKS>, cudaFuncAttributeMaxDynamicSharedMemorySize, split8::SMEM);
        // clusters do not fill every SM (a group of SMs holds whole clusters only): what the device says it runs at once
        cudaLaunchConfig_t c = {};
        cudaLaunchAttribute size[1];
        size[0].id = cudaLaunchAttributeClusterDimension;
        size[0].val.clusterDim.y = size[0].val.clusterDim.z = 1;
        c.attrs = size;
        c.numAttrs = 1;
        for (int i = 0; i < 4 && e == cudaSuccess; ++i) {
            size[0].val.clusterDim.x = 1 << i;
            c.gridDim = dim3(8);
            c.blockDim = dim3(split8::THREADS);
            c.dynamicSmemBytes = split8::SMEM;
            e = cudaOccupancyMaxActiveClusters(&slots[dev].clusters[i], fp8_gemm_split_kernel<TO, CHUNKS>, &c);
        }
        if (e == cudaSuccess) {
            size[0].val.clusterDim.x = 2;
            c.blockDim = dim3(pair8::THREADS);
            c.dynamicSmemBytes = pair8::SMEM;
            e = cudaOccupancyMaxActiveClusters(&slots[dev].pairs, fp8_gemm_kernel<TO, CHUNKS>, &c);
        }
        NVFP4_REQUIRE(e == cudaSuccess && slots[dev].pairs > 0, NVFP4_ERR_LAUNCH, "nvfp4_fp8_gemm: cannot configure the kernels: %s", cudaGetErrorString(e));
        configured[dev] = true;
    }
    const int splits = split_for(g, slots[dev]);
    CUtensorMap ma;
    NVFP4_REQUIRE(operand_map(&ma, a, g.M, g.k_tiles * static_cast<int64_t>(G8_BK), splits ? g.a_rows : 128), NVFP4_ERR_LAUNCH,
                  "nvfp4_fp8_gemm: cuTensorMapEncodeTiled failed or is unavailable");
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaError_t e;
    if (splits == 0) {
        g.tiles_m = (g.M + 255) / 256;
        g.tiles_n = (g.N + 255) / 256;
        CUtensorMap mo = ma;           // unused without tma_store, but the parameter must hold a valid map
        constexpr int ESZ = sizeof(TO);
        g.tma_store = aligned(g.out, 16) && g.ldo * ESZ % 16 == 0 &&
                      map_2d(&mo, ESZ == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, g.out, g.N, g.M, g.ldo * ESZ, 16, 32,
                             ESZ == 4 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B);
        attr[0].val.clusterDim.x = 2;
        cfg.gridDim = dim3(static_cast<unsigned>(2 * std::min<int64_t>(static_cast<int64_t>(g.tiles_m) * g.tiles_n, slots[dev].pairs)));
        cfg.blockDim = dim3(pair8::THREADS);
        cfg.dynamicSmemBytes = pair8::SMEM;
        e = cudaLaunchKernelEx(&cfg, fp8_gemm_kernel<TO, CHUNKS>, ma, mb, msa, msb, mo, g);
    } else {
        g.tiles_m = (g.M + 127) / 128;
        g.tiles_n = (g.N + 127) / 128;
        attr[0].val.clusterDim.x = splits;
        cfg.gridDim = dim3(static_cast<unsigned>(g.tiles_m * g.tiles_n * splits));
        cfg.blockDim = dim3(split8::THREADS);
        cfg.dynamicSmemBytes = split8::SMEM;
        e = cudaLaunchKernelEx(&cfg, fp8_gemm_split_kernel<TO, CHUNKS>, ma, mb, msa, msb, g, splits);
    }
    NVFP4_REQUIRE(e == cudaSuccess, NVFP4_ERR_LAUNCH, "nvfp4_fp8_gemm: cluster launch failed: %s", cudaGetErrorString(e));
    return launch_status("nvfp4_fp8_gemm");
}

}  // namespace nvfp4

using namespace nvfp4;

extern "C" int nvfp4_fp8_gemm(const uint8_t* a, const uint8_t* a_scales, const uint8_t* b, const uint8_t* b_scales, int64_t M, int64_t N, int64_t K,
                              const void* bias, int bias_dtype, void* out, int out_dtype, int64_t ldo, int* status, nvfp4_stream_t stream) {
    NVFP4_REQUIRE(a && a_scales && b && b_scales && out, NVFP4_ERR_ARG, "nvfp4_fp8_gemm: null pointer");
    NVFP4_REQUIRE(M > 0 && N > 0 && K > 0 && K % 128 == 0 && ldo >= N, NVFP4_ERR_ARG,
                  "nvfp4_fp8_gemm: M, N and K must be positive, K a multiple of 128, ldo at least N (got %lld %lld %lld %lld)", (long long)M, (long long)N,
                  (long long)K, (long long)ldo);
    // tile coordinates and scale-block indices are 32-bit
    NVFP4_REQUIRE(M < (1LL << 30) && N < (1LL << 30) && K < (1LL << 30) && ((M + 255) / 128 + 1) * (K / 128) < (1LL << 31) &&
                  ((N + 255) / 128 + 1) * (K / 128) < (1LL << 31) && ((M + 127) / 128) * ((N + 127) / 128) < (1LL << 27), NVFP4_ERR_ARG,
                  "nvfp4_fp8_gemm: sizes exceed the tile index range");
    NVFP4_REQUIRE(is_float_dtype(out_dtype) && (!bias || is_float_dtype(bias_dtype)), NVFP4_ERR_DTYPE, "nvfp4_fp8_gemm: FP32, BF16 or FP16 result and bias");
    for (const void* p : {static_cast<const void*>(a), static_cast<const void*>(a_scales), static_cast<const void*>(b), static_cast<const void*>(b_scales)})
        NVFP4_REQUIRE(aligned(p, 16), NVFP4_ERR_ALIGN, "nvfp4_fp8_gemm: operands and scales must be 16-byte aligned");
    NVFP4_REQUIRE(aligned(out, dtype_size(out_dtype)) && aligned(bias, bias ? dtype_size(bias_dtype) : 1), NVFP4_ERR_ALIGN,
                  "nvfp4_fp8_gemm: result and bias must be aligned to their elements");
    Gemm8Args g{bias, out, status, ldo, bias_dtype, static_cast<int>(M), static_cast<int>(N), static_cast<int>(K / 128), 0, 0, 0, 128};
    g.a_rows = M < 128 ? static_cast<int>((M + 15) / 16 * 16) : 128;
    CUtensorMap mb, msa, msb;
    NVFP4_REQUIRE(operand_map(&mb, b, N, K, 128) && scale_map(&msa, a_scales, M, K) && scale_map(&msb, b_scales, N, K),
                  NVFP4_ERR_LAUNCH, "nvfp4_fp8_gemm: cuTensorMapEncodeTiled failed or is unavailable");
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const bool chunks = g.k_tiles > CHUNK<__half>;
    if (out_dtype == NVFP4_BF16) return chunks ? launch_gemm8<__nv_bfloat16, true>(g, a, mb, msa, msb, st) : launch_gemm8<__nv_bfloat16, false>(g, a, mb, msa, msb, st);
    if (out_dtype == NVFP4_F16) return chunks ? launch_gemm8<__half, true>(g, a, mb, msa, msb, st) : launch_gemm8<__half, false>(g, a, mb, msa, msb, st);
    return launch_gemm8<float, true>(g, a, mb, msa, msb, st);
}

extern "C" int64_t nvfp4_fp8_packing_bytes(int64_t rows, int64_t k) {
    const int64_t kp = round128(k);
    return rows * kp + round128(rows) / 128 * (kp / 128) * G8_SF;
}

static uint8_t* scales_of(const uint8_t* packing, int64_t rows, int64_t k) { return const_cast<uint8_t*>(packing) + rows * round128(k); }

extern "C" int nvfp4_fp8_linear(const void* x, int x_dtype, int64_t m, int64_t k, int64_t x_pitch, const void* w, int w_dtype, int64_t n,
                                int64_t w_pitch, const void* bias, int bias_dtype, void* y, uint8_t* work, uint8_t* x_t, uint8_t* w_t, int* status,
                                nvfp4_stream_t stream) {
    NVFP4_REQUIRE(x && w && y && work, NVFP4_ERR_ARG, "nvfp4_fp8_linear: null pointer");
    NVFP4_REQUIRE(m > 0 && n > 0 && k > 0, NVFP4_ERR_ARG, "nvfp4_fp8_linear: sizes must be positive");
    const bool packed = w_dtype == NVFP4_E4M3;
    NVFP4_REQUIRE(!packed || !w_t, NVFP4_ERR_ARG, "nvfp4_fp8_linear: a packed weight has its transpose already");
    uint8_t* wq = packed ? static_cast<uint8_t*>(const_cast<void*>(w)) : work + nvfp4_fp8_packing_bytes(m, k);
    int rc = nvfp4_fp8_quantize(x, x_dtype, m, k, x_pitch, 0, work, scales_of(work, m, k), x_t, x_t ? scales_of(x_t, k, m) : nullptr, nullptr, stream);
    if (!rc && !packed)
        rc = nvfp4_fp8_quantize(w, w_dtype, n, k, w_pitch, 1, wq, scales_of(wq, n, k), w_t, w_t ? scales_of(w_t, k, n) : nullptr, nullptr, stream);
    if (!rc)
        rc = nvfp4_fp8_gemm(work, scales_of(work, m, k), wq, scales_of(wq, n, k), m, n, round128(k), bias, bias_dtype, y, x_dtype, n, status, stream);
    return rc;
}

extern "C" int nvfp4_fp8_linear_bwd(const void* dy, int dtype, int64_t m, int64_t n, int64_t k, int64_t dy_pitch, const uint8_t* x_t,
                                    const uint8_t* w_t, void* dx, void* dw, int dw_dtype, void* dbias, int dbias_dtype, uint8_t* work, int* status,
                                    nvfp4_stream_t stream) {
    NVFP4_REQUIRE(dy && work && (dx || dw || dbias) && (!dx || w_t) && (!dw || x_t), NVFP4_ERR_ARG, "nvfp4_fp8_linear_bwd: null pointer");
    NVFP4_REQUIRE(m > 0 && n > 0 && k > 0, NVFP4_ERR_ARG, "nvfp4_fp8_linear_bwd: sizes must be positive");
    uint8_t* g = dx ? work : nullptr;
    uint8_t* g_t = dw || dbias ? work + (dx ? nvfp4_fp8_packing_bytes(m, n) : 0) : nullptr;
    float* sums = dbias ? reinterpret_cast<float*>(g_t + nvfp4_fp8_packing_bytes(n, m)) : nullptr;
    int rc = nvfp4_fp8_quantize(dy, dtype, m, n, dy_pitch, 0, g, g ? scales_of(g, m, n) : nullptr, g_t, g_t ? scales_of(g_t, n, m) : nullptr, sums, stream);
    if (!rc && dx) rc = nvfp4_fp8_gemm(g, scales_of(g, m, n), w_t, scales_of(w_t, k, n), m, k, round128(n), nullptr, 0, dx, dtype, k, status, stream);
    if (!rc && dw) rc = nvfp4_fp8_gemm(g_t, scales_of(g_t, n, m), x_t, scales_of(x_t, k, m), n, k, round128(m), nullptr, 0, dw, dw_dtype, k, status, stream);
    if (!rc && dbias) rc = nvfp4_column_sums(sums, round128(m) / 128, n, dbias, dbias_dtype, stream);
    return rc;
}
