// e4m3 codes with one power-of-two scale for each block of 128, both contraction directions from one read of the source.
//
//   e = smallest integer with max|x| / 2^e <= 448 = 1.75 * 2^8 over the block (at least -127; 0 for a block of zeros),
//   code = e4m3(x * 2^-e), round to nearest even.  2^-e is exact and so is the product (above e4m3's subnormals), hence one
//   rounding per element and no saturation.  Integer maxima of the magnitude bits give max|x|; they order NaN above
//   infinity above every number, and a block whose maximum is not finite gets NaN for every code.
//
// HBM is the bound: 2 bytes in and 1 out per element and direction (BF16).  A CTA owns a 128 x 128 tile, the shape in which a
// row of the tile is a 1 x 128 block, a column of it a transposed block and the tile a square block; the whole tile is in
// registers after one round of loads (32 KB in flight per CTA), eight rows of one 16-byte column group per lane.  Row codes go
// straight out (128-byte segments); transposed codes pass through shared memory as 8-byte pieces (eight rows of a column),
// placed with their index exclusive-ored by the column group so that neither side has bank conflicts.  Both packings of
// 16384 x 14336 BF16 take 162 us (0.90 of the measured HBM rate), the row packing alone 107 us (1.0); of 8192 x 4096 28 us
// (0.74: 3.5 waves of tiles), of such a weight in 128 x 128 blocks 23.5 us (0.89).
#include "bf16x8.cuh"
#include "vec.cuh"

#include <algorithm>

namespace nvfp4 {

constexpr int F8_THREADS = 256;

struct Fp8Args {
    const void* x;
    uint8_t *codes, *scales, *codes_t, *scales_t;
    float* column_sums;
    int64_t rows, cols, pitch, rows_p, cols_p, col_blocks, row_blocks;
    int vector;                    // rows start on 16-byte boundaries
};

struct Fp8Scale { float inverse; uint32_t word; };      // 2^-e, and the UE8M0 byte of 2^e four times
__device__ __forceinline__ Fp8Scale fp8_scale(float amax) {
    const uint32_t bits = __float_as_uint(amax);
    if (bits >= 0x7f800000u) return {__uint_as_float(0x7fffffffu), 0x7f7f7f7fu};
    int e = static_cast<int>(bits >> 23) - 135 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    e = bits == 0 ? 0 : max(e, -127);
    return {__uint_as_float(static_cast<uint32_t>(127 - e) << 23), static_cast<uint32_t>(e + 127) * 0x01010101u};
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {       // four codes, a in the low byte
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return static_cast<uint32_t>(lo) | static_cast<uint32_t>(hi) << 16;
}
__device__ __forceinline__ float max_bits(float a, float b) { return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b))); }

// E: elements per 16-byte vector; a row is L lanes, a warp holds 32 / L rows side by side and I of them per lane.
template <typename T> struct Fp8Map {
    static constexpr int E = 16 / sizeof(T), L = 128 / E, I = 16 * L / 32;
    static constexpr int CTAS = sizeof(T) == 2 ? 4 : 2;      // per SM: 32 or 64 registers hold the tile's share of a thread
};

// Magnitude maxima as integers: 16-bit types two to a register, FP32 one.
template <typename T> struct Magnitude {
    static constexpr int PER = sizeof(T) == 2 ? 2 : 1;                 // per register
    static __device__ __forceinline__ uint32_t of(uint32_t w) { return w & (PER == 2 ? 0x7fff7fffu : 0x7fffffffu); }
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return PER == 2 ? __vmaxu2(a, b) : max(a, b); }
    static __device__ __forceinline__ uint32_t single(uint32_t m) { return PER == 2 ? max(m & 0xffffu, m >> 16) : m; }      // of a register's two
    static __device__ __forceinline__ float value(uint32_t bits) {     // FP32 of one element's magnitude bits
        if constexpr (sizeof(T) == 4) return __uint_as_float(bits);
        else if constexpr (Code<T>::value == NVFP4_BF16) return __uint_as_float(bits << 16);
        else return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
    }
};

template <typename T, bool COL, bool SQUARE>
__global__ void __launch_bounds__(F8_THREADS, Fp8Map<T>::CTAS) fp8_quantize_kernel(const Fp8Args a) {
    using M = Fp8Map<T>;
    using Mag = Magnitude<T>;
    constexpr int E = M::E, L = M::L, I = M::I;
    __shared__ __align__(16) uint8_t turned[COL ? 128 * 128 : 16];
    __shared__ float warp_cols[COL ? 8 : 1][COL ? 128 : 1], col_inverse[128], row_inverse[128];
    __shared__ uint32_t warp_best[8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
    const int64_t rb = blockIdx.x / a.col_blocks, cb = blockIdx.x - rb * a.col_blocks;
    const int cl = lane % L, part = lane / L;                 // column group, and which run of I rows of the warp's sixteen
    const int row_in = warp * 16 + part * I, col_in = cl * E;
    const int64_t row0 = rb * 128 + row_in, col0 = cb * 128 + col_in;
    const int rows_left = static_cast<int>(min(max(a.rows - row0, static_cast<int64_t>(0)), static_cast<int64_t>(I)));

    Pack<T, E> v[I];
    const T* src = static_cast<const T*>(a.x) + row0 * a.pitch + col0;
    const bool whole = a.vector && col0 + E <= a.cols;
    if (whole && rows_left == I) {
#pragma unroll
        for (int i = 0; i < I; ++i) v[i] = load_pack<T, E>(src + i * a.pitch);
    } else {
#pragma unroll
        for (int i = 0; i < I; ++i) {
            v[i] = Pack<T, E>{};
            if (i >= rows_left) continue;
            if (whole) v[i] = load_pack<T, E>(src + i * a.pitch);
            else {
#pragma unroll
                for (int j = 0; j < E; ++j)
                    if (col0 + j < a.cols) set_element(v[i], j, src[i * a.pitch + j]);
            }
        }
    }
    uint32_t row_best[I];
#pragma unroll
    for (int i = 0; i < I; ++i) {
        row_best[i] = Mag::larger(Mag::larger(Mag::of(v[i].w[0]), Mag::of(v[i].w[1])), Mag::larger(Mag::of(v[i].w[2]), Mag::of(v[i].w[3])));
    }
    Fp8Scale square{};
    if constexpr (SQUARE) {
        uint32_t best = row_best[0];
#pragma unroll
        for (int i = 1; i < I; ++i) best = Mag::larger(best, row_best[i]);
        best = __reduce_max_sync(0xffffffffu, Mag::single(best));
        if (lane == 0) warp_best[warp] = best;
        __syncthreads();
        best = 0;
#pragma unroll
        for (int w = 0; w < 8; ++w) best = max(best, warp_best[w]);
        square = fp8_scale(Mag::value(best));
    } else if (a.codes) {
        // The I rows' maxima over their L lanes, halving the rows a lane carries at each exchange: afterwards lane cl holds
        // the maximum of row cl * I / L of its run, forms its scale once, and the run's lanes read it from shared memory.
#pragma unroll
        for (int d = L / 2, n = I; d > 0; d >>= 1) {
            if (n > 1) {
                n >>= 1;
                const bool upper = cl & d;
#pragma unroll
                for (int i = 0; i < n; ++i) {
                    const uint32_t keep = upper ? row_best[i + n] : row_best[i], send = upper ? row_best[i] : row_best[i + n];
                    row_best[i] = Mag::larger(keep, __shfl_xor_sync(0xffffffffu, send, d));
                }
            } else {
                row_best[0] = Mag::larger(row_best[0], __shfl_xor_sync(0xffffffffu, row_best[0], d));
            }
        }
        const Fp8Scale s = fp8_scale(Mag::value(Mag::single(row_best[0])));
        if (cl % (L / I) == 0) {
            const int r = row_in + cl / (L / I);
            row_inverse[r] = s.inverse;
            *reinterpret_cast<uint32_t*>(a.scales + (rb * a.col_blocks + cb) * 512 + (r & 31) * 16 + (r >> 5) * 4) = s.word;
        }
        __syncwarp();
    }
    if (COL && a.column_sums) {                                // each lane's rows, then the warps' in order
#pragma unroll
        for (int j = 0; j < E; ++j) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < I; ++i) sum += element(v[i], j);
            if (L == 16) sum += __shfl_xor_sync(0xffffffffu, sum, 16);
            if (part == 0) warp_cols[warp][col_in + j] = sum;
        }
        __syncthreads();
        if (tid < 128 && cb * 128 + tid < a.cols) {
            float t = 0.f;
#pragma unroll
            for (int w = 0; w < 8; ++w) t += warp_cols[w][tid];
            a.column_sums[rb * a.cols + cb * 128 + tid] = t;
        }
        __syncthreads();
    }
    if constexpr (COL && !SQUARE) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            uint32_t best = Mag::of(v[0].w[k]);
#pragma unroll
            for (int i = 1; i < I; ++i) best = Mag::larger(best, Mag::of(v[i].w[k]));
            if (L == 16) best = Mag::larger(best, __shfl_xor_sync(0xffffffffu, best, 16));
            if (part == 0) {
                if constexpr (Mag::PER == 2) {
                    warp_cols[warp][col_in + 2 * k] = Mag::value(best & 0xffffu);
                    warp_cols[warp][col_in + 2 * k + 1] = Mag::value(best >> 16);
                } else {
                    warp_cols[warp][col_in + k] = Mag::value(best);
                }
            }
        }
    }
    if (a.codes) {
        uint8_t* out = a.codes + row0 * a.cols_p + col0;
#pragma unroll
        for (int i = 0; i < I; ++i, out += a.cols_p) {
            const float inverse = SQUARE ? square.inverse : row_inverse[row_in + i];
            float f[E];
            unpack(v[i], f);
#pragma unroll
            for (int j = 0; j < E; ++j) f[j] *= inverse;
            if (i < rows_left) {
                if constexpr (E == 8) *reinterpret_cast<uint2*>(out) = make_uint2(e4m3x4(f[0], f[1], f[2], f[3]), e4m3x4(f[4], f[5], f[6], f[7]));
                else *reinterpret_cast<uint32_t*>(out) = e4m3x4(f[0], f[1], f[2], f[3]);
            }
        }
        if (SQUARE && tid < 128) *reinterpret_cast<uint32_t*>(a.scales + (rb * a.col_blocks + cb) * 512 + tid * 4) = square.word;
    }
    if constexpr (COL) {
        if constexpr (SQUARE) {
            if (tid < 128) *reinterpret_cast<uint32_t*>(a.scales_t + (cb * a.row_blocks + rb) * 512 + tid * 4) = square.word;
        } else {
            __syncthreads();
            if (tid < 128) {
                float best = 0.f;
#pragma unroll
                for (int w = 0; w < 8; ++w) best = max_bits(best, warp_cols[w][tid]);
                const Fp8Scale s = fp8_scale(best);
                col_inverse[tid] = s.inverse;
                *reinterpret_cast<uint32_t*>(a.scales_t + (cb * a.row_blocks + rb) * 512 + (tid & 31) * 16 + (tid >> 5) * 4) = s.word;
            }
            __syncthreads();
        }
        // column c's 128 rows are sixteen 8-byte pieces; piece p lies at p ^ (c / 8)
#pragma unroll
        for (int j = 0; j < E; ++j) {
            const int c = col_in + j;
            const float inv = SQUARE ? square.inverse : col_inverse[c];
#pragma unroll
            for (int p = 0; p < I / 8; ++p) {
                float f[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = element(v[p * 8 + i], j) * inv;
                const int piece = (row_in >> 3) + p;
                *reinterpret_cast<uint2*>(turned + c * 128 + ((piece ^ (c >> 3)) & 15) * 8) =
                    make_uint2(e4m3x4(f[0], f[1], f[2], f[3]), e4m3x4(f[4], f[5], f[6], f[7]));
            }
        }
        __syncthreads();
        const int first = warp * 2 + (lane >> 4), piece = lane & 15;
        const int cols_left = static_cast<int>(min(a.cols - cb * 128, static_cast<int64_t>(128))) - first;
        uint8_t* out = a.codes_t + (cb * 128 + first) * a.rows_p + rb * 128 + piece * 8;
#pragma unroll
        for (int k = 0; k < 8; ++k, out += 16 * a.rows_p) {
            const int c = k * 16 + first;
            if (k * 16 < cols_left) *reinterpret_cast<uint2*>(out) = *reinterpret_cast<const uint2*>(turned + c * 128 + ((piece ^ (c >> 3)) & 15) * 8);
        }
    }
}

template <typename T>
static void launch_fp8(const Fp8Args& a, bool square, cudaStream_t st) {
    const unsigned grid = static_cast<unsigned>(a.row_blocks * a.col_blocks);
    if (square) {
        if (a.codes_t) fp8_quantize_kernel<T, true, true><<<grid, F8_THREADS, 0, st>>>(a);
        else fp8_quantize_kernel<T, false, true><<<grid, F8_THREADS, 0, st>>>(a);
    } else {
        if (a.codes_t) fp8_quantize_kernel<T, true, false><<<grid, F8_THREADS, 0, st>>>(a);
        else fp8_quantize_kernel<T, false, false><<<grid, F8_THREADS, 0, st>>>(a);
    }
}

}  // namespace nvfp4

using namespace nvfp4;

extern "C" int nvfp4_fp8_quantize(const void* x, int dtype, int64_t rows, int64_t cols, int64_t pitch, int square, uint8_t* codes,
                                  uint8_t* scales, uint8_t* codes_t, uint8_t* scales_t, float* column_sums, nvfp4_stream_t stream) {
    NVFP4_REQUIRE(x && (codes || codes_t) && (codes == nullptr) == (scales == nullptr) && (codes_t == nullptr) == (scales_t == nullptr),
                  NVFP4_ERR_ARG, "nvfp4_fp8_quantize: null pointer");
    NVFP4_REQUIRE(!column_sums || codes_t, NVFP4_ERR_ARG, "nvfp4_fp8_quantize: column sums come with the transposed packing");
    NVFP4_REQUIRE(rows > 0 && cols > 0 && rows < (1LL << 31) && cols < (1LL << 31) && pitch >= cols, NVFP4_ERR_ARG,
                  "nvfp4_fp8_quantize: sizes must be positive and below 2^31, the row pitch at least cols");
    NVFP4_REQUIRE(is_float_dtype(dtype), NVFP4_ERR_DTYPE, "nvfp4_fp8_quantize: FP32, BF16 or FP16 source");
    for (const void* p : {static_cast<const void*>(codes), static_cast<const void*>(scales), static_cast<const void*>(codes_t), static_cast<const void*>(scales_t)})
        NVFP4_REQUIRE(aligned(p, 16), NVFP4_ERR_ALIGN, "nvfp4_fp8_quantize: codes and scales must be 16-byte aligned");
    Fp8Args a{x, codes, scales, codes_t, scales_t, column_sums, rows, cols, pitch, round128(rows), round128(cols), (cols + 127) / 128,
              (rows + 127) / 128, aligned(x, 16) && pitch * dtype_size(dtype) % 16 == 0};
    NVFP4_REQUIRE(a.row_blocks * a.col_blocks < (1LL << 31), NVFP4_ERR_ARG, "nvfp4_fp8_quantize: more than 2^31 blocks");
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (dtype == NVFP4_BF16) launch_fp8<__nv_bfloat16>(a, square != 0, st);
    else if (dtype == NVFP4_F16) launch_fp8<__half>(a, square != 0, st);
    else launch_fp8<float>(a, square != 0, st);
    return launch_status("nvfp4_fp8_quantize");
}
