// Layer norm with the residual sum in front of it, forward and backward.
//
//   total = x + delta,  h = (total - mean) * rstd * w + b,   mean, var over the row, rstd = 1 / sqrt(var + eps)
//   with z = (total - mean) * rstd, u = dh * w:   dx = rstd * (u - mean(u) - z * mean(u z)) + dsum,  dw = sum dh z,  db = sum dh
//
// Both directions stream: every operand is read once and every result written once, so HBM is the bound.  A row stays in
// registers between the sweeps over it (sum, centred squares, result), held by one warp up to 256 vectors of 16 bytes and by
// one CTA above that; the centred second sweep keeps the variance exact where the mean is large against the spread.  All
// statistics are FP32; a result is rounded once, except that h is formed from the total as it is stored (the backward pass
// reads that one too).
#include "bf16x8.cuh"
#include "vec.cuh"

#include <algorithm>

namespace nvfp4 {

struct NormArgs {
    const void *x, *delta, *weight, *bias;
    void *sum, *h;
    float *mean, *rstd, *amax;
    int64_t x_pitch, delta_pitch, rows;
    int cols, delta_bf16, weight_dtype;   // delta_bf16: a BF16 delta beside an FP32 x
    float eps;
};

// Sum over the CTA in a fixed order, every thread gets it.  One barrier: callers alternate between two `slots` arrays, and
// the barrier of the other one lies between a slot's last read and its next write.
__device__ __forceinline__ float cta_sum(float v, float* slots) {
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    v = warp_sum(v);
    if (lane == 0) slots[threadIdx.x >> 5] = v;
    __syncthreads();
    return warp_sum(lane < warps ? slots[lane] : 0.f);
}

// V elements of total at column c of row r (stored, too, when there is a delta), as FP32
template <typename TX, int V>
__device__ __forceinline__ void load_total(const NormArgs& a, int64_t r, int c, float (&f)[V]) {
    Pack<TX, V> p = load_pack<TX, V>(static_cast<const TX*>(a.x) + r * a.x_pitch + c);
    unpack(p, f);
    if (a.delta) {
        float d[V];
        if (sizeof(TX) == 4 && a.delta_bf16) unpack(load_pack<__nv_bfloat16, V>(static_cast<const __nv_bfloat16*>(a.delta) + r * a.delta_pitch + c), d);
        else unpack(load_pack<TX, V>(static_cast<const TX*>(a.delta) + r * a.delta_pitch + c), d);
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] += d[j];
        p = pack<TX, V>(f);
        store_pack(static_cast<TX*>(a.sum) + r * a.cols + c, p);
        unpack(p, f);
    }
}
template <typename TO, int V>
__device__ __forceinline__ float store_normed(const NormArgs& a, int64_t r, int c, const float (&f)[V], float mean, float rstd) {
    float o[V], p[V];
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = (f[j] - mean) * rstd;
    if (a.weight) {
        load_param<V>(a.weight, a.weight_dtype, c, p);
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] *= p[j];
    }
    if (a.bias) {
        load_param<V>(a.bias, a.weight_dtype, c, p);
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] += p[j];
    }
    const Pack<TO, V> q = pack<TO, V>(o);
    store_pack(static_cast<TO*>(a.h) + r * a.cols + c, q);
    return abs_max(q);
}

// N vectors of V elements per thread; ROW_CTA: a CTA per row, else a warp per row.
template <typename TX, typename TO, int V, int N, bool ROW_CTA>
__global__ void __launch_bounds__(ROW_CTA ? 1024 : 256) norm_fwd_kernel(const NormArgs a) {
    __shared__ float slots[2][32];
    const int tid = ROW_CTA ? threadIdx.x : (threadIdx.x & 31), step = ROW_CTA ? blockDim.x : 32;
    const int64_t row0 = ROW_CTA ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const int64_t row_step = ROW_CTA ? gridDim.x : static_cast<int64_t>(gridDim.x) * 8;
    const int vectors = a.cols / V;
    const float inv_n = 1.f / static_cast<float>(a.cols);
    float best = 0.f;
    for (int64_t r = row0; r < a.rows; r += row_step) {
        float f[N][V];
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = tid + i * step;
            if (c < vectors) {
                load_total<TX, V>(a, r, c * V, f[i]);
#pragma unroll
                for (int j = 0; j < V; ++j) s += f[i][j];
            }
        }
        const float mean = (ROW_CTA ? cta_sum(s, slots[0]) : warp_sum(s)) * inv_n;
        float sq = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (tid + i * step < vectors) {
#pragma unroll
                for (int j = 0; j < V; ++j) { const float d = f[i][j] - mean; sq = fmaf(d, d, sq); }
            }
        const float rstd = rsqrtf((ROW_CTA ? cta_sum(sq, slots[1]) : warp_sum(sq)) * inv_n + a.eps);
        if (tid == 0 && a.mean) { a.mean[r] = mean; a.rstd[r] = rstd; }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = tid + i * step;
            if (c < vectors) best = fmaxf(best, store_normed<TO, V>(a, r, c * V, f[i], mean, rstd));
        }
    }
    if (a.amax) block_atomic_amax(a.amax, best);
}

// Any width: a CTA per row, one element at a time, the row read again for each sweep (from L1 / L2).
template <typename TX, typename TO>
__global__ void __launch_bounds__(256) norm_fwd_any_kernel(const NormArgs a) {
    __shared__ float slots[2][32];
    float best = 0.f;
    const TX* total = static_cast<const TX*>(a.delta ? a.sum : a.x);
    const int64_t pitch = a.delta ? a.cols : a.x_pitch;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        float s = 0.f, sq = 0.f;
        for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
            float f[1];
            load_total<TX, 1>(a, r, c, f);
            s += f[0];
        }
        const float mean = cta_sum(s, slots[0]) / static_cast<float>(a.cols);
        for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {       // a thread reads back only what it wrote itself
            const float d = to_float(total[r * pitch + c]) - mean;
            sq = fmaf(d, d, sq);
        }
        const float rstd = rsqrtf(cta_sum(sq, slots[1]) / static_cast<float>(a.cols) + a.eps);
        if (threadIdx.x == 0 && a.mean) { a.mean[r] = mean; a.rstd[r] = rstd; }
        for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
            const float f[1] = {to_float(total[r * pitch + c])};
            best = fmaxf(best, store_normed<TO, 1>(a, r, c, f, mean, rstd));
        }
    }
    if (a.amax) block_atomic_amax(a.amax, best);
}

// ---- backward ---------------------------------------------------------------------------------------------------------
struct NormBwdArgs {
    const void *dh, *total, *weight, *dsum;
    const float *mean, *rstd;
    void *dx, *ddelta;
    float *partial, *amax;     // partial: [parts][2][cols], null when neither dw nor db is asked for
    int64_t dh_pitch, total_pitch, dsum_pitch, rows;
    int cols, weight_dtype;
};

// dx of V elements from the row's two means; returns max |what the producer of x's branch receives|
template <typename TX, int V>
__device__ __forceinline__ float store_dx(const NormBwdArgs& a, int64_t r, int c, const float (&u)[V], const float (&z)[V], float rstd,
                                          float mean_u, float mean_uz, const Pack<TX, V>& dsum) {
    float o[V], d[V];
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = rstd * (u[j] - mean_u - z[j] * mean_uz);
    if (a.dsum) {
        unpack(dsum, d);
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] += d[j];
    }
    const Pack<TX, V> q = pack<TX, V>(o);
    store_pack(static_cast<TX*>(a.dx) + r * a.cols + c, q);
    if (sizeof(TX) == 4 && a.ddelta) {
        const Pack<__nv_bfloat16, V> qd = pack<__nv_bfloat16, V>(o);
        store_pack(static_cast<__nv_bfloat16*>(a.ddelta) + r * a.cols + c, qd);
        return abs_max(qd);
    }
    return abs_max(q);
}

// Every thread owns N vectors of V columns for all rows its group (a warp, or the CTA) takes, so the column sums stay in
// registers; a group has R rows in flight.  The CTA's sums go out as one partial row, added up in a fixed order by
// column_sums_kernel.
template <typename TX, typename TH, int V, int N, int R, bool ROW_CTA>
__global__ void __launch_bounds__(ROW_CTA ? 512 : 256) norm_bwd_kernel(const NormBwdArgs a) {
    __shared__ float slots[2][2 * R][16];
    __shared__ float cols_sum[ROW_CTA ? 1 : 2 * 32 * N * V];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int tid = ROW_CTA ? threadIdx.x : lane, step = ROW_CTA ? blockDim.x : 32;
    const int64_t row0 = (ROW_CTA ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * warps + warp) * R;
    const int64_t row_step = (ROW_CTA ? gridDim.x : static_cast<int64_t>(gridDim.x) * warps) * R;
    const int vectors = a.cols / V;
    const float inv_n = 1.f / static_cast<float>(a.cols);
    float acc_w[N][V], acc_b[N][V];
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) acc_w[i][j] = acc_b[i][j] = 0.f;
    float best = 0.f;
    int phase = 0;
    for (int64_t r0 = row0; r0 < a.rows; r0 += row_step, phase ^= 1) {
        Pack<TH, V> pg[R][N];
        Pack<TX, V> ps[R][N], pd[R][N];
        float mean[R], rstd[R];
#pragma unroll
        for (int k = 0; k < R; ++k) {
            const int64_t r = r0 + k;
            mean[k] = r < a.rows ? a.mean[r] : 0.f;
            rstd[k] = r < a.rows ? a.rstd[r] : 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int c = tid + i * step;
                const bool live = r < a.rows && c < vectors;
                pg[k][i] = Pack<TH, V>{}; ps[k][i] = Pack<TX, V>{}; pd[k][i] = Pack<TX, V>{};
                if (live) {
                    pg[k][i] = load_pack<TH, V>(static_cast<const TH*>(a.dh) + r * a.dh_pitch + c * V);
                    ps[k][i] = load_pack<TX, V>(static_cast<const TX*>(a.total) + r * a.total_pitch + c * V);
                    if (a.dsum) pd[k][i] = load_pack<TX, V>(static_cast<const TX*>(a.dsum) + r * a.dsum_pitch + c * V);
                }
            }
        }
        auto weights = [&](int i, float (&w)[V]) {
#pragma unroll
            for (int j = 0; j < V; ++j) w[j] = 1.f;
            if (a.weight && tid + i * step < vectors) load_param<V>(a.weight, a.weight_dtype, (tid + i * step) * V, w);
        };
        float su[R], suz[R];
#pragma unroll
        for (int k = 0; k < R; ++k) su[k] = suz[k] = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float w[V];
            weights(i, w);
#pragma unroll
            for (int k = 0; k < R; ++k) {
                float g[V], s[V];
                unpack(pg[k][i], g); unpack(ps[k][i], s);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float z = (s[j] - mean[k]) * rstd[k], u = g[j] * w[j];
                    su[k] += u;
                    suz[k] = fmaf(u, z, suz[k]);
                    acc_w[i][j] = fmaf(g[j], z, acc_w[i][j]);
                    acc_b[i][j] += g[j];
                }
            }
        }
#pragma unroll
        for (int k = 0; k < R; ++k) {
            su[k] = warp_sum(su[k]); suz[k] = warp_sum(suz[k]);
            if (ROW_CTA && lane == 0) { slots[phase][2 * k][warp] = su[k]; slots[phase][2 * k + 1][warp] = suz[k]; }
        }
        if constexpr (ROW_CTA) {      // one barrier a round: the next round writes the other half of `slots`
            __syncthreads();
#pragma unroll
            for (int k = 0; k < R; ++k) {
                su[k] = warp_sum(lane < warps ? slots[phase][2 * k][lane & 15] : 0.f);
                suz[k] = warp_sum(lane < warps ? slots[phase][2 * k + 1][lane & 15] : 0.f);
            }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = tid + i * step;
            if (c >= vectors) continue;
            float w[V];
            weights(i, w);
#pragma unroll
            for (int k = 0; k < R; ++k) {
                if (r0 + k >= a.rows) continue;
                float u[V], z[V];
                unpack(pg[k][i], u); unpack(ps[k][i], z);
#pragma unroll
                for (int j = 0; j < V; ++j) { u[j] *= w[j]; z[j] = (z[j] - mean[k]) * rstd[k]; }
                best = fmaxf(best, store_dx<TX, V>(a, r0 + k, c * V, u, z, rstd[k], su[k] * inv_n, suz[k] * inv_n, pd[k][i]));
            }
        }
    }
    if (a.amax) block_atomic_amax(a.amax, best);
    if (!a.partial) return;
    float* out = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * a.cols;
    if constexpr (ROW_CTA) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = tid + i * step;
            if (c >= vectors) continue;
#pragma unroll
            for (int j = 0; j < V; ++j) { out[c * V + j] = acc_w[i][j]; out[a.cols + c * V + j] = acc_b[i][j]; }
        }
    } else {
        for (int w = 0; w < warps; ++w) {       // the warps' sums are added in warp order
            if (warp == w) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int c = lane + i * 32;
                    if (c >= vectors) continue;
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        float* sw = cols_sum + c * V + j;
                        float* sb = sw + 32 * N * V;
                        *sw = w ? *sw + acc_w[i][j] : acc_w[i][j];
                        *sb = w ? *sb + acc_b[i][j] : acc_b[i][j];
                    }
                }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < a.cols; c += blockDim.x) { out[c] = cols_sum[c]; out[a.cols + c] = cols_sum[32 * N * V + c]; }
    }
}

// Any width: dx by a CTA per row, the row read twice; the column sums by a pass of their own.
template <typename TX, typename TH>
__global__ void __launch_bounds__(256) norm_bwd_any_kernel(const NormBwdArgs a) {
    __shared__ float slots[2][32];
    const float inv_n = 1.f / static_cast<float>(a.cols);
    float best = 0.f;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const float mean = a.mean[r], rstd = a.rstd[r];
        const TH* dh = static_cast<const TH*>(a.dh) + r * a.dh_pitch;
        const TX* total = static_cast<const TX*>(a.total) + r * a.total_pitch;
        auto uz = [&](int c, float& u, float& z) {
            float w[1] = {1.f};
            if (a.weight) load_param<1>(a.weight, a.weight_dtype, c, w);
            u = to_float(dh[c]) * w[0];
            z = (to_float(total[c]) - mean) * rstd;
        };
        float su = 0.f, suz = 0.f;
        for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
            float u, z;
            uz(c, u, z);
            su += u;
            suz = fmaf(u, z, suz);
        }
        su = cta_sum(su, slots[0]) * inv_n;
        suz = cta_sum(suz, slots[1]) * inv_n;
        for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
            float u[1], z[1];
            uz(c, u[0], z[0]);
            Pack<TX, 1> d{};
            if (a.dsum) d = load_pack<TX, 1>(static_cast<const TX*>(a.dsum) + r * a.dsum_pitch + c);
            best = fmaxf(best, store_dx<TX, 1>(a, r, c, u, z, rstd, su, suz, d));
        }
    }
    if (a.amax) block_atomic_amax(a.amax, best);
}
template <typename TX, typename TH>
__global__ void __launch_bounds__(256) norm_bwd_columns_kernel(const NormBwdArgs a) {
    __shared__ float subtotal[2][8][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + lane;
    float sw = 0.f, sb = 0.f;
    if (c < a.cols) {
#pragma unroll 4
        for (int64_t r = static_cast<int64_t>(blockIdx.y) * 8 + warp; r < a.rows; r += static_cast<int64_t>(gridDim.y) * 8) {
            const float g = to_float(static_cast<const TH*>(a.dh)[r * a.dh_pitch + c]);
            const float z = (to_float(static_cast<const TX*>(a.total)[r * a.total_pitch + c]) - a.mean[r]) * a.rstd[r];
            sw = fmaf(g, z, sw);
            sb += g;
        }
    }
    subtotal[0][warp][lane] = sw;
    subtotal[1][warp][lane] = sb;
    __syncthreads();
    if (warp < 2 && c < a.cols) {
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) t += subtotal[warp][w][lane];
        a.partial[(static_cast<int64_t>(blockIdx.y) * 2 + warp) * a.cols + c] = t;
    }
}

// out[c] = sum of `parts` rows of `width` floats, columns [0, cols) to out0 and [cols, 2 cols) to out1 (either may be null).
// A CTA takes 32 columns, its eight warps every eighth row each, the eight subtotals are added in warp order.
__global__ void __launch_bounds__(256) column_sums_kernel(const float* __restrict__ partial, int64_t parts, int64_t width, int64_t cols,
                                                          void* out0, void* out1, int dtype) {
    __shared__ float subtotal[8][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    float t = 0.f;
    if (c < width) {
#pragma unroll 8
        for (int64_t p = warp; p < parts; p += 8) t += partial[p * width + c];
    }
    subtotal[warp][lane] = t;
    __syncthreads();
    if (warp != 0 || c >= width) return;
    float total = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) total += subtotal[w][lane];
    void* out = c < cols ? out0 : out1;
    if (out) store_param(out, dtype, c < cols ? c : c - cols, total);
}

constexpr int64_t NORM_MAX_PARTS = 148 * 4;
constexpr int64_t MAX_GRID = 1 << 30;

static int round32(int n) { return (n + 31) / 32 * 32; }

template <typename TX, typename TO, int V>
static bool launch_fwd(const NormArgs& a, cudaStream_t st) {
    const int vectors = a.cols / V;
    auto by_warp = [&](auto kernel) { kernel<<<static_cast<unsigned>(std::min((a.rows + 7) / 8, MAX_GRID)), 256, 0, st>>>(a); return true; };
    auto by_cta = [&](auto kernel, int n) {
        kernel<<<static_cast<unsigned>(std::min(a.rows, MAX_GRID)), round32((vectors + n - 1) / n), 0, st>>>(a);
        return true;
    };
    if (vectors <= 32) return by_warp(norm_fwd_kernel<TX, TO, V, 1, false>);
    if (vectors <= 64) return by_warp(norm_fwd_kernel<TX, TO, V, 2, false>);
    if (vectors <= 128) return by_warp(norm_fwd_kernel<TX, TO, V, 4, false>);
    if (vectors <= 256) return by_warp(norm_fwd_kernel<TX, TO, V, 8, false>);
    if (vectors <= 4 * 1024) return by_cta(norm_fwd_kernel<TX, TO, V, 4, true>, 4);
    return false;
}

template <typename TX, typename TO>
static void forward(const NormArgs& a, bool vector, cudaStream_t st) {
    constexpr int V = 16 / sizeof(TX);
    if (vector ? launch_fwd<TX, TO, V>(a, st) : launch_fwd<TX, TO, 1>(a, st)) return;
    norm_fwd_any_kernel<TX, TO><<<static_cast<unsigned>(std::min(a.rows, MAX_GRID)), 256, 0, st>>>(a);
}

// Returns the number of partial rows, or 0 when the width does not fit the register kernels.
template <typename TX, typename TH, int V>
static int64_t launch_bwd(const NormBwdArgs& a, cudaStream_t st) {
    const int vectors = a.cols / V;
    auto by_warp = [&](auto kernel) {
        const int64_t parts = std::min<int64_t>((a.rows + 7) / 8, 148 * 2);
        kernel<<<static_cast<unsigned>(parts), 256, 0, st>>>(a);
        return parts;
    };
    auto by_cta = [&](auto kernel, int n) {
        const int threads = round32((vectors + n - 1) / n);
        const int64_t parts = std::min<int64_t>(a.rows, 148 * (threads <= 256 ? 3 : threads <= 384 ? 2 : 1));
        kernel<<<static_cast<unsigned>(parts), threads, 0, st>>>(a);
        return parts;
    };
    constexpr int U = 8 / V;        // vectors that make eight columns
    if (vectors <= 32 * U) return by_warp(norm_bwd_kernel<TX, TH, V, U, 1, false>);
    if (vectors <= 64 * U) return by_warp(norm_bwd_kernel<TX, TH, V, 2 * U, 1, false>);
    if (vectors <= 96 * U) return by_warp(norm_bwd_kernel<TX, TH, V, 3 * U, 1, false>);
    if (vectors <= 512 * U) return by_cta(norm_bwd_kernel<TX, TH, V, U, 1, true>, U);
    if (vectors <= 1024 * U) return by_cta(norm_bwd_kernel<TX, TH, V, 2 * U, 1, true>, 2 * U);
    return 0;
}

template <typename TX, typename TH>
static int64_t backward(const NormBwdArgs& a, bool vector, cudaStream_t st) {
    constexpr int V = 16 / sizeof(TX);
    if (const int64_t parts = vector ? launch_bwd<TX, TH, V>(a, st) : launch_bwd<TX, TH, 1>(a, st)) return parts;
    norm_bwd_any_kernel<TX, TH><<<static_cast<unsigned>(std::min(a.rows, MAX_GRID)), 256, 0, st>>>(a);
    if (!a.partial) return 1;
    const int64_t blocks = (a.cols + 31) / 32;
    const int64_t parts = std::min<int64_t>({(a.rows + 31) / 32, NORM_MAX_PARTS, std::max<int64_t>(1, 148 * 16 / blocks)});
    norm_bwd_columns_kernel<TX, TH><<<dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(parts)), 256, 0, st>>>(a);
    return parts;
}

}  // namespace nvfp4

using namespace nvfp4;

extern "C" int nvfp4_layer_norm(const void* x, int x_dtype, int64_t x_pitch, const void* delta, int delta_dtype, int64_t delta_pitch,
                                const void* weight, const void* bias, int weight_dtype, float eps, int64_t rows, int64_t cols,
                                void* sum_out, void* h_out, int h_dtype, float* mean_out, float* rstd_out, float* amax,
                                nvfp4_stream_t stream) {
    NVFP4_REQUIRE(x && h_out && (!delta || sum_out) && (mean_out == nullptr) == (rstd_out == nullptr), NVFP4_ERR_ARG, "nvfp4_layer_norm: null pointer");
    NVFP4_REQUIRE(rows > 0 && cols > 0 && cols < (1LL << 30) && x_pitch >= cols && (!delta || delta_pitch >= cols), NVFP4_ERR_ARG,
                  "nvfp4_layer_norm: rows and cols must be positive and the row pitches at least cols");
    NVFP4_REQUIRE(is_float_dtype(x_dtype) && is_float_dtype(h_dtype) && ((!weight && !bias) || is_float_dtype(weight_dtype)), NVFP4_ERR_DTYPE,
                  "nvfp4_layer_norm: FP32, BF16 or FP16 tensors");
    NVFP4_REQUIRE(h_dtype == x_dtype || (x_dtype == NVFP4_F32 && h_dtype == NVFP4_BF16), NVFP4_ERR_DTYPE,
                  "nvfp4_layer_norm: the result has the input's type, or BF16 beside an FP32 input");
    NVFP4_REQUIRE(!delta || delta_dtype == x_dtype || (x_dtype == NVFP4_F32 && delta_dtype == NVFP4_BF16), NVFP4_ERR_DTYPE,
                  "nvfp4_layer_norm: the second summand has the input's type, or BF16 beside an FP32 input");
    NormArgs a{x, delta, weight, bias, sum_out, h_out, mean_out, rstd_out, amax, x_pitch, delta_pitch, rows, static_cast<int>(cols),
               delta && delta_dtype != x_dtype, weight_dtype, eps};
    // 16-byte vectors of x need every operand's rows to start on a multiple of its own share of them
    const int v = 16 / dtype_size(x_dtype);
    auto fits = [&](const void* p, int dtype, int64_t pitch) { return !p || (aligned(p, std::min(16, v * dtype_size(dtype))) && pitch % v == 0); };
    const bool vector = cols % v == 0 && fits(x, x_dtype, x_pitch) && fits(delta, delta_dtype, delta_pitch) && fits(sum_out, x_dtype, cols) &&
                        fits(h_out, h_dtype, cols) && fits(weight, weight_dtype, 0) && fits(bias, weight_dtype, 0);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (x_dtype == NVFP4_BF16) forward<__nv_bfloat16, __nv_bfloat16>(a, vector, st);
    else if (x_dtype == NVFP4_F16) forward<__half, __half>(a, vector, st);
    else if (h_dtype == NVFP4_F32) forward<float, float>(a, vector, st);
    else forward<float, __nv_bfloat16>(a, vector, st);
    return launch_status("nvfp4_layer_norm");
}

extern "C" int64_t nvfp4_layer_norm_bwd_partials(int64_t rows, int64_t) { return std::max<int64_t>(1, std::min(rows, NORM_MAX_PARTS)); }

extern "C" int nvfp4_layer_norm_bwd(const void* dh, int h_dtype, int64_t dh_pitch, const void* total, int x_dtype, int64_t total_pitch,
                                    const float* mean, const float* rstd, const void* weight, int weight_dtype, const void* dsum,
                                    int64_t dsum_pitch, int64_t rows, int64_t cols, void* dx, void* ddelta, float* partial, void* dweight,
                                    void* dbias, float* amax, nvfp4_stream_t stream) {
    NVFP4_REQUIRE(dh && total && mean && rstd && dx && ((!dweight && !dbias) || partial), NVFP4_ERR_ARG, "nvfp4_layer_norm_bwd: null pointer");
    NVFP4_REQUIRE(rows > 0 && cols > 0 && cols < (1LL << 30) && dh_pitch >= cols && total_pitch >= cols && (!dsum || dsum_pitch >= cols), NVFP4_ERR_ARG,
                  "nvfp4_layer_norm_bwd: rows and cols must be positive and the row pitches at least cols");
    NVFP4_REQUIRE(is_float_dtype(x_dtype) && (h_dtype == x_dtype || (x_dtype == NVFP4_F32 && h_dtype == NVFP4_BF16)) &&
                  ((!weight && !dweight && !dbias) || is_float_dtype(weight_dtype)), NVFP4_ERR_DTYPE, "nvfp4_layer_norm_bwd: FP32, BF16 or FP16 tensors");
    NVFP4_REQUIRE(!ddelta || x_dtype == NVFP4_F32, NVFP4_ERR_DTYPE, "nvfp4_layer_norm_bwd: ddelta is the BF16 copy of an FP32 dx");
    NormBwdArgs a{dh, total, weight, dsum, mean, rstd, dx, ddelta, (dweight || dbias) ? partial : nullptr, amax, dh_pitch, total_pitch, dsum_pitch,
                  rows, static_cast<int>(cols), weight_dtype};
    const int v = 16 / dtype_size(x_dtype);
    auto fits = [&](const void* p, int dtype, int64_t pitch) { return !p || (aligned(p, std::min(16, v * dtype_size(dtype))) && pitch % v == 0); };
    const bool vector = cols % v == 0 && fits(dh, h_dtype, dh_pitch) && fits(total, x_dtype, total_pitch) && fits(dsum, x_dtype, dsum_pitch) &&
                        fits(dx, x_dtype, cols) && fits(ddelta, NVFP4_BF16, cols) && fits(weight, weight_dtype, 0);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    int64_t parts;
    if (x_dtype == NVFP4_BF16) parts = backward<__nv_bfloat16, __nv_bfloat16>(a, vector, st);
    else if (x_dtype == NVFP4_F16) parts = backward<__half, __half>(a, vector, st);
    else if (h_dtype == NVFP4_F32) parts = backward<float, float>(a, vector, st);
    else parts = backward<float, __nv_bfloat16>(a, vector, st);
    if (a.partial)
        column_sums_kernel<<<static_cast<unsigned>((2 * cols + 31) / 32), 256, 0, st>>>(partial, parts, 2 * cols, cols, dweight, dbias, weight_dtype);
    return launch_status("nvfp4_layer_norm_bwd");
}

extern "C" int nvfp4_column_sums(const float* partial, int64_t parts, int64_t cols, void* out, int out_dtype, nvfp4_stream_t stream) {
    NVFP4_REQUIRE(partial && out && parts > 0 && cols > 0 && cols < (1LL << 31), NVFP4_ERR_ARG, "nvfp4_column_sums: null pointer or empty size");
    NVFP4_REQUIRE(is_float_dtype(out_dtype), NVFP4_ERR_DTYPE, "nvfp4_column_sums: FP32, BF16 or FP16 result");
    column_sums_kernel<<<static_cast<unsigned>((cols + 31) / 32), 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
        partial, parts, cols, cols, out, nullptr, out_dtype);
    return launch_status("nvfp4_column_sums");
}
