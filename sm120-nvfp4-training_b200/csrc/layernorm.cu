// Layer norm with the residual sum in front of it, forward and backward.
//
//   total = x + delta,  h = (total - mean) * rstd * w + b,   mean, var over the row, rstd = 1 / sqrt(var + eps)
//   with z = (total - mean) * rstd, u = dh * w:   dx = rstd * (u - mean(u) - z * mean(u z)) + dsum,  dw = sum dh z,  db = sum dh
//
// Both directions stream: every operand is read once and every result written once, so HBM is the bound.  A row stays in
// registers between the sweeps over it (sum, centred squares, result); squares are taken around a mean, never as a difference of
// sums, which keeps the variance exact where the mean is large against the spread, and means are rounded once (Reciprocal
// below): a constant row whose sum FP32 holds gives differences of exactly zero.  All statistics are FP32; a result is
// rounded once, except that h is formed from the total as it is stored (the backward pass reads that one too).  Rows that
// bulk copies can fetch go through the ring further down (16384 x 5120 BF16 with the residual sum: forward 106 us, 0.98 of the
// measured HBM rate, backward 142 us, 0.73); the kernels before it take the odd widths, the unaligned rows and the widest.
#include "async.cuh"
#include "bf16x8.cuh"
#include "vec.cuh"

#include <algorithm>

namespace nvfp4 {

struct NormArgs {
    const void *x, *delta, *weight, *bias;
    void *sum, *h;
    float *mean, *rstd, *amax;
    int* status;
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

// 1 / n in two parts, so that a sum's mean is off by 2^-46 before its one rounding: where the quotient is a float, as for constant
// rows, it is that float.  (One product more than with a rounded 1 / n; a division for each mean took 122 instead of 106 us for
// 16384 x 5120 BF16, 22.6 instead of 13.9 for 32768 x 256.)
struct Reciprocal {
    float high, low;
    __device__ __forceinline__ explicit Reciprocal(float n) : high(1.f / n), low(fmaf(-high, n, 1.f) * high) {}
    __device__ __forceinline__ float of(float sum) const { return fmaf(sum, high, sum * low); }
};

// V elements of total at column c of row r (stored, too, when there is a delta), as FP32
template <typename TX, int V>
__device__ __forceinline__ void load_total(const NormArgs& a, int64_t r, int c, float (&f)[V]) {
    Pack<TX, V> p = load_const<TX, V>(static_cast<const TX*>(a.x) + r * a.x_pitch + c);
    unpack(p, f);
    if (a.delta) {
        float d[V];
        if (sizeof(TX) == 4 && a.delta_bf16) unpack(load_const<__nv_bfloat16, V>(static_cast<const __nv_bfloat16*>(a.delta) + r * a.delta_pitch + c), d);
        else unpack(load_const<TX, V>(static_cast<const TX*>(a.delta) + r * a.delta_pitch + c), d);
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
    return a.amax ? abs_max(q) : 0.f;
}

// A row in registers, N vectors of V elements per thread; ROW_CTA: a CTA per row, else a warp per row.
template <typename TX, typename TO, int V, int N, bool ROW_CTA>
__global__ void __launch_bounds__(ROW_CTA ? 1024 : 256) norm_fwd_kernel(const NormArgs a) {
    __shared__ float slots[2][32];
    const int tid = ROW_CTA ? threadIdx.x : (threadIdx.x & 31), step = ROW_CTA ? blockDim.x : 32;
    const int64_t row0 = ROW_CTA ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const int64_t row_step = ROW_CTA ? gridDim.x : static_cast<int64_t>(gridDim.x) * 8;
    const int vectors = a.cols / V;
    const Reciprocal inv_n(static_cast<float>(a.cols));
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
        const float mean = inv_n.of(ROW_CTA ? cta_sum(s, slots[0]) : warp_sum(s));
        float sq = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (tid + i * step < vectors) {
#pragma unroll
                for (int j = 0; j < V; ++j) { const float d = f[i][j] - mean; sq = fmaf(d, d, sq); }
            }
        const float rstd = rsqrtf((ROW_CTA ? cta_sum(sq, slots[1]) : warp_sum(sq)) * inv_n.high + a.eps);
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
    int* status;
    float *partial, *amax;     // partial: [parts][2][cols], null when neither dw nor db is asked for
    int64_t dh_pitch, total_pitch, dsum_pitch, rows;
    int cols, weight_dtype;
};

// dx of V elements from the row's two means; returns max |what the producer of x's branch receives|
template <typename TX, int V>
__device__ __forceinline__ float store_dx(const NormBwdArgs& a, int64_t r, int c, const float (&u)[V], const float (&z)[V], float rstd,
                                          float mean_u, float mean_uz, const Pack<TX, V>& dsum) {
    float o[V], d[V];
    const float k1 = -rstd * mean_u, k2 = -rstd * mean_uz;
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = fmaf(u[j], rstd, fmaf(z[j], k2, k1));
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
        return a.amax ? abs_max(qd) : 0.f;
    }
    return a.amax ? abs_max(q) : 0.f;
}

// Every thread owns N columns for all rows its group (a warp, or the CTA) takes, so the column sums stay in registers.  The CTA's sums go out as one partial row, added up in a fixed order by
// column_sums_kernel.
template <typename TX, typename TH, int N, bool ROW_CTA>
__global__ void __launch_bounds__(ROW_CTA ? 512 : 256) norm_bwd_kernel(const NormBwdArgs a) {
    constexpr int V = 1, R = 1;       // single elements, one row at a time
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
// A CTA takes 32 columns, its 16 warps every 16th row each, the subtotals are added in warp order.  (32 warps a CTA leave a
// second wave of CTAs at 2 * 5120 columns.)
constexpr int SUM_WARPS = 16;
__global__ void __launch_bounds__(SUM_WARPS * 32) column_sums_kernel(const float* __restrict__ partial, int64_t parts, int64_t width, int64_t cols,
                                                                     void* out0, void* out1, int dtype) {
    __shared__ float subtotal[SUM_WARPS][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    float t = 0.f;
    if (c < width) {
#pragma unroll 8
        for (int64_t p = warp; p < parts; p += SUM_WARPS) t += partial[p * width + c];
    }
    subtotal[warp][lane] = t;
    __syncthreads();
    if (warp != 0 || c >= width) return;
    t = 0.f;
#pragma unroll
    for (int w = 0; w < SUM_WARPS; ++w) t += subtotal[w][lane];
    void* out = c < cols ? out0 : out1;
    if (out) store_param(out, dtype, c < cols ? c : c - cols, t);
}

// ====================================================================================================================
// rows through a ring in shared memory
// ====================================================================================================================
// With its operands in registers alone a CTA loads a row, waits, reduces, waits, and stores: 0.3 to 0.6 of HBM, all of it load
// latency (long-scoreboard stalls 10 of 16 cycles per instruction).  Here one thread keeps bulk copies of the next rows in
// flight into a ring of stages, and a stage is refilled as soon as the CTA's first barrier behind its reads has passed.  CTAs
// are persistent, so weight and bias (and the backward pass's column sums) stay in registers: C columns per thread as 16-byte
// vectors of x, up to 8192 columns.  Narrow rows have several groups of threads side by side in a CTA; R rows of each group
// share the barriers of a round.
namespace ring {
constexpr int MAX_STAGES = 8;
constexpr int BYTES_PER_SM = 228 * 1024, ASIDE = 2560;      // of it a CTA's own 1024 bytes and its static arrays
struct Plan { int row_threads, threads, stages, stage_bytes, ctas, parked; };      // parked: bytes behind the stages
}  // namespace ring

struct RingOperand { const uint8_t* base; int64_t pitch; uint32_t bytes; };       // pitch and row length in bytes; base null: absent

// Runs of `per_stage` rows of up to OPS operands through the ring; thread 0 is the producer.  What only it needs lies in shared
// memory (held in registers by every thread it cost 20 of them).  Every wait is bounded: when one runs out, all later ones
// return at once, the loops end over stale data, and the status word says so.
template <int OPS>
struct RowRing {
    RingOperand op[OPS];
    int64_t rows, groups;
    uint32_t row_bytes;
    int per_stage, stages, abort_flag;
    uint64_t full[ring::MAX_STAGES];
};
struct RingCursor { int slot; uint32_t phase; };

template <int OPS>
__device__ __forceinline__ void ring_fill(RowRing<OPS>& q, uint8_t* data, int64_t group, int into) {
    const int64_t r0 = group * q.per_stage;
    const int live = static_cast<int>(q.rows - r0 < q.per_stage ? q.rows - r0 : q.per_stage);
    aop::mbar_expect_tx(&q.full[into], live * q.row_bytes);
    uint8_t* dst = data + static_cast<size_t>(into) * q.per_stage * q.row_bytes;
    for (int o = 0; o < OPS; ++o) {
        const RingOperand op = q.op[o];
        if (!op.base) continue;
        const uint8_t* src = op.base + r0 * op.pitch;
        if (op.pitch == op.bytes) aop::bulk_load(dst, src, live * op.bytes, &q.full[into]);
        else for (int k = 0; k < live; ++k) aop::bulk_load(dst + k * op.bytes, src + k * op.pitch, op.bytes, &q.full[into]);
        dst += q.per_stage * op.bytes;
    }
}
// by thread 0, which has set the operands, rows, per_stage and stages
template <int OPS>
__device__ __forceinline__ void ring_start(RowRing<OPS>& q, uint8_t* data) {
    q.groups = (q.rows + q.per_stage - 1) / q.per_stage;
    q.row_bytes = 0;
    for (int o = 0; o < OPS; ++o) q.row_bytes += q.op[o].base ? q.op[o].bytes : 0;
    for (int s = 0; s < q.stages; ++s) aop::mbar_init(&q.full[s], 1);
    q.abort_flag = 0;
    aop::fence_barrier_init();
    for (int s = 0; s < q.stages; ++s) {
        const int64_t group = blockIdx.x + static_cast<int64_t>(s) * gridDim.x;
        if (group < q.groups) ring_fill(q, data, group, s);
    }
}
// behind a barrier that follows every read of the present stage
template <int OPS>
__device__ __forceinline__ void ring_advance(RowRing<OPS>& q, uint8_t* data, RingCursor& at, int stages, int64_t group) {
    if (threadIdx.x == 0) {
        const int64_t next = group + static_cast<int64_t>(stages) * gridDim.x;
        if (next < q.groups && !*static_cast<volatile int*>(&q.abort_flag)) ring_fill(q, data, next, at.slot);
    }
    if (++at.slot == stages) { at.slot = 0; at.phase ^= 1; }
}
// after the last barrier: a bounded wait for copies that nobody read
template <int OPS>
__device__ __forceinline__ void ring_finish(RowRing<OPS>& q, int* status) {
    if (threadIdx.x == 0 && *static_cast<volatile int*>(&q.abort_flag)) {
        const long long t0 = clock64();
        for (int s = 0; s < q.stages; ++s)
            while (!aop::mbar_try(&q.full[s], 0) && !aop::mbar_try(&q.full[s], 1) && clock64() - t0 < aop::WAIT_LIMIT_CYCLES / 8) {}
        while (clock64() - t0 < 400000) {}
        if (status) atomicExch(status, NVFP4_ERR_TIMEOUT);
    }
}

// C sums over a group of `warps` warps from `first` on, in a fixed order; every thread gets all of them; one barrier of the CTA
// (see cta_sum).  The lanes of a warp fold the C values together, halving what each carries at every exchange, so that lane l
// ends with the warp's sum of value l C / 32; each warp then adds the group's warps, 32 / C at a time.
template <int C>
__device__ __forceinline__ void group_sums(float (&a)[C], float (*slots)[C], int first, int warps) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int d = 16, n = C; d > 0; d >>= 1) {
        if (n > 1) {
            n >>= 1;
            const bool upper = lane & d;
#pragma unroll
            for (int i = 0; i < n; ++i) {
                const float keep = upper ? a[i + n] : a[i], send = upper ? a[i] : a[i + n];
                a[i] = keep + __shfl_xor_sync(0xffffffffu, send, d);
            }
        } else {
            a[0] += __shfl_xor_sync(0xffffffffu, a[0], d);
        }
    }
    if (lane % (32 / C) == 0) slots[threadIdx.x >> 5][lane / (32 / C)] = a[0];
    __syncthreads();
    float t = 0.f;
    for (int w = lane / C; w < warps; w += 32 / C) t += slots[first + w][lane % C];
#pragma unroll
    for (int d = C; d < 32; d <<= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
#pragma unroll
    for (int i = 0; i < C; ++i) a[i] = __shfl_sync(0xffffffffu, t, i);
}

template <typename T, int V> __device__ __forceinline__ void load_or(const void* p, int dtype, int c, bool live, float otherwise, T (&f)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = otherwise;
    if (p && live) load_param<V>(p, dtype, c, f);
}

template <typename TX, typename TD, typename TO, int C, int R, int MAXT, int CTAS>
__global__ void __launch_bounds__(MAXT, CTAS) norm_fwd_ring_kernel(const NormArgs a, int stages, int row_threads) {
    constexpr int V = 16 / sizeof(TX), N = C / V;
    extern __shared__ __align__(128) uint8_t ring_data[];
    __shared__ float2 slots[2][R][32];           // a warp's sum and its squares around its own mean
    __shared__ RowRing<2> q;
    const int group = threadIdx.x / row_threads, tid = threadIdx.x - group * row_threads, step = row_threads, vectors = a.cols / V;
    const int per_stage = blockDim.x / row_threads * R, first_warp = group * (row_threads >> 5);
    const uint32_t x_bytes = a.cols * sizeof(TX), d_bytes = a.delta ? a.cols * sizeof(TD) : 0;
    if (threadIdx.x == 0) {
        q.op[0] = {static_cast<const uint8_t*>(a.x), a.x_pitch * static_cast<int64_t>(sizeof(TX)), x_bytes};
        q.op[1] = {static_cast<const uint8_t*>(a.delta), a.delta_pitch * static_cast<int64_t>(sizeof(TD)), d_bytes};
        q.rows = a.rows;
        q.per_stage = per_stage;
        q.stages = stages;
        ring_start(q, ring_data);
    }
    __syncthreads();
    const int64_t runs = q.groups;
    const uint32_t stage_bytes = per_stage * q.row_bytes;
    RingCursor at{0, 0};
    float w[N][V], b[N][V];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = tid + i * step;
        load_or(a.weight, a.weight_dtype, c * V, c < vectors, 1.f, w[i]);
        load_or(a.bias, a.weight_dtype, c * V, c < vectors, 0.f, b[i]);
    }
    // columns of this warp, and of warp `lane` of the group (what the gather below needs)
    const int lane = threadIdx.x & 31, warps = step >> 5;
    float mine = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) mine += tid + i * step < vectors ? static_cast<float>(V) : 0.f;
    mine = warp_sum(mine);
    if (lane == 0) slots[0][0][threadIdx.x >> 5].x = mine;
    __syncthreads();
    const float theirs = lane < warps ? slots[0][0][first_warp + lane].x : 0.f;
    // (a warp without columns has sums of zero)
    const Reciprocal inv_mine(fmaxf(mine, 1.f)), inv_theirs(fmaxf(theirs, 1.f)), inv_n(static_cast<float>(a.cols));
    int half = 1;
    float best = 0.f;
    for (int64_t g = blockIdx.x; g < runs; g += gridDim.x, half ^= 1) {
        aop::mbar_wait(&q.full[at.slot], at.phase, &q.abort_flag);
        const uint8_t* stage = ring_data + at.slot * stage_bytes;
        float f[R][N][V], sums[R];
#pragma unroll
        for (int k = 0; k < R; ++k) {
            const int64_t r = g * per_stage + group * R + k;
            sums[k] = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int c = tid + i * step;
                if (c >= vectors || r >= a.rows) continue;
                unpack(load_pack<TX, V>(reinterpret_cast<const TX*>(stage + (group * R + k) * x_bytes) + c * V), f[k][i]);
                if (a.delta) {
                    float d[V];
                    unpack(load_pack<TD, V>(reinterpret_cast<const TD*>(stage + per_stage * x_bytes + (group * R + k) * d_bytes) + c * V), d);
#pragma unroll
                    for (int j = 0; j < V; ++j) f[k][i][j] += d[j];
                    const Pack<TX, V> p = pack<TX, V>(f[k][i]);
                    store_pack(static_cast<TX*>(a.sum) + r * a.cols + c * V, p);
                    unpack(p, f[k][i]);
                }
#pragma unroll
                for (int j = 0; j < V; ++j) sums[k] += f[k][i][j];
            }
        }
        // the warp's mean and squares around it, then the group's from the warps': one barrier, no cancellation
        float squares[R], mean[R];
#pragma unroll
        for (int k = 0; k < R; ++k) sums[k] = warp_sum(sums[k]);
#pragma unroll
        for (int k = 0; k < R; ++k) {
            const float m = inv_mine.of(sums[k]);
            squares[k] = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (tid + i * step < vectors) {
#pragma unroll
                    for (int j = 0; j < V; ++j) { const float d = f[k][i][j] - m; squares[k] = fmaf(d, d, squares[k]); }
                }
        }
#pragma unroll
        for (int k = 0; k < R; ++k) {
            squares[k] = warp_sum(squares[k]);
            if (lane == 0) slots[half][k][threadIdx.x >> 5] = make_float2(sums[k], squares[k]);
        }
        __syncthreads();
        ring_advance(q, ring_data, at, stages, g);
        if (warps > 1) {
            float2 part[R];
#pragma unroll
            for (int k = 0; k < R; ++k) {
                part[k] = lane < warps ? slots[half][k][first_warp + lane] : make_float2(0.f, 0.f);
                sums[k] = warp_sum(part[k].x);
            }
#pragma unroll
            for (int k = 0; k < R; ++k) {
                mean[k] = inv_n.of(sums[k]);
                const float d = inv_theirs.of(part[k].x) - mean[k];
                squares[k] = warp_sum(fmaf(theirs * d, d, part[k].y));
            }
        } else {
#pragma unroll
            for (int k = 0; k < R; ++k) mean[k] = inv_n.of(sums[k]);
        }
#pragma unroll
        for (int k = 0; k < R; ++k) {
            const int64_t r = g * per_stage + group * R + k;
            if (r >= a.rows) continue;
            const float rstd = rsqrtf(squares[k] * inv_n.high + a.eps);
            if (tid == 0 && a.mean) { a.mean[r] = mean[k]; a.rstd[r] = rstd; }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int c = tid + i * step;
                if (c >= vectors) continue;
                float o[V];
#pragma unroll
                for (int j = 0; j < V; ++j) o[j] = fmaf((f[k][i][j] - mean[k]) * rstd, w[i][j], b[i][j]);
                const Pack<TO, V> q = pack<TO, V>(o);
                store_pack(static_cast<TO*>(a.h) + r * a.cols + c * V, q);
                if (a.amax) best = fmaxf(best, abs_max(q));
            }
        }
    }
    if (a.amax) block_atomic_amax(a.amax, best);
    ring_finish(q, a.status);
}

__device__ __forceinline__ float4 shared_again(const float4* p) {      // a load that stays where it is written
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(aop::smem_u32(p)));
    return v;
}

template <typename TX, typename TH, int C, int R, int MAXT, int CTAS>
__global__ void __launch_bounds__(MAXT, CTAS) norm_bwd_ring_kernel(const NormBwdArgs a, int stages, int row_threads) {
    constexpr int V = 16 / sizeof(TX), N = C / V;
    extern __shared__ __align__(128) uint8_t ring_data[];
    __shared__ float slots[2][32][2 * R];
    __shared__ RowRing<3> q;
    const int group = threadIdx.x / row_threads, tid = threadIdx.x - group * row_threads, step = row_threads, vectors = a.cols / V;
    const int per_stage = blockDim.x / row_threads * R, first_warp = group * (row_threads >> 5);
    const uint32_t h_bytes = a.cols * sizeof(TH), x_bytes = a.cols * sizeof(TX), s_bytes = a.dsum ? x_bytes : 0;
    if (threadIdx.x == 0) {
        q.op[0] = {static_cast<const uint8_t*>(a.dh), a.dh_pitch * static_cast<int64_t>(sizeof(TH)), h_bytes};
        q.op[1] = {static_cast<const uint8_t*>(a.total), a.total_pitch * static_cast<int64_t>(sizeof(TX)), x_bytes};
        q.op[2] = {static_cast<const uint8_t*>(a.dsum), a.dsum_pitch * static_cast<int64_t>(sizeof(TX)), s_bytes};
        q.rows = a.rows;
        q.per_stage = per_stage;
        q.stages = stages;
        ring_start(q, ring_data);
    }
    __syncthreads();
    const int64_t runs = q.groups;
    const uint32_t stage_bytes = per_stage * q.row_bytes;
    RingCursor at{0, 0};
    // With sixteen columns a thread keeps its weights in shared memory, in registers they would spill.
    constexpr bool PARKED = C == 16;
    float w[N][V], acc_w[N][V], acc_b[N][V];
    float4* parked = reinterpret_cast<float4*>(ring_data + stages * stage_bytes) + threadIdx.x;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        load_or(a.weight, a.weight_dtype, (tid + i * step) * V, tid + i * step < vectors, 1.f, w[i]);
#pragma unroll
        for (int j = 0; j < V; ++j) acc_w[i][j] = acc_b[i][j] = 0.f;
        if constexpr (PARKED) {
#pragma unroll
            for (int j = 0; j < V; j += 4) parked[(i * V + j) / 4 * blockDim.x] = make_float4(w[i][j], w[i][j + 1], w[i][j + 2], w[i][j + 3]);
        }
    }
    const float inv_n = 1.f / static_cast<float>(a.cols);
    float best = 0.f, mean[R], rstd[R];          // of the next group, fetched one round ahead
    auto statistics = [&](int64_t g) {
#pragma unroll
        for (int k = 0; k < R; ++k) {
            const int64_t r = g * per_stage + group * R + k;
            mean[k] = r < a.rows ? __ldg(a.mean + r) : 0.f;
            rstd[k] = r < a.rows ? __ldg(a.rstd + r) : 0.f;
        }
    };
    statistics(blockIdx.x);
    int half = 0;
    for (int64_t g = blockIdx.x; g < runs; g += gridDim.x, half ^= 1) {
        aop::mbar_wait(&q.full[at.slot], at.phase, &q.abort_flag);
        const uint8_t* stage = ring_data + at.slot * stage_bytes;
        float u[R][N][V], z[R][N][V], sums[2 * R], rs[R];
        Pack<TX, V> res[R][N];
#pragma unroll
        for (int k = 0; k < R; ++k) {
            rs[k] = rstd[k];
            sums[2 * k] = sums[2 * k + 1] = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int c = tid + i * step, row = group * R + k;
                if (c >= vectors || g * per_stage + row >= a.rows) continue;
                unpack(load_pack<TH, V>(reinterpret_cast<const TH*>(stage + row * h_bytes) + c * V), u[k][i]);
                unpack(load_pack<TX, V>(reinterpret_cast<const TX*>(stage + per_stage * h_bytes + row * x_bytes) + c * V), z[k][i]);
                if constexpr (PARKED) {
#pragma unroll
                    for (int j = 0; j < V; j += 4) {
                        const float4 t = shared_again(parked + (i * V + j) / 4 * blockDim.x);
                        w[i][j] = t.x; w[i][j + 1] = t.y; w[i][j + 2] = t.z; w[i][j + 3] = t.w;
                    }
                }
                if (a.dsum) res[k][i] = load_pack<TX, V>(reinterpret_cast<const TX*>(stage + per_stage * (h_bytes + x_bytes) + row * s_bytes) + c * V);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float dh = u[k][i][j];
                    z[k][i][j] = (z[k][i][j] - mean[k]) * rs[k];      // not x rstd - mean rstd, whose rounding is large where the mean is
                    acc_w[i][j] = fmaf(dh, z[k][i][j], acc_w[i][j]);
                    acc_b[i][j] += dh;
                    u[k][i][j] = dh * w[i][j];
                    sums[2 * k] += u[k][i][j];
                    sums[2 * k + 1] = fmaf(u[k][i][j], z[k][i][j], sums[2 * k + 1]);
                }
            }
        }
        statistics(g + gridDim.x);
        group_sums(sums, slots[half], first_warp, step >> 5);
        ring_advance(q, ring_data, at, stages, g);
#pragma unroll
        for (int k = 0; k < R; ++k) {
            const int64_t r = g * per_stage + group * R + k;
            if (r >= a.rows) continue;
            const float mean_u = sums[2 * k] * inv_n, mean_uz = sums[2 * k + 1] * inv_n;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int c = tid + i * step;
                if (c < vectors) best = fmaxf(best, store_dx<TX, V>(a, r, c * V, u[k][i], z[k][i], rs[k], mean_u, mean_uz, res[k][i]));
            }
        }
    }
    if (a.amax) block_atomic_amax(a.amax, best);
    ring_finish(q, a.status);
    if (!a.partial) return;
    // the groups' sums meet in shared memory (the ring is empty) and are added in group order
    float* out = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * a.cols;
    const bool alone = step == blockDim.x;
    float* meet = reinterpret_cast<float*>(ring_data) + static_cast<int64_t>(group) * 2 * a.cols;
    float* mine = alone ? out : meet;
    if (!alone) __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = tid + i * step;
        if (c >= vectors) continue;
        store_pack(mine + c * V, pack<float, V>(acc_w[i]));
        store_pack(mine + a.cols + c * V, pack<float, V>(acc_b[i]));
    }
    if (alone) return;
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * a.cols; c += blockDim.x) {
        float t = 0.f;
        for (int q = 0; q < static_cast<int>(blockDim.x) / step; ++q) t += reinterpret_cast<const float*>(ring_data)[static_cast<int64_t>(q) * 2 * a.cols + c];
        out[c] = t;
    }
}

constexpr int64_t SMS = 148;
constexpr int64_t MAX_GRID = 1 << 30;

static int round32(int n) { return (n + 31) / 32 * 32; }

// Sixteen columns a thread from 2048 columns on, eight below: a round costs a thread about 150 instructions whatever it holds
// (waiting, two reductions, addresses), which sixteen columns halve (16384 x 5120 BF16: 179 -> 109 us forward, 165 -> 137
// backward when it was made); below, the rows would not fill a warp.  Narrow rows stand in groups that make 256 threads.  As many
// CTAs per SM as the registers allow (threads_that_fit) and as leave each of them three stages, within a budget of threads: 1024
// forward and 512 backward with eight columns a thread, 640 with sixteen.  A CTA more than fits would run behind the others with
// its share of the rows, on stages cut to its size: backward, 2304 columns BF16 (160 threads of 128 registers), 159 us with four
// CTAs planned, 112 with the three that fit.
static int columns_per_thread(int64_t cols) { return cols >= 2048 ? 16 : 8; }
static int round_threads(int64_t cols) { return round32(static_cast<int>((cols + columns_per_thread(cols) - 1) / columns_per_thread(cols))); }
static int bwd_threads_per_sm(int64_t cols) { return columns_per_thread(cols) == 8 ? 512 : 640; }

// Partial rows of dw and db at most, which is what the caller's scratch holds: every way the backward pass may go at this width
// keeps to it.  Wide rows are summed by a pass of their own, in about 16 CTAs per SM of 32 columns each.
static int64_t column_pass_parts(int64_t rows, int64_t cols) {
    return std::min<int64_t>({(rows + 31) / 32, SMS * 4, std::max<int64_t>(1, SMS * 16 / ((cols + 31) / 32))});
}
static int64_t bwd_parts_limit(int64_t rows, int64_t cols) {
    if (cols > 8192) return column_pass_parts(rows, cols);
    const int row_threads = round_threads(cols), threads = row_threads * std::max(1, 256 / row_threads);
    const int64_t ring = SMS * std::max(1, bwd_threads_per_sm(cols) / threads);
    const int64_t other = cols <= 768 ? SMS * 2 : cols <= 4096 ? SMS * 3 : column_pass_parts(rows, cols);
    return std::min(rows, std::max(ring, other));
}
static ring::Plan ring_plan(int64_t rows, int64_t cols, int rows_per_group, int row_bytes, int sms, int threads_per_sm, bool backward) {
    ring::Plan p;
    const int per_thread = columns_per_thread(cols);
    p.row_threads = round_threads(cols);
    // few rows: no group without one
    const int64_t want = std::max<int64_t>(1, (rows + static_cast<int64_t>(rows_per_group) * sms - 1) / (static_cast<int64_t>(rows_per_group) * sms));
    const int groups = static_cast<int>(std::min<int64_t>(std::max(1, 256 / p.row_threads), want));
    p.threads = p.row_threads * groups;
    p.stage_bytes = groups * rows_per_group * row_bytes;
    p.parked = backward && per_thread == 16 ? p.threads * 16 * 4 : 0;
    const int aside = p.parked + ring::ASIDE;
    p.ctas = std::max(1, std::min(threads_per_sm / p.threads, ring::BYTES_PER_SM / (3 * p.stage_bytes + aside)));
    p.stages = std::max(2, std::min(ring::MAX_STAGES, (ring::BYTES_PER_SM / p.ctas - aside) / p.stage_bytes));
    // the groups' column sums of the backward pass (8 bytes a column) meet in the stages
    if (backward) while (p.stages * p.stage_bytes < groups * 8 * cols) ++p.stages;
    const int64_t all = (rows + static_cast<int64_t>(groups) * rows_per_group - 1) / (static_cast<int64_t>(groups) * rows_per_group);
    p.ctas = static_cast<int>(std::min<int64_t>({all, static_cast<int64_t>(p.ctas) * sms, backward ? bwd_parts_limit(rows, cols) : all}));
    return p;
}
static bool ring_operand(const void* p, int dtype, int64_t pitch, int64_t cols) {       // rows that bulk copies can fetch
    return !p || (aligned(p, 16) && pitch * dtype_size(dtype) % 16 == 0 && cols * dtype_size(dtype) % 16 == 0);
}
static int sm_count() {
    static int count[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return 148;
    if (!count[dev]) cudaDeviceGetAttribute(&count[dev], cudaDevAttrMultiProcessorCount, dev);
    return count[dev];
}
// Threads of KERNEL that the registers of an SM hold (allocated by eights a thread), asked once per kernel; 512 at 128 registers.
template <typename Args>
static int threads_that_fit(void (*kernel)(Args, int, int), int& known) {
    if (!known) {
        cudaFuncAttributes f;
        known = cudaFuncGetAttributes(&f, kernel) == cudaSuccess && f.numRegs > 0 ? 65536 / ((f.numRegs + 7) / 8 * 8) : 512;
    }
    return known;
}
// One launch of a ring kernel; KERNEL's shared-memory limit is raised once per device.
template <typename Args>
static bool launch_ring(void (*kernel)(Args, int, int), bool (&ready)[64], const Args& a, const ring::Plan& p, cudaStream_t st) {
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return false;
    if (!ready[dev]) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, ring::BYTES_PER_SM - ring::ASIDE) != cudaSuccess) return false;
        ready[dev] = true;
    }
    kernel<<<p.ctas, p.threads, p.stages * p.stage_bytes + p.parked, st>>>(a, p.stages, p.row_threads);
    return true;
}
template <typename TX, typename TD, typename TO, int C, int R, int MAXT, int CTAS>
static bool fwd_ring(const NormArgs& a, int row_bytes, int threads_per_sm, cudaStream_t st) {
    static bool ready[64] = {};
    static int fit = 0;
    const auto kernel = norm_fwd_ring_kernel<TX, TD, TO, C, R, MAXT, CTAS>;
    const ring::Plan p = ring_plan(a.rows, a.cols, R, row_bytes, sm_count(), std::min(threads_per_sm, threads_that_fit<NormArgs>(kernel, fit)), false);
    return launch_ring<NormArgs>(kernel, ready, a, p, st);
}
template <typename TX, typename TD, typename TO>
static bool fwd_ring_sized(const NormArgs& a, cudaStream_t st) {
    const int row_bytes = a.cols * static_cast<int>(sizeof(TX) + (a.delta ? sizeof(TD) : 0));
    const int row_threads = round_threads(a.cols);
    if (columns_per_thread(a.cols) == 8) return fwd_ring<TX, TD, TO, 8, 2, 256, 4>(a, row_bytes, 1024, st);
    if (row_threads <= 256) return fwd_ring<TX, TD, TO, 16, 1, 256, 2>(a, row_bytes, 640, st);
    return row_threads <= 320 ? fwd_ring<TX, TD, TO, 16, 1, 320, 2>(a, row_bytes, 640, st) : fwd_ring<TX, TD, TO, 16, 1, 512, 1>(a, row_bytes, 640, st);
}
template <typename TX, typename TH, int C, int R, int MAXT, int CTAS>
static int64_t bwd_ring(const NormBwdArgs& a, int row_bytes, cudaStream_t st) {
    static bool ready[64] = {};
    static int fit = 0;
    const auto kernel = norm_bwd_ring_kernel<TX, TH, C, R, MAXT, CTAS>;
    const int threads = std::min(bwd_threads_per_sm(a.cols), threads_that_fit<NormBwdArgs>(kernel, fit));
    const ring::Plan p = ring_plan(a.rows, a.cols, R, row_bytes, sm_count(), threads, true);
    return launch_ring<NormBwdArgs>(kernel, ready, a, p, st) ? p.ctas : 0;
}
template <typename TX, typename TH>
static int64_t bwd_ring_sized(const NormBwdArgs& a, cudaStream_t st) {
    const int row_bytes = a.cols * static_cast<int>(sizeof(TH) + sizeof(TX) * (a.dsum ? 2 : 1));
    const int row_threads = round_threads(a.cols);
    if (columns_per_thread(a.cols) == 8) return bwd_ring<TX, TH, 8, 2, 256, 2>(a, row_bytes, st);
    if (row_threads <= 256) return bwd_ring<TX, TH, 16, 1, 256, 2>(a, row_bytes, st);
    return row_threads <= 320 ? bwd_ring<TX, TH, 16, 1, 320, 2>(a, row_bytes, st) : bwd_ring<TX, TH, 16, 1, 512, 1>(a, row_bytes, st);
}

// Rows that bulk copies cannot fetch, or wider than the ring's threads hold: odd widths and unaligned rows element by element in
// registers up to 4096 columns, aligned rows of more than 8192 in vectors, the rest from memory each time.
template <typename TX, typename TO>
static void forward(const NormArgs& a, bool vector, bool ring, cudaStream_t st) {
    constexpr int V = 16 / sizeof(TX);
    if (ring) {
        if constexpr (sizeof(TX) == 4) {
            if (a.delta_bf16 ? fwd_ring_sized<TX, __nv_bfloat16, TO>(a, st) : fwd_ring_sized<TX, TX, TO>(a, st)) return;
        } else if (fwd_ring_sized<TX, TX, TO>(a, st)) {
            return;
        }
    }
    auto by_warp = [&](auto kernel) { kernel<<<static_cast<unsigned>(std::min((a.rows + 7) / 8, MAX_GRID)), 256, 0, st>>>(a); };
    auto by_cta = [&](auto kernel, int threads) { kernel<<<static_cast<unsigned>(std::min(a.rows, MAX_GRID)), threads, 0, st>>>(a); };
    if (a.cols <= 64) by_warp(norm_fwd_kernel<TX, TO, 1, 2, false>);
    else if (a.cols <= 256) by_warp(norm_fwd_kernel<TX, TO, 1, 8, false>);
    else if (a.cols <= 4096) by_cta(norm_fwd_kernel<TX, TO, 1, 4, true>, round32((a.cols + 3) / 4));
    else if (vector && a.cols <= 4 * V * 1024) by_cta(norm_fwd_kernel<TX, TO, V, 4, true>, round32((a.cols / V + 3) / 4));
    else by_cta(norm_fwd_any_kernel<TX, TO>, 256);
}

// Returns the number of partial rows.
template <typename TX, typename TH>
static int64_t backward(const NormBwdArgs& a, bool ring, cudaStream_t st) {
    if (ring)
        if (const int64_t parts = bwd_ring_sized<TX, TH>(a, st)) return parts;
    auto by_warp = [&](auto kernel) {
        const int64_t parts = std::min<int64_t>((a.rows + 7) / 8, SMS * 2);
        kernel<<<static_cast<unsigned>(parts), 256, 0, st>>>(a);
        return parts;
    };
    if (a.cols <= 256) return by_warp(norm_bwd_kernel<TX, TH, 8, false>);
    if (a.cols <= 768) return by_warp(norm_bwd_kernel<TX, TH, 24, false>);
    if (a.cols <= 4096) {
        const int threads = round32((a.cols + 7) / 8);
        const int64_t parts = std::min<int64_t>(a.rows, SMS * (threads <= 256 ? 3 : threads <= 384 ? 2 : 1));
        norm_bwd_kernel<TX, TH, 8, true><<<static_cast<unsigned>(parts), threads, 0, st>>>(a);
        return parts;
    }
    norm_bwd_any_kernel<TX, TH><<<static_cast<unsigned>(std::min(a.rows, MAX_GRID)), 256, 0, st>>>(a);
    if (!a.partial) return 1;
    const int64_t parts = column_pass_parts(a.rows, a.cols);
    norm_bwd_columns_kernel<TX, TH><<<dim3(static_cast<unsigned>((a.cols + 31) / 32), static_cast<unsigned>(parts)), 256, 0, st>>>(a);
    return parts;
}

}  // namespace nvfp4

using namespace nvfp4;

extern "C" int nvfp4_layer_norm(const void* x, int x_dtype, int64_t x_pitch, const void* delta, int delta_dtype, int64_t delta_pitch,
                                const void* weight, const void* bias, int weight_dtype, float eps, int64_t rows, int64_t cols,
                                void* sum_out, void* h_out, int h_dtype, float* mean_out, float* rstd_out, float* amax,
                                int* status, nvfp4_stream_t stream) {
    NVFP4_REQUIRE(x && h_out && (!delta || sum_out) && (mean_out == nullptr) == (rstd_out == nullptr), NVFP4_ERR_ARG, "nvfp4_layer_norm: null pointer");
    NVFP4_REQUIRE(rows > 0 && cols > 0 && cols < (1LL << 30) && x_pitch >= cols && (!delta || delta_pitch >= cols), NVFP4_ERR_ARG,
                  "nvfp4_layer_norm: rows and cols must be positive and the row pitches at least cols");
    NVFP4_REQUIRE(is_float_dtype(x_dtype) && is_float_dtype(h_dtype) && ((!weight && !bias) || is_float_dtype(weight_dtype)), NVFP4_ERR_DTYPE,
                  "nvfp4_layer_norm: FP32, BF16 or FP16 tensors");
    NVFP4_REQUIRE(h_dtype == x_dtype || (x_dtype == NVFP4_F32 && h_dtype == NVFP4_BF16), NVFP4_ERR_DTYPE,
                  "nvfp4_layer_norm: the result has the input's type, or BF16 beside an FP32 input");
    NVFP4_REQUIRE(!delta || delta_dtype == x_dtype || (x_dtype == NVFP4_F32 && delta_dtype == NVFP4_BF16), NVFP4_ERR_DTYPE,
                  "nvfp4_layer_norm: the second summand has the input's type, or BF16 beside an FP32 input");
    NormArgs a{x, delta, weight, bias, sum_out, h_out, mean_out, rstd_out, amax, status, x_pitch, delta_pitch, rows, static_cast<int>(cols),
               delta && delta_dtype != x_dtype, weight_dtype, eps};
    // 16-byte vectors of x need every operand's rows to start on a multiple of its own share of them
    const int v = 16 / dtype_size(x_dtype);
    auto fits = [&](const void* p, int dtype, int64_t pitch) { return !p || (aligned(p, std::min(16, v * dtype_size(dtype))) && pitch % v == 0); };
    const bool vector = cols % v == 0 && fits(x, x_dtype, x_pitch) && fits(delta, delta_dtype, delta_pitch) && fits(sum_out, x_dtype, cols) &&
                        fits(h_out, h_dtype, cols) && fits(weight, weight_dtype, 0) && fits(bias, weight_dtype, 0);
    const bool ring = vector && cols <= 8192 && ring_operand(x, x_dtype, x_pitch, cols) && ring_operand(delta, delta_dtype, delta_pitch, cols);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (x_dtype == NVFP4_BF16) forward<__nv_bfloat16, __nv_bfloat16>(a, vector, ring, st);
    else if (x_dtype == NVFP4_F16) forward<__half, __half>(a, vector, ring, st);
    else if (h_dtype == NVFP4_F32) forward<float, float>(a, vector, ring, st);
    else forward<float, __nv_bfloat16>(a, vector, ring, st);
    return launch_status("nvfp4_layer_norm");
}

extern "C" int64_t nvfp4_layer_norm_bwd_partials(int64_t rows, int64_t cols) {
    return rows > 0 && cols > 0 ? std::max<int64_t>(1, bwd_parts_limit(rows, std::min<int64_t>(cols, 1 << 30))) : 1;
}

extern "C" int nvfp4_layer_norm_bwd(const void* dh, int h_dtype, int64_t dh_pitch, const void* total, int x_dtype, int64_t total_pitch,
                                    const float* mean, const float* rstd, const void* weight, int weight_dtype, const void* dsum,
                                    int64_t dsum_pitch, int64_t rows, int64_t cols, void* dx, void* ddelta, float* partial, void* dweight,
                                    void* dbias, float* amax, int* status, nvfp4_stream_t stream) {
    NVFP4_REQUIRE(dh && total && mean && rstd && dx && ((!dweight && !dbias) || partial), NVFP4_ERR_ARG, "nvfp4_layer_norm_bwd: null pointer");
    NVFP4_REQUIRE(rows > 0 && cols > 0 && cols < (1LL << 30) && dh_pitch >= cols && total_pitch >= cols && (!dsum || dsum_pitch >= cols), NVFP4_ERR_ARG,
                  "nvfp4_layer_norm_bwd: rows and cols must be positive and the row pitches at least cols");
    NVFP4_REQUIRE(is_float_dtype(x_dtype) && (h_dtype == x_dtype || (x_dtype == NVFP4_F32 && h_dtype == NVFP4_BF16)) &&
                  ((!weight && !dweight && !dbias) || is_float_dtype(weight_dtype)), NVFP4_ERR_DTYPE, "nvfp4_layer_norm_bwd: FP32, BF16 or FP16 tensors");
    NVFP4_REQUIRE(!ddelta || x_dtype == NVFP4_F32, NVFP4_ERR_DTYPE, "nvfp4_layer_norm_bwd: ddelta is the BF16 copy of an FP32 dx");
    NormBwdArgs a{dh, total, weight, dsum, mean, rstd, dx, ddelta, status, (dweight || dbias) ? partial : nullptr, amax, dh_pitch, total_pitch, dsum_pitch,
                  rows, static_cast<int>(cols), weight_dtype};
    const int v = 16 / dtype_size(x_dtype);
    auto fits = [&](const void* p, int dtype, int64_t pitch) { return !p || (aligned(p, std::min(16, v * dtype_size(dtype))) && pitch % v == 0); };
    bool ring = cols % v == 0 && cols <= 8192 && fits(dh, h_dtype, dh_pitch) && fits(total, x_dtype, total_pitch) && fits(dsum, x_dtype, dsum_pitch) &&
                        fits(dx, x_dtype, cols) && fits(ddelta, NVFP4_BF16, cols) && fits(weight, weight_dtype, 0) && aligned(partial, 16);
    ring = ring && ring_operand(dh, h_dtype, dh_pitch, cols) && ring_operand(total, x_dtype, total_pitch, cols) && ring_operand(dsum, x_dtype, dsum_pitch, cols);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    int64_t parts;
    if (x_dtype == NVFP4_BF16) parts = backward<__nv_bfloat16, __nv_bfloat16>(a, ring, st);
    else if (x_dtype == NVFP4_F16) parts = backward<__half, __half>(a, ring, st);
    else if (h_dtype == NVFP4_F32) parts = backward<float, float>(a, ring, st);
    else parts = backward<float, __nv_bfloat16>(a, ring, st);
    if (a.partial)
        column_sums_kernel<<<static_cast<unsigned>((2 * cols + 31) / 32), SUM_WARPS * 32, 0, st>>>(partial, parts, 2 * cols, cols, dweight, dbias, weight_dtype);
    return launch_status("nvfp4_layer_norm_bwd");
}

extern "C" int nvfp4_column_sums(const float* partial, int64_t parts, int64_t cols, void* out, int out_dtype, nvfp4_stream_t stream) {
    NVFP4_REQUIRE(partial && out && parts > 0 && cols > 0 && cols < (1LL << 31), NVFP4_ERR_ARG, "nvfp4_column_sums: null pointer or empty size");
    NVFP4_REQUIRE(is_float_dtype(out_dtype), NVFP4_ERR_DTYPE, "nvfp4_column_sums: FP32, BF16 or FP16 result");
    column_sums_kernel<<<static_cast<unsigned>((cols + 31) / 32), SUM_WARPS * 32, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
        partial, parts, cols, cols, out, nullptr, out_dtype);
    return launch_status("nvfp4_column_sums");
}
