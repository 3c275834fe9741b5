// Rotary positions over several axes (time, height, width): pair j of a head turns by position[token][axis(j)] * frequency(j).
//
// A warp takes a token (or a share of its heads).  Its lanes first form the sines and cosines of the token's pairs, once for
// all heads of q and k: the angle in FP64 as a number of full turns, then sincospi in FP32 on its fraction.  The frequency and its
// product with the position are rounded to 53 bits, an error of about |position * frequency| * 2^-52 of an angle in radians (2^-21
// at 2^31, 2^-12 at 2^40); the fraction of that product is exact but for its rounding to FP32, another 2^-24.  Every lane then keeps the values of its own chunk of a head in registers and streams
// that chunk of head after head: two vectors per head, V pairs.  No table is read, and q, k (and v, where a fused projection's
// gradient is put together) cross HBM once each way, which is the bound: 75600 tokens x 80 heads of 128 in BF16 take 471 us, the
// measured HBM rate.
#include "bf16x8.cuh"
#include "vec.cuh"

#include <algorithm>

namespace nvfp4 {

constexpr int ROT_WARPS = 8;
// Heads whose loads a lane has in flight.  Three of them leave registers for three CTAs per SM: four (two CTAs) took 85 against
// 78 us for 17408 tokens x 48 heads of 128 and 16.4 against 11.8 us for 3063 x 32 of 72 in FP32; two (four CTAs) took 79 and 11.9.
constexpr int ROT_AHEAD = 3;

struct RotaryArgs {
    const void* x[3];
    void* out[3];
    int64_t xs[3][3], os[3][3];        // [tensor][batch, seq, head]
    int first[4];                        // tensor t holds heads first[t] .. first[t + 1] - 1 of the joint head index
    int turn[3];
    const void* positions;
    int64_t ps[3];
    float* amax;
    int64_t batch, seq, items;
    int dim, pairs, splits, heads_per_split, position_kind;
    float sign;
    double turns[NVFP4_ROTARY_MAX_PAIRS];
    uint8_t axis[NVFP4_ROTARY_MAX_PAIRS];
};

__device__ __forceinline__ double position_at(const RotaryArgs& a, int64_t i) {
    if (a.position_kind == 0) return static_cast<double>(static_cast<const int64_t*>(a.positions)[i]);
    if (a.position_kind == 1) return static_cast<double>(static_cast<const int32_t*>(a.positions)[i]);
    if (a.position_kind == 2) return static_cast<double>(static_cast<const float*>(a.positions)[i]);
    return static_cast<const double*>(a.positions)[i];
}

// INTER: pair j is features (2j, 2j + 1), else (j, j + pairs).  A lane's chunk c is the vectors at c V and pairs + c V either
// way (V divides pairs): V pairs (c V + i) in the split layout, V / 2 pairs of each vector in the interleaved one.  With
// V == 1 the interleaved chunk is the two features 2c, 2c + 1.
template <typename T, int V, bool INTER>
__global__ void __launch_bounds__(ROT_WARPS * 32, 3) rotary_axes_kernel(const __grid_constant__ RotaryArgs a) {
    __shared__ float2 table[ROT_WARPS][NVFP4_ROTARY_MAX_PAIRS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int chunks = a.pairs / V;
    const int off_b = (INTER && V == 1) ? 1 : a.pairs;
    const int rest0 = 2 * a.pairs, rest = (a.dim - rest0) / V;     // vectors behind the turned features
    float best = 0.f;
    for (int64_t item = static_cast<int64_t>(blockIdx.x) * ROT_WARPS + warp; item < a.items; item += static_cast<int64_t>(gridDim.x) * ROT_WARPS) {
        const int64_t token = item / a.splits;
        const int h0 = static_cast<int>(item - token * a.splits) * a.heads_per_split, h1 = min(h0 + a.heads_per_split, a.first[3]);
        const int64_t b = token / a.seq, s = token - b * a.seq;
        __syncwarp();
        for (int j = lane; j < a.pairs; j += 32) {
            const double t = position_at(a, b * a.ps[0] + s * a.ps[1] + a.axis[j] * a.ps[2]) * a.turns[j];
            float sn, cs;
            sincospif(static_cast<float>(2.0 * (t - rint(t))), &sn, &cs);
            table[warp][j] = make_float2(cs, sn * a.sign);
        }
        __syncwarp();
        auto address = [&](int h, int64_t& in, int64_t& out, int& which) {
            which = h < a.first[1] ? 0 : h < a.first[2] ? 1 : 2;
            const int local = h - (which == 0 ? 0 : which == 1 ? a.first[1] : a.first[2]);
            in = b * a.xs[which][0] + s * a.xs[which][1] + local * a.xs[which][2];
            out = b * a.os[which][0] + s * a.os[which][1] + local * a.os[which][2];
        };
        for (int c0 = 0; c0 < chunks; c0 += 32) {
            const int here = min(chunks - c0, 32), abreast = 32 / here;      // heads side by side in the warp
            const int c = c0 + lane % here, slot = lane / here;
            if (slot >= abreast) continue;
            const int at = (INTER && V == 1) ? 2 * c : c * V;
            float cs[V], sn[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int pair = !INTER ? c * V + i : V == 1 ? c : (i < V / 2 ? c * V / 2 + i : a.pairs / 2 + c * V / 2 + i - V / 2);
                const float2 e = table[warp][pair];
                cs[i] = e.x; sn[i] = e.y;
            }
            for (int h = h0 + slot; h < h1; h += abreast * ROT_AHEAD) {
                Pack<T, V> pa[ROT_AHEAD], pb[ROT_AHEAD];
                int64_t out[ROT_AHEAD];
                int which[ROT_AHEAD];
#pragma unroll
                for (int k = 0; k < ROT_AHEAD; ++k) {
                    const int hk = h + k * abreast;
                    if (hk < h1) {
                        int64_t in;
                        address(hk, in, out[k], which[k]);
                        const T* x = static_cast<const T*>(a.x[which[k]]) + in + at;
                        pa[k] = load_pack<T, V>(x);
                        pb[k] = load_pack<T, V>(x + off_b);
                    }
                }
#pragma unroll
                for (int k = 0; k < ROT_AHEAD; ++k) {
                    if (h + k * abreast >= h1) continue;
                    if (a.turn[which[k]]) {
                        float fa[V], fb[V], ra[V], rb[V];
                        unpack(pa[k], fa); unpack(pb[k], fb);
                        if constexpr (!INTER || V == 1) {
#pragma unroll
                            for (int i = 0; i < V; ++i) {
                                ra[i] = fa[i] * cs[i] - fb[i] * sn[i];
                                rb[i] = fb[i] * cs[i] + fa[i] * sn[i];
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < V / 2; ++i) {
                                ra[2 * i] = fa[2 * i] * cs[i] - fa[2 * i + 1] * sn[i];
                                ra[2 * i + 1] = fa[2 * i + 1] * cs[i] + fa[2 * i] * sn[i];
                                rb[2 * i] = fb[2 * i] * cs[V / 2 + i] - fb[2 * i + 1] * sn[V / 2 + i];
                                rb[2 * i + 1] = fb[2 * i + 1] * cs[V / 2 + i] + fb[2 * i] * sn[V / 2 + i];
                            }
                        }
                        pa[k] = pack<T, V>(ra); pb[k] = pack<T, V>(rb);
                    }
                    T* o = static_cast<T*>(a.out[which[k]]) + out[k] + at;
                    store_pack(o, pa[k]);
                    store_pack(o + off_b, pb[k]);
                    if (a.amax) best = fmaxf(best, fmaxf(abs_max(pa[k]), abs_max(pb[k])));
                }
            }
        }
        for (int i = lane; i < (h1 - h0) * rest; i += 32) {
            int64_t in, out;
            int which;
            address(h0 + i / rest, in, out, which);
            const int at = rest0 + i % rest * V;
            const Pack<T, V> p = load_pack<T, V>(static_cast<const T*>(a.x[which]) + in + at);
            store_pack(static_cast<T*>(a.out[which]) + out + at, p);
            if (a.amax) best = fmaxf(best, abs_max(p));
        }
    }
    if (a.amax) block_atomic_amax(a.amax, best);
}

template <typename T, int V>
static void launch_rotary(const RotaryArgs& a, bool interleaved, cudaStream_t st) {
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>((a.items + ROT_WARPS - 1) / ROT_WARPS, 148 * 32));
    if (interleaved) rotary_axes_kernel<T, V, true><<<grid, ROT_WARPS * 32, 0, st>>>(a);
    else rotary_axes_kernel<T, V, false><<<grid, ROT_WARPS * 32, 0, st>>>(a);
}

template <typename T>
static void rotary(const RotaryArgs& a, int v, bool interleaved, cudaStream_t st) {
    if (sizeof(T) == 2 && v == 8) launch_rotary<T, sizeof(T) == 2 ? 8 : 4>(a, interleaved, st);
    else if (v == 4) launch_rotary<T, 4>(a, interleaved, st);
    else if (v == 2) launch_rotary<T, 2>(a, interleaved, st);
    else launch_rotary<T, 1>(a, interleaved, st);
}

}  // namespace nvfp4

using namespace nvfp4;

extern "C" int nvfp4_rotary_axes(const nvfp4_rotary_tensor* tensors, int count, int dtype, int64_t batch, int64_t seq, int dim,
                                 const void* positions, int position_kind, const int64_t* position_stride, int axes, const double* turns,
                                 const uint8_t* axis, int pairs, int interleaved, int inverse, float* amax, nvfp4_stream_t stream) {
    NVFP4_REQUIRE(tensors && positions && position_stride && turns && axis, NVFP4_ERR_ARG, "nvfp4_rotary_axes: null pointer");
    NVFP4_REQUIRE(count >= 1 && count <= 3 && batch > 0 && seq > 0 && dim > 0 && axes > 0, NVFP4_ERR_ARG, "nvfp4_rotary_axes: one to three tensors of positive sizes");
    NVFP4_REQUIRE(pairs > 0 && pairs <= NVFP4_ROTARY_MAX_PAIRS && 2 * pairs <= dim, NVFP4_ERR_ARG,
                  "nvfp4_rotary_axes: between 1 and %d pairs, at most half of the head dimension", NVFP4_ROTARY_MAX_PAIRS);
    NVFP4_REQUIRE(is_float_dtype(dtype), NVFP4_ERR_DTYPE, "nvfp4_rotary_axes: FP32, BF16 or FP16 tensors");
    NVFP4_REQUIRE(position_kind >= 0 && position_kind <= 3, NVFP4_ERR_DTYPE, "nvfp4_rotary_axes: int64, int32, FP32 or FP64 positions");
    NVFP4_REQUIRE(batch < (1LL << 31) && seq < (1LL << 31), NVFP4_ERR_ARG, "nvfp4_rotary_axes: batch and seq must be below 2^31");
    RotaryArgs a{};
    int heads = 0;
    // the widest vector that divides the halves and the rest of a head, and that every row starts on
    int v = 16 / dtype_size(dtype);
    auto narrow = [&](int64_t n) { while (n % v) v >>= 1; };
    narrow(pairs);
    narrow(dim - 2 * pairs);
    for (int t = 0; t < 3; ++t) {
        a.first[t] = heads;
        if (t >= count) continue;
        const nvfp4_rotary_tensor& q = tensors[t];
        NVFP4_REQUIRE(q.x && q.out && q.heads > 0 && q.heads < (1 << 20), NVFP4_ERR_ARG, "nvfp4_rotary_axes: null pointer or no heads");
        a.x[t] = q.x; a.out[t] = q.out; a.turn[t] = q.turn;
        heads += q.heads;
        for (int i = 0; i < 3; ++i) {
            a.xs[t][i] = q.x_stride[i]; a.os[t][i] = q.out_stride[i];
            // a stride along an extent of one is never taken
            const bool taken = i == 0 ? batch > 1 : i == 1 ? seq > 1 : q.heads > 1;
            if (taken) { narrow(q.x_stride[i]); narrow(q.out_stride[i]); }
        }
        while (!aligned(q.x, v * dtype_size(dtype)) || !aligned(q.out, v * dtype_size(dtype))) {
            NVFP4_REQUIRE(v > 1, NVFP4_ERR_ALIGN, "nvfp4_rotary_axes: tensors must be aligned to their elements");
            v >>= 1;
        }
    }
    a.first[3] = heads;
    NVFP4_REQUIRE(static_cast<int64_t>(heads) * dim < (1LL << 30), NVFP4_ERR_ARG, "nvfp4_rotary_axes: the heads of a token must have fewer than 2^30 features in all");
    for (int j = 0; j < pairs; ++j) {
        NVFP4_REQUIRE(axis[j] < axes, NVFP4_ERR_ARG, "nvfp4_rotary_axes: a pair names an axis that the positions do not have");
        a.turns[j] = turns[j];
        a.axis[j] = axis[j];
    }
    a.positions = positions;
    for (int i = 0; i < 3; ++i) a.ps[i] = position_stride[i];
    a.amax = amax; a.batch = batch; a.seq = seq; a.dim = dim; a.pairs = pairs; a.position_kind = position_kind;
    a.sign = inverse ? -1.f : 1.f;
    // few tokens: several warps share a token's heads until about 16 warps per SM have work, each with at least four heads
    const int64_t tokens = batch * seq, want = 148 * 16;
    a.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(want / tokens, heads / 4)));
    a.heads_per_split = (heads + a.splits - 1) / a.splits;
    a.splits = (heads + a.heads_per_split - 1) / a.heads_per_split;
    a.items = tokens * a.splits;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (dtype == NVFP4_BF16) rotary<__nv_bfloat16>(a, v, interleaved != 0, st);
    else if (dtype == NVFP4_F16) rotary<__half>(a, v, interleaved != 0, st);
    else rotary<float>(a, v, interleaved != 0, st);
    return launch_status("nvfp4_rotary_axes");
}
