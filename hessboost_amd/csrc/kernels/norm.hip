// Root-mean-square norm of rows and its gradient, and rows to 8 bits and back.
//
//   s = x + residual; inv = 1 / sqrt(mean s^2 + eps); n = s inv; out = n weight
//   g = dout weight; dx = inv (g - n mean(g n)) + dtotal; dweight = sum over rows dout n
//
// A row lies on `lanes` lanes and stays in their registers between its sum and
// its results: it is read once and written once. A lane's columns are the same
// in every row, so that the weights are loaded once and the weights' gradient is
// summed in registers, joined in LDS and over the workgroups in order.
#include "rows8.h"

namespace hbr {

template <typename E, int V>
__device__ __forceinline__ void load_up(const void *p, uint64_t at, float (&v)[V]) {
    const Vec<typename E::type, V> x = *reinterpret_cast<const Vec<typename E::type, V> *>(static_cast<const typename E::type *>(p) + at);
#pragma unroll
    for (int k = 0; k < V; k++) v[k] = E::up(x.v[k]);
}

template <typename E, int V>
__device__ __forceinline__ void store_down(void *p, uint64_t at, const float (&v)[V]) {
    Vec<typename E::type, V> x;
#pragma unroll
    for (int k = 0; k < V; k++) x.v[k] = E::down(v[k]);
    *reinterpret_cast<Vec<typename E::type, V> *>(static_cast<typename E::type *>(p) + at) = x;
}

// The sum over a row's lanes, the same bits in each. More than a wave's lanes
// are the workgroup's, and all of it calls.
template <typename T>
__device__ __forceinline__ T row_sum(T v, uint32_t lanes) {
    __shared__ T wave_sum[2][16];
    static_assert(sizeof(T) <= 8, "a register or two");
    for (uint32_t d = min(lanes, (uint32_t)kWave) / 2; d; d /= 2) v += __shfl_xor(v, d, kWave);
    if (lanes <= (uint32_t)kWave) return v;
    const uint32_t wave = threadIdx.x / kWave, waves = lanes / kWave;
    __syncthreads();
    if (lane_id() == 0) wave_sum[0][wave] = v;
    __syncthreads();
    v = wave_sum[0][0];
    for (uint32_t w = 1; w < waves; w++) v += wave_sum[0][w];
    return v;
}

// A sum of squares that f32 does not hold is taken again in f64.
__device__ __forceinline__ bool beyond_f32(float sum, float eps) {
    return !(sum < INFINITY) || (sum < 1e-30f && eps < 1e-30f);
}
__device__ __forceinline__ float inverse_of(float sum, float mean, float eps) {
    return __builtin_amdgcn_rsqf(__builtin_fmaf(sum, mean, eps));
}
__device__ __forceinline__ float inverse_of(double sum, uint32_t dim, float eps) {
    return (float)(1.0 / __builtin_sqrt(sum / (double)dim + (double)eps));
}

// The largest magnitude of 32 columns, on the lanes that hold them.
template <int V>
__device__ __forceinline__ float block_largest(const float (&v)[V]) {
    float m = 0.0f;
#pragma unroll
    for (int k = 0; k < V; k++) m = fmaxf(m, magnitude(v[k]));
#pragma unroll
    for (int d = 1; d < (int)kPackBlock / V; d *= 2) m = fmaxf(m, __shfl_xor(m, d, kWave));
    return m;
}

// One vector of a row into codes, the block's first lane writing its power. `is`: within the row.
template <int V>
__device__ __forceinline__ void put_codes(uint8_t *codes, uint8_t *scales, uint32_t vec, bool is, const float (&v)[V]) {
    const int32_t power = power_of(block_largest<V>(v));
    if (!is) return;
    *reinterpret_cast<Vec<uint8_t, V> *>(codes + vec * V) = codes_of<V>(v, exp2_of(-power));
    if (vec % (kPackBlock / V) == 0) scales[vec / (kPackBlock / V)] = (uint8_t)(power + kPowerBias);
}

template <int V>
__device__ __forceinline__ void get_codes(const uint8_t *codes, const uint8_t *scales, uint32_t vec, float (&v)[V]) {
    const float power = exp2_of((int32_t)scales[vec / (kPackBlock / V)] - kPowerBias);
    values_of<V>(*reinterpret_cast<const Vec<uint8_t, V> *>(codes + vec * V), power, v);
}

// U vectors a lane in registers; 0: any number, read again where they are used.
template <typename E, int V, int U>
__device__ __forceinline__ void rms_norm(const NormArgs &a) {
    constexpr int kHeld = U ? U : 1;
    const uint32_t lanes = a.lanes, in = threadIdx.x & (lanes - 1), per = blockDim.x / lanes;
    const uint32_t rounds = U ? U : (a.vecs + lanes - 1) / lanes;
    float s[kHeld][V], w[kHeld][V];
    auto weights = [&](uint32_t i, float (&to)[V]) {
#pragma unroll
        for (int k = 0; k < V; k++) to[k] = 1.0f;
        if (a.weight && i < a.vecs) load_up<F32, V>(a.weight, (uint64_t)i * V, to);
    };
    if constexpr (U != 0) {
#pragma unroll
        for (int u = 0; u < U; u++) weights(in + u * lanes, w[u]);
    }
    for (uint64_t r0 = (uint64_t)blockIdx.x * per; r0 < a.n_rows; r0 += (uint64_t)gridDim.x * per) {
        const uint64_t r = r0 + threadIdx.x / lanes;
        const bool live = r < a.n_rows;
        auto read = [&](uint32_t i, float (&to)[V]) {
#pragma unroll
            for (int k = 0; k < V; k++) to[k] = 0.0f;
            if (!live || i >= a.vecs) return;
            load_up<E, V>(a.x, r * a.x_stride + (uint64_t)i * V, to);
            if (a.residual) {
                float more[V];
                load_up<E, V>(a.residual, r * a.residual_stride + (uint64_t)i * V, more);
#pragma unroll
                for (int k = 0; k < V; k++) to[k] += more[k];
            }
        };
        float sum = 0.0f;
        auto squares = [&](const float (&v)[V]) {
#pragma unroll
            for (int k = 0; k < V; k++) sum = __builtin_fmaf(v[k], v[k], sum);
        };
        if constexpr (U != 0) {
#pragma unroll
            for (int u = 0; u < U; u++) read(in + u * lanes, s[u]);
#pragma unroll
            for (int u = 0; u < U; u++) squares(s[u]);
        } else {
            for (uint32_t u = 0; u < rounds; u++) read(in + u * lanes, s[0]), squares(s[0]);
        }
        sum = row_sum(sum, lanes);
        float inv = inverse_of(sum, a.mean, a.eps);
        if (beyond_f32(sum, a.eps)) {
            double far = 0.0;
            auto far_squares = [&](const float (&v)[V]) {
#pragma unroll
                for (int k = 0; k < V; k++) far = __builtin_fma((double)v[k], (double)v[k], far);
            };
            if constexpr (U != 0) {
#pragma unroll
                for (int u = 0; u < U; u++) far_squares(s[u]);
            } else {
                for (uint32_t u = 0; u < rounds; u++) read(in + u * lanes, s[0]), far_squares(s[0]);
            }
            inv = inverse_of(row_sum(far, lanes), a.dim, a.eps);
        }
        if (a.inv && live && in == 0) a.inv[r] = inv;
        auto write = [&](uint32_t i, float (&v)[V], const float (&by)[V]) {
            const bool is = live && i < a.vecs;
            if (a.total && is) store_down<E, V>(a.total, r * a.total_stride + (uint64_t)i * V, v);
            float out[V];
#pragma unroll
            for (int k = 0; k < V; k++) {
                v[k] *= inv;
                out[k] = v[k] * by[k];
            }
            if (a.out && is) store_down<E, V>(a.out, r * a.out_stride + (uint64_t)i * V, out);
            if (!a.codes) return;
            if (!is) {  // (an inv that is no number makes none of the zeros past the row)
#pragma unroll
                for (int k = 0; k < V; k++) v[k] = out[k] = 0.0f;
            }
            uint8_t *codes = a.codes + r * a.codes_stride, *scales = a.scales + r * a.scales_stride;
            if (a.normed) put_codes<V>(codes, scales, i, is, v);
            else put_codes<V>(codes, scales, i, is, out);
        };
        if constexpr (U != 0) {
#pragma unroll
            for (int u = 0; u < U; u++) write(in + u * lanes, s[u], w[u]);
        } else {
            for (uint32_t u = 0; u < rounds; u++) {
                read(in + u * lanes, s[0]);
                weights(in + u * lanes, w[0]);
                write(in + u * lanes, s[0], w[0]);
            }
        }
    }
}

template <typename E, int V, int U>
__device__ __forceinline__ void rms_norm_grad(const NormGradArgs &a) {
    constexpr int kHeld = U ? U : 1;
    // the rows' sums of a workgroup of 256 threads
    __shared__ float sums[U ? 256 * U * V : 1];
    const uint32_t lanes = a.lanes, in = threadIdx.x & (lanes - 1), per = blockDim.x / lanes;
    const uint32_t rounds = U ? U : (a.vecs + lanes - 1) / lanes;
    float n[kHeld][V], d[kHeld][V], w[kHeld][V], acc[kHeld][V] = {};
    auto weights = [&](uint32_t i, float (&to)[V]) {
#pragma unroll
        for (int k = 0; k < V; k++) to[k] = 1.0f;
        if (a.weight && i < a.vecs) load_up<F32, V>(a.weight, (uint64_t)i * V, to);
    };
    if constexpr (U != 0) {
#pragma unroll
        for (int u = 0; u < U; u++) weights(in + u * lanes, w[u]);
    }
    float *part = a.part ? a.part + (uint64_t)blockIdx.x * a.dim : nullptr;
    bool first = true;
    for (uint64_t r0 = (uint64_t)blockIdx.x * per; r0 < a.n_rows; r0 += (uint64_t)gridDim.x * per) {
        const uint64_t r = r0 + threadIdx.x / lanes;
        const bool live = r < a.n_rows;
        auto rows = [&](uint32_t i, float (&to)[V]) {
#pragma unroll
            for (int k = 0; k < V; k++) to[k] = 0.0f;
            if (!live || i >= a.vecs) return;
            if (a.codes) get_codes<V>(a.codes + r * a.codes_stride, a.scales + r * a.scales_stride, i, to);
            else load_up<E, V>(a.x, r * a.x_stride + (uint64_t)i * V, to);
        };
        auto douts = [&](uint32_t i, float (&to)[V]) {
#pragma unroll
            for (int k = 0; k < V; k++) to[k] = 0.0f;
            if (live && i < a.vecs) load_up<E, V>(a.dout, r * a.dout_stride + (uint64_t)i * V, to);
        };
        if constexpr (U != 0) {
#pragma unroll
            for (int u = 0; u < U; u++) rows(in + u * lanes, n[u]);
#pragma unroll
            for (int u = 0; u < U; u++) douts(in + u * lanes, d[u]);
        }
        float inv = a.inv && live ? a.inv[r] : 1.0f;
        if (!a.inv) {
            float sum = 0.0f;
            auto squares = [&](const float (&v)[V]) {
#pragma unroll
                for (int k = 0; k < V; k++) sum = __builtin_fmaf(v[k], v[k], sum);
            };
            if constexpr (U != 0) {
#pragma unroll
                for (int u = 0; u < U; u++) squares(n[u]);
            } else {
                for (uint32_t u = 0; u < rounds; u++) rows(in + u * lanes, n[0]), squares(n[0]);
            }
            sum = row_sum(sum, lanes);
            inv = inverse_of(sum, a.mean, a.eps);
            if (beyond_f32(sum, a.eps)) {
                double far = 0.0;
                auto far_squares = [&](const float (&v)[V]) {
#pragma unroll
                    for (int k = 0; k < V; k++) far = __builtin_fma((double)v[k], (double)v[k], far);
                };
                if constexpr (U != 0) {
#pragma unroll
                    for (int u = 0; u < U; u++) far_squares(n[u]);
                } else {
                    for (uint32_t u = 0; u < rounds; u++) rows(in + u * lanes, n[0]), far_squares(n[0]);
                }
                inv = inverse_of(row_sum(far, lanes), a.dim, a.eps);
            }
        }
        // codes hold the rows as they were normalised
        const float by = a.codes ? 1.0f : inv;
        float along = 0.0f;
        auto add = [&](float (&v)[V], const float (&dy)[V], const float (&of)[V]) {
#pragma unroll
            for (int k = 0; k < V; k++) {
                v[k] *= by;
                along = __builtin_fmaf(dy[k] * of[k], v[k], along);
            }
        };
        if constexpr (U != 0) {
#pragma unroll
            for (int u = 0; u < U; u++) add(n[u], d[u], w[u]);
        } else {
            for (uint32_t u = 0; u < rounds; u++) {
                rows(in + u * lanes, n[0]);
                douts(in + u * lanes, d[0]);
                weights(in + u * lanes, w[0]);
                add(n[0], d[0], w[0]);
            }
        }
        along = row_sum(along, lanes) * a.mean;
        auto write = [&](uint32_t i, const float (&v)[V], const float (&dy)[V], const float (&of)[V], float (&total)[V]) {
            const bool is = live && i < a.vecs;
            if (!is) return;
            float dx[V];
#pragma unroll
            for (int k = 0; k < V; k++) {
                total[k] = __builtin_fmaf(dy[k], v[k], total[k]);
                dx[k] = inv * __builtin_fmaf(-v[k], along, dy[k] * of[k]);
            }
            if (!a.dx) return;
            if (a.dtotal) {
                float more[V];
                load_up<E, V>(a.dtotal, r * a.dtotal_stride + (uint64_t)i * V, more);
#pragma unroll
                for (int k = 0; k < V; k++) dx[k] += more[k];
            }
            store_down<E, V>(a.dx, r * a.dx_stride + (uint64_t)i * V, dx);
        };
        if constexpr (U != 0) {
#pragma unroll
            for (int u = 0; u < U; u++) write(in + u * lanes, n[u], d[u], w[u], acc[u]);
        } else {
            for (uint32_t u = 0; u < rounds; u++) {
                const uint32_t i = in + u * lanes;
                rows(i, n[0]);
                douts(i, d[0]);
                weights(i, w[0]);
#pragma unroll
                for (int k = 0; k < V; k++) n[0][k] *= by, acc[0][k] = 0.0f;
                // a lane's columns of its workgroup's sums are its own
                if (part && !first && i < a.vecs) load_up<F32, V>(part, (uint64_t)i * V, acc[0]);
                write(i, n[0], d[0], w[0], acc[0]);
                if (part && i < a.vecs) store_down<F32, V>(part, (uint64_t)i * V, acc[0]);
            }
            first = false;
        }
    }
    if (U == 0 || !part) return;
    if (lanes > (uint32_t)kWave) {
#pragma unroll
        for (int u = 0; u < kHeld; u++)
            if (in + u * lanes < a.vecs) store_down<F32, V>(part, (uint64_t)(in + u * lanes) * V, acc[u]);
        return;
    }
    const uint32_t cols = lanes * kHeld * V;  // of a row's sums
#pragma unroll
    for (int u = 0; u < kHeld; u++)
#pragma unroll
        for (int k = 0; k < V; k++) sums[threadIdx.x / lanes * cols + (in + u * lanes) * V + k] = acc[u][k];
    __syncthreads();
    for (uint32_t c = threadIdx.x; c < a.dim; c += blockDim.x) {
        float sum = sums[c];
        for (uint32_t g = 1; g < per; g++) sum += sums[g * cols + c];
        part[c] = sum;
    }
}

template <typename E, int V>
__device__ __forceinline__ void pack_rows(const PackArgs &a) {
    const uint32_t lanes = a.lanes, in = threadIdx.x & (lanes - 1), per = blockDim.x / lanes;
    const uint32_t first = blockIdx.y * a.each * lanes, end = min(first + a.each * lanes, (a.vecs + 31) / 32 * 32);
    for (uint64_t r0 = (uint64_t)blockIdx.x * per; r0 < a.n_rows; r0 += (uint64_t)gridDim.x * per) {
        const uint64_t r = r0 + threadIdx.x / lanes;
        for (uint32_t i0 = first; i0 < end; i0 += lanes) {
            const uint32_t i = i0 + in;
            const bool is = r < a.n_rows && i < a.vecs;
            float v[V] = {};
            if (is) load_up<E, V>(a.x, r * a.x_stride + (uint64_t)i * V, v);
            put_codes<V>(a.codes + r * a.codes_stride, a.scales + r * a.scales_stride, i, is, v);
        }
    }
}

template <typename E, int V>
__device__ __forceinline__ void unpack_rows(const PackArgs &a) {
    const uint32_t lanes = a.lanes, in = threadIdx.x & (lanes - 1), per = blockDim.x / lanes;
    const uint32_t first = blockIdx.y * a.each * lanes, end = min(first + a.each * lanes, a.vecs);
    for (uint64_t r = (uint64_t)blockIdx.x * per + threadIdx.x / lanes; r < a.n_rows; r += (uint64_t)gridDim.x * per)
        for (uint32_t i = first + in; i < end; i += lanes) {
            float v[V];
            get_codes<V>(a.codes + r * a.codes_stride, a.scales + r * a.scales_stride, i, v);
            if (a.weight) {
                float w[V];
                load_up<F32, V>(a.weight, (uint64_t)i * V, w);
#pragma unroll
                for (int k = 0; k < V; k++) v[k] *= w[k];
            }
            store_down<E, V>(a.x, r * a.x_stride + (uint64_t)i * V, v);
        }
}

}  // namespace hbr

using namespace hbr;

#define HBR_NORM(suffix, E, V, U)                                                                                      \
    extern "C" __global__ __launch_bounds__(1024) void hbr_rms_norm_##suffix(NormArgs a) { rms_norm<E, V, U>(a); }     \
    extern "C" __global__ __launch_bounds__(1024) void hbr_rms_norm_grad_##suffix(NormGradArgs a) { rms_norm_grad<E, V, U>(a); }
#define HBR_ROWS(t, E, V)                                                                                    \
    HBR_NORM(t##_##V##_0, E, V, 0)                                                                           \
    HBR_NORM(t##_##V##_1, E, V, 1)                                                                           \
    HBR_NORM(t##_##V##_2, E, V, 2)                                                                           \
    extern "C" __global__ __launch_bounds__(256) void hbr_pack_##t##_##V(PackArgs a) { pack_rows<E, V>(a); } \
    extern "C" __global__ __launch_bounds__(256) void hbr_unpack_##t##_##V(PackArgs a) { unpack_rows<E, V>(a); }
HBR_ROWS(f32, F32, 1)
HBR_ROWS(f32, F32, 2)
HBR_ROWS(f32, F32, 4)
HBR_ROWS(bf16, Bf16, 1)
HBR_ROWS(bf16, Bf16, 2)
HBR_ROWS(bf16, Bf16, 4)
HBR_ROWS(bf16, Bf16, 8)
HBR_NORM(f32_1_4, F32, 1, 4)
HBR_NORM(f32_2_4, F32, 2, 4)
HBR_NORM(f32_4_4, F32, 4, 4)
HBR_NORM(bf16_1_4, Bf16, 1, 4)
HBR_NORM(bf16_2_4, Bf16, 2, 4)
HBR_NORM(bf16_4_4, Bf16, 4, 4)
