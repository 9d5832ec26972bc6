// Root-mean-square norm of rows and its gradient, and rows to 8 bits and back.
//
//   s = x + residual; inv = 1 / sqrt(mean s^2 + eps); n = s inv; out = n weight
//   g = dout weight; dx = inv (g - n mean(g n)) + dtotal; dweight = sum over rows dout n
//
// A row lies on `lanes` lanes and stays in their registers between its sum and
// its results: up to 16,384 columns of bf16 and 8,192 of f32 it is read once and
// written once, beyond it is read again for every use. A lane's columns are the same
// in every row, so that the weights are loaded once and the weights' gradient is
// summed in registers, joined in LDS and over the workgroups in order.
//
// Memory bounds all of it. Measured, against a large copy's 5.15 TB/s: 65,537 rows
// of 1,024 bf16 with a residual, their sum and codes written too and the codes read
// back, 167 us (157 at the copy's rate); the gradient out of the codes, with dtotal,
// 108 us (92); 262,144 x 1,024 bf16 into codes and back 287 us (317: some of the codes
// come out of a cache); one row 9 us, all of it the launch. Rows of other than whole
// vectors: 10,058 x 6,661 bf16 the same 226 us (157), the gradient out of the rows
// 149 (104).
#include "rows8.h"

namespace hbr {

// A lane's vector `i` of a row. A row need not lie on its vectors' size, nor,
// Ragged, be of whole ones: its last vector reaches back into the one before it,
// of whose columns the lane reads zeros and writes none. (Element by element
// instead, the gradient of 10,058 rows of 6,661 bf16 took 822 us, now 148.)
template <int V, bool Ragged>
struct Place {
    uint32_t at, back;  // the first column, and how many of the vector's are not its own
    bool is;            // within the row
    __device__ __forceinline__ Place(uint32_t i, uint32_t vecs, uint32_t dim) {
        at = Ragged ? min(i * V, dim - V) : i * V;
        back = Ragged ? i * V - at : 0;
        is = i < vecs;
    }
    __device__ __forceinline__ bool own(int k) const { return !Ragged || k >= (int)back; }
    // an element as it is, or zero (by its bits: behind a choice the compiler
    // loads a vector in pieces)
    __device__ __forceinline__ float of(int k, float v) const {
        if constexpr (!Ragged) return v;
        const int32_t keep = ((int32_t)back - 1 - k) >> 31;
        return __uint_as_float(__float_as_uint(v) & (uint32_t)keep);
    }
};

// Vectors in one access wherever they lie.
template <int Bytes>
struct Anywhere;
template <>
struct Anywhere<16> {
    typedef int type __attribute__((ext_vector_type(4), aligned(1)));
};
template <>
struct Anywhere<8> {
    typedef int type __attribute__((ext_vector_type(2), aligned(1)));
};
template <>
struct Anywhere<4> {
    typedef int type __attribute__((aligned(1)));
};
template <>
struct Anywhere<2> {
    typedef short type;
};
template <>
struct Anywhere<1> {
    typedef char type;
};
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load(const T *p) {
    if constexpr (sizeof(T) * V == 32) {
        const Vec<T, V / 2> x = load<T, V / 2>(p), y = load<T, V / 2>(p + V / 2);
        Vec<T, V> v;
#pragma unroll
        for (int k = 0; k < V; k++) v.v[k] = k < V / 2 ? x.v[k] : y.v[k - V / 2];
        return v;
    } else {
        using A = typename Anywhere<sizeof(T) * V>::type;
        return __builtin_bit_cast(Vec<T, V>, *reinterpret_cast<const A *>(p));
    }
}

template <typename E, int V, bool Ragged>
__device__ __forceinline__ void load_up(const void *row, const Place<V, Ragged> &c, float (&v)[V]) {
    using T = typename E::type;
    const Vec<T, V> x = load<T, V>(static_cast<const T *>(row) + c.at);
#pragma unroll
    for (int k = 0; k < V; k++) v[k] = c.of(k, E::up(x.v[k]));
}

template <typename T, int V, bool Ragged>
__device__ __forceinline__ void store(void *row, const Place<V, Ragged> &c, const Vec<T, V> &x) {
    T *to = static_cast<T *>(row) + c.at;
    if (!Ragged || c.back == 0) {
        if constexpr (sizeof(T) * V == 32) {
            *reinterpret_cast<typename Anywhere<16>::type *>(to) = *reinterpret_cast<const typename Anywhere<16>::type *>(&x.v[0]);
            *reinterpret_cast<typename Anywhere<16>::type *>(to + V / 2) = *reinterpret_cast<const typename Anywhere<16>::type *>(&x.v[V / 2]);
        } else {
            using A = typename Anywhere<sizeof(T) * V>::type;
            *reinterpret_cast<A *>(to) = __builtin_bit_cast(A, x);
        }
    } else {
#pragma unroll
        for (int k = 0; k < V; k++)
            if (c.own(k)) to[k] = x.v[k];
    }
}

template <typename E, int V, bool Ragged>
__device__ __forceinline__ void store_down(void *row, const Place<V, Ragged> &c, const float (&v)[V]) {
    Vec<typename E::type, V> x;
#pragma unroll
    for (int k = 0; k < V; k++) x.v[k] = E::down(v[k]);
    store(row, c, x);
}

// The sum over a row's lanes, the same bits in each. More than a wave's lanes
// are the workgroup's, and all of it calls.
template <typename T>
__device__ __forceinline__ T row_sum(T v, uint32_t lanes) {
    __shared__ T wave_sum[16];
    for (uint32_t d = min(lanes, (uint32_t)kWave) / 2; d; d /= 2) v += __shfl_xor(v, d, kWave);
    if (lanes <= (uint32_t)kWave) return v;
    const uint32_t wave = threadIdx.x / kWave, waves = lanes / kWave;
    __syncthreads();
    if (lane_id() == 0) wave_sum[wave] = v;
    __syncthreads();
    v = wave_sum[0];
    for (uint32_t w = 1; w < waves; w++) v += wave_sum[w];
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

// One vector of a row into codes, the block's first lane writing its power.
template <int V, bool Ragged>
__device__ __forceinline__ void put_codes(uint8_t *codes, uint8_t *scales, uint32_t i, const Place<V, Ragged> &c, const float (&v)[V]) {
    const int32_t power = power_of(block_largest<V>(v));
    if (!c.is) return;
    store(codes, c, codes_of<V>(v, exp2_of(-power)));
    if (i % (kPackBlock / V) == 0) scales[i / (kPackBlock / V)] = (uint8_t)(power + kPowerBias);
}

template <int V, bool Ragged>
__device__ __forceinline__ void get_codes(const uint8_t *codes, const uint8_t *scales, uint32_t i, const Place<V, Ragged> &c, float (&v)[V]) {
    const float power = exp2_of((int32_t)scales[i / (kPackBlock / V)] - kPowerBias);
    values_of<V>(load<uint8_t, V>(codes + c.at), power, v);
#pragma unroll
    for (int k = 0; k < V; k++) v[k] = c.of(k, v[k]);
}

// A row of an array of E.
template <typename E>
__device__ __forceinline__ const void *row_of(const void *p, uint64_t r, uint64_t stride) { return static_cast<const typename E::type *>(p) + r * stride; }
template <typename E>
__device__ __forceinline__ void *row_of(void *p, uint64_t r, uint64_t stride) { return static_cast<typename E::type *>(p) + r * stride; }

// U vectors a lane in registers; 0: any number, read again where they are used.
template <typename E, int V, int U, bool R>
__device__ __forceinline__ void rms_norm(const NormArgs &a) {
    constexpr int kHeld = U ? U : 1;
    const uint32_t lanes = a.lanes, in = threadIdx.x & (lanes - 1), per = blockDim.x / lanes;
    const uint32_t rounds = U ? U : (a.vecs + lanes - 1) / lanes;
    float s[kHeld][V], w[kHeld][V];
    auto weights = [&](uint32_t i, float (&to)[V]) {
#pragma unroll
        for (int k = 0; k < V; k++) to[k] = 1.0f;
        const Place<V, R> c(i, a.vecs, a.dim);
        if (a.weight && c.is) load_up<F32>(a.weight, c, to);
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
            const Place<V, R> c(i, a.vecs, a.dim);
            if (!live || !c.is) return;
            load_up<E>(row_of<E>(a.x, r, a.x_stride), c, to);
            if (a.residual) {
                float more[V];
                load_up<E>(row_of<E>(a.residual, r, a.residual_stride), c, more);
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
            Place<V, R> c(i, a.vecs, a.dim);
            c.is = c.is && live;
            if (a.total && c.is) store_down<E>(row_of<E>(a.total, r, a.total_stride), c, v);
            float out[V];
#pragma unroll
            for (int k = 0; k < V; k++) {
                v[k] *= inv;
                out[k] = v[k] * by[k];
            }
            if (a.out && c.is) store_down<E>(row_of<E>(a.out, r, a.out_stride), c, out);
            if (!a.codes) return;
            // (an inv that is no number makes none of the zeros in columns of no one)
#pragma unroll
            for (int k = 0; k < V; k++)
                if (!c.is || !c.own(k)) v[k] = out[k] = 0.0f;
            uint8_t *codes = a.codes + r * a.codes_stride, *scales = a.scales + r * a.scales_stride;
            if (a.normed) put_codes(codes, scales, i, c, v);
            else put_codes(codes, scales, i, c, out);
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

template <typename E, int V, int U, bool R>
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
        const Place<V, R> c(i, a.vecs, a.dim);
        if (a.weight && c.is) load_up<F32>(a.weight, c, to);
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
            const Place<V, R> c(i, a.vecs, a.dim);
            if (!live || !c.is) return;
            if (a.codes) get_codes(a.codes + r * a.codes_stride, a.scales + r * a.scales_stride, i, c, to);
            else load_up<E>(row_of<E>(a.x, r, a.x_stride), c, to);
        };
        auto douts = [&](uint32_t i, float (&to)[V]) {
#pragma unroll
            for (int k = 0; k < V; k++) to[k] = 0.0f;
            const Place<V, R> c(i, a.vecs, a.dim);
            if (live && c.is) load_up<E>(row_of<E>(a.dout, r, a.dout_stride), c, to);
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
            const Place<V, R> c(i, a.vecs, a.dim);
            if (!live || !c.is) return;
            float dx[V];
#pragma unroll
            for (int k = 0; k < V; k++) {
                total[k] = __builtin_fmaf(dy[k], v[k], total[k]);
                dx[k] = inv * __builtin_fmaf(-v[k], along, dy[k] * of[k]);
            }
            if (!a.dx) return;
            if (a.dtotal) {
                float more[V];
                load_up<E>(row_of<E>(a.dtotal, r, a.dtotal_stride), c, more);
#pragma unroll
                for (int k = 0; k < V; k++) dx[k] += more[k];
            }
            store_down<E>(row_of<E>(a.dx, r, a.dx_stride), c, dx);
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
                const Place<V, R> c(i, a.vecs, a.dim);
                if (part && !first && c.is) load_up<F32>(part, c, acc[0]);
                write(i, n[0], d[0], w[0], acc[0]);
                if (part && c.is) store_down<F32>(part, c, acc[0]);
            }
            first = false;
        }
    }
    if (U == 0 || !part) return;
    if (lanes > (uint32_t)kWave) {
#pragma unroll
        for (int u = 0; u < kHeld; u++) {
            const Place<V, R> c(in + u * lanes, a.vecs, a.dim);
            if (c.is) store_down<F32>(part, c, acc[u]);
        }
        return;
    }
    const uint32_t cols = lanes * kHeld * V;  // of a row's sums
#pragma unroll
    for (int u = 0; u < kHeld; u++) {
        const Place<V, R> c(in + u * lanes, a.vecs, a.dim);
#pragma unroll
        for (int k = 0; k < V; k++)
            if (c.is && c.own(k)) sums[threadIdx.x / lanes * cols + c.at + k] = acc[u][k];
    }
    __syncthreads();
    for (uint32_t c = threadIdx.x; c < a.dim; c += blockDim.x) {
        float sum = sums[c];
        for (uint32_t g = 1; g < per; g++) sum += sums[g * cols + c];
        part[c] = sum;
    }
}

template <typename E, int V, bool R>
__device__ __forceinline__ void pack_rows(const PackArgs &a) {
    const uint32_t lanes = a.lanes, in = threadIdx.x & (lanes - 1), per = blockDim.x / lanes;
    const uint32_t first = blockIdx.y * a.each * lanes, end = min(first + a.each * lanes, (a.vecs + 31) / 32 * 32);
    for (uint64_t r0 = (uint64_t)blockIdx.x * per; r0 < a.n_rows; r0 += (uint64_t)gridDim.x * per) {
        const uint64_t r = r0 + threadIdx.x / lanes;
        for (uint32_t i0 = first; i0 < end; i0 += lanes) {
            const uint32_t i = i0 + in;
            Place<V, R> c(i, a.vecs, a.dim);
            c.is = c.is && r < a.n_rows;
            float v[V] = {};
            if (c.is) load_up<E>(row_of<E>(a.x, r, a.x_stride), c, v);
            put_codes(a.codes + r * a.codes_stride, a.scales + r * a.scales_stride, i, c, v);
        }
    }
}

template <typename E, int V, bool R>
__device__ __forceinline__ void unpack_rows(const PackArgs &a) {
    const uint32_t lanes = a.lanes, in = threadIdx.x & (lanes - 1), per = blockDim.x / lanes;
    const uint32_t first = blockIdx.y * a.each * lanes, end = min(first + a.each * lanes, a.vecs);
    for (uint64_t r = (uint64_t)blockIdx.x * per + threadIdx.x / lanes; r < a.n_rows; r += (uint64_t)gridDim.x * per)
        for (uint32_t i = first + in; i < end; i += lanes) {
            const Place<V, R> c(i, a.vecs, a.dim);
            float v[V];
            get_codes(a.codes + r * a.codes_stride, a.scales + r * a.scales_stride, i, c, v);
            if (a.weight) {
                float w[V];
                load_up<F32>(a.weight, c, w);
#pragma unroll
                for (int k = 0; k < V; k++) v[k] *= w[k];
            }
            store_down<E>(row_of<E>(a.x, r, a.x_stride), c, v);
        }
}

}  // namespace hbr

using namespace hbr;

// V: 16 bytes, or 8 for short rows of f32 of whole such, or one element for rows
// shorter than a vector; R: rows of other than whole vectors
#define HBR_NORM(suffix, E, V, U, R)                                                                                   \
    extern "C" __global__ __launch_bounds__(1024) void hbr_rms_norm_##suffix(NormArgs a) { rms_norm<E, V, U, R>(a); }  \
    extern "C" __global__ __launch_bounds__(1024) void hbr_rms_norm_grad_##suffix(NormGradArgs a) { rms_norm_grad<E, V, U, R>(a); }
#define HBR_PACK(suffix, E, V, R)                                                                                    \
    extern "C" __global__ __launch_bounds__(256) void hbr_pack_##suffix(PackArgs a) { pack_rows<E, V, R>(a); }       \
    extern "C" __global__ __launch_bounds__(256) void hbr_unpack_##suffix(PackArgs a) { unpack_rows<E, V, R>(a); }
#define HBR_NORMS(suffix, E, V, R)   \
    HBR_NORM(suffix##_1, E, V, 1, R) \
    HBR_NORM(suffix##_2, E, V, 2, R) \
    HBR_NORM(suffix##_0, E, V, 0, R)
HBR_NORM(f32_1_1, F32, 1, 1, false)
HBR_NORM(bf16_1_1, Bf16, 1, 1, false)
HBR_NORM(f32_2_1, F32, 2, 1, false)
HBR_NORM(f32_2_2, F32, 2, 2, false)
HBR_NORMS(f32_4, F32, 4, false)
HBR_NORMS(f32_4r, F32, 4, true)
HBR_NORMS(bf16_8, Bf16, 8, false)
HBR_NORMS(bf16_8r, Bf16, 8, true)
// (four vectors a lane: the norm's alone, by workgroups of 256)
extern "C" __global__ __launch_bounds__(256) void hbr_rms_norm_f32_2_4(NormArgs a) { rms_norm<F32, 2, 4, false>(a); }
extern "C" __global__ __launch_bounds__(256) void hbr_rms_norm_f32_4_4(NormArgs a) { rms_norm<F32, 4, 4, false>(a); }
extern "C" __global__ __launch_bounds__(256) void hbr_rms_norm_f32_4r_4(NormArgs a) { rms_norm<F32, 4, 4, true>(a); }
HBR_PACK(f32_1, F32, 1, false)
HBR_PACK(f32_4, F32, 4, false)
HBR_PACK(f32_4r, F32, 4, true)
HBR_PACK(bf16_1, Bf16, 1, false)
HBR_PACK(bf16_8, Bf16, 8, false)
HBR_PACK(bf16_8r, Bf16, 8, true)
