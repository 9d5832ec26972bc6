// The softmax head over few classes (kFewClasses at most): a row's scores fit
// the lanes' registers, so one pass over the rows gives loss and pairs, and a
// second the products with them. Both passes are bound by the rows' traffic:
// h is read twice and dh written once, w and the pairs are small. No LDS: a
// fragment is what its lanes load, 16 bytes of a row each or an element of a
// column each, and the L1 serves what waves of a workgroup share.
//
// f32 is multiplied as f32 (v_mfma_f32_32x32x2_f32), whose rate the traffic
// does not reach.
//
// 200,003 rows of 50 f32 and ten classes: scores 29 us (h read at 1.4 TB/s:
// a wave's own chain of loads and exponentials), products 36 (108 MB with the
// pairs, 3 TB/s), sums 5. 100,000 rows of 256 bf16 and ten classes 64 us in all
// (the kernels for many classes 111).
#include "common.h"

namespace hbr {

// The products' operands by type: a fragment of kStep products holds kEach of
// them a lane, those from kEach (lane / 32) on.
struct FewF32 {
    using E = F32;
    static constexpr int kStep = 8, kEach = 4;
    using Frag = Vec<float, 4>;
    static __device__ __forceinline__ f32x16 mul(const Frag &a, const Frag &b, f32x16 c) {
#pragma unroll
        for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[i], b.v[i], c, 0, 0, 0);
        return c;
    }
};
struct FewBf16 {
    using E = Bf16;
    static constexpr int kStep = 16, kEach = 8;
    using Frag = Vec<uint16_t, 8>;
    static __device__ __forceinline__ f32x16 mul(const Frag &a, const Frag &b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};

// kEach elements of a row of at least as many, from k on, zeros past its dim: a
// vector (of no more than its elements' alignment) from where one still fits
// the row, so that no load waits on a condition, which few_tail then shifts to
// its place.
template <typename F>
__device__ __forceinline__ typename F::Frag few_row(const typename F::E::type *row, uint32_t k, uint32_t dim) {
    typename F::Frag f;
    __builtin_memcpy(&f, row + min(k, dim - F::kEach), sizeof f);
    return f;
}
template <typename F>
__device__ __forceinline__ void few_tail(typename F::Frag &f, uint32_t k, uint32_t dim) {
    const uint32_t by = k - min(k, dim - F::kEach);
#pragma unroll
    for (int b = 1; b < F::kEach; b *= 2)
        if (by & b)
#pragma unroll
            for (int i = 0; i < F::kEach; i++) f.v[i] = i + b < F::kEach ? f.v[i + b < F::kEach ? i + b : 0] : (typename F::E::type)0;
    if (by >= (uint32_t)F::kEach) f = typename F::Frag{};
}
// A shorter row, by element.
template <typename F>
__device__ __forceinline__ typename F::Frag few_short(const typename F::E::type *row, uint32_t k, uint32_t dim) {
    typename F::Frag f{};
#pragma unroll
    for (int i = 0; i < F::kEach; i++)
        if (k + i < dim) f.v[i] = row[k + i];
    return f;
}

// A wave takes 32 rows at a time; a lane holds its row's classes 32 kt +
// row_of(e), the lane of the other half of the wave the row's others.
template <typename F, int KT>
__device__ __forceinline__ void few_scores(const FewArgs &a) {
    using T = typename F::E::type;
    __shared__ __align__(16) float bias[32 * KT];
    if (threadIdx.x < 32 * KT)
        bias[threadIdx.x] = threadIdx.x >= a.classes ? -INFINITY : a.bias ? a.bias[threadIdx.x] : 0.0f;
    __syncthreads();
    const uint32_t lane = lane_id(), wave = blockIdx.x * 4 + threadIdx.x / kWave, waves = gridDim.x * 4;
    const uint32_t groups = (uint32_t)((a.rows + 31) / 32);
    const T *w[KT];
#pragma unroll
    for (int t = 0; t < KT; t++) w[t] = static_cast<const T *>(a.w) + min(32 * t + lane % 32, a.classes - 1) * a.w_stride;
    float db[KT][16] = {};
    for (uint32_t g = wave; g < groups; g += waves) {
        const uint64_t r = (uint64_t)g * 32 + lane % 32;
        const bool in = r < a.rows;
        const T *h = static_cast<const T *>(a.h) + min(r, a.rows - 1) * a.h_stride;
        f32x16 acc[KT];
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[t][e] = 0.0f;
        constexpr int kAhead = 4;  // loads of as many steps in flight
        if (a.dim < (uint32_t)F::kEach) {
            const uint32_t k = lane / 32 * F::kEach;
            const typename F::Frag fh = few_short<F>(h, k, a.dim);
#pragma unroll
            for (int t = 0; t < KT; t++) acc[t] = F::mul(few_short<F>(w[t], k, a.dim), fh, acc[t]);
        } else {
            for (uint32_t k0 = 0; k0 < a.dim; k0 += kAhead * F::kStep) {
                typename F::Frag fh[kAhead], fw[kAhead][KT];
#pragma unroll
                for (int u = 0; u < kAhead; u++) {
                    const uint32_t k = k0 + u * F::kStep + lane / 32 * F::kEach;
                    fh[u] = few_row<F>(h, k, a.dim);
#pragma unroll
                    for (int t = 0; t < KT; t++) fw[u][t] = few_row<F>(w[t], k, a.dim);
                }
                __builtin_amdgcn_sched_barrier(0);  // all loads out before the first is waited for
                if (k0 + kAhead * F::kStep > a.dim) {
#pragma unroll
                    for (int u = 0; u < kAhead; u++) {
                        const uint32_t k = k0 + u * F::kStep + lane / 32 * F::kEach;
                        few_tail<F>(fh[u], k, a.dim);
#pragma unroll
                        for (int t = 0; t < KT; t++) few_tail<F>(fw[u][t], k, a.dim);
                    }
                }
#pragma unroll
                for (int u = 0; u < kAhead; u++)
#pragma unroll
                    for (int t = 0; t < KT; t++) acc[t] = F::mul(fw[u][t], fh[u], acc[t]);
            }
        }
        const int32_t y = a.labels && in ? a.labels[r] : -1;
        float top = -INFINITY, at_label = 0.0f;
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const uint32_t c = 32 * t + row_of(e);
                const float z = c < a.classes ? acc[t][e] + bias[c] : -INFINITY;
                acc[t][e] = z;
                top = fmaxf(top, z);
                if (y == (int32_t)c) at_label = z;
            }
        top = fmaxf(top, __shfl_xor(top, 32, kWave));
        const float shift = shift_of(top);
        float sum = 0.0f;
        int32_t best = 0x7fffffff;
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                if (acc[t][e] == top) best = min(best, (int32_t)(32 * t + row_of(e)));
                acc[t][e] = exp_of(acc[t][e] - shift);
                sum += acc[t][e];
            }
        sum += __shfl_xor(sum, 32, kWave);
        at_label += __shfl_xor(at_label, 32, kWave);
        best = min(best, __shfl_xor(best, 32, kWave));
        // a label that is no class: neither a loss nor a gradient
        const bool no_class = y >= 0 && (uint32_t)y >= a.classes;
        const float more = no_class ? NAN : __builtin_amdgcn_logf(sum) * kLn2;
        const float weight = in && a.weight ? a.weight[r] : 1.0f;
        if (in && lane < 32) {
            if (a.lse) a.lse[r] = shift + more;
            if (a.best) a.best[r] = best < (int32_t)a.classes ? best : 0;
            if (a.loss)
                a.loss[r] = !a.labels ? (shift - top) + more : y < 0 ? 0.0f : no_class ? NAN : weight * ((shift - at_label) + more);
        }
        if (!a.g) continue;
        const uint64_t kept = __ballot(y >= 0);
        if (lane == 0) a.keep[g] = (uint32_t)kept;
        const float share = no_class ? NAN : 1.0f / sum;
        T *out = static_cast<T *>(a.g) + r * a.g_stride;
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                Vec<T, 4> v;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int e = 4 * q + i;
                    float p = acc[t][e] * share;
                    if (y == (int32_t)(32 * t + row_of(e))) p -= 1.0f;
                    p = y < 0 ? 0.0f : p * weight;
                    db[t][e] += p;
                    v.v[i] = F::E::down(p);
                }
                const uint32_t c = 32 * t + 8 * q + 4 * (lane / 32);
                if (in && c < a.g_stride) *reinterpret_cast<Vec<T, 4> *>(out + c) = v;
            }
    }
    if (!a.g) return;
#pragma unroll
    for (int t = 0; t < KT; t++)
#pragma unroll
        for (int e = 0; e < 16; e++) {
            float s = db[t][e];
            for (int d = 16; d >= 1; d >>= 1) s += __shfl_xor(s, d, kWave);
            const uint32_t c = 32 * t + row_of(e);
            if (lane % 32 == 0 && c < a.classes) a.part_db[(uint64_t)wave * a.classes + c] = s;
        }
}

// A wave takes 32 columns of h and every chunks-th group of 32 rows: dh = g w
// with its part of w in registers throughout, dw = g^T h summed in registers
// over its rows.
template <typename F, int KT>
__device__ __forceinline__ void few_products(const FewArgs &a) {
    using T = typename F::E::type;
    using Frag = typename F::Frag;
    constexpr int kSteps = 32 * KT / F::kStep, kRowSteps = 32 / F::kStep;
    const uint32_t lane = lane_id(), wave = blockIdx.x * 4 + threadIdx.x / kWave, half = lane / 32;
    const uint32_t chunk = wave / a.col_tiles, d = wave % a.col_tiles * 32 + lane % 32;
    if (chunk >= a.chunks) return;
    const uint32_t groups = (uint32_t)((a.rows + 31) / 32), dd = min(d, a.dim - 1);
    Frag w[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; s++)
#pragma unroll
        for (int i = 0; i < F::kEach; i++) {
            const uint32_t k = s * F::kStep + half * F::kEach + i;
            w[s].v[i] = k < a.classes ? static_cast<const T *>(a.w)[k * a.w_stride + dd] : (T)0;
        }
    f32x16 dw[KT];
#pragma unroll
    for (int t = 0; t < KT; t++)
#pragma unroll
        for (int e = 0; e < 16; e++) dw[t][e] = 0.0f;
    // A group's loads are out before the one before it is worked on: without
    // conditions (a row past the last is the last again), and what rows that
    // take no part hold is dropped behind them. (100,000 rows of 256 bf16: ten
    // classes 64 us, 150 with a wait at each load; 48 classes 114, 155 with the
    // loads at the group itself.)
    T h[kRowSteps][F::kEach], p[KT][kRowSteps][F::kEach];
    Frag row[kSteps];
    uint32_t kept = 0;
    auto load = [&](uint32_t g) {
        const uint64_t r0 = (uint64_t)g * 32;
        const uint32_t m = (uint32_t)min((uint64_t)32, a.rows - r0);
        const T *pairs = static_cast<const T *>(a.g) + r0 * a.g_stride, *from = static_cast<const T *>(a.h) + r0 * a.h_stride + dd;
        if (a.dw) {
            kept = a.keep[g];
#pragma unroll
            for (int s = 0; s < kRowSteps; s++)
#pragma unroll
                for (int i = 0; i < F::kEach; i++) {
                    const uint32_t r = min(s * F::kStep + half * F::kEach + i, m - 1);
                    h[s][i] = from[r * a.h_stride];
#pragma unroll
                    for (int t = 0; t < KT; t++) p[t][s][i] = pairs[r * a.g_stride + min(32 * t + lane % 32, (uint32_t)a.g_stride - 1)];
                }
        }
        if (a.dh)
#pragma unroll
            for (int s = 0; s < kSteps; s++)  // past the pairs' columns the last again, times w's zeros
                row[s] = *reinterpret_cast<const Frag *>(pairs + min(lane % 32, m - 1) * a.g_stride +
                                                         min((uint32_t)(s * F::kStep), (uint32_t)a.g_stride - F::kStep) + half * F::kEach);
    };
    if (chunk < groups) load(chunk);
    for (uint32_t g = chunk; g < groups; g += a.chunks) {
        const uint64_t r0 = (uint64_t)g * 32;
        const uint32_t m = (uint32_t)min((uint64_t)32, a.rows - r0);
        Frag fh[kRowSteps], fp[KT][kRowSteps], fr[kSteps];
#pragma unroll
        for (int s = 0; s < kRowSteps; s++)
#pragma unroll
            for (int i = 0; i < F::kEach; i++) {
                const bool in = (kept >> (s * F::kStep + half * F::kEach + i)) & 1u;
                fh[s].v[i] = in ? h[s][i] : (T)0;
#pragma unroll
                for (int t = 0; t < KT; t++) fp[t][s].v[i] = in ? p[t][s][i] : (T)0;
            }
#pragma unroll
        for (int s = 0; s < kSteps; s++) fr[s] = row[s];
        __builtin_amdgcn_sched_barrier(0);
        load(min(g + a.chunks, groups - 1));
        __builtin_amdgcn_sched_barrier(0);
        if (a.dw)
#pragma unroll
            for (int s = 0; s < kRowSteps; s++)
#pragma unroll
                for (int t = 0; t < KT; t++) dw[t] = F::mul(fp[t][s], fh[s], dw[t]);
        if (a.dh) {
            f32x16 acc;
#pragma unroll
            for (int e = 0; e < 16; e++) acc[e] = 0.0f;
#pragma unroll
            for (int s = 0; s < kSteps; s++) acc = F::mul(fr[s], w[s], acc);
            T *out = static_cast<T *>(a.dh) + r0 * a.dh_stride + d;
            if (d < a.dim) {
#pragma unroll
                for (int e = 0; e < 16; e++)
                    if (row_of(e) < m) out[row_of(e) * a.dh_stride] = F::E::down(acc[e] * a.scale);
            }
        }
    }
    if (!a.dw || d >= a.dim) return;
#pragma unroll
    for (int t = 0; t < KT; t++)
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const uint32_t c = 32 * t + row_of(e);
            if (c < a.classes) a.part_dw[((uint64_t)chunk * a.classes + c) * a.dim + d] = dw[t][e];
        }
}

// dw and db from their parts: a workgroup takes 16 cells, its 64 groups of 16
// lanes an even share of the parts each, joined in order.
template <typename E>
__device__ __forceinline__ void few_sums(const FewSumsArgs &a) {
    __shared__ float sum_of[64][16];
    const bool dw = blockIdx.x < a.dw_blocks;
    const uint32_t lane = threadIdx.x % 16, group = threadIdx.x / 16;
    const uint32_t cells = dw ? a.classes * a.dim : a.classes, parts = dw ? a.shares : a.waves;
    const uint32_t i = (dw ? blockIdx.x : blockIdx.x - a.dw_blocks) * 16 + lane;
    const uint32_t p0 = (uint32_t)((uint64_t)parts * group / 64), p1 = (uint32_t)((uint64_t)parts * (group + 1) / 64);
    float s = 0.0f;
    if (i < cells) {
        const float *part = (dw ? a.part_dw : a.part_db) + i;
#pragma unroll 8
        for (uint32_t p = p0; p < p1; p++) s += part[(uint64_t)p * cells];
    }
    sum_of[group][lane] = s;
    __syncthreads();
    if (group || i >= cells) return;
    for (int g = 1; g < 64; g++) s += sum_of[g][lane];
    s *= a.scale;
    if (dw) static_cast<typename E::type *>(a.dw)[i / a.dim * a.dw_stride + i % a.dim] = E::down(s);
    else a.db[i] = s;
}

}  // namespace hbr

using namespace hbr;

#define HBR_FEW(suffix, F, KT)                                                                                    \
    extern "C" __global__ __launch_bounds__(256) void hbr_few_scores_##suffix(FewArgs a) { few_scores<F, KT>(a); } \
    extern "C" __global__ __launch_bounds__(256) void hbr_few_products_##suffix(FewArgs a) { few_products<F, KT>(a); }
HBR_FEW(f32_1, FewF32, 1)
HBR_FEW(f32_2, FewF32, 2)
HBR_FEW(bf16_1, FewBf16, 1)
HBR_FEW(bf16_2, FewBf16, 2)
extern "C" __global__ __launch_bounds__(1024) void hbr_few_sums_f32(FewSumsArgs a) { few_sums<F32>(a); }
extern "C" __global__ __launch_bounds__(1024) void hbr_few_sums_bf16(FewSumsArgs a) { few_sums<Bf16>(a); }
