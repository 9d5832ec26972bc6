// The softmax cross entropy of a linear layer over many classes and its
// gradients, the scores made tile by tile and never kept.
//
//   z = h W^T + b; lse = log sum exp z; loss = a (lse - z_y)
//   g = c a (exp(z - lse) - [k = y]); dh = g W; dW = g^T h; db = sum g
#include "common.h"

namespace hbr {

constexpr uint32_t kHeadDepth = 16;

// One 64 x 64 tile of C[m][n] = sum_k A(m, k) B(n, k): 256 threads of 4 x 4
// sums in f32, the operands staged in LDS as f32. A product's k that `skip`
// marks is taken as zero on both sides, whatever stands there.
template <typename E>
__device__ __forceinline__ void head_tile(const HeadArgs &a, uint64_t m0, uint64_t n0, float (&acc)[4][4]) {
    using T = typename E::type;
    __shared__ float sa[kHeadDepth][kHeadTile + 4], sb[kHeadDepth][kHeadTile + 4];
    const uint32_t tm = threadIdx.x / 16 * 4, tn = threadIdx.x % 16 * 4;
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = 0.0f;
    for (uint64_t k0 = 0; k0 < a.k; k0 += kHeadDepth) {
        for (uint32_t q = threadIdx.x; q < kHeadTile * kHeadDepth; q += 256) {
            // along the axis that is contiguous in memory
            const uint32_t am = a.a_k == 1 ? q / kHeadDepth : q % kHeadTile, ak = a.a_k == 1 ? q % kHeadDepth : q / kHeadTile;
            const uint32_t bn = a.b_k == 1 ? q / kHeadDepth : q % kHeadTile, bk = a.b_k == 1 ? q % kHeadDepth : q / kHeadTile;
            const uint64_t m = m0 + am, n = n0 + bn, ka = k0 + ak, kb = k0 + bk;
            float va = 0.0f, vb = 0.0f;
            if (m < a.m && ka < a.k && (!a.skip || a.skip[ka] >= 0))
                va = E::up(static_cast<const T *>(a.a)[m * a.a_m + ka * a.a_k]);
            if (n < a.n && kb < a.k && (!a.skip || a.skip[kb] >= 0))
                vb = E::up(static_cast<const T *>(a.b)[n * a.b_n + kb * a.b_k]);
            sa[ak][am] = va;
            sb[bk][bn] = vb;
        }
        __syncthreads();
#pragma unroll
        for (uint32_t k = 0; k < kHeadDepth; k++) {
            float va[4], vb[4];
#pragma unroll
            for (int i = 0; i < 4; i++) va[i] = sa[k][tm + i], vb[i] = sb[k][tn + i];
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = __builtin_fmaf(va[i], vb[j], acc[i][j]);
        }
        __syncthreads();
    }
}

// A running maximum's shift: a tile with no open class sums to zero.
__device__ __forceinline__ float shift_of(float m) { return m == -INFINITY ? 0.0f : m; }

__device__ __forceinline__ float exp_f32(float x) { return expf(x); }

template <typename E>
__device__ __forceinline__ void head_scores(const HeadArgs &a) {
    const uint64_t m0 = (uint64_t)blockIdx.x * kHeadTile, n0 = (uint64_t)blockIdx.y * kHeadTile;
    float acc[4][4];
    head_tile<E>(a, m0, n0, acc);
    const uint32_t tm = threadIdx.x / 16 * 4, tn = threadIdx.x % 16 * 4;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint64_t r = m0 + tm + i;
        const int32_t y = a.labels && r < a.m ? a.labels[r] : -1;
        float top = -INFINITY;
        int32_t best = (int32_t)n0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint64_t k = n0 + tn + j;
            float z = acc[i][j] + (a.bias && k < a.n ? a.bias[k] : 0.0f);
            if (k >= a.n) z = -INFINITY;
            acc[i][j] = z;
            if (y >= 0 && (uint64_t)y == k && k < a.n) a.label_margin[r] = z;
            if (z > top) top = z, best = (int32_t)k;
        }
        for (int d = 1; d < 16; d <<= 1) {
            const float t = __shfl_xor(top, d, kWave);
            const int32_t b = __shfl_xor(best, d, kWave);
            if (t > top || (t == top && b < best)) top = t, best = b;
        }
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; j++) sum += exp_f32(acc[i][j] - shift_of(top));
        for (int d = 1; d < 16; d <<= 1) sum += __shfl_xor(sum, d, kWave);
        if (threadIdx.x % 16 == 0 && r < a.m) {
            const uint64_t at = (uint64_t)blockIdx.y * a.rows + r;
            a.part_max[at] = top;
            a.part_sum[at] = sum;
            if (a.part_best) a.part_best[at] = best;
        }
    }
}

template <typename E>
__device__ __forceinline__ void head_pairs(const HeadArgs &a) {
    using T = typename E::type;
    __shared__ float column[16][kHeadTile];
    const uint64_t m0 = (uint64_t)blockIdx.x * kHeadTile, n0 = (uint64_t)blockIdx.y * kHeadTile;
    float acc[4][4];
    head_tile<E>(a, m0, n0, acc);
    const uint32_t tm = threadIdx.x / 16 * 4, tn = threadIdx.x % 16 * 4;
    float db[4] = {};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint64_t r = m0 + tm + i;
        if (r >= a.m) continue;
        const int32_t y = a.labels[r];
        const float by = a.grad_scale * (a.weight ? a.weight[r] : 1.0f), lse = a.lse[r];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint64_t k = n0 + tn + j;
            if (k >= a.n) continue;
            const float z = acc[i][j] + (a.bias ? a.bias[a.first + k] : 0.0f);
            float g = exp_f32(z - lse) - ((uint64_t)(int64_t)y == a.first + k ? 1.0f : 0.0f);
            g = y < 0 ? 0.0f : g * by;
            static_cast<T *>(a.g)[r * a.g_stride + k] = E::down(g);
            db[j] += g;
        }
    }
#pragma unroll
    for (int j = 0; j < 4; j++) column[threadIdx.x / 16][tn + j] = db[j];
    __syncthreads();
    if (threadIdx.x < kHeadTile && n0 + threadIdx.x < a.n) {
        float s = 0.0f;
        for (int i = 0; i < 16; i++) s += column[i][threadIdx.x];
        a.part_db[(uint64_t)blockIdx.x * a.n + n0 + threadIdx.x] = s;
    }
}

// c in f32, or rounded to the type.
template <typename E, bool Sum>
__device__ __forceinline__ void head_product(const HeadArgs &a) {
    using T = typename E::type;
    const uint64_t m0 = (uint64_t)blockIdx.x * kHeadTile, n0 = (uint64_t)blockIdx.y * kHeadTile;
    float acc[4][4];
    head_tile<E>(a, m0, n0, acc);
    const uint32_t tm = threadIdx.x / 16 * 4, tn = threadIdx.x % 16 * 4;
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint64_t m = m0 + tm + i, n = n0 + tn + j;
            if (m >= a.m || n >= a.n) continue;
            if (Sum) {
                float *c = static_cast<float *>(a.c) + m * a.c_stride + n;
                *c = a.accumulate ? *c + acc[i][j] : acc[i][j];
            } else {
                static_cast<T *>(a.c)[m * a.c_stride + n] = E::down(acc[i][j]);
            }
        }
}

template <typename E>
__device__ __forceinline__ void head_sum(const HeadSumArgs &a) {
    const uint64_t cells = a.rows * a.cols;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < cells; i += (uint64_t)gridDim.x * 256) {
        float s = 0.0f;
        for (uint32_t p = 0; p < a.parts; p++) s += a.part[p * a.part_stride + i];
        const uint64_t r = i / a.cols;
        static_cast<typename E::type *>(a.dst)[r * a.dst_stride + (i - r * a.cols)] = E::down(s);
    }
}

}  // namespace hbr

using namespace hbr;

#define HBR_HEAD(suffix, E)                                                                                       \
    extern "C" __global__ __launch_bounds__(256) void hbr_head_scores_##suffix(HeadArgs a) { head_scores<E>(a); } \
    extern "C" __global__ __launch_bounds__(256) void hbr_head_pairs_##suffix(HeadArgs a) { head_pairs<E>(a); }   \
    extern "C" __global__ __launch_bounds__(256) void hbr_head_add_##suffix(HeadArgs a) { head_product<E, true>(a); } \
    extern "C" __global__ __launch_bounds__(256) void hbr_head_out_##suffix(HeadArgs a) { head_product<E, false>(a); } \
    extern "C" __global__ __launch_bounds__(256) void hbr_head_sum_##suffix(HeadSumArgs a) { head_sum<E>(a); }
HBR_HEAD(f32, F32)
HBR_HEAD(bf16, Bf16)

// A row's tiles joined: 64 rows a workgroup, its 16 waves a share of the
// class tiles each, in order within a wave and over the waves.
extern "C" __global__ __launch_bounds__(1024) void hbr_head_finish(HeadFinishArgs a) {
    constexpr uint32_t kWaves = 16;
    __shared__ float top_of[kWaves][kWave], sum_of[kWaves][kWave];
    __shared__ int32_t best_of[kWaves][kWave];
    const uint32_t lane = lane_id(), wave = threadIdx.x / kWave;
    const uint64_t r = (uint64_t)blockIdx.x * kWave + lane;
    const uint32_t share = (a.tiles + kWaves - 1) / kWaves;
    float top = -INFINITY, sum = 0.0f;
    int32_t best = 0;
    bool any = false;
    if (r < a.rows) {
        for (uint32_t t = wave * share; t < min(a.tiles, (wave + 1) * share); t++) {
            const float m = a.part_max[t * a.rows + r], s = a.part_sum[t * a.rows + r];
            if (!any || m > top) {
                sum = sum * exp_f32(top - shift_of(m)) + s;
                top = m;
                if (a.part_best) best = a.part_best[t * a.rows + r];
            } else {
                sum += s * exp_f32(m - shift_of(top));
            }
            any = true;
        }
    }
    top_of[wave][lane] = any ? top : -INFINITY;
    sum_of[wave][lane] = sum;
    best_of[wave][lane] = best;
    __syncthreads();
    if (wave != 0 || r >= a.rows) return;
    for (uint32_t w = 1; w < kWaves; w++) {
        if (w * share >= a.tiles) break;
        const float m = top_of[w][lane], s = sum_of[w][lane];
        if (m > top) {
            sum = sum * exp_f32(top - shift_of(m)) + s;
            top = m;
            best = best_of[w][lane];
        } else {
            sum += s * exp_f32(m - shift_of(top));
        }
    }
    const int32_t y = a.labels ? a.labels[r] : -1;
    // a label that is no class: neither a loss nor a gradient
    const float lse = y >= 0 && (uint64_t)y >= a.classes ? NAN : shift_of(top) + logf(sum);
    a.lse[r] = lse;
    if (a.best) a.best[r] = best;
    if (!a.loss) return;
    if (!a.labels) {
        a.loss[r] = lse - top;
        return;
    }
    const float by = a.weight ? a.weight[r] : 1.0f;
    a.loss[r] = y < 0 ? 0.0f : (uint64_t)y >= a.classes ? NAN : by * (lse - a.label_margin[r]);
}
