// Gradient clipping: the norm of a set of tensors, and the set scaled to a
// largest norm,
//
//   norm = sqrt(sum g^2), out = g min(1, max / (norm + 1e-6)).
//
// Two passes, since the factor needs every square: blocks of kClipElems
// elements, the tensors' one behind the other, go round kClipBlocks workgroups,
// whose sums lie in order and are added in order by every workgroup of the
// second pass, so that the bits do not depend on the schedule and no third
// launch joins them. The records of 96 tensors travel as the kernel's
// argument: nothing is copied to the device. Bound by HBM: 400,000,003 bf16
// elements take 164 us (4.9 TB/s) and 279 us (5.7, part of it out of the last
// level's cache); 40 tensors of 300,001 f32 in all 5.7 and 5.3 us, their launches.
#include "common.h"

namespace hbr {

constexpr uint64_t kClipBlock = kClipElems;

__device__ __forceinline__ uint32_t clip_tensor(const ClipArgs &a, uint32_t block) {
    uint32_t lo = 0, hi = a.tensors;  // the last tensor whose first block is not past it
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (a.t[mid].block <= block) lo = mid;
        else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ double block_sum(double v) {
    __shared__ double wave_sum[256 / kWave];
    for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d, kWave);
    if (lane_id() == 0) wave_sum[threadIdx.x / kWave] = v;
    __syncthreads();
    double s = 0.0;
    for (int w = 0; w < 256 / kWave; w++) s += wave_sum[w];
    return s;
}

// One block's squares. Each is exact in f64 (an f32's square has 48 bits).
template <typename E>
__device__ __forceinline__ double clip_squares(const ClipTensor &t, uint64_t at, uint64_t n) {
    using T = typename E::type;
    constexpr int V = 16 / sizeof(T);
    const T *p = static_cast<const T *>(t.data) + at;
    double acc = 0.0;
    uint64_t i = 0;
    if ((reinterpret_cast<uint64_t>(p) & 15u) == 0) {
        const uint64_t vecs = n / V;
        for (uint64_t k = threadIdx.x; k < vecs; k += 256) {
            const Vec<T, V> v = reinterpret_cast<const Vec<T, V> *>(p)[k];
#pragma unroll
            for (int j = 0; j < V; j++) {
                const double x = (double)E::up(v.v[j]);
                acc = __builtin_fma(x, x, acc);
            }
        }
        i = vecs * V;
    }
    for (i += threadIdx.x; i < n; i += 256) {
        const double x = (double)E::up(p[i]);
        acc = __builtin_fma(x, x, acc);
    }
    return acc;
}

template <typename E>
__device__ __forceinline__ void clip_scale(const ClipTensor &t, uint64_t at, uint64_t n, float by) {
    using T = typename E::type;
    constexpr int V = 16 / sizeof(T);
    const T *p = static_cast<const T *>(t.data) + at;
    T *o = static_cast<T *>(t.out) + at;
    uint64_t i = 0;
    if (((reinterpret_cast<uint64_t>(p) | reinterpret_cast<uint64_t>(o)) & 15u) == 0) {
        const uint64_t vecs = n / V;
        for (uint64_t k = threadIdx.x; k < vecs; k += 256) {
            Vec<T, V> v = reinterpret_cast<const Vec<T, V> *>(p)[k];
#pragma unroll
            for (int j = 0; j < V; j++) v.v[j] = E::down(E::up(v.v[j]) * by);
            reinterpret_cast<Vec<T, V> *>(o)[k] = v;
        }
        i = vecs * V;
    }
    for (i += threadIdx.x; i < n; i += 256) o[i] = E::down(E::up(p[i]) * by);
}

}  // namespace hbr

using namespace hbr;

extern "C" __global__ __launch_bounds__(256) void hbr_clip_norm(ClipArgs a) {
    double acc = 0.0;
    for (uint32_t b = blockIdx.x; b < a.blocks; b += gridDim.x) {
        const ClipTensor &t = a.t[clip_tensor(a, b)];
        const uint64_t at = (b - t.block) * kClipBlock, n = min(kClipBlock, t.len - at);
        acc += t.dtype == kBf16 ? clip_squares<Bf16>(t, at, n) : clip_squares<F32>(t, at, n);
    }
    acc = block_sum(acc);
    if (threadIdx.x == 0) a.part[a.first_part + blockIdx.x] = acc;
}

extern "C" __global__ __launch_bounds__(256) void hbr_clip_scale(ClipArgs a) {
    double acc = 0.0;
    for (uint32_t i = threadIdx.x; i < a.parts; i += 256) acc += a.part[i];
    // the norm and the factor in f64, each rounded once; a norm that is not
    // a number gives a factor that is none
    const double norm = __builtin_sqrt(block_sum(acc));
    const double by = a.max_norm / (norm + 1e-6);
    const float factor = (float)(by > 1.0 ? 1.0 : by);
    if (a.norm && a.first_part == 0 && blockIdx.x == 0 && threadIdx.x == 0) *a.norm = (float)norm;
    for (uint32_t b = blockIdx.x; b < a.blocks; b += gridDim.x) {
        const ClipTensor &t = a.t[clip_tensor(a, b)];
        const uint64_t at = (b - t.block) * kClipBlock, n = min(kClipBlock, t.len - at);
        if (t.dtype == kBf16) clip_scale<Bf16>(t, at, n, factor);
        else clip_scale<F32>(t, at, n, factor);
    }
}
