// The softmax head's gradients over short inputs (kNarrowDim elements at
// most): the scores' gradients are made where they are used and never
// written. Either side of the product is held: a wave has 32 rows (for dh) or
// 32 classes (for dw) in registers and walks all of the other side,
//
//   out[x] = sum over y of p(z[y][x]) Y[y],   z[y][x] = <Y[y], X[x]>,
//
// so that the scores are made twice more and no pair is stored. What is
// saved is the pairs' traffic, 6 bytes a score in bf16 and 30 in f32's parts
// (written once, read twice), against 2 dim operations. Bound by the
// exponentials and their surroundings, about ten instructions a score: 16,384 x
// 8,192 scores of 64 bf16, made three times, take 184 us, 2.2e12 a second.
//
// The first product leaves a lane one x and, of sixteen y, the eight that the
// second product's operand takes from it, in an order that the transposing
// reads of Y follow: the scores' gradients pass from the one to the other
// without leaving the lane.
#include "product.h"

namespace hbr {

constexpr int kNarrowY = 64, kNarrowWaves = 4, kNarrowX = 32 * kNarrowWaves;

// kScores holds rows as kRows does, and keeps each row's running maximum and
// sum in the place of the second product.
enum NarrowMode { kScores, kRows, kClasses };

template <NarrowMode Mode, int Parts, int DT>
__device__ __forceinline__ void head_narrow(const NarrowArgs &a, char *lds) {
    constexpr bool Rows = Mode != kClasses;
    constexpr int kChunk = kNarrowY * 64, kStage = Parts * DT * kChunk, kSteps = 2 * DT, kSegments = Parts == 1 ? 1 : 6;
    __shared__ float u_of[2][kNarrowY], weight_of[2][kNarrowY];
    __shared__ int32_t label_of[2][kNarrowY];
    const uint32_t lane = lane_id(), wave = uniform(threadIdx.x / kWave), half = lane / 32;
    const uint32_t split = blockIdx.x / a.x_tiles, x_tile = blockIdx.x % a.x_tiles;
    const uint32_t x = x_tile * kNarrowX + wave * 32 + lane % 32;
    const bool in = x < a.nx;
    // the held side
    bf16x8 xf[Parts][kSteps];
#pragma unroll
    for (int q = 0; q < Parts; q++)
#pragma unroll
        for (int k = 0; k < kSteps; k++) {
            i32x4 v = {0, 0, 0, 0};
            if (in)
                v = *reinterpret_cast<const i32x4 *>(static_cast<const char *>(a.x) + q * a.x_part + k / 2 * a.x_chunk +
                                                     (uint64_t)x * 64 + (k % 2 * 2 + half) * 16);
            xf[q][k] = __builtin_bit_cast(bf16x8, v);
        }
    float v_x = 0.0f, weight_x = 1.0f;
    int32_t label_x = -1;
    if (Mode == kScores) {
        if (in && a.labels) label_x = a.labels[x];
    } else if (Rows && in) {
        label_x = a.labels[x];
        v_x = label_x < 0 ? -INFINITY : -a.lse2[x];
        if (a.weight && label_x >= 0) weight_x = a.weight[x];
    } else if (in && a.bias) {
        v_x = a.bias[x];
    }
    f32x16 out[DT];
#pragma unroll
    for (int t = 0; t < DT; t++)
#pragma unroll
        for (int e = 0; e < 16; e++) out[t][e] = 0.0f;
    float db = 0.0f;
    float top = -INFINITY, total = 0.0f;  // kScores
    int32_t best = 0x7fffffff;
    const uint32_t steps = (a.ny + kNarrowY - 1) / kNarrowY;
    const uint32_t s0 = (uint32_t)((uint64_t)steps * split / a.splits), s1 = (uint32_t)((uint64_t)steps * (split + 1) / a.splits);
    // a wave's share of a stage: 16 rows of every chunk, their 16-byte pieces
    // exchanged within a row for the reads along the rows (the transposing
    // ones read whole rows, in any order)
    const uint32_t row = wave * 16 + lane / 4, off = row * 64 + (lane % 4 ^ ((row >> 2) & 3u)) * 16;
    float next_u = -INFINITY, next_weight = 0.0f;
    int32_t next_label = -1;
    auto load = [&](uint32_t s) {
        const uint32_t y0 = s * kNarrowY, left = s < s1 ? min(a.ny - y0, (uint32_t)kNarrowY) : 0;
        const uint32_t to = (uint32_t)(uintptr_t)(HBR_LDS char *)lds + s % 2 * kStage + wave * 1024;
#pragma unroll
        for (int q = 0; q < Parts; q++)
#pragma unroll
            for (int c = 0; c < DT; c++) {
                const uint64_t from = reinterpret_cast<uint64_t>(a.y) + q * a.y_part + c * a.y_chunk + (uint64_t)y0 * 64;
                const i32x4 r = {uniform((uint32_t)from), uniform((uint32_t)(from >> 32)) & 0xffff, uniform(left * 64), 0x00020000};
                asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                             :
                             : "s"(uniform(to + (q * DT + c) * kChunk)), "v"(off), "s"(r)
                             : "memory");
            }
        // the y's own numbers, a thread each
        if (threadIdx.x < kNarrowY) {
            const uint32_t y = y0 + threadIdx.x;
            next_u = -INFINITY;
            next_weight = 0.0f;
            next_label = -1;
            if (threadIdx.x < left) {
                if (Rows) {
                    next_u = a.bias ? a.bias[y] : 0.0f;
                } else {
                    next_label = a.labels[y];
                    next_u = next_label < 0 ? -INFINITY : -a.lse2[y];
                    next_weight = next_label < 0 ? 0.0f : a.weight ? a.weight[y] : 1.0f;
                }
            }
        }
    };
    auto meet = [&](uint32_t s) {  // stage s is whole, and the other is read
        if (threadIdx.x < kNarrowY) {
            u_of[s % 2][threadIdx.x] = next_u;
            if (!Rows) {
                weight_of[s % 2][threadIdx.x] = next_weight;
                label_of[s % 2][threadIdx.x] = next_label;
            }
        }
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    load(s0);
    for (uint32_t s = s0; s < s1; s++) {
        meet(s);
        load(s + 1);
        const char *stage = lds + s % 2 * kStage;
#pragma unroll 1
        for (uint32_t b = 0; b < kNarrowY / 32; b++) {
            f32x16 z;
#pragma unroll
            for (int e = 0; e < 16; e++) z[e] = 0.0f;
#pragma unroll
            for (int g = 0; g < kSegments; g++) {
                const int of = Parts == 1 ? 10 : 2 * g, pa = kPartA >> of & 3u, pb = kPartB >> of & 3u;
#pragma unroll
                for (int k = 0; k < kSteps; k++) {
                    const uint32_t y = b * 32 + lane % 32, piece = (k % 2 * 2 + half) ^ ((y >> 2) & 3u);
                    const bf16x8 f = *reinterpret_cast<const bf16x8 *>(stage + (pa * DT + k / 2) * kChunk + y * 64 + piece * 16);
                    z = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f, xf[pb][k], z, 0, 0, 0);
                }
            }
            const uint32_t y0 = s * kNarrowY + b * 32;
            if constexpr (Mode == kScores) {
                if (y0 + 32 > a.ny)  // past the last class: zeros, which make no number of an infinite input
#pragma unroll
                    for (int e = 0; e < 16; e++)
                        if (y0 + row_of(e) >= a.ny) z[e] = 0.0f;
                float most = -INFINITY;
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    z[e] += u_of[s % 2][b * 32 + row_of(e)];
                    most = fmaxf(most, z[e]);
                }
                if (__ballot((uint32_t)label_x - y0 < 32u))
#pragma unroll
                    for (int e = 0; e < 16; e++)
                        if (label_x == (int32_t)(y0 + row_of(e)) && (uint32_t)label_x < a.ny) a.label_margin[x] = z[e];
                if (a.part_best && __ballot(most > top)) {
                    int32_t at = 0x7fffffff;
#pragma unroll
                    for (int e = 15; e >= 0; e--)
                        if (z[e] == most) at = (int32_t)(y0 + row_of(e));
                    if (most > top) best = at;
                }
                const float both = fmaxf(top, most), shift = shift_of(both);
                float sum = 0.0f;
#pragma unroll
                for (int e = 0; e < 16; e++) sum += exp_of(z[e] - shift);
                total = total * exp_of(top - shift) + sum;
                top = both;
                continue;
            }
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const float u = u_of[s % 2][b * 32 + row_of(e)];
                // the class's bias and the row's -lse log2 e are one each of u and v_x
                z[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(z[e] + (Rows ? u : v_x), kLog2e, Rows ? v_x : u));
            }
            // one less where the row's label is the class, if that is anywhere here
            if (Rows) {
                if (__ballot((uint32_t)label_x - y0 < 32u))
#pragma unroll
                    for (int e = 0; e < 16; e++)
                        if (label_x == (int32_t)(y0 + row_of(e))) z[e] -= 1.0f;
            } else {
                const uint32_t x0 = x - lane % 32;
                if (__ballot((uint32_t)label_of[s % 2][b * 32 + lane % 32] - x0 < 32u))
#pragma unroll
                    for (int e = 0; e < 16; e++)
                        if (label_of[s % 2][b * 32 + row_of(e)] == (int32_t)x) z[e] -= 1.0f;
                if (a.weight)
#pragma unroll
                    for (int e = 0; e < 16; e++) z[e] *= weight_of[s % 2][b * 32 + row_of(e)];
                auto sum_of = [&] {  // of the block alone: the running sum may be far larger
                    float sum = 0.0f;
#pragma unroll
                    for (int e = 0; e < 16; e++) sum += z[e];
                    return sum;
                };
                float sum = sum_of();
                if (__ballot(sum != sum)) {
                    // a row that takes no part may have any score: past f32's
                    // range, less infinity, it is no number
#pragma unroll
                    for (int e = 0; e < 16; e++)
                        if (label_of[s % 2][b * 32 + row_of(e)] < 0) z[e] = 0.0f;
                    sum = sum_of();
                }
                db += sum;
            }
            // sixteen y a fragment, of which a lane has eight: its elements
            // 8 k to 8 k + 7, y 16 k + 4 half + 0..3 and 8 more
            union Frag {
                uint16_t v[8];
                bf16x8 f;
            } pf[Parts][2];
#pragma unroll
            for (int e = 0; e < 16; e++) {
                if (Parts == 1) {
                    pf[0][e / 8].v[e % 8] = to_bf16(z[e]);
                } else {
                    uint16_t part[3];
                    split3(z[e], part);
#pragma unroll
                    for (int q = 0; q < Parts; q++) pf[q][e / 8].v[e % 8] = part[q];
                }
            }
#pragma unroll
            for (int t = 0; t < DT; t++)
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    bf16x8 f[Parts];
#pragma unroll
                    for (int q = 0; q < Parts; q++) {
                        union {
                            s16x4 h[2];
                            bf16x8 v;
                        } w;
#pragma unroll
                        for (int p = 0; p < 2; p++) {
                            const uint32_t y = b * 32 + k * 16 + p * 8 + half * 4 + lane % 16 / 4;
                            const uint32_t piece = (lane / 16 % 2 * 2 + lane % 4 / 2) ^ ((y >> 2) & 3u);
                            w.h[p] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                (HBR_LDS s16x4 *)(stage + (q * DT + t) * kChunk + y * 64 + piece * 16 + lane % 2 * 8));
                        }
                        f[q] = w.v;
                    }
#pragma unroll
                    for (int g = 0; g < kSegments; g++) {
                        const int of = Parts == 1 ? 10 : 2 * g;
                        out[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[kPartA >> of & 3u], pf[kPartB >> of & 3u][k].f, out[t], 0, 0, 0);
                    }
                }
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if constexpr (Mode == kScores) {
        const float t = __shfl_xor(top, 32, kWave), sum = __shfl_xor(total, 32, kWave);
        const int32_t b = __shfl_xor(best, 32, kWave);
        const float both = fmaxf(top, t), shift = shift_of(both);
        if (!in || half) return;
        const uint64_t at = (uint64_t)split * a.nx + x;
        a.part_max[at] = both;
        a.part_sum[at] = total * exp_of(top - shift) + sum * exp_of(t - shift);
        if (a.part_best) a.part_best[at] = top > t ? best : t > top ? b : min(best, b);
        return;
    }
    if (!Rows) db += __shfl_xor(db, 32, kWave);
    if (!in) return;
    if (!Rows && a.part_db && half == 0) a.part_db[(uint64_t)split * a.nx + x] = db;
    float *part = a.part + ((uint64_t)split * a.nx + x) * a.dim;
#pragma unroll
    for (int t = 0; t < DT; t++)
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const uint32_t d = 32 * t + row_of(e);
            if (d < a.dim) part[d] = Rows && label_x < 0 ? 0.0f : out[t][e] * weight_x;
        }
}

}  // namespace hbr

using namespace hbr;

#define HBR_NARROW_MODE(name, Mode, Parts, DT)                                      \
    extern "C" __global__ __launch_bounds__(256, 2) void name(NarrowArgs a) {       \
        __shared__ __align__(1024) char lds[2 * Parts * DT * kNarrowY * 64];        \
        head_narrow<Mode, Parts, DT>(a, lds);                                       \
    }
#define HBR_NARROW(suffix, Parts, DT)                                               \
    HBR_NARROW_MODE(hbr_head_narrow_scores_##suffix, kScores, Parts, DT)            \
    HBR_NARROW_MODE(hbr_head_narrow_dh_##suffix, kRows, Parts, DT)                  \
    HBR_NARROW_MODE(hbr_head_narrow_dw_##suffix, kClasses, Parts, DT)
HBR_NARROW(bf16_1, 1, 1)
HBR_NARROW(bf16_2, 1, 2)
HBR_NARROW(bf16_3, 1, 3)
HBR_NARROW(f32_1, 3, 1)
HBR_NARROW(f32_2, 3, 2)
