// Projections of rows, with each row's low-rank adapter beside them, and their gradients.
//
//   out = x w^T + bias + scale[a] (x down[a]^T) up[a]^T, a = ids[row]
//   dx = dout w; dw = (dout^T x) weight; db = sum over rows dout
//
// The products are product.h's tiles. An f32 operand is three bf16 parts; rows in
// 8 bits are one (a code times its power is a bf16), so that f32 gradients of
// theirs take three products and not six.
#include <type_traits>

#include "product.h"
#include "rows8.h"

namespace hbr {

// A tile's cells: E what c holds, f32 parts of the sums as they are, or the
// result: times the column's factor, and its bias added.
template <typename Tile, typename E, bool Part>
__device__ __forceinline__ void linear_store(const HeadArgs &a, Tile &t) {
    using T = typename E::type;
    const uint32_t lane = lane_id();
    const uint64_t from = reinterpret_cast<uint64_t>(static_cast<T *>(a.c) + t.split * a.c_split + t.m0 * a.c_stride + t.n0);
    const uint32_t stride = (uint32_t)a.c_stride * sizeof(T);
    const uint32_t rows = min(a.rows > t.m0 ? a.rows - t.m0 : 0u, (uint32_t)Tile::kM);
    const uint32_t size = rows ? (rows - 1) * stride + min(a.n - t.n0, (uint32_t)Tile::kN) * (uint32_t)sizeof(T) : 0u;
    // a buffer that ends with the tile's last cell
    __amdgpu_buffer_rsrc_t c = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void *>(from), 0, size, 0x00020000);
#pragma unroll
    for (int j = 0; j < Tile::kJ; j++) {
        const uint32_t n = t.wave_n + 32 * j + lane % 32;
        const bool in = t.n0 + n < a.n;
        const uint32_t at = in ? (t.wave_m + lane / 32 * 4) * stride + n * (uint32_t)sizeof(T) : kNowhere;
        const float by = !Part && in && a.weight ? a.weight[t.n0 + n] : 1.0f;
        const float bias = !Part && in && a.bias ? a.bias[t.n0 + n] : 0.0f;
#pragma unroll
        for (int i = 0; i < Tile::kI; i++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const uint32_t to = at + (32 * i + 8 * (e / 4) + e % 4) * stride;
                const float v = Part ? t.acc[i][j][e] : __builtin_fmaf(t.acc[i][j][e], by, bias);
                if constexpr (sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), c, to, 0, 0);
                else __builtin_amdgcn_raw_buffer_store_b16(to_bf16(v), c, to, 0, 0);
            }
    }
}

// The tile's adapters: more products, over the pairs (adapter of the tile, rank)
// one behind the other. A row's low values stand at its own adapter's places and
// zeros at the others', so that any order of the rows is right, and rows of few
// adapters take few steps: an adapter's rows next to each other are one slot,
// and in tiles of many slots the same adapter's are joined.
//
// In bf16 the low values are rounded once to bf16, as any product's operand
// is: half a step each of the adapters' part. In f32 all is in three parts.
template <typename Tile, typename E>
__device__ __forceinline__ void linear_adapters(const LinearArgs &a, char *lds, Tile &t) {
    using T = typename E::type;
    constexpr int kParts = sizeof(T) == 4 ? 3 : 1, kPairs = kParts == 3 ? 6 : 1;
    constexpr uint32_t kM = Tile::kM, kNone = 0xffffu, kWaves = Tile::kThreads / kWave;
    using Op = Operand<false, Tile::kW>;
    // the first stage holds a step's operands, the second the slots
    int32_t *slot_id = reinterpret_cast<int32_t *>(lds + Tile::kStage);          // [kM] a slot's adapter
    uint16_t *slot_of = reinterpret_cast<uint16_t *>(slot_id + kM);              // [kM] a row's slot
    uint16_t *joined = slot_of + kM;                                             // [kM] a slot's place among the joined
    uint32_t *counts = reinterpret_cast<uint32_t *>(joined + kM);                // [kWaves]
    static_assert(kM * 8 + kWaves * 4 <= (uint32_t)Tile::kStage && kM <= (uint32_t)Tile::kThreads, "the slots fit a stage");
    const uint32_t m = threadIdx.x, lane = lane_id(), wave = threadIdx.x / kWave;
    auto adapter = [&](uint32_t row) {
        const int32_t id = row < a.p.m ? a.ids[row] : -1;
        return id >= 0 && (uint32_t)id < a.adapters ? id : -1;
    };
    const int32_t id = m < kM ? adapter(t.m0 + m) : -1;
    const bool starts = id >= 0 && (m == 0 || adapter(t.m0 + m - 1) != id);
    const uint64_t start = __ballot(starts);
    if (lane == 0) counts[wave] = (uint32_t)__popcll(start);
    __syncthreads();
    uint32_t slots = 0, before = 0;
    for (uint32_t w = 0; w < kWaves; w++) {
        before += w < wave ? counts[w] : 0;
        slots += counts[w];
    }
    const uint32_t slot = before + (uint32_t)__popcll(start & (~0ull >> (63 - lane))) - 1;  // of the last start up to here
    if (m < kM) slot_of[m] = (uint16_t)(id >= 0 ? slot : kNone);
    if (starts) slot_id[slot] = id;
    __syncthreads();
    slots = (uint32_t)uniform(slots);
    if (slots > 8) {
        // the first slot of the same adapter, and its place among the first ones
        uint32_t first = kNone, place = 0;
        int32_t mine = 0;
        if (m < slots) {
            mine = slot_id[m];
            first = 0;
            while (slot_id[first] != mine) first++;
        }
        const bool is = first == m;
        const uint64_t some = __ballot(is);
        __syncthreads();
        if (lane == 0) counts[wave] = (uint32_t)__popcll(some);
        __syncthreads();
        slots = 0;
        for (uint32_t w = 0; w < kWaves; w++) {
            place += w < wave ? counts[w] : 0;
            slots += counts[w];
        }
        place += (uint32_t)__popcll(some & ((1ull << lane) - 1));
        if (is) joined[m] = (uint16_t)place, slot_id[place] = mine;  // (place <= m, and every slot_id has been read)
        __syncthreads();
        if (first != kNone && !is) joined[m] = joined[first];
        __syncthreads();
        if (m < kM && slot_of[m] != kNone) slot_of[m] = joined[slot_of[m]];
        __syncthreads();
        slots = (uint32_t)uniform(slots);
    }
    const uint32_t all = slots * a.rank;
    const bool wide = (a.up_stride % 8 == 0) && reinterpret_cast<uint64_t>(a.up) % 16 == 0;
    for (uint32_t k0 = 0; k0 < all; k0 += kHeadK) {
        for (int pair = 0; pair < kPairs; pair++) {
            const int pa = kParts == 1 ? 0 : kPartA >> 2 * pair & 3u, pb = kParts == 1 ? 0 : kPartB >> 2 * pair & 3u;
            // pieces of eight products of a row: of the rows' low values, and of the outputs' second factors
            for (uint32_t q = threadIdx.x; q < (kM + Tile::kN) * 4; q += Tile::kThreads) {
                const bool second = q >= kM * 4;
                const uint32_t at = second ? q - kM * 4 : q, row = at / 4, piece = at % 4, k = k0 + piece * 8;
                float v[8] = {};
                uint32_t s = k / a.rank, rho = k - s * a.rank;
                if (second) {
                    if (t.n0 + row < a.p.n) {
                        const T *up = static_cast<const T *>(a.up);
                        if (wide && kParts == 1 && rho + 8 <= a.rank && rho % 8 == 0 && k < all) {
                            const Vec<T, 8> x = *reinterpret_cast<const Vec<T, 8> *>(
                                up + ((uint64_t)slot_id[s] * a.p.n + t.n0 + row) * a.up_stride + rho);
#pragma unroll
                            for (int j = 0; j < 8; j++) v[j] = E::up(x.v[j]);
                        } else {
#pragma unroll
                            for (int j = 0; j < 8; j++) {
                                if (k + j < all) v[j] = E::up(up[((uint64_t)slot_id[s] * a.p.n + t.n0 + row) * a.up_stride + rho]);
                                if (++rho == a.rank) rho = 0, s++;
                            }
                        }
                    }
                } else {
                    const uint32_t own = slot_of[row];
                    if (own != kNone) {
                        const float *low = a.low + (uint64_t)(t.m0 + row) * a.rank;
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            if (k + j < all && s == own) v[j] = low[rho];
                            if (++rho == a.rank) rho = 0, s++;
                        }
                    }
                }
                Vec<uint16_t, 8> out;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    if constexpr (kParts == 1) {
                        out.v[j] = to_bf16(v[j]);
                    } else {
                        uint16_t p[3];
                        split3(v[j], p);
                        const int part = second ? pb : pa;
                        out.v[j] = part == 0 ? p[0] : part == 1 ? p[1] : p[2];
                    }
                }
                char *to = lds + (second ? Op::kBytes : 0) + row * (kHeadK * 2) + (piece ^ ((row >> 2) & 3u)) * 16;
                *reinterpret_cast<Vec<uint16_t, 8> *>(to) = out;
            }
            __syncthreads();
#pragma unroll
            for (int kk = 0; kk < (int)kHeadK / 16; kk++) {
                bf16x8 fa[Tile::kI], fb[Tile::kJ];
#pragma unroll
                for (int i = 0; i < Tile::kI; i++) fa[i] = Op::fragment(lds, t.wave_m + 32 * i, kk);
#pragma unroll
                for (int j = 0; j < Tile::kJ; j++) fb[j] = Op::fragment(lds + Op::kBytes, t.wave_n + 32 * j, kk);
#pragma unroll
                for (int i = 0; i < Tile::kI; i++)
#pragma unroll
                    for (int j = 0; j < Tile::kJ; j++)
                        t.acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[i], fb[j], t.acc[i][j], 0, 0, 0);
            }
            __syncthreads();
        }
    }
}

// E: the inputs' type; Part: f32 sums of a share of the steps
template <typename Tile, typename E, bool Part>
__device__ __forceinline__ void linear_y(const LinearArgs &a, char *lds) {
    Tile t;
    head_place(a.p, t);
    head_product<false, false>(a.p, lds, t);
    if (a.low && (!Part || t.split == 0)) linear_adapters<Tile, E>(a, lds, t);
    linear_store<Tile, std::conditional_t<Part, F32, E>, Part>(a.p, t);
}

// The gradients' products: of the inputs (AT false) and of the weights. E: what c holds.
template <typename Tile, typename E, bool AT, bool Part>
__device__ __forceinline__ void linear_d(const LinearArgs &a, char *lds) {
    Tile t;
    head_place(a.p, t);
    head_product<AT, true>(a.p, lds, t);
    linear_store<Tile, E, Part>(a.p, t);
}

template <typename E>
__device__ __forceinline__ void linear_join(const LinearJoinArgs &a) {
    const uint64_t cells = a.rows * a.cols;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < cells; i += (uint64_t)gridDim.x * 256) {
        const uint64_t r = i / a.cols, c = i - r * a.cols;
        float s = 0.0f;
#pragma unroll 8
        for (uint32_t p = 0; p < a.parts; p++) s += a.part[p * a.part_stride + i];
        s = __builtin_fmaf(s, a.weight ? a.weight[c] : 1.0f, a.bias ? a.bias[c] : 0.0f);
        static_cast<typename E::type *>(a.dst)[r * a.dst_stride + c] = E::down(s);
    }
}

// A wave a row.
template <typename E>
__device__ __forceinline__ void linear_low(const LinearLowArgs &a) {
    using T = typename E::type;
    const uint32_t lane = lane_id();
    for (uint64_t r = (uint64_t)blockIdx.x * 4 + threadIdx.x / kWave; r < a.n_rows; r += (uint64_t)gridDim.x * 4) {
        const int32_t id = a.ids[r];
        if (id < 0 || (uint32_t)id >= a.adapters) continue;
        const float by = a.scale ? a.scale[id] : 1.0f;
        const T *x = static_cast<const T *>(a.x) + r * a.x_stride;
        for (uint32_t rho = 0; rho < a.rank; rho++) {
            const T *down = static_cast<const T *>(a.down) + ((uint64_t)id * a.rank + rho) * a.down_stride;
            float s = 0.0f;
            for (uint32_t c = lane; c < a.dim; c += kWave) s = __builtin_fmaf(E::up(x[c]), E::up(down[c]), s);
            for (int d = 32; d; d /= 2) s += __shfl_xor(s, d, kWave);
            if (lane == 0) a.low[r * a.rank + rho] = s * by;
        }
    }
}

// Eight columns of a row a thread, a wave 16 rows of a chunk.
__device__ __forceinline__ void lay_codes(const LayCodesArgs &a) {
    const uint64_t cells = a.rows * a.chunks * 4;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < cells; i += (uint64_t)gridDim.x * 256) {
        const uint64_t block = i / (a.rows * 16);
        const uint32_t wide = min(4u, a.chunks - (uint32_t)block * 4);
        const uint64_t in = i - block * a.rows * 16, r = in / (wide * 4);
        const uint32_t chunk = (uint32_t)block * 4 + (uint32_t)(in % (wide * 4)) / 4, c = chunk * 32 + in % 4 * 8;
        const uint8_t *src = a.codes + r * a.codes_stride + c;
        Vec<uint8_t, 8> codes{};
        if (c + 8 <= a.cols) {
            __builtin_memcpy(&codes, src, 8);
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (c + k < a.cols) codes.v[k] = src[k];
        }
        float v[8];
        values_of<8>(codes, exp2_of((int32_t)a.scales[r * a.scales_stride + chunk] - kPowerBias), v);
        Vec<uint16_t, 8> out;
#pragma unroll
        for (int k = 0; k < 8; k++) out.v[k] = (uint16_t)(__float_as_uint(v[k]) >> 16);
        *reinterpret_cast<Vec<uint16_t, 8> *>(a.dst + chunk * a.chunk + r * 32 + in % 4 * 8) = out;
    }
}

// A column a thread, a share of the rows a workgroup.
template <typename E>
__device__ __forceinline__ void column_sum(const ColumnSumArgs &a) {
    const uint32_t tiles = (a.cols + 255) / 256, share = blockIdx.x / tiles, c = blockIdx.x % tiles * 256 + threadIdx.x;
    if (c >= a.cols) return;
    const uint64_t r0 = a.rows * share / a.shares, r1 = a.rows * (share + 1) / a.shares;
    const typename E::type *x = static_cast<const typename E::type *>(a.x) + c;
    float s = 0.0f;
#pragma unroll 8
    for (uint64_t r = r0; r < r1; r++) s += E::up(x[r * a.x_stride]);
    a.part[(uint64_t)share * a.cols + c] = s;
}

}  // namespace hbr

using namespace hbr;

#define HBR_LINEAR(name, W, waves, ...)                                                             \
    extern "C" __global__ __launch_bounds__(HeadTile<W>::kThreads, waves) void name(LinearArgs a) { \
        __shared__ __align__(1024) char lds[HeadTile<W>::kLds];                                     \
        __VA_ARGS__(a, lds);                                                                        \
    }
#define HBR_LINEARS(suffix, W, waves)                                                               \
    HBR_LINEAR(hbr_linear_y_f32_##suffix, W, waves, linear_y<HeadTile<W>, F32, false>)              \
    HBR_LINEAR(hbr_linear_y_bf16_##suffix, W, waves, linear_y<HeadTile<W>, Bf16, false>)            \
    HBR_LINEAR(hbr_linear_y_part_f32_##suffix, W, waves, linear_y<HeadTile<W>, F32, true>)          \
    HBR_LINEAR(hbr_linear_y_part_bf16_##suffix, W, waves, linear_y<HeadTile<W>, Bf16, true>)        \
    HBR_LINEAR(hbr_linear_dx_f32_##suffix, W, waves, linear_d<HeadTile<W>, F32, false, false>)      \
    HBR_LINEAR(hbr_linear_dx_bf16_##suffix, W, waves, linear_d<HeadTile<W>, Bf16, false, false>)    \
    HBR_LINEAR(hbr_linear_dx_part_##suffix, W, waves, linear_d<HeadTile<W>, F32, false, true>)      \
    HBR_LINEAR(hbr_linear_dw_f32_##suffix, W, waves, linear_d<HeadTile<W>, F32, true, false>)       \
    HBR_LINEAR(hbr_linear_dw_bf16_##suffix, W, waves, linear_d<HeadTile<W>, Bf16, true, false>)     \
    HBR_LINEAR(hbr_linear_dw_part_##suffix, W, waves, linear_d<HeadTile<W>, F32, true, true>)
HBR_LINEARS(256, 8, 2)
HBR_LINEARS(128, 4, 4)

extern "C" __global__ __launch_bounds__(256) void hbr_linear_join_f32(LinearJoinArgs a) { linear_join<F32>(a); }
extern "C" __global__ __launch_bounds__(256) void hbr_linear_join_bf16(LinearJoinArgs a) { linear_join<Bf16>(a); }
extern "C" __global__ __launch_bounds__(256) void hbr_linear_low_f32(LinearLowArgs a) { linear_low<F32>(a); }
extern "C" __global__ __launch_bounds__(256) void hbr_linear_low_bf16(LinearLowArgs a) { linear_low<Bf16>(a); }
extern "C" __global__ __launch_bounds__(256) void hbr_lay_codes(LayCodesArgs a) { lay_codes(a); }
extern "C" __global__ __launch_bounds__(256) void hbr_column_sum_f32(ColumnSumArgs a) { column_sum<F32>(a); }
extern "C" __global__ __launch_bounds__(256) void hbr_column_sum_bf16(ColumnSumArgs a) { column_sum<Bf16>(a); }
