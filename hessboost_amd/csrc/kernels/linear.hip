// Projections of rows, with each row's low-rank adapter beside them, and their gradients.
//
//   out = x w^T + bias + scale[a] (x down[a]^T) up[a]^T, a = ids[row]
//   dx = dout w; dw = (dout^T x) weight; db = sum over rows dout
//
// The products are tile_product.h's. An f32 operand is three bf16 parts; rows in
// 8 bits are one (a code times its power is a bf16), so that f32 gradients of
// theirs take three products and not six.
//
// Measured (us, and what a large product's 1,361 TFLOP/s would take): 65,536 rows of
// 1,024 by 4,096 bf16, both gradients out of rows in 8 bits 944 to 990 (808), of
// which dx 446 to 511, dw 459 to 535, codes laid out 46 to 51, shares joined 20 to 22;
// 8,191 rows forward 73 to 78 (50), with 64 adapters of rank 16 in 50 runs 94 to 99
// (52), in random order 297 to 308; 7 rows, each its own adapter, 15 for the call, 5 a
// kernel; 4,001 x 250 by 333 f32, both gradients, 36 in three short kernels.
#include <type_traits>

#include "tile_product.h"
#include "rows8.h"

namespace hbr {

// A lane's four columns of a row: cells e = 4 g to 4 g + 3 of acc[i][j].
template <typename Tile>
__device__ __forceinline__ uint32_t column_of(const Tile &t, int i, int g) { return t.m0 + t.wave_m + 32 * i + 8 * g + 4 * (lane_id() / 32); }

// What a lane's columns are multiplied by (a weight) or have added (a bias), read
// before the products and waited for behind them. Null: nothing.
template <typename Tile>
struct Columns {
    float v[Tile::kI][4][4];
    __device__ __forceinline__ void read(const Tile &t, const float *p, uint32_t cols, float otherwise) {
#pragma unroll
        for (int i = 0; i < Tile::kI; i++)
#pragma unroll
            for (int g = 0; g < 4; g++)
#pragma unroll
                for (int k = 0; k < 4; k++) v[i][g][k] = p ? p[min(column_of(t, i, g) + k, cols - 1)] : otherwise;
    }
};
struct NoColumns {};

// The sums stay in the accumulators' registers until they are used.
template <typename Tile>
__device__ __forceinline__ void hold(Tile &t) {
#pragma unroll
    for (int i = 0; i < Tile::kI; i++)
#pragma unroll
        for (int j = 0; j < Tile::kJ; j++) {
            if constexpr (Tile::kI == 4) asm volatile("" : "+a"(t.acc[i][j]));
        }
}

// The tile's result, through LDS to stores of 16 bytes: 64 of a wave's rows by
// 128 bytes of columns at a time, in its own 8 KiB. A row's pieces of 16 bytes are
// exchanged by the row's bits, so that rows meet different banks.
template <typename Tile, typename E, bool Weighted, typename More>
__device__ __forceinline__ void linear_store(const LinearArgs &a, char *room, Tile &t, const More &more) {
    using T = typename E::type;
    constexpr int kSize = sizeof(T), kBlocks = 4 / kSize, kV = 16 / kSize;  // blocks of 32 columns at a time; columns a piece
    static_assert(Tile::kI % kBlocks == 0 && Tile::kJ % 2 == 0, "whole blocks");
    const uint32_t lane = lane_id();
    const uint32_t own = (uint32_t)(uintptr_t)(HBR_LDS char *)room + uniform(threadIdx.x / kWave) * 8192;
    // a lane's cells of a row lie at one piece, exchanged by constants
    uint32_t in = own + lane % 32 * 128 + (kSize == 4 ? (lane % 8 ^ lane / 32) * 16 : lane % 8 * 16 + lane / 32 * 8);
    uint32_t back = own + lane / 8 * 128 + (lane % 8 ^ lane / 8) * 16;
    asm volatile("" : "+v"(in), "+v"(back));  // (no address of theirs is kept from tile to tile)
    const bool whole = a.out_stride % kV == 0 && reinterpret_cast<uint64_t>(a.out) % 16 == 0 && t.m0 + Tile::kM <= a.cols;
#pragma unroll
    for (int i0 = 0; i0 < Tile::kI; i0 += kBlocks)
#pragma unroll
        for (int j0 = 0; j0 < Tile::kJ; j0 += 2) {
            hold(t);
#pragma unroll
            for (int b = 0; b < kBlocks; b++)
#pragma unroll
                for (int g = 0; g < 4; g++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        Vec<T, 4> v;
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            float x = t.acc[i0 + b][j0 + j][4 * g + k];
                            if constexpr (!std::is_same_v<More, NoColumns>) {
                                if constexpr (Weighted) x *= more.v[i0 + b][g][k];
                                else x += more.v[i0 + b][g][k];
                            }
                            if constexpr (kSize == 4) v.v[k] = x;
                            else v.v[k] = to_bf16(x);
                        }
                        *(HBR_LDS Vec<T, 4> *)((in ^ (uint32_t)(kSize == 4 ? 2 * g : 4 * b + g) * 16) + 4096 * j) = v;
                    }
            const uint32_t r = t.n0 + t.wave_n + 32 * j0 + lane / 8, c = t.m0 + t.wave_m + 32 * i0 + lane % 8 * kV;
            T *to = static_cast<T *>(a.out) + (uint64_t)r * a.out_stride + c;
            auto piece = [&](int q) { return *(HBR_LDS const Vec<T, kV> *)(back + q * 1024); };
            if (whole) {
#pragma unroll
                for (int q = 0; q < 8; q++, to += 8 * a.out_stride)
                    if (r + 8 * q < a.rows) *reinterpret_cast<Vec<T, kV> *>(to) = piece(q);
            } else {
                for (int q = 0; q < 8; q++, to += 8 * a.out_stride) {
                    const Vec<T, kV> v = piece(q);
#pragma unroll
                    for (int k = 0; k < kV; k++)
                        if (r + 8 * q < a.rows && c + k < a.cols) to[k] = v.v[k];
                }
            }
            asm volatile("" ::: "memory");  // the pieces are read before the next ones are written
        }
}

// Where a tile's sums lie among the parts, in fours.
template <typename Tile>
__device__ __forceinline__ uint64_t part_at(const HeadArgs &p, uint64_t tile, uint32_t cell) {
    return (tile * (Tile::kI * Tile::kJ * 4) + cell) * Tile::kThreads + threadIdx.x;
}

template <typename Tile>
__device__ __forceinline__ void linear_store_part(const LinearArgs &a, Tile &t) {
    const uint64_t tile = ((uint64_t)t.split * a.p.m_tiles + t.m0 / Tile::kM) * a.p.n_tiles + t.n0 / Tile::kN;
#pragma unroll
    for (int i = 0; i < Tile::kI; i++)
#pragma unroll
        for (int j = 0; j < Tile::kJ; j++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                Vec<float, 4> v;
#pragma unroll
                for (int k = 0; k < 4; k++) v.v[k] = t.acc[i][j][4 * g + k];
                reinterpret_cast<Vec<float, 4> *>(a.part)[part_at<Tile>(a.p, tile, (i * Tile::kJ + j) * 4 + g)] = v;
            }
}

// The tile's adapters: more products, over the pairs (adapter of the tile, rank)
// one behind the other. A row's low values stand at its own adapter's places and
// zeros at the others', so that any order of the rows is right, and rows of few
// adapters take few steps.
//
// The low values are f32 sums and stay so, in three bf16 parts; `up` is one part in
// bf16 and three in f32. (As one bf16 each they took less time, 8,191 rows of 1,024
// by 4,096 with 64 adapters in 50 runs 94 us and now 99, in random order 256 and
// 308; but few rows and shares' joins add f32 values, and a row's outputs depended
// on how many rows stood beside it.)
//
// An adapter is its own rows' alone: an element of `up` that is no finite number
// would make no number of the others' zeros, so a one of its sign stands in its
// place (so that an infinite low value stays infinite), and a tile that met one
// goes over its adapters four times more, once for either sign of low values and
// of such elements, with a product of the largest numbers, infinite, where a row's
// own adapter has the pair. What is zero or no number counts for both signs:
// infinity less infinity, no number, as the formula has it.
template <typename Tile, typename E>
struct Adapters {
    using T = typename E::type;
    static constexpr int kUps = sizeof(T) == 4 ? 3 : 1, kLows = 3, kPairs = kUps == 3 ? 6 : 3;
    // A step is 32 products, in f32 16, of all their parts
    static constexpr uint32_t kM = Tile::kM, kStep = kUps == 1 ? 32 : 16, kRow = kStep * 2, kPart = kM * kRow, kIn = kStep / 8;
    static constexpr uint32_t kStage = (kUps + kLows) * kPart;
    static constexpr int kPieces = kM * kIn / Tile::kThreads;  // of eight products of a row, of either operand
    static_assert(Tile::kM == Tile::kN && kM * kIn % Tile::kThreads == 0, "as many pieces of each a thread");
    static_assert(2 * kStage <= (uint32_t)Tile::kLds, "two steps fit the stages");
    static_assert(Tile::kThreads == 4 * kWave, "four waves' flags");
    uint32_t all, own[kPieces];
    const int32_t *slot_id;
    bool eights, wide;

    __device__ __forceinline__ Adapters(const LinearArgs &a, const Tile &t) {
        const uint32_t tile = t.n0 / Tile::kN;
        all = uniform(a.slots[tile]) * a.rank;
        slot_id = a.slot_id + (uint64_t)tile * Tile::kN;
        eights = a.rank % 8 == 0;
        wide = eights && a.up_stride % 8 == 0 && reinterpret_cast<uint64_t>(a.up) % 16 == 0;
#pragma unroll
        for (int q = 0; q < kPieces; q++) own[q] = a.slot_of[min(t.n0 + (q * Tile::kThreads + threadIdx.x) / kIn, a.rows - 1)];
    }
    // Whether any of eight elements is no finite number: their exponents, two at a
    // time in 16 bits, carried into the sign's place.
    template <typename B>
    static __device__ __forceinline__ bool not_finite(const Vec<B, 8> &v) {
        constexpr uint32_t kExponents = sizeof(B) == 4 ? 0x7f800000u : 0x7f807f80u, kOne = sizeof(B) == 4 ? 0x00800000u : 0x00800080u;
        const auto words = __builtin_bit_cast(Vec<uint32_t, 2 * sizeof(B)>, v);
        uint32_t carried = 0;
#pragma unroll
        for (uint32_t i = 0; i < 2 * sizeof(B); i++) carried |= (words.v[i] & kExponents) + kOne;
        return (carried & ~kExponents & (kExponents << 1)) != 0;
    }
    static __device__ __forceinline__ bool finite(float v) { return (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u; }
    // A step's operands as they are read, beside the products of the step before
    // (64 adapters in random order took an eighth less time so than read behind
    // them), and which pieces of `low` and `up` count: nothing waits
    // for them before they are put into LDS.
    struct Step {
        float low[kPieces][8];
        Vec<T, 8> up[kPieces];
        bool mine[kPieces], some[kPieces];
        uint32_t slot, rho;  // of the next read, whose adapter is known by then
        int32_t id;
    };
    // (a piece of eight is one slot's, and all of a thread's pieces are the same one's)
    __device__ __forceinline__ void look(const LinearArgs &a, uint32_t k0, Step &to) {
        const uint32_t kc = min(k0 + threadIdx.x % kIn * 8, all - 1);
        to.slot = kc / a.rank;
        to.rho = (kc - to.slot * a.rank) & ~7u;
        to.id = slot_id[to.slot];
    }
    // Every load is made, from within its array.
    __device__ __forceinline__ void read(const LinearArgs &a, const Tile &t, uint32_t k0, Step &to) {
        const T *ups = static_cast<const T *>(a.up);
        auto lows = [&](int q) { return a.low + (uint64_t)(min(t.n0 + (q * Tile::kThreads + threadIdx.x) / kIn, a.rows - 1)) * a.rank; };
        auto from = [&](int q, int32_t id) {
            const uint64_t out = min(t.m0 + (q * Tile::kThreads + threadIdx.x) / kIn, a.cols - 1);
            return ups + ((uint64_t)id * a.cols + out) * a.up_stride;
        };
        if (eights) {
            const uint32_t k = k0 + threadIdx.x % kIn * 8, s = to.slot, rho = to.rho;
            const int32_t id = to.id;
            look(a, k0 + kStep, to);
#pragma unroll
            for (int q = 0; q < kPieces; q++) {
                const Vec<float, 4> l0 = *reinterpret_cast<const Vec<float, 4> *>(lows(q) + rho),
                                    l1 = *reinterpret_cast<const Vec<float, 4> *>(lows(q) + rho + 4);
#pragma unroll
                for (int j = 0; j < 8; j++) to.low[q][j] = j < 4 ? l0.v[j % 4] : l1.v[j % 4];
                to.some[q] = k < all;
                to.mine[q] = k < all && s == own[q];
            }
            if (wide) {
#pragma unroll
                for (int q = 0; q < kPieces; q++) to.up[q] = *reinterpret_cast<const Vec<T, 8> *>(from(q, id) + rho);
            } else {
#pragma unroll
                for (int q = 0; q < kPieces; q++)
#pragma unroll
                    for (int j = 0; j < 8; j++) to.up[q].v[j] = from(q, id)[rho + j];
            }
            return;
        }
#pragma unroll
        for (int q = 0; q < kPieces; q++) {
            const uint32_t k = k0 + threadIdx.x % kIn * 8, kc = min(k, all - 1);
            uint32_t s = kc / a.rank, rho = kc - s * a.rank;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const bool some = k + j < all;
                const float l = lows(q)[rho];
                const T u = from(q, slot_id[s])[rho];
                to.low[q][j] = some && s == own[q] ? l : 0.0f;
                to.up[q].v[j] = some ? u : (T)0;
                if (++rho == a.rank) {
                    rho = 0;
                    s += k + j + 1 < all;
                }
            }
            to.some[q] = to.mine[q] = true;
        }
    }
    // a piece's place: the rows that LDS serves at once meet different banks
    static __device__ __forceinline__ uint32_t place(uint32_t row, uint32_t piece) {
        return row * kRow + (piece ^ ((row >> (kIn == 4 ? 2 : 3)) & (kIn - 1))) * 16;
    }
    template <int Parts>
    static __device__ __forceinline__ void put(char *to, const float (&v)[8]) {
        Vec<uint16_t, 8> out[Parts];
        float rest[8];
#pragma unroll
        for (int j = 0; j < 8; j++) rest[j] = v[j];
#pragma unroll
        for (int q = 0; q < Parts; q++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                out[q].v[j] = to_bf16(rest[j]);
                rest[j] -= bf16_f32(out[q].v[j]);
            }
        // (what does not round to a finite number is split by itself)
        if (Parts == 3 && not_finite(out[0])) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                uint16_t p[3];
                split3(v[j], p);
#pragma unroll
                for (int q = 0; q < Parts; q++) out[q].v[j] = p[q];
            }
        }
#pragma unroll
        for (int q = 0; q < Parts; q++) *reinterpret_cast<Vec<uint16_t, 8> *>(to + q * kPart) = out[q];
    }
    // What stands in the operands' places of the passes behind the first: the
    // largest bf16, whose square f32 does not hold.
    static constexpr float kLargest = 0x1.fep127f;
    __device__ __forceinline__ void mark(const LinearArgs &a, const Tile &t, uint32_t k0, int q, float sign_low, float sign_up, float (&low)[8],
                                         float (&up)[8]) {
        const uint32_t at = q * Tile::kThreads + threadIdx.x, row = at / kIn;
        const uint64_t out = min(t.m0 + row, a.cols - 1), in = min(t.n0 + row, a.rows - 1);
        for (int j = 0; j < 8; j++) {
            const uint32_t k = k0 + at % kIn * 8 + j, kc = min(k, all - 1), s = kc / a.rank, rho = kc - s * a.rank;
            const float u = E::up(static_cast<const T *>(a.up)[((uint64_t)slot_id[s] * a.cols + out) * a.up_stride + rho]);
            const bool mine = k < all && s == own[q];
            low[j] = mine && !(a.low[in * a.rank + rho] * sign_low < 0.0f) ? kLargest : 0.0f;
            up[j] = k < all && !finite(u) && !(u * sign_up < 0.0f) ? kLargest * sign_low * sign_up : 0.0f;
        }
    }
    // a pass over the adapters; whether a thread's elements are all finite
    template <bool First>
    __device__ __forceinline__ bool pass(const LinearArgs &a, char *stages, Tile &t, float sign_low = 0.0f, float sign_up = 0.0f) {
        const uint32_t lane = lane_id();
        bool all_finite = true;
        Step step;
        if constexpr (First) {
            look(a, 0, step);
            read(a, t, 0, step);
        }
        for (uint32_t k0 = 0, turn = 0; k0 < all; k0 += kStep, turn ^= 1) {
            char *lds = stages + turn * kStage;
#pragma unroll
            for (int q = 0; q < kPieces; q++) {
                const uint32_t at = q * Tile::kThreads + threadIdx.x;
                char *to = lds + place(at / kIn, at % kIn);
                float v[8], low[8];
                if constexpr (First) {
                    Vec<T, 8> &u = step.up[q];
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        low[j] = step.mine[q] ? step.low[q][j] : 0.0f;
                        u.v[j] = step.some[q] ? u.v[j] : (T)0;
                    }
                    if (not_finite(u)) {
                        all_finite = false;
#pragma unroll
                        for (int j = 0; j < 8; j++) u.v[j] = finite(E::up(u.v[j])) ? u.v[j] : E::down(__builtin_copysignf(1.0f, E::up(u.v[j])));
                    }
                    if constexpr (kUps == 1) {
                        *reinterpret_cast<Vec<T, 8> *>(to) = u;
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; j++) v[j] = u.v[j];
                        put<kUps>(to, v);
                    }
                } else {
                    mark(a, t, k0, q, sign_low, sign_up, low, v);
                    put<kUps>(to, v);
                }
                if (!First || __ballot(step.mine[q])) {
                    put<kLows>(to + kUps * kPart, low);
                } else {  // zeros need no parts
#pragma unroll
                    for (int part = 0; part < kLows; part++) *reinterpret_cast<Vec<uint16_t, 8> *>(to + (kUps + part) * kPart) = {};
                }
                __builtin_amdgcn_sched_barrier(0);  // and one piece's parts
            }
            __syncthreads();  // (the step before the last has been read by all that come here)
            if constexpr (First)
                if (k0 + kStep < all) read(a, t, k0 + kStep, step);  // beside the products
#pragma unroll
            for (uint32_t kk = 0; kk < kStep / 16; kk++) {
                const uint32_t piece = kk * 2 + lane / 32;
                auto fragment = [&](uint32_t part, uint32_t row) {
                    return *reinterpret_cast<const bf16x8 *>(lds + part * kPart + place(row + lane % 32, piece));
                };
                bf16x8 fa[kUps][Tile::kI], first[Tile::kJ];
#pragma unroll
                for (int j = 0; j < Tile::kJ; j++) first[j] = fragment(kUps, t.wave_n + 32 * j);
#pragma unroll
                for (int part = 0; part < kUps; part++)
#pragma unroll
                    for (int i = 0; i < Tile::kI; i++) fa[part][i] = fragment(part, t.wave_m + 32 * i);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int j = 0; j < Tile::kJ; j++) {
                    // (where none of the 32 rows has the adapters of these products nothing is added)
                    const auto words = __builtin_bit_cast(i32x4, first[j]);
                    if (!__ballot((words[0] | words[1] | words[2] | words[3]) != 0)) continue;
                    // the other parts are read under the products with the first
                    const bf16x8 fb[kLows] = {first[j], fragment(kUps + 1, t.wave_n + 32 * j), fragment(kUps + 2, t.wave_n + 32 * j)};
#pragma unroll
                    for (int pair = kPairs - 1; pair >= 0; pair--) {
                        const uint32_t pa = kUps == 1 ? 0 : kPartB >> 2 * pair & 3u, pb = (kUps == 1 ? kPartsByOne : kPartA) >> 2 * pair & 3u;
#pragma unroll
                        for (int i = 0; i < Tile::kI; i++)
                            t.acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[pa][i], fb[pb], t.acc[i][j], 0, 0, 0);
                    }
                }
            }
        }
        __syncthreads();
        return all_finite;
    }
    __device__ __forceinline__ void add(const LinearArgs &a, char *stages, Tile &t) {
        if (all == 0) return;
        const uint64_t some = __ballot(!pass<true>(a, stages, t));
        uint32_t *met = reinterpret_cast<uint32_t *>(stages);
        if (lane_id() == 0) met[threadIdx.x / kWave] = some != 0;
        __syncthreads();
        const uint32_t any = uniform(met[0] | met[1] | met[2] | met[3]);
        __syncthreads();
        if (!any) return;
        for (uint32_t signs = 0; signs < 4; signs++) pass<false>(a, stages, t, signs & 1 ? -1.0f : 1.0f, signs & 2 ? -1.0f : 1.0f);
    }
};

// The adapters of a tile's rows, each once, in order of their first rows.
__device__ __forceinline__ void tile_slots(const LinearLowArgs &a, uint32_t tile) {
    __shared__ int32_t start_id[256];
    __shared__ uint16_t start_slot[256];
    __shared__ uint32_t counts[4];
    const uint32_t m = threadIdx.x, lane = lane_id(), wave = m / kWave;
    const uint64_t r0 = (uint64_t)tile * a.tile;
    auto adapter = [&](uint32_t in) {
        const int32_t id = in < a.tile && r0 + in < a.n_rows ? a.ids[r0 + in] : -1;
        return id >= 0 && (uint32_t)id < a.adapters ? id : -1;
    };
    // a count over the threads up to this one
    auto place = [&](bool is, uint32_t &all) {
        const uint64_t some = __ballot(is);
        __syncthreads();
        if (lane == 0) counts[wave] = (uint32_t)__popcll(some);
        __syncthreads();
        uint32_t before = 0;
        all = 0;
        for (uint32_t w = 0; w < 4; w++) {
            before += w < wave ? counts[w] : 0;
            all += counts[w];
        }
        return before + (uint32_t)__popcll(some & (~0ull >> (63 - lane)));
    };
    // rows of one adapter next to each other are one start
    const int32_t id = adapter(m), before = m ? adapter(m - 1) : -1;
    const bool starts = id >= 0 && before != id;
    uint32_t all, slots;
    const uint32_t start = place(starts, all) - 1;
    if (starts) start_id[start] = id;
    __syncthreads();
    // the first start of the same adapter
    uint32_t first = kNoSlot;
    if (m < all) {
        first = 0;
        while (start_id[first] != start_id[m]) first++;
    }
    const uint32_t slot = place(first == m, slots) - 1;
    if (first == m) start_slot[m] = (uint16_t)slot;
    __syncthreads();
    if (m < all && first != m) start_slot[m] = start_slot[first];
    __syncthreads();
    if (m < a.tile && r0 + m < a.n_rows) a.slot_of[r0 + m] = id >= 0 ? start_slot[start] : (uint16_t)kNoSlot;
    if (first == m) a.slot_id[r0 + slot] = start_id[m];
    if (m == 0) a.slots[tile] = slots;
}

// A workgroup's tiles, one after the other: the next one's first steps are loaded
// while the last one's cells are written. `Work` has what is done before a tile's
// products, beside them, behind them in the stages, and with its cells.
template <bool AT, bool BT, typename Tile, typename Work>
__device__ __forceinline__ void linear_tiles(const LinearArgs &a, char *lds, uint32_t first, uint32_t groups) {
    const uint32_t all = a.p.m_tiles * a.p.n_tiles * a.p.splits;
    char *room = lds + Tile::kRoom;
    TileProduct<AT, BT, Tile> product(a.p, lds);
    Tile t;
    const uint32_t wave = uniform(threadIdx.x / kWave);
    t.wave_m = wave / Tile::kWavesN * Tile::kWaveM;
    t.wave_n = wave % Tile::kWavesN * Tile::kWaveN;
    Spot next = tile_spot<Tile>(a.p, first, all);
    product.prime(next);
    for (uint32_t index = first;;) {
        static_cast<Spot &>(t) = next;
        Work work(a, t);
        product.run(t, work.beside());
        hold(t);
        work.behind(a, lds, t);
        index += groups;
        const bool more = Tile::kSeveral && index < all;
        if (more) {
            next = tile_spot<Tile>(a.p, index, all);
            product.prime(next);
        }
        work.store(a, room, t);
        if (!more) return;
    }
}

template <typename Tile, typename E>
struct LinearY {
    Columns<Tile> bias;
    __device__ __forceinline__ LinearY(const LinearArgs &a, const Tile &t) { bias.read(t, a.bias, a.cols, 0.0f); }
    __device__ __forceinline__ NothingElse beside() { return {}; }
    __device__ __forceinline__ void behind(const LinearArgs &, char *, Tile &) {}
    __device__ __forceinline__ void store(const LinearArgs &a, char *room, Tile &t) { linear_store<Tile, E, false>(a, room, t, bias); }
};

// With adapters, whose operands take the registers that fragments had: the biases
// are read with them, behind the products, and of small tiles, of which a SIMD has
// two waves, behind theirs too. (The first step's operands read before the products
// spilled: 98 us against 83, 8,191 rows of 1,024 by 4,096.)
template <typename Tile, typename E>
struct LinearYa {
    Adapters<Tile, E> adapters;
    Columns<Tile> bias;
    __device__ __forceinline__ LinearYa(const LinearArgs &a, const Tile &t) : adapters(a, t) {}
    __device__ __forceinline__ NothingElse beside() { return {}; }
    __device__ __forceinline__ void behind(const LinearArgs &a, char *lds, Tile &t) {
        if constexpr (Tile::kI == 4) bias.read(t, a.bias, a.cols, 0.0f);
        adapters.add(a, lds, t);
        if constexpr (Tile::kI != 4) bias.read(t, a.bias, a.cols, 0.0f);
    }
    __device__ __forceinline__ void store(const LinearArgs &a, char *room, Tile &t) { linear_store<Tile, E, false>(a, room, t, bias); }
};

// A share of a projection's steps.
template <typename Tile>
struct LinearPart {
    __device__ __forceinline__ LinearPart(const LinearArgs &, const Tile &) {}
    __device__ __forceinline__ NothingElse beside() { return {}; }
    __device__ __forceinline__ void behind(const LinearArgs &, char *, Tile &) {}
    __device__ __forceinline__ void store(const LinearArgs &a, char *, Tile &t) { linear_store_part(a, t); }
};

// The sums of dout's rows, out of the fragments that the products with it read:
// of the workgroups of the same rows each takes its turn of the steps, and of
// the waves that read the same fragments each one of them. f32 parts count with
// the first part of what they meet, once each.
template <typename Tile>
struct RowSums {
    static constexpr int kOf = Tile::kJ / Tile::kWavesM;  // a wave's fragments of each sixteenth
    static_assert(Tile::kJ % Tile::kWavesM == 0, "the waves share the fragments evenly");
    uint32_t per, order, m_tiles, wave;
    uint32_t at, seg, turn;  // of the step at hand
    bool counts = false, wanted;
    float sum[kOf] = {};
    __device__ __forceinline__ RowSums(const LinearArgs &a, const Tile &t) {
        per = (a.p.k + 63) / 64;
        const uint32_t s0 = (uint32_t)((uint64_t)per * a.p.segments * t.split / a.p.splits);
        order = a.p.a_order;
        m_tiles = a.p.m_tiles;
        wave = t.wave_m / Tile::kWaveM;
        wanted = a.part_b != nullptr;
        at = s0 % per;
        seg = s0 / per;
        turn = (s0 + m_tiles - t.m0 / Tile::kM) % m_tiles;
    }
    __device__ __forceinline__ void operator()(const bf16x8 (&fb)[Tile::kJ], uint32_t kk) {
        if (kk == 0) {
            counts = wanted && turn == 0 && (order >> 2 * seg & 3u) == 0;
            if (++turn == m_tiles) turn = 0;
            if (++at == per) at = 0, seg++;
        }
        if (!counts) return;
#pragma unroll
        for (int q = 0; q < kOf; q++) {
            bf16x8 f = fb[q];
#pragma unroll
            for (int w = 1; w < Tile::kWavesM; w++) f = wave == (uint32_t)w ? fb[w * kOf + q] : f;
#pragma unroll
            for (int k = 0; k < 8; k++) sum[q] += (float)f[k];
        }
    }
};

// The gradients of the inputs and of the weights.
template <typename Tile, typename E>
struct LinearDx {
    __device__ __forceinline__ LinearDx(const LinearArgs &, const Tile &) {}
    __device__ __forceinline__ NothingElse beside() { return {}; }
    __device__ __forceinline__ void behind(const LinearArgs &, char *, Tile &) {}
    __device__ __forceinline__ void store(const LinearArgs &a, char *room, Tile &t) {
        if (a.part) linear_store_part(a, t);
        else linear_store<Tile, E, false>(a, room, t, NoColumns{});
    }
};

template <typename Tile, typename E>
struct LinearDw {
    RowSums<Tile> sums;
    __device__ __forceinline__ LinearDw(const LinearArgs &a, const Tile &t) : sums(a, t) {}
    __device__ __forceinline__ RowSums<Tile> &beside() { return sums; }
    __device__ __forceinline__ void behind(const LinearArgs &a, char *, Tile &t) {
        if (!a.part_b) return;
#pragma unroll
        for (int q = 0; q < RowSums<Tile>::kOf; q++) {
            const float sum = sums.sum[q] + __shfl_xor(sums.sum[q], 32, kWave);
            const uint32_t r = t.n0 + t.wave_n + 32 * (sums.wave * RowSums<Tile>::kOf + q) + lane_id() % 32;
            if (lane_id() < 32 && r < a.rows) a.part_b[((uint64_t)t.split * a.p.m_tiles + t.m0 / Tile::kM) * a.rows + r] = sum;
        }
    }
    __device__ __forceinline__ void store(const LinearArgs &a, char *room, Tile &t) {
        if (a.part) {
            linear_store_part(a, t);
            return;
        }
        Columns<Tile> weight;
        weight.read(t, a.weight, a.cols, 1.0f);
        linear_store<Tile, E, true>(a, room, t, weight);
    }
};

// A row's adapter in C neighbouring outputs (of `up`'s rows), sixteen ranks of
// loads at a time.
template <typename E, int C>
__device__ __forceinline__ void adapter_cells(const float *low, const typename E::type *const (&up)[C], uint32_t rank, float (&more)[C]) {
#pragma unroll
    for (int c = 0; c < C; c++) more[c] = 0.0f;
    for (uint32_t rho0 = 0; rho0 < rank; rho0 += 16) {
        float l[16], u[C][16];
#pragma unroll
        for (uint32_t k = 0; k < 16; k++) {
            const uint32_t rho = min(rho0 + k, rank - 1);
            l[k] = low[rho];
#pragma unroll
            for (int c = 0; c < C; c++) u[c][k] = E::up(up[c][rho]);
        }
#pragma unroll
        for (uint32_t k = 0; k < 16; k++)
#pragma unroll
            for (int c = 0; c < C; c++) more[c] = rho0 + k < rank ? __builtin_fmaf(l[k], u[c][k], more[c]) : more[c];
    }
}

// The shares joined: a thread takes the four columns of a row that a lane held,
// adds the shares in order and, of a projection, the row's adapter.
template <typename Tile, typename E>
__device__ __forceinline__ void linear_join(const LinearArgs &a, uint32_t block) {
    using T = typename E::type;
    constexpr uint32_t kCells = Tile::kI * Tile::kJ * 4;
    const uint64_t tiles = (uint64_t)a.p.m_tiles * a.p.n_tiles, tile = block / kCells;
    const uint32_t cell = block % kCells, g = cell % 4, j = cell / 4 % Tile::kJ, i = cell / 4 / Tile::kJ;
    Tile t;
    t.m0 = (uint32_t)(tile / a.p.n_tiles) * Tile::kM;
    t.n0 = (uint32_t)(tile % a.p.n_tiles) * Tile::kN;
    const uint32_t wave = threadIdx.x / kWave;
    t.wave_m = wave / Tile::kWavesN * Tile::kWaveM;
    t.wave_n = wave % Tile::kWavesN * Tile::kWaveN;
    const uint32_t c = column_of(t, i, g), r = t.n0 + t.wave_n + 32 * j + lane_id() % 32;
    if (r >= a.rows || c >= a.cols) return;
    float s[4] = {};
#pragma unroll 4
    for (uint32_t p = 0; p < a.p.splits; p++) {
        const Vec<float, 4> v = reinterpret_cast<const Vec<float, 4> *>(a.part)[part_at<Tile>(a.p, p * tiles + tile, cell)];
#pragma unroll
        for (int k = 0; k < 4; k++) s[k] += v.v[k];
    }
    if (a.low) {
        const int32_t id = a.ids[r];
        if (id >= 0 && (uint32_t)id < a.adapters) {
            const float *low = a.low + (uint64_t)r * a.rank;
            const T *up[4];
            float more[4];
#pragma unroll
            for (int k = 0; k < 4; k++) up[k] = static_cast<const T *>(a.up) + ((uint64_t)id * a.cols + min(c + k, a.cols - 1)) * a.up_stride;
            adapter_cells<E, 4>(low, up, a.rank, more);
#pragma unroll
            for (int k = 0; k < 4; k++) s[k] += more[k];
        }
    }
    Vec<T, 4> v;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const uint32_t column = min(c + k, a.cols - 1);
        v.v[k] = E::down((a.weight ? s[k] * a.weight[column] : s[k]) + (a.bias ? a.bias[column] : 0.0f));
    }
    T *to = static_cast<T *>(a.out) + (uint64_t)r * a.out_stride + c;
    if (c + 4 <= a.cols && a.out_stride % 4 == 0 && reinterpret_cast<uint64_t>(a.out) % (4 * sizeof(T)) == 0) {
        *reinterpret_cast<Vec<T, 4> *>(to) = v;
        return;
    }
#pragma unroll
    for (int k = 0; k < 4; k++)
        if (c + k < a.cols) to[k] = v.v[k];
}

// Columns' parts joined: 16 columns a workgroup, a thread a column and a share of the parts.
template <uint32_t Shares>
__device__ __forceinline__ void column_join(const float *part, uint32_t parts, uint32_t cols, float *dst, uint32_t block) {
    __shared__ float sum_of[Shares][16];
    const uint32_t in = threadIdx.x % 16, share = threadIdx.x / 16, c = block * 16 + in;
    float s = 0.0f;
    if (c < cols) {
#pragma unroll 8
        for (uint32_t p = share; p < parts; p += Shares) s += part[(uint64_t)p * cols + c];
    }
    sum_of[share][in] = s;
    __syncthreads();
    if (share || c >= cols) return;
    for (uint32_t w = 1; w < Shares; w++) s += sum_of[w][in];
    dst[c] = s;
}

// Either product's shares, by its tile, and db.
template <typename E>
__device__ __forceinline__ void linear_joins(const LinearPairArgs &a) {
    uint32_t block = blockIdx.x;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        if (block < a.groups[i]) {
            if (a.of[i].large) linear_join<ProductTile<256, 2, true>, E>(a.of[i], block);
            else linear_join<ProductTile<128, 2, false>, E>(a.of[i], block);
            return;
        }
        block -= a.groups[i];
    }
    column_join<16>(a.part_b, a.b_parts, a.outs, a.db, block);
}

// Operands laid out in chunks: eight columns of a row a thread, a wave eight rows
// of a chunk. The arrays' workgroups stand one behind the other.
template <uint32_t Kind>
__device__ __forceinline__ void lay(const LayArray &a, uint32_t block) {
    using E = std::conditional_t<Kind == kLayF32, F32, Bf16>;
    using T = typename E::type;
    const uint64_t cells = a.rows * a.chunks * 8;
    for (uint64_t i = (uint64_t)block * 256 + threadIdx.x; i < cells; i += (uint64_t)a.blocks * 256) {
        // two chunks of a row by neighbouring threads
        const uint64_t group = i / (a.rows * 16);
        const uint32_t wide = min(2u, a.chunks - (uint32_t)group * 2);
        const uint64_t in = i - group * a.rows * 16, r = in / (wide * 8);
        const uint32_t chunk = (uint32_t)group * 2 + (uint32_t)(in % (wide * 8)) / 8, c = chunk * 64 + in % 8 * 8;
        uint16_t *dst = a.dst + chunk * a.chunk + r * 64 + in % 8 * 8;
        Vec<uint16_t, 8> out;
        if constexpr (Kind == kLayCodes) {
            const uint8_t *src = static_cast<const uint8_t *>(a.src) + r * a.stride + c;
            Vec<uint8_t, 8> codes{};
            if (c + 8 <= a.cols) {
                __builtin_memcpy(&codes, src, 8);
            } else {
#pragma unroll
                for (int k = 0; k < 8; k++)
                    if (c + k < a.cols) codes.v[k] = src[k];
            }
            float v[8];
            values_of<8>(codes, exp2_of((int32_t)a.scales[r * a.scales_stride + min(c, a.cols - 1) / kPackBlock] - kPowerBias), v);
#pragma unroll
            for (int k = 0; k < 8; k++) out.v[k] = (uint16_t)(__float_as_uint(v[k]) >> 16);
            *reinterpret_cast<Vec<uint16_t, 8> *>(dst) = out;
        } else {
            const T *src = static_cast<const T *>(a.src) + r * a.stride + c;
            Vec<T, 8> v{};
            if (c + 8 <= a.cols) {
                __builtin_memcpy(&v, src, sizeof v);
            } else {
#pragma unroll
                for (int k = 0; k < 8; k++)
                    if (c + k < a.cols) v.v[k] = src[k];
            }
            if constexpr (Kind == kLayBf16) {
#pragma unroll
                for (int k = 0; k < 8; k++) out.v[k] = v.v[k];
                *reinterpret_cast<Vec<uint16_t, 8> *>(dst) = out;
            } else {
                Vec<uint16_t, 8> parts[3];
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    uint16_t p[3];
                    split3(v.v[k], p);
#pragma unroll
                    for (int q = 0; q < 3; q++) parts[q].v[k] = p[q];
                }
#pragma unroll
                for (int q = 0; q < 3; q++) *reinterpret_cast<Vec<uint16_t, 8> *>(dst + q * a.part) = parts[q];
            }
        }
    }
}

__device__ __forceinline__ void lay_all(const LayArgs &a, uint32_t block) {
    // (by constant places: an argument read at a variable one goes through memory)
    LayArray of = a.of[0];
    if (block >= of.blocks) {
        block -= of.blocks;
        of = a.of[1];
        if (block >= of.blocks) {
            block -= of.blocks;
            of = a.of[2];
        }
    }
    if (of.kind == kLayF32) lay<kLayF32>(of, block);
    else if (of.kind == kLayBf16) lay<kLayBf16>(of, block);
    else lay<kLayCodes>(of, block);
}

// ---- sixteen rows against sixteen, without LDS ------------------------------------------------

typedef float f32x4 __attribute__((ext_vector_type(4)));

// A lane's 16 bytes of its row (lane % 16) for a step of 4 x 16 bytes of products:
// those from its quarter on, zeros past the row's end. Wide: rows of whole 16 bytes,
// on 16 bytes; else element by element. Every load is made, from within the row
// whatever the place, so that no branch stands between the loads.
template <typename E, bool Wide>
struct Strip {
    using T = typename E::type;
    static constexpr uint32_t kV = 16 / sizeof(T), kStep = 4 * kV;  // products a lane and step, products a step
    static __device__ __forceinline__ Vec<T, kV> load(const T *row, uint32_t c, uint32_t dim) {
        Vec<T, kV> v;
        if constexpr (Wide) {
            v = *reinterpret_cast<const Vec<T, kV> *>(row + min(c, dim - kV));
        } else {
#pragma unroll
            for (uint32_t k = 0; k < kV; k++) v.v[k] = row[min(c + k, dim - 1)];
        }
#pragma unroll
        for (uint32_t k = 0; k < kV; k++) v.v[k] = c + (Wide ? 0 : k) < dim ? v.v[k] : (T)0;
        return v;
    }
    // acc: row 4 (lane / 16) + e of a, row lane % 16 of b
    static __device__ __forceinline__ void multiply(const Vec<T, kV> &a, const Vec<T, kV> &b, f32x4 &acc) {
        if constexpr (sizeof(T) == 2) {
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
        } else {
#pragma unroll
            for (uint32_t k = 0; k < kV; k++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[k], b.v[k], acc, 0, 0, 0);
        }
    }
};

// The rows' low values: a workgroup takes 16 rows and all ranks of their
// adapters, each adapter once, 32 of those rows of `down` at a time; its waves
// share the steps (16 of them where few workgroups have the CUs to themselves).
// A cell counts where the row's adapter is the column's.
template <typename E, bool Wide, uint32_t kWaves>
__device__ __forceinline__ void linear_low(const LinearLowArgs &a) {
    using T = typename E::type;
    using S = Strip<E, Wide>;
    constexpr uint32_t kRows = 16, kCols = 2, kAhead = kWaves == 4 ? sizeof(T) == 2 && Wide ? 8 : 4 : 2;
    __shared__ int32_t slot_id[kRows], slot_of[kRows];
    __shared__ f32x4 part[kWaves][kCols][kWave];
    if (blockIdx.x >= a.groups * a.shares) {
        const uint32_t block = blockIdx.x - a.groups * a.shares;
        if constexpr (kWaves == 4) {
            if (block < a.tiles) tile_slots(a, block);
            else lay_all(a.lay, block - a.tiles);
        }
        return;
    }
    const uint32_t share = blockIdx.x / a.groups;
    const uint32_t lane = lane_id(), wave = threadIdx.x / kWave, in = lane % 16, quarter = lane / 16;
    const uint64_t r0 = (uint64_t)(blockIdx.x % a.groups) * kRows;
    const T *x = static_cast<const T *>(a.x) + min(r0 + in, (uint64_t)a.n_rows - 1) * a.x_stride;
    int32_t id = r0 + in < a.n_rows ? a.ids[r0 + in] : -1;
    Vec<T, S::kV> fx[kAhead];  // of the rows' first steps, which wait for no id
    auto read_x = [&](uint32_t c0) {
#pragma unroll
        for (uint32_t k = 0; k < kAhead; k++) fx[k] = S::load(x, c0 + k * S::kStep + quarter * S::kV, a.dim);
    };
    read_x(wave * kAhead * S::kStep);
    // every wave finds the slots: the rows' adapters in order of their first rows
    if (id < 0 || (uint32_t)id >= a.adapters) id = -1;
    uint32_t first = in;
#pragma unroll
    for (int o = kRows - 1; o >= 0; o--)
        if (__builtin_amdgcn_readlane(id, o) == id) first = min(first, (uint32_t)o);
    const uint64_t firsts = __ballot(lane < kRows && id >= 0 && first == in);
    const uint32_t slots = (uint32_t)__popcll(firsts), slot = (uint32_t)__popcll(firsts & ((1ull << first) - 1));
    if (wave == 0 && lane < kRows) {
        slot_of[lane] = id >= 0 ? (int32_t)slot : -1;
        if (id >= 0 && first == lane) slot_id[slot] = id;
    }
    __syncthreads();
    const uint32_t all = slots * a.rank;
    bool fresh = true;  // fx holds the wave's first steps
    for (uint32_t v0 = share * kCols * 16; v0 < all; v0 += a.shares * kCols * 16) {
        const T *down[kCols];
#pragma unroll
        for (uint32_t q = 0; q < kCols; q++) {
            const uint32_t v = min(v0 + q * 16 + in, all - 1), s = v / a.rank;
            down[q] = static_cast<const T *>(a.down) + ((uint64_t)slot_id[s] * a.rank + (v - s * a.rank)) * a.down_stride;
        }
        f32x4 acc[kCols] = {};
        for (uint32_t c0 = wave * kAhead * S::kStep; c0 < a.dim; c0 += kWaves * kAhead * S::kStep) {
            Vec<T, S::kV> fd[kAhead][kCols];
            if (!fresh) read_x(c0);
            fresh = false;
#pragma unroll
            for (uint32_t k = 0; k < kAhead; k++) {
                const uint32_t c = c0 + k * S::kStep + quarter * S::kV;
#pragma unroll
                for (uint32_t q = 0; q < kCols; q++) fd[k][q] = S::load(down[q], c, a.dim);
            }
#pragma unroll
            for (uint32_t k = 0; k < kAhead; k++)
#pragma unroll
                for (uint32_t q = 0; q < kCols; q++) S::multiply(fx[k], fd[k][q], acc[q]);
        }
#pragma unroll
        for (uint32_t q = 0; q < kCols; q++) part[wave][q][lane] = acc[q];
        __syncthreads();
        if (wave < kCols) {
            f32x4 s = part[0][wave][lane];
            for (uint32_t w = 1; w < kWaves; w++) s += part[w][wave][lane];
            const uint32_t v = v0 + wave * 16 + in, of = v / a.rank;
            if (v < all) {
                const float by = a.scale ? a.scale[slot_id[of]] : 1.0f;
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) {
                    const uint32_t row = quarter * 4 + e;
                    if (slot_of[row] == (int32_t)of) a.low[(r0 + row) * a.rank + (v - of * a.rank)] = s[e] * by;
                }
            }
        }
        __syncthreads();
    }
}

// Few rows: a workgroup takes 16 outputs and all rows, 16 R of them; w is read
// once, straight into the operands' registers, the four waves sharing the steps.
// Then a thread a cell joins the waves' sums and adds the bias and the adapter.
template <typename E, int R, bool Wide>
__device__ __forceinline__ void linear_few(const LinearFewArgs &a) {
    using T = typename E::type;
    using S = Strip<E, Wide>;
    constexpr uint32_t kWaves = 4, kAhead = R == 4 ? 4 : 8;
    __shared__ f32x4 part[kWaves][R][kWave];
    const uint32_t lane = lane_id(), wave = threadIdx.x / kWave, in = lane % 16, quarter = lane / 16;
    const uint32_t o0 = blockIdx.x * 16;
    const T *w = static_cast<const T *>(a.w) + (uint64_t)min(o0 + in, a.outs - 1) * a.w_stride;
    f32x4 acc[R] = {};
    for (uint32_t c0 = wave * kAhead * S::kStep; c0 < a.dim; c0 += kWaves * kAhead * S::kStep) {
        Vec<T, S::kV> fw[kAhead], fx[kAhead][R];
#pragma unroll
        for (uint32_t k = 0; k < kAhead; k++) {
            const uint32_t c = c0 + k * S::kStep + quarter * S::kV;
            fw[k] = S::load(w, c, a.dim);
        }
#pragma unroll
        for (uint32_t k = 0; k < kAhead; k++) {
            const uint32_t c = c0 + k * S::kStep + quarter * S::kV;
#pragma unroll
            for (uint32_t q = 0; q < (uint32_t)R; q++) {
                // (a row past the last is the last again, and its cells are not written)
                const uint32_t r = min(q * 16 + in, a.n_rows - 1);
                fx[k][q] = S::load(static_cast<const T *>(a.x) + (uint64_t)r * a.x_stride, c, a.dim);
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < kAhead; k++)
#pragma unroll
            for (uint32_t q = 0; q < (uint32_t)R; q++) S::multiply(fw[k], fx[k][q], acc[q]);
    }
#pragma unroll
    for (uint32_t q = 0; q < (uint32_t)R; q++) part[wave][q][lane] = acc[q];
    __syncthreads();
    // cell (output o0 + t % 16, row q 16 + t / 16)
    const uint32_t o = threadIdx.x % 16, row = threadIdx.x / 16;
    if (o0 + o >= a.outs) return;
    const float bias = a.bias ? a.bias[o0 + o] : 0.0f;
#pragma unroll
    for (uint32_t q = 0; q < (uint32_t)R; q++) {
        const uint32_t r = q * 16 + row;
        if (r >= a.n_rows) return;
        const uint32_t at = row + o / 4 * 16;
        float s = part[0][q][at][o % 4];
        for (uint32_t v = 1; v < kWaves; v++) s += part[v][q][at][o % 4];
        if (a.low) {
            const int32_t id = a.ids[r];
            if (id >= 0 && (uint32_t)id < a.adapters) {
                const T *const up[1] = {static_cast<const T *>(a.up) + ((uint64_t)id * a.outs + o0 + o) * a.up_stride};
                float more[1];
                adapter_cells<E, 1>(a.low + (uint64_t)r * a.rank, up, a.rank, more);
                s += more[0];
            }
        }
        static_cast<T *>(a.out)[(uint64_t)r * a.out_stride + o0 + o] = E::down(s + bias);
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

// waves: a SIMD's, at least
#define HBR_LINEAR(name, Tile, waves, AT, BT, ...)                                           \
    extern "C" __global__ __launch_bounds__(Tile::kThreads, waves) void name(LinearArgs a) { \
        __shared__ __align__(1024) char lds[Tile::kLds];                                  \
        linear_tiles<AT, BT, Tile, __VA_ARGS__>(a, lds, blockIdx.x, gridDim.x);              \
    }
#define HBR_LINEARS(suffix, Tile, waves)                                                             \
    HBR_LINEAR(hbr_linear_y_f32_##suffix, Tile, waves, false, false, LinearY<Tile, F32>)             \
    HBR_LINEAR(hbr_linear_y_bf16_##suffix, Tile, waves, false, false, LinearY<Tile, Bf16>)           \
    HBR_LINEAR(hbr_linear_ya_f32_##suffix, Tile, waves, false, false, LinearYa<Tile, F32>)           \
    HBR_LINEAR(hbr_linear_ya_bf16_##suffix, Tile, waves, false, false, LinearYa<Tile, Bf16>)         \
    HBR_LINEAR(hbr_linear_y_part_##suffix, Tile, waves, false, false, LinearPart<Tile>)              \
    HBR_LINEAR(hbr_linear_dx_f32_##suffix, Tile, waves, true, false, LinearDx<Tile, F32>)            \
    HBR_LINEAR(hbr_linear_dx_bf16_##suffix, Tile, waves, true, false, LinearDx<Tile, Bf16>)          \
    HBR_LINEAR(hbr_linear_dw_f32_##suffix, Tile, waves, true, true, LinearDw<Tile, F32>)             \
    HBR_LINEAR(hbr_linear_dw_bf16_##suffix, Tile, waves, true, true, LinearDw<Tile, Bf16>)
using Tile256 = ProductTile<256, 2, true>;
using Tile128 = ProductTile<128, 2, false>;
using Tile128Deep = ProductTile<128, 4, false>;
HBR_LINEARS(256, Tile256, 1)
HBR_LINEARS(128, Tile128, 2)
HBR_LINEARS(128_deep, Tile128Deep, 1)

#define HBR_PAIR(t, E)                                                                                                \
    extern "C" __global__ __launch_bounds__(256, 2) void hbr_linear_pair_##t(LinearPairArgs a) {                      \
        __shared__ __align__(1024) char lds[Tile128::kLds];                                                           \
        if (blockIdx.x < a.groups[0]) linear_tiles<true, false, Tile128, LinearDx<Tile128, E>>(a.of[0], lds, blockIdx.x, 1); \
        else linear_tiles<true, true, Tile128, LinearDw<Tile128, E>>(a.of[1], lds, blockIdx.x - a.groups[0], 1);      \
    }                                                                                                                 \
    extern "C" __global__ __launch_bounds__(256) void hbr_linear_joins_##t(LinearPairArgs a) { linear_joins<E>(a); }
HBR_PAIR(f32, F32)
HBR_PAIR(bf16, Bf16)

#define HBR_STRIPS(t, E, v, Wide)                                                                                                   \
    extern "C" __global__ __launch_bounds__(256) void hbr_linear_low_##t##_##v(LinearLowArgs a) { linear_low<E, Wide, 4>(a); }      \
    extern "C" __global__ __launch_bounds__(1024) void hbr_linear_low_##t##_##v##_16(LinearLowArgs a) { linear_low<E, Wide, 16>(a); } \
    extern "C" __global__ __launch_bounds__(256) void hbr_linear_few_##t##_##v##_16(LinearFewArgs a) { linear_few<E, 1, Wide>(a); } \
    extern "C" __global__ __launch_bounds__(256) void hbr_linear_few_##t##_##v##_32(LinearFewArgs a) { linear_few<E, 2, Wide>(a); } \
    extern "C" __global__ __launch_bounds__(256) void hbr_linear_few_##t##_##v##_64(LinearFewArgs a) { linear_few<E, 4, Wide>(a); }
HBR_STRIPS(f32, F32, 1, false)
HBR_STRIPS(f32, F32, 4, true)
HBR_STRIPS(bf16, Bf16, 1, false)
HBR_STRIPS(bf16, Bf16, 8, true)
extern "C" __global__ __launch_bounds__(256) void hbr_lay(LayArgs a) { lay_all(a, blockIdx.x); }
extern "C" __global__ __launch_bounds__(1024) void hbr_column_join(ColumnJoinArgs a) { column_join<64>(a.part, a.parts, a.cols, a.dst, blockIdx.x); }
extern "C" __global__ __launch_bounds__(256) void hbr_column_sum_f32(ColumnSumArgs a) { column_sum<F32>(a); }
extern "C" __global__ __launch_bounds__(256) void hbr_column_sum_bf16(ColumnSumArgs a) { column_sum<Bf16>(a); }
