// Products on the matrix cores, C(m, n) = sum over k of A(m, k) B(n, k): tiles
// of bf16 operands (f32 ones in three bf16 parts) fed through LDS.
#pragma once
#include "elements.h"

namespace hbr {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
#define HBR_LDS __attribute__((address_space(3)))

constexpr uint32_t kNowhere = 0x80000000u;  // past every buffer: reads as zero

__device__ __forceinline__ int32_t uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane((int32_t)v); }

__device__ __forceinline__ uint16_t to_bf16(float v) {
    const __bf16 b = (__bf16)v;
    return __builtin_bit_cast(uint16_t, b);
}

// An f32 as the sum of three bf16 values, exactly: each takes the next eight
// bits of what is left. One that rounds to infinity is cut off instead. An
// infinity is its sign's 1, 0 and infinity: of the six products with another
// value's parts the last part meets only the first, which has the value's sign
// and is zero only with it, so that their sum is what infinity times the value
// is. (As the first part it would meet zeros, and be no number.)
__device__ __forceinline__ void split3(float v, uint16_t (&p)[3]) {
    p[0] = to_bf16(v);
    if ((p[0] & 0x7f80u) == 0x7f80u) {
        if ((__float_as_uint(v) & 0x7f800000u) == 0x7f800000u) {
            const bool none = (p[0] & 0x7fu) != 0;
            p[2] = none ? 0 : p[0];
            if (!none) p[0] = (p[0] & 0x8000u) | 0x3f80u;
            p[1] = 0;
            return;
        }
        p[0] = (uint16_t)(__float_as_uint(v) >> 16);
    }
    const float rest = v - bf16_f32(p[0]);
    p[1] = to_bf16(rest);
    p[2] = to_bf16(rest - bf16_f32(p[1]));
}

// ---- one operand's tile in LDS ---------------------------------------------------------
//
// An operand lies in chunks of 32 columns: rows row_step bytes apart, chunks
// chunk_step. What the products read often is laid out so (a chunk's rows of
// 64 bytes one behind the other), and 16 rows of a chunk are the 1 KiB that
// one load of a wave fills; plain rows are the same with other steps.
//
// A tile is 32 W rows x kHeadK (W waves), or, transposed, kHeadK rows x 32 W
// in W chunks, filled by 16-byte loads that go to LDS without registers. A wave's
// load fills LDS in lane order, so the layout is that of the loads. Of a tile
// read along its rows the 16-byte pieces of a row are exchanged by their
// source addresses: a piece's place is xored with its row's bits, so that the
// 16 lanes that LDS serves at once meet all 64 banks. The transposing reads
// meet them anyway (four rows of 64 bytes).
template <bool T, int W>
struct Operand {
    static constexpr int kBytes = 32 * W * kHeadK * 2;
    static constexpr int kLoads = kBytes / 1024 / W;  // a wave's, a step
    uint64_t at, step;      // where the wave's next step begins, and from step to step
    uint32_t off[kLoads];   // a lane's source, bytes from there
    uint32_t k_at[kLoads];  // and its first k within the step (not transposed)

    // first: the tile's first row (m or n); size: how many there are (to the
    // end of the last chunk, transposed)
    __device__ __forceinline__ void init(uint64_t row_step, uint64_t chunk_step, uint32_t first, uint32_t size, const int32_t *labels) {
        const uint32_t lane = lane_id(), wave = threadIdx.x / kWave;
        step = T ? kHeadK * row_step : chunk_step;
#pragma unroll
        for (int j = 0; j < kLoads; j++) {
            if (T) {  // a wave loads a chunk
                const uint32_t row = j * 16 + lane / 4, col = wave * 32 + lane % 4 * 8;
                off[j] = first + col < size ? (uint32_t)(row * row_step) + lane % 4 * 16 : kNowhere;
            } else {
                const uint32_t row = (wave * kLoads + j) * 16 + lane / 4, piece = lane % 4 ^ ((row >> 2) & 3u);
                const bool in = first + row < size && (!labels || labels[first + row] >= 0);
                off[j] = in ? (uint32_t)(row * row_step) + piece * 16 : kNowhere;
                k_at[j] = piece * 8;
            }
        }
        static_assert(kLoads == 2, "a wave loads a chunk's 32 rows");
    }
    // To step s of the operand at p.
    __device__ __forceinline__ void seek(const void *p, uint64_t row_step, uint64_t chunk_step, uint32_t first, uint32_t s) {
        const uint32_t wave = uniform(threadIdx.x / kWave);
        at = reinterpret_cast<uint64_t>(p) + (T ? (first / 32 + wave) * chunk_step : first * row_step) + s * step;
    }
    // The next step, of which `left` k are left (0: nothing is read). The
    // loads are not the compiler's: it would wait for them before any read of
    // LDS, and the pipeline's own waits know which stage they fill.
    // Transposed, the buffer ends with the last k; else what lies past it is
    // zeros, or `check`ed.
    __device__ __forceinline__ void load(uint32_t lds, uint32_t left, uint64_t row_step, bool check) {
        const uint32_t to = uniform(lds + threadIdx.x / kWave * (kLoads * 1024));
        const uint32_t size = T ? (left >= kHeadK ? 0x7fffffffu : left * (uint32_t)row_step) : left ? 0x7fffffffu : 0u;
        const i32x4 r = {uniform((uint32_t)at), uniform((uint32_t)(at >> 32)) & 0xffff, uniform(size), 0x00020000};
        uint32_t from[kLoads];
#pragma unroll
        for (int j = 0; j < kLoads; j++) from[j] = off[j];
        if (!T && check && left < kHeadK) {
#pragma unroll
            for (int j = 0; j < kLoads; j++)
                if (k_at[j] >= left) from[j] = kNowhere;
        }
#pragma unroll
        for (int j = 0; j < kLoads; j++)
            // (m0 is the compiler's to set before each use of its own, and nothing
            // here keeps a value in it)
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                         :
                         : "s"(to + j * 1024), "v"(from[j]), "s"(r)
                         : "memory");
        at += step;
    }
    // Rows [row, row + 32) and products [16 kk, 16 kk + 16) of the tile: a
    // lane's row is lane % 32, its products the eight from 8 (lane / 32) on.
    static __device__ __forceinline__ bf16x8 fragment(const char *lds, uint32_t row, uint32_t kk) {
        const uint32_t lane = lane_id();
        if (T) {
            // two transposing reads of four products: sixteen lanes read four
            // rows of the tile, four elements each, and get a column each
            const uint32_t k = kk * 16 + lane / 32 * 8 + lane % 16 / 4;
            const char *p = lds + row / 32 * 2048 + k * 64 + lane / 16 % 2 * 32 + lane % 4 * 8;
            union {
                s16x4 h[2];
                bf16x8 v;
            } u;
            u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((HBR_LDS s16x4 *)p);
            u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((HBR_LDS s16x4 *)(p + 4 * 64));
            return u.v;
        }
        const uint32_t m = row + lane % 32, piece = (kk * 2 + lane / 32) ^ ((m >> 2) & 3u);
        return *reinterpret_cast<const bf16x8 *>(lds + m * (kHeadK * 2) + piece * 16);
    }
};

// A workgroup's tile of the product: 32 W x 32 W of W waves, 2 x W / 2, the
// operands of two steps in LDS.
template <int W>
struct HeadTile {
    static constexpr int kW = W, kM = 32 * W, kN = 32 * W, kWavesM = 2, kWavesN = W / 2, kThreads = W * kWave;
    static constexpr int kWaveM = kM / kWavesM, kWaveN = kN / kWavesN, kI = kWaveM / 32, kJ = kWaveN / 32;
    static constexpr int kStage = (kM + kN) * kHeadK * 2, kLds = 2 * kStage;
    uint32_t m0, n0, split;  // the tile's first row and column, and its share of the steps
    // element e of acc[i][j]: row wave_m + 32 i + row_of(e), column wave_n + 32 j + lane % 32
    f32x16 acc[kI][kJ];
    uint32_t wave_m, wave_n;
};

__device__ __forceinline__ uint32_t row_of(int e) { return 8 * (e / 4) + 4 * (lane_id() / 32) + e % 4; }

// A workgroup's tile: neighbours in the launch go to different XCDs, so each
// XCD takes a contiguous share of the tiles, in groups of eight rows of tiles
// whose operands its L2 holds.
template <typename Tile>
__device__ __forceinline__ void head_place(const HeadArgs &a, Tile &t) {
    const uint32_t all = gridDim.x, per = all / 8, rest = all % 8, xcd = blockIdx.x % 8;
    uint32_t id = xcd * per + min(xcd, rest) + blockIdx.x / 8;
    const uint32_t tiles = a.m_tiles * a.n_tiles;
    t.split = id / tiles;
    id -= t.split * tiles;
    constexpr uint32_t kGroup = 8;
    const uint32_t group = id / (kGroup * a.n_tiles), first = group * kGroup;
    const uint32_t rows = min(kGroup, a.m_tiles - first), in = id - group * kGroup * a.n_tiles;
    t.m0 = (first + in % rows) * Tile::kM;
    t.n0 = in / rows * Tile::kN;
    const uint32_t wave = threadIdx.x / kWave;
    t.wave_m = wave / Tile::kWavesN * Tile::kWaveM;
    t.wave_n = wave % Tile::kWavesN * Tile::kWaveN;
}

// The tile's products. A step's fragments are read one sixteenth of products
// ahead of the matrix instructions that use them, across the steps too: the
// last sixteenth's are in registers when the waves meet, so that the next
// step's loads may overwrite its stage and its first fragments be read
// behind the meeting, both under the last sixteenth's products.
template <bool AT, bool BT, typename Tile>
__device__ __forceinline__ void head_product(const HeadArgs &a, char *lds, Tile &t, const int32_t *a_labels = nullptr) {
    using A = Operand<AT, Tile::kW>;
    using B = Operand<BT, Tile::kW>;
    constexpr int kI = Tile::kI, kJ = Tile::kJ, kSixteenths = kHeadK / 16;
    A oa;
    B ob;
    oa.init(a.a_row, a.a_chunk, t.m0, a.m, a_labels);
    ob.init(a.b_row, a.b_chunk, t.n0, a.n, nullptr);
#pragma unroll
    for (int i = 0; i < kI; i++)
#pragma unroll
        for (int j = 0; j < kJ; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) t.acc[i][j][e] = 0.0f;
    const uint32_t per = (a.k + kHeadK - 1) / kHeadK, steps = per * a.segments;
    const uint32_t s0 = (uint32_t)((uint64_t)steps * t.split / a.splits),
                   s1 = (uint32_t)((uint64_t)steps * (t.split + 1) / a.splits);
    uint32_t seg = s0 / per, at = s0 % per;
    auto seek = [&] {
        // (past the last segment its loads read nothing)
        oa.seek(static_cast<const char *>(a.a) + (a.a_order >> 2 * seg & 3u) * a.a_part, a.a_row, a.a_chunk, t.m0, at);
        ob.seek(static_cast<const char *>(a.b) + (a.b_order >> 2 * seg & 3u) * a.b_part, a.b_row, a.b_chunk, t.n0, at);
    };
    seek();
    // past the last step the loads read nothing
    auto load = [&](uint32_t s) {
        const uint32_t left = s < s1 ? a.k - at * kHeadK : 0;
        const uint32_t to = (uint32_t)(uintptr_t)(HBR_LDS char *)lds + s % 2 * Tile::kStage;
        oa.load(to, left, a.a_row, a.check != 0);
        ob.load(to + A::kBytes, left, a.b_row, a.check != 0);
        if (++at == per) {
            at = 0, seg++;
            seek();
        }
    };
    bf16x8 fa[2][kI], fb[2][kJ];
    auto read = [&](int set, uint32_t s, uint32_t kk) {
        const char *from = lds + s % 2 * Tile::kStage;
#pragma unroll
        for (int i = 0; i < kI; i++) fa[set][i] = A::fragment(from, t.wave_m + 32 * i, kk);
#pragma unroll
        for (int j = 0; j < kJ; j++) fb[set][j] = B::fragment(from + A::kBytes, t.wave_n + 32 * j, kk);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto multiply = [&](int set) {
        __builtin_amdgcn_s_setprio(1);  // before the other waves' reads and addresses
#pragma unroll
        for (int i = 0; i < kI; i++)
#pragma unroll
            for (int j = 0; j < kJ; j++)
                t.acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[set][i], fb[set][j], t.acc[i][j], 0, 0, 0);
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto meet = [&] {  // the wave's loads have landed and its reads are in registers; so have all others'
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    load(s0);
    meet();
    load(s0 + 1);
    read(0, s0, 0);
    for (uint32_t s = s0; s < s1; s++) {
#pragma unroll
        for (int kk = 0; kk + 1 < kSixteenths; kk++) {
            read((kk + 1) & 1, s, kk + 1);
            multiply(kk & 1);
        }
        meet();
        load(s + 2);
        read(kSixteenths & 1, s + 1, 0);
        multiply((kSixteenths - 1) & 1);
    }
    meet();  // the loads ahead have landed before the LDS or the workgroup ends
}

}  // namespace hbr
