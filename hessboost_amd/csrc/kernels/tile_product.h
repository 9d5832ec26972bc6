// A projection's products on the matrix cores, C(m, n) = sum over k of A(m, k)
// B(n, k): tiles of 256 x 256 or 128 x 128 of bf16 operands (f32 ones in three
// bf16 parts), 64 products a step, on four waves.
//
// What the matrix instructions wait for is LDS and the L2, so both are asked for
// as little as can be: a wave's tile is half the workgroup's each way (128 x 128:
// a fragment serves four instructions, and the waves read 32 KiB of LDS a
// sixteenth where eight waves of 128 x 64 read 48), and a row's 64 products are
// one line of 128 bytes (with 32 the L2 answered twice as many requests). One wave
// a SIMD has no other to fill its gaps: whatever feeds the matrix instructions
// is put between them. The matrix cores are busy 63 to 68% of a large product's
// cycles, and power holds their clock: matrix instructions alone, nothing loaded,
// take 76% of the time (8,192 x 4,096 x 4,096: 214 us of 281).
#pragma once
#include "product.h"

namespace hbr {

// An operand's tile: Rows rows of 64 products, or, transposed, 64 rows of Rows
// columns, in chunks of 64. In memory an operand lies in chunks of 64 columns, rows
// row_step bytes apart and chunks chunk_step; plain rows are the same with other
// steps. A wave's load of 1 KiB goes to LDS without registers and fills eight
// rows of 128 bytes in lane order; their pieces are exchanged by the loads'
// source addresses, so that the lanes that LDS serves at once meet all banks:
// read along the rows a piece of 16 bytes by three bits of its row (16 rows meet
// all banks), read across them a piece of 64 by one bit (four rows do).
template <bool T, int Rows>
struct TileOperand {
    static constexpr int kWaves = 4, kBytes = Rows * 128, kLoads = kBytes / 1024 / kWaves;  // a wave's, a step
    static constexpr int kSharers = kWaves / (Rows / 64) > 0 ? kWaves / (Rows / 64) : 1;    // waves of a chunk (transposed)
    static_assert(Rows == 128 || Rows == 256, "a wave loads whole shares of chunks");
    uint64_t at, step;  // where the wave's next step begins, and from step to step
    uint32_t off[2];    // a lane's source, bytes from there, of even loads and of odd ones
    uint32_t k_at;      // and an even load's first k within the step (not transposed; an odd one's is 32 from it)
    uint32_t rows;      // of the wave's that there are (not transposed)
    uint32_t row_step;

    // first: the tile's first row (m or n); size: how many there are
    __device__ __forceinline__ void init(uint64_t row_bytes, uint64_t chunk_step, uint32_t first, uint32_t size) {
        const uint32_t lane = lane_id(), wave = uniform(threadIdx.x / kWave);
        row_step = (uint32_t)row_bytes;
        step = T ? 64 * row_bytes : chunk_step;
        if (T) {
            const uint32_t piece = lane % 8 ^ lane / 16 % 2 * 4, col = wave / kSharers * 64 + piece * 8;
            off[0] = off[1] = first + col < size ? lane / 8 * row_step + piece * 16 : kNowhere;
        } else {
            const uint32_t piece = lane % 8 ^ lane / 16, from = first + wave * (Rows / kWaves);
            off[0] = lane / 8 * row_step + piece * 16;
            off[1] = lane / 8 * row_step + (piece ^ 4) * 16;
            k_at = piece * 8;
            rows = size > from ? min(size - from, (uint32_t)(Rows / kWaves)) : 0;
        }
    }
    // To step s of the operand at p.
    __device__ __forceinline__ void seek(const void *p, uint64_t chunk_step, uint32_t first, uint32_t s) {
        const uint32_t wave = uniform(threadIdx.x / kWave);
        at = reinterpret_cast<uint64_t>(p) + s * step;
        if (T) at += (first / 64 + wave / kSharers) * chunk_step + wave % kSharers * (64 / kSharers) * row_step;
        else at += (uint64_t)(first + wave * (Rows / kWaves)) * row_step;
    }
    // Load j of the step, of which `left` k are left (0: nothing is read). The
    // loads are not the compiler's: it would wait for them before any read of
    // LDS, and the pipeline's own waits know which stage they fill. The buffer
    // ends with the last row's last k of the step; what lies past a row's last
    // within it reads as zeros.
    __device__ __forceinline__ i32x4 buffer(uint32_t left) const {
        uint32_t size;
        if (T) {
            const uint32_t k0 = uniform(threadIdx.x / kWave) % kSharers * (64 / kSharers);
            size = (left > k0 ? min(left - k0, 64u) : 0) * row_step;
        } else {
            size = rows && left ? (rows - 1) * row_step + min((left * 2 + 15) / 16 * 16, 128u) : 0;
        }
        return {uniform((uint32_t)at), uniform((uint32_t)(at >> 32)) & 0xffff, uniform(size), 0x00020000};
    }
    __device__ __forceinline__ void sources(uint32_t left, uint32_t (&from)[2]) const {
        from[0] = !T && left < 64 && k_at >= left ? kNowhere : off[0];
        from[1] = !T && left < 64 && (k_at ^ 32) >= left ? kNowhere : off[1];
    }
    static __device__ __forceinline__ uint32_t destination(uint32_t lds) { return lds + uniform(threadIdx.x / kWave) * (kLoads * 1024); }
    __device__ __forceinline__ void load(int j, const i32x4 &from, const uint32_t (&source)[2], uint32_t to) const {
        // (m0 is the compiler's to set before each use of its own, and nothing
        // here keeps a value in it)
        // (the rows' distance is added to the lanes' offsets: a buffer's end is
        // not checked against a scalar one)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                     :
                     : "s"(uniform(to + j * 1024)), "v"(source[j % 2] + j * 8 * row_step), "s"(from)
                     : "memory");
    }

    // A lane's places of the fragments in a stage: rows [row, row + 32) of the
    // tile, 16 kk to 16 kk + 15 of the step; its row is lane % 32, its products the
    // eight from 8 (lane / 32) on.
    struct Places {
        uint32_t of[4];  // by kk; transposed: the two reads of either half of a chunk
        __device__ __forceinline__ void init(uint32_t lds, uint32_t row) {
            const uint32_t lane = lane_id();
            if (T) {
                // two transposing reads of four products: sixteen lanes read four
                // rows of the tile, four elements each, and get a column each
#pragma unroll
                for (int h = 0; h < 4; h++) {
                    const uint32_t k = lane / 32 * 8 + lane % 16 / 4 + h % 2 * 4, half = (h / 2) ^ (k / 2 % 2);
                    of[h] = lds + row / 64 * 8192 + k * 128 + half * 64 + lane / 16 % 2 * 32 + lane % 4 * 8;
                }
            } else {
#pragma unroll
                for (int kk = 0; kk < 4; kk++)
                    of[kk] = lds + (row + lane % 32) * 128 + ((kk * 2 + lane / 32) ^ lane / 2 % 8) * 16;
            }
        }
        // to the other of two stages `stage` bytes apart, or one on
        __device__ __forceinline__ void move(uint32_t by) {
#pragma unroll
            for (int q = 0; q < 4; q++) of[q] += by;
        }
        // the fragment of rows 32 i on
        __device__ __forceinline__ bf16x8 read(int i, int kk) const {
            if (T) {
                union {
                    s16x4 h[2];
                    bf16x8 v;
                } u;
#pragma unroll
                for (int h = 0; h < 2; h++)
                    u.h[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (HBR_LDS s16x4 *)(of[i % 2 * 2 + h] + i / 2 * 8192 + kk * 2048));
                return u.v;
            }
            return *(HBR_LDS const bf16x8 *)(of[kk] + i * 4096);
        }
    };
};

// Where a tile lies, and its share of the steps.
struct Spot {
    uint32_t m0, n0, split;
};

// A workgroup's tile: kM x kN on 2 x 2 waves, in LDS the operands of Stages steps,
// and of A of one more. Several: a workgroup takes one tile after the other, and
// the room in which its cells are written is A's last stage, which the next one's
// first steps do not take.
template <int Size, int Stages, bool Several>
struct ProductTile : Spot {
    static constexpr bool kSeveral = Several;
    static constexpr int kWaves = 4, kM = Size, kN = Size, kWavesM = 2, kWavesN = 2, kThreads = kWaves * kWave;
    static constexpr int kWaveM = kM / kWavesM, kWaveN = kN / kWavesN, kI = kWaveM / 32, kJ = kWaveN / 32;
    static constexpr int kStages = Stages, kBytes = Size * 128;  // of an operand's step
    static constexpr int kB = (Stages + 1) * kBytes, kLds = kB + Stages * kBytes;  // B's stages stand behind A's
    static constexpr int kRoom = Several ? Stages * kBytes : 0;
    // element e of acc[i][j]: row wave_m + 32 i + row_of(e), column wave_n + 32 j + lane % 32
    f32x16 acc[kI][kJ];
    uint32_t wave_m, wave_n;
};

// `also` sees each sixteenth's fragments of B before its products.
struct NothingElse {
    template <typename F>
    __device__ __forceinline__ void operator()(const F &, uint32_t) const {}
};

// An operand's steps, loaded one after the other into its ring of stages.
template <bool T, int Rows, int Stages>
struct TileStream {
    using O = TileOperand<T, Rows>;
    O o;
    const char *base;
    uint64_t row_bytes, chunk_step, part;
    uint32_t order, first, per, k, seg, at, left_steps, lds, stage;
    i32x4 from;  // of the step at hand; past the last nothing is read
    uint32_t source[2], to;

    __device__ __forceinline__ void init(const void *p, uint64_t row, uint64_t chunk, uint64_t part_step, uint32_t parts, uint32_t products,
                                         uint32_t ring) {
        base = static_cast<const char *>(p);
        row_bytes = row;
        chunk_step = chunk;
        part = part_step;
        order = parts;
        k = products;
        per = (products + 63) / 64;
        lds = O::destination(ring);
    }
    // To steps [s0, s1) of the tile from row `of` on.
    __device__ __forceinline__ void open(uint32_t of, uint32_t size, uint32_t s0, uint32_t s1) {
        first = of;
        o.init(row_bytes, chunk_step, of, size);
        seg = s0 / per;
        at = s0 - seg * per;
        left_steps = s1 - s0;
        stage = 0;
        seek();
    }
    __device__ __forceinline__ void seek() {
        // (past the last segment nothing is read)
        o.seek(base + (order >> 2 * seg & 3u) * part, chunk_step, first, at);
    }
    __device__ __forceinline__ void begin() {
        const uint32_t left = left_steps ? k - at * 64 : 0;
        left_steps -= left_steps != 0;
        from = o.buffer(left);
        o.sources(left, source);
        to = lds + stage * (Rows * 128);
        if (++stage == Stages) stage = 0;
        o.at += o.step;
        if (++at == per) {
            at = 0, seg++;
            seek();
        }
    }
    __device__ __forceinline__ void load(int j) { o.load(j, from, source, to); }
};

// A tile's products. The matrix units are kept busy by what stands between their
// rows of instructions: a share of the next sixteenth's reads and one load of a
// later step. All waves have read a step by its last sixteenth; B's stage is
// loaded again from there, and A's, which has one stage more, in the next step, so
// that the loads are spread evenly. The waves wait for the next step's loads
// alone. A tile's first steps may be loaded (prime) while the cells of the one
// before it are written.
template <bool AT, bool BT, typename Tile>
struct TileProduct {
    using A = TileOperand<AT, Tile::kM>;
    using B = TileOperand<BT, Tile::kN>;
    static constexpr int kI = Tile::kI, kJ = Tile::kJ, kL = A::kLoads, kS = Tile::kStages;
    static constexpr int kShare = kL / kI / 2;  // loads behind a row
    static_assert(kI == kJ && A::kLoads == B::kLoads && kL == 2 * kI * kShare, "even shares between the rows");
    const HeadArgs &a;
    const uint32_t lds;
    TileStream<AT, Tile::kM, kS + 1> sa;
    TileStream<BT, Tile::kN, kS> sb;
    uint32_t steps;

    __device__ __forceinline__ TileProduct(const HeadArgs &args, char *stages)
        : a(args), lds((uint32_t)(uintptr_t)(HBR_LDS char *)stages) {
        sa.init(a.a, a.a_row, a.a_chunk, a.a_part, a.a_order, a.k, lds);
        sb.init(a.b, a.b_row, a.b_chunk, a.b_part, a.b_order, a.k, lds + Tile::kB);
    }
    // The tile's first steps, and half of B's step behind them, into stages that no wave reads.
    __device__ __forceinline__ void prime(const Spot &t) {
        const uint32_t all = sa.per * a.segments;
        const uint32_t s0 = (uint32_t)((uint64_t)all * t.split / a.splits), s1 = (uint32_t)((uint64_t)all * (t.split + 1) / a.splits);
        steps = s1 - s0;
        sa.open(t.m0, a.m, s0, s1);
        sb.open(t.n0, a.n, s0, s1);
#pragma unroll
        for (int s = 0; s < kS; s++) {
            sa.begin();
            sb.begin();
#pragma unroll
            for (int j = 0; j < kL; j++) sa.load(j);
#pragma unroll
            for (int j = 0; j < (s + 1 < kS ? kL : kL / 2); j++) sb.load(j);
        }
    }
    // InFlight: the wave's loads behind those that have to have landed
    template <int InFlight>
    static __device__ __forceinline__ void meet() {  // they have, and the wave's reads are in registers; so have all others'
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(InFlight) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    }
    template <typename Also>
    __device__ __forceinline__ void run(Tile &t, Also &&also) {
        constexpr int kBehind = (2 * kS - 3) * kL;  // loads behind those of B's next step
#pragma unroll
        for (int i = 0; i < kI; i++)
#pragma unroll
            for (int j = 0; j < kJ; j++)
#pragma unroll
                for (int e = 0; e < 16; e++) t.acc[i][j][e] = 0.0f;
        uint32_t stage_a = 0, stage_b = 0;
        typename A::Places pa;
        typename B::Places pb;
        pa.init(lds, t.wave_m);
        pb.init(lds + Tile::kB, t.wave_n);
        bf16x8 fa[2][kI], fb[2][kJ];
        // a share of the fragments: B's first, which the first row meets all of
        auto read = [&](int q, int set, int kk) {
#pragma unroll
            for (int f = 2 * q; f < 2 * q + 2; f++) {
                if (f < kJ) fb[set][f] = pb.read(f, kk);
                else fa[set][f - kJ] = pa.read(f - kJ, kk);
            }
        };
        auto row = [&](int i, int set) {
#pragma unroll
            for (int j = 0; j < kJ; j++)
                t.acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[set][i], fb[set][j], t.acc[i][j], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        };
        meet<kBehind + kL / 2>();
#pragma unroll
        for (int q = 0; q < kI; q++) read(q, 0, 0);
        for (uint32_t s = 0; s < steps; s++) {
#pragma unroll
            for (int kk = 0; kk < 3; kk++) {
                also(fb[kk & 1], kk);
#pragma unroll
                for (int i = 0; i < kI; i++) {
                    row(i, kk & 1);
                    read(i, ~kk & 1, kk + 1);
#pragma unroll
                    for (int j = 0; j < kShare; j++) {
                        if (kk == 0) sb.load(kL / 2 + i * kShare + j);
                        else sa.load((kk - 1) * (kL / 2) + i * kShare + j);
                    }
                    if (kk == 0 && i == 0) sa.begin();
                    if (kk == 2 && i == 0) sb.begin();
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            also(fb[1], 3);
            const bool last_a = ++stage_a == kS + 1, last_b = ++stage_b == kS;
            if (last_a) stage_a = 0;
            if (last_b) stage_b = 0;
            pa.move(last_a ? (uint32_t)(-kS * Tile::kBytes) : (uint32_t)Tile::kBytes);
            pb.move(last_b ? (uint32_t)((1 - kS) * Tile::kBytes) : (uint32_t)Tile::kBytes);
            meet<kBehind>();
#pragma unroll
            for (int i = 0; i < kI; i++) {
                row(i, 1);
                read(i, 0, 0);
#pragma unroll
                for (int j = 0; j < kShare; j++) sb.load(i * kShare + j);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        meet<0>();  // the loads ahead have landed before the stages or the workgroup end
    }
};

// A workgroup's tile `id` of `all`: neighbours in the launch go to different
// XCDs, so each XCD takes a contiguous share of the tiles, in groups of eight
// columns of tiles whose operands its L2 holds.
template <typename Tile>
__device__ __forceinline__ Spot tile_spot(const HeadArgs &a, uint32_t index, uint32_t all) {
    Spot t;
    const uint32_t per = all / 8, rest = all % 8, xcd = index % 8;
    uint32_t id = xcd * per + min(xcd, rest) + index / 8;
    const uint32_t tiles = a.m_tiles * a.n_tiles;
    t.split = id / tiles;
    id -= t.split * tiles;
    constexpr uint32_t kGroup = 8;
    const uint32_t group = id / (kGroup * a.n_tiles), first = group * kGroup;
    const uint32_t rows = min(kGroup, a.m_tiles - first), in = id - group * kGroup * a.n_tiles;
    t.m0 = (first + in % rows) * Tile::kM;
    t.n0 = in / rows * Tile::kN;
    return t;
}

}  // namespace hbr
