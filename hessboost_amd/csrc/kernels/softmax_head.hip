// The softmax cross entropy of a linear layer over many classes and its
// gradients, the scores made tile by tile and never kept.
//
//   z = h W^T + b; lse = log sum exp z; loss = a (lse - z_y)
//   g = a (exp(z - lse) - [k = y]); dh = c g W; dW = c g^T h; db = c sum g
//
// In bf16 the pairs g are rounded once to bf16 for the products, as a layer's
// output gradient in mixed precision is: half a step each, of the size of the
// result's own rounding. They hold no c, so that a row without a weight has
// its label's pair near -1, which bf16 holds well, and not near -c.
//
// A row's maximum is kept in the scores' own units and the sum of its
// exponentials relative to it: the largest score counts exactly one, two scores
// that differ by a bit stay apart, and lse and loss are rounded at the size of
// the scores' differences. (In units of log2 throughout an exponential has one
// instruction less, and neighbours fall together: z log2 e rounds again.)
//
// 8 n K D operations with the gradients: the scores once for the sums and once
// for the pairs (6 if they were kept, which takes 4 bytes a score), and both
// products with the pairs. Bound by the products' pipeline, whose every step of
// 32 waits for its last load (the matrix cores are busy 57% of the cycles, 45%
// in the pairs), and by the exponentials between: 16,384 x 131,072 x 1,024 bf16
// scores 4.4 ms (1.0 PFLOP/s), pairs 5.1 (0.86), dw 4.0 and dh 3.9 (1.1). f32
// operands are three bf16 parts, of whose nine products the six that matter are
// made: 4,096 x 5,003 x 256 scores 68 us (154 TFLOP/s of f32, a library product's
// in f32), pairs 84, dw 74, dh 71. One row against 131,072 classes of 1,024 bf16: 56 us,
// w read at 4.8 TB/s.
#include "common.h"

namespace hbr {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
#define HBR_LDS __attribute__((address_space(3)))

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLn2 = 0.693147180559945309f;
constexpr int kPairsMore = 2048;  // LDS of the pairs beyond the stages
constexpr uint32_t kNowhere = 0x80000000u;  // past every buffer: reads as zero

__device__ __forceinline__ int32_t uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane((int32_t)v); }

// A running maximum's shift: a tile with no open class sums to zero.
__device__ __forceinline__ float shift_of(float m) { return m == -INFINITY ? 0.0f : m; }

// exp of a difference of scores (-infinity: 0).
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

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

// The pairs of parts of a product of two f32 operands, smallest first: (2, 0),
// (0, 2), (1, 1), (1, 0), (0, 1), (0, 0), two bits a segment.
constexpr uint32_t kPartA = 2u | 0u << 2 | 1u << 4 | 1u << 6 | 0u << 8 | 0u << 10;
constexpr uint32_t kPartB = 0u | 2u << 2 | 1u << 4 | 0u << 6 | 1u << 8 | 0u << 10;

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
        const uint32_t of = a.segments == 1 ? 10 : 2 * min(seg, 5u);
        oa.seek(static_cast<const char *>(a.a) + (kPartA >> of & 3u) * a.a_part, a.a_row, a.a_chunk, t.m0, at);
        ob.seek(static_cast<const char *>(a.b) + (kPartB >> of & 3u) * a.b_part, a.b_row, a.b_chunk, t.n0, at);
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

// ---- the scores' maxima and sums -----------------------------------------------------------

// m: classes, n: rows. A lane holds its wave's classes of kJ rows: maxima and
// sums stay in its registers but for the other half of the wave and the other
// waves of the same rows.
template <typename Tile>
__device__ __forceinline__ void head_scores(const HeadArgs &a, char *lds) {
    __shared__ float bias[Tile::kM];
    __shared__ float top_of[Tile::kWavesM][Tile::kN], sum_of[Tile::kWavesM][Tile::kN];
    __shared__ int32_t best_of[Tile::kWavesM][Tile::kN];
    Tile t;
    head_place(a, t);
    for (uint32_t i = threadIdx.x; i < Tile::kM; i += Tile::kThreads) {
        const uint32_t c = t.m0 + i;
        bias[i] = c >= a.m ? -INFINITY : a.bias ? a.bias[c] : 0.0f;
    }
    head_product<false, false>(a, lds, t);
    const uint32_t lane = lane_id(), wm = t.wave_m / Tile::kWaveM;
    if (t.m0 + Tile::kM > a.m) {  // classes past the last are zeros, which make no number of an infinite input
#pragma unroll
        for (int i = 0; i < Tile::kI; i++)
#pragma unroll
            for (int e = 0; e < 16; e++)
                if (t.m0 + t.wave_m + 32 * i + row_of(e) >= a.m)
#pragma unroll
                    for (int j = 0; j < Tile::kJ; j++) t.acc[i][j][e] = 0.0f;
    }
#pragma unroll
    for (int j = 0; j < Tile::kJ; j++) {
        const uint32_t in = t.wave_n + 32 * j + lane % 32, r = t.n0 + in;
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < Tile::kI; i++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const float z = t.acc[i][j][e] + bias[t.wave_m + 32 * i + row_of(e)];
                t.acc[i][j][e] = z;
                top = fmaxf(top, z);
            }
        top = fmaxf(top, __shfl_xor(top, 32, kWave));
        const float shift = shift_of(top);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < Tile::kI; i++)
#pragma unroll
            for (int e = 0; e < 16; e++) sum += exp_of(t.acc[i][j][e] - shift);
        sum += __shfl_xor(sum, 32, kWave);
        // the label's class, where it is one of the wave's
        const int64_t y = a.labels && r < a.n ? (int64_t)a.labels[r] - t.m0 - t.wave_m : -1;
        if (__ballot(y >= 0 && y < Tile::kWaveM)) {
#pragma unroll
            for (int i = 0; i < Tile::kI; i++)
#pragma unroll
                for (int e = 0; e < 16; e++)
                    if (y == 32 * i + row_of(e) && t.m0 + t.wave_m + y < a.m) a.label_margin[r] = t.acc[i][j][e];
        }
        int32_t best = 0x7fffffff;
        if (a.part_best) {
#pragma unroll
            for (int i = 0; i < Tile::kI; i++)
#pragma unroll
                for (int e = 0; e < 16; e++)
                    if (t.acc[i][j][e] == top) best = min(best, (int32_t)(t.m0 + t.wave_m + 32 * i + row_of(e)));
            best = min(best, __shfl_xor(best, 32, kWave));
        }
        if (lane < 32) {
            top_of[wm][in] = top;
            sum_of[wm][in] = sum;
            best_of[wm][in] = best;
        }
    }
    __syncthreads();
    const uint32_t in = threadIdx.x, r = t.n0 + in;
    if (in >= Tile::kN || r >= a.n) return;
    static_assert(Tile::kN <= Tile::kThreads && Tile::kWavesM == 2, "a thread a row, two waves of its classes");
    const float t0 = top_of[0][in], t1 = top_of[1][in], top = fmaxf(t0, t1), shift = shift_of(top);
    const uint64_t at = (uint64_t)(t.m0 / Tile::kM) * a.n + r;
    a.part_max[at] = top;
    a.part_sum[at] = sum_of[0][in] * exp_of(t0 - shift) + sum_of[1][in] * exp_of(t1 - shift);
    if (a.part_best) a.part_best[at] = best_of[t1 > t0 ? 1 : 0][in];
}

// ---- the scores' gradients --------------------------------------------------------------------

// m: rows, n: classes. A lane holds its wave's rows of kJ classes, so a
// class's sum over the rows stays in its registers; a row whose label is below
// 0 is read as zeros and has no gradient. Past the classes g is zero up to its
// stride.
template <typename Tile, int Parts>
__device__ __forceinline__ void head_pairs(const HeadArgs &a, char *lds) {
    __shared__ float lse_of[Tile::kM], by_of[Tile::kM];
    __shared__ int32_t label_of[Tile::kM];
    __shared__ float db_of[Tile::kWavesM][Tile::kN];
    Tile t;
    head_place(a, t);
    for (uint32_t i = threadIdx.x; i < Tile::kM; i += Tile::kThreads) {
        const uint32_t r = t.m0 + i;
        const int32_t y = r < a.m ? a.labels[r] : -1;
        const bool live = y >= 0;
        lse_of[i] = live ? a.lse2[r] : INFINITY;
        by_of[i] = live ? a.weight ? a.weight[r] : 1.0f : 0.0f;
        const int64_t in = (int64_t)y - (int64_t)a.first - t.n0;
        label_of[i] = live && in >= 0 && in < (int64_t)Tile::kN ? (int32_t)in : -0x10000;
    }
    head_product<false, false>(a, lds, t, a.labels);
    const uint32_t lane = lane_id(), wm = t.wave_m / Tile::kWaveM;
    float bias[Tile::kJ], db[Tile::kJ];
#pragma unroll
    for (int j = 0; j < Tile::kJ; j++) {
        const uint32_t c = t.n0 + t.wave_n + 32 * j + lane % 32;
        bias[j] = c >= a.n ? -INFINITY : a.bias ? a.bias[c] : 0.0f;
        db[j] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < Tile::kI; i++) {
        __builtin_amdgcn_sched_barrier(0);  // the rows' values of one i at a time in registers
        // does a row of these 32 have its label among the wave's classes?
        const uint32_t y = (uint32_t)label_of[t.wave_m + 32 * i + lane % 32] - t.wave_n;
        const bool labelled = __ballot(y < (uint32_t)Tile::kWaveN) != 0;
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const uint32_t m = t.wave_m + 32 * i + row_of(e);
            const float lse = lse_of[m], by = by_of[m];
#pragma unroll
            for (int j = 0; j < Tile::kJ; j++)
                t.acc[i][j][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(t.acc[i][j][e] + bias[j], kLog2e, -lse)) * by;
        }
        if (labelled) {
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const uint32_t m = t.wave_m + 32 * i + row_of(e);
                const int32_t at = label_of[m] - (int32_t)(t.wave_n + lane % 32);
                const float by = by_of[m];
#pragma unroll
                for (int j = 0; j < Tile::kJ; j++)
                    if (at == 32 * j) t.acc[i][j][e] -= by;
            }
        }
        // a row of zeros and an infinite weight are no number: there is none
        // in the gradients of a row that takes no part
        float sum[Tile::kJ] = {}, any = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; e++)
#pragma unroll
            for (int j = 0; j < Tile::kJ; j++) sum[j] += t.acc[i][j][e];
#pragma unroll
        for (int j = 0; j < Tile::kJ; j++) any += sum[j];
        if (__ballot(any != any)) {
#pragma unroll
            for (int j = 0; j < Tile::kJ; j++) sum[j] = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const bool dead = lse_of[t.wave_m + 32 * i + row_of(e)] == INFINITY;
#pragma unroll
                for (int j = 0; j < Tile::kJ; j++) {
                    if (dead) t.acc[i][j][e] = 0.0f;
                    sum[j] += t.acc[i][j][e];
                }
            }
        }
#pragma unroll
        for (int j = 0; j < Tile::kJ; j++) db[j] += sum[j];
    }
#pragma unroll
    for (int j = 0; j < Tile::kJ; j++) {
        db[j] += __shfl_xor(db[j], 32, kWave);
        if (lane < 32) db_of[wm][t.wave_n + 32 * j + lane % 32] = db[j];
    }
    // through LDS to stores of 16 bytes: bf16 whole, f32 in two halves of each
    // wave's rows, split on the way out. A row of LDS is 16 bytes longer than
    // the tile's, so that the wave's two rows of a write meet different banks.
    constexpr int kHalves = Parts == 1 ? 1 : 2, kSize = Parts == 1 ? 2 : 4, kI = Tile::kI / kHalves;
    constexpr uint32_t kRow = Tile::kN * kSize + 16, kRows = Tile::kM / kHalves, kWaveRows = Tile::kWaveM / kHalves;
    static_assert(kRows * kRow <= Tile::kLds + kPairsMore, "the pairs fit LDS");
#pragma unroll
    for (int half = 0; half < kHalves; half++) {
        if (half) __syncthreads();
#pragma unroll
        for (int i = 0; i < kI; i++) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < 16; e++)
#pragma unroll
                for (int j = 0; j < Tile::kJ; j++) {
                    char *to = lds + (wm * kWaveRows + 32 * i + row_of(e)) * kRow + (t.wave_n + 32 * j + lane % 32) * kSize;
                    const float v = t.acc[half * kI + i][j][e];
                    if constexpr (Parts == 1) *reinterpret_cast<uint16_t *>(to) = to_bf16(v);
                    else *reinterpret_cast<float *>(to) = v;
                }
        }
        __syncthreads();
        // a wave writes 16 rows of a chunk at a time
        for (uint32_t i = threadIdx.x; i < kRows * (Tile::kN / 8); i += Tile::kThreads) {
            const uint32_t chunk = i / (kRows * 4), m = i / 4 % kRows, col = chunk * 32 + i % 4 * 8;
            const uint64_t r = t.m0 + m / kWaveRows * Tile::kWaveM + half * kWaveRows + m % kWaveRows;
            if (r >= a.m || t.n0 + col >= a.g_stride) continue;
            uint16_t *g = static_cast<uint16_t *>(a.g) + (t.n0 / 32 + chunk) * a.g_chunk + r * 32 + i % 4 * 8;
            if constexpr (Parts == 1) {
                *reinterpret_cast<i32x4 *>(g) = *reinterpret_cast<const i32x4 *>(lds + m * kRow + col * 2);
            } else {
                Vec<float, 4> v[2];
#pragma unroll
                for (int k = 0; k < 2; k++)
                    v[k] = *reinterpret_cast<const Vec<float, 4> *>(lds + m * kRow + (col + 4 * k) * 4);
                Vec<uint16_t, 8> out[3];
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    uint16_t s[3];
                    split3(v[k / 4].v[k % 4], s);
#pragma unroll
                    for (int q = 0; q < 3; q++) out[q].v[k] = s[q];
                }
#pragma unroll
                for (int q = 0; q < 3; q++) *reinterpret_cast<Vec<uint16_t, 8> *>(g + q * a.g_part) = out[q];
            }
        }
    }
    const uint32_t c = t.n0 + threadIdx.x;
    if (threadIdx.x < Tile::kN && c < a.n) {
        float sum = 0.0f;
        for (int w = 0; w < Tile::kWavesM; w++) sum += db_of[w][threadIdx.x];
        a.part_db[(uint64_t)(t.m0 / Tile::kM) * a.g_stride + c] = sum;
    }
}

// ---- the products with the gradients ---------------------------------------------------------------

// E: what c holds: f32 sums (a share's, added to or not) or the result.
template <typename Tile, typename E, bool AT>
__device__ __forceinline__ void head_sums(const HeadArgs &a, char *lds) {
    using T = typename E::type;
    Tile t;
    head_place(a, t);
    head_product<AT, true>(a, lds, t);
    const uint32_t lane = lane_id();
    // the tile's rows as a buffer that ends with its last: what lies past the
    // rows or the columns is neither read nor written
    const uint64_t from = reinterpret_cast<uint64_t>(static_cast<T *>(a.c) + t.split * a.c_split + t.m0 * a.c_stride + t.n0);
    const uint32_t stride = (uint32_t)a.c_stride * sizeof(T);
    const uint32_t rows = min(a.rows > t.m0 ? a.rows - t.m0 : 0u, (uint32_t)Tile::kM);
    const uint32_t size = rows ? (rows - 1) * stride + min(a.n - t.n0, (uint32_t)Tile::kN) * (uint32_t)sizeof(T) : 0u;
    __amdgpu_buffer_rsrc_t c = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void *>(from), 0, size, 0x00020000);
#pragma unroll
    for (int j = 0; j < Tile::kJ; j++) {
        const uint32_t n = t.wave_n + 32 * j + lane % 32;
        const uint32_t at = t.n0 + n < a.n ? (t.wave_m + lane / 32 * 4) * stride + n * (uint32_t)sizeof(T) : kNowhere;
#pragma unroll
        for (int i = 0; i < Tile::kI; i++) {
            if constexpr (sizeof(T) == 4) {
                if (a.accumulate) {
                    float before[16];
#pragma unroll
                    for (int e = 0; e < 16; e++)
                        before[e] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(
                            c, at + (32 * i + 8 * (e / 4) + e % 4) * stride, 0, 0));
#pragma unroll
                    for (int e = 0; e < 16; e++) t.acc[i][j][e] += before[e];
                }
            }
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const uint32_t to = at + (32 * i + 8 * (e / 4) + e % 4) * stride;
                if constexpr (sizeof(T) == 4)
                    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(t.acc[i][j][e] * a.scale), c, to, 0, 0);
                else
                    __builtin_amdgcn_raw_buffer_store_b16(to_bf16(t.acc[i][j][e] * a.scale), c, to, 0, 0);
            }
        }
    }
}

// A workgroup sums 64 cells a wave; with several shares its waves take shares
// of the same cells' parts, joined in order.
template <typename E>
__device__ __forceinline__ void head_sum(const HeadSumArgs &a) {
    __shared__ float sum_of[16][kWave];
    const uint64_t cells = a.rows * a.cols;
    const uint32_t lane = lane_id(), wave = threadIdx.x / kWave, waves = blockDim.x / kWave;
    const uint32_t share = wave % a.shares, each = waves / a.shares;
    const uint32_t p0 = (uint32_t)((uint64_t)a.parts * share / a.shares), p1 = (uint32_t)((uint64_t)a.parts * (share + 1) / a.shares);
    for (uint64_t at = (uint64_t)blockIdx.x * each * kWave; at < cells; at += (uint64_t)gridDim.x * each * kWave) {
        const uint64_t i = at + wave / a.shares * kWave + lane;
        float s = 0.0f;
        if (i < cells) {
            const float *part = a.part + i;
#pragma unroll 8
            for (uint32_t p = p0; p < p1; p++) s += part[p * a.part_stride];
        }
        if (a.shares > 1) {
            __syncthreads();
            sum_of[wave][lane] = s;
            __syncthreads();
            if (share) continue;
            for (uint32_t w = 1; w < a.shares; w++) s += sum_of[wave + w][lane];
        }
        if (i >= cells) continue;
        const uint64_t r = i / a.cols;
        static_cast<typename E::type *>(a.dst)[r * a.dst_stride + (i - r * a.cols)] = E::down(s * a.scale);
    }
}

// Rows into chunks of 32 columns (zeros past the last): eight elements of a
// row a thread, a wave 16 rows of a chunk.
template <typename E, int Parts>
__device__ __forceinline__ void head_parts(const HeadPartsArgs &a) {
    using T = typename E::type;
    const uint64_t cells = a.rows * a.chunks * 4;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < cells; i += (uint64_t)gridDim.x * 256) {
        // four chunks (256 bytes of a bf16 row) of a row by neighbouring threads
        const uint64_t block = i / (a.rows * 16);
        const uint32_t wide = min(4u, a.chunks - (uint32_t)block * 4);
        const uint64_t in = i - block * a.rows * 16, r = in / (wide * 4);
        const uint32_t chunk = (uint32_t)block * 4 + (uint32_t)(in % (wide * 4)) / 4, c = chunk * 32 + in % 4 * 8;
        const T *src = static_cast<const T *>(a.src) + r * a.src_stride + c;
        Vec<T, 8> v{};
        if (c + 8 <= a.cols) {
            __builtin_memcpy(&v, src, sizeof v);
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (c + k < a.cols) v.v[k] = src[k];
        }
        // a row that takes no part may hold anything: finite, so that its
        // gradient of zero adds nothing
        if (a.labels && a.labels[r] < 0)
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (!(__builtin_fabsf(E::up(v.v[k])) < INFINITY)) v.v[k] = (T)0;
        Vec<uint16_t, 8> out[Parts];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            if (Parts == 1) {
                out[0].v[k] = (uint16_t)v.v[k];
            } else {
                uint16_t s[3];
                split3(E::up(v.v[k]), s);
#pragma unroll
                for (int q = 0; q < Parts; q++) out[q].v[k] = s[q];
            }
        }
#pragma unroll
        for (int q = 0; q < Parts; q++)
            *reinterpret_cast<Vec<uint16_t, 8> *>(a.dst + q * a.part + chunk * a.chunk + r * 32 + in % 4 * 8) = out[q];
    }
}

}  // namespace hbr

using namespace hbr;

// waves: a SIMD's, at least
#define HBR_HEAD(name, W, waves, more, ...)                                                       \
    extern "C" __global__ __launch_bounds__(HeadTile<W>::kThreads, waves) void name(HeadArgs a) { \
        __shared__ __align__(1024) char lds[HeadTile<W>::kLds + more];                            \
        __VA_ARGS__(a, lds);                                                                      \
    }
#define HBR_HEADS(suffix, W, waves)                                                                 \
    HBR_HEAD(hbr_head_dh_part_##suffix, W, waves, 0, head_sums<HeadTile<W>, F32, false>)            \
    HBR_HEAD(hbr_head_dh_bf16_##suffix, W, waves, 0, head_sums<HeadTile<W>, Bf16, false>)           \
    HBR_HEAD(hbr_head_dw_part_##suffix, W, waves, 0, head_sums<HeadTile<W>, F32, true>)             \
    HBR_HEAD(hbr_head_dw_bf16_##suffix, W, waves, 0, head_sums<HeadTile<W>, Bf16, true>)
HBR_HEAD(hbr_head_scores_128, 4, 3, 0, head_scores<HeadTile<4>>)
HBR_HEAD(hbr_head_pairs_bf16_128, 4, 4, kPairsMore, head_pairs<HeadTile<4>, 1>)
HBR_HEAD(hbr_head_pairs_f32_128, 4, 4, kPairsMore, head_pairs<HeadTile<4>, 3>)
HBR_HEADS(256, 8, 2)
HBR_HEADS(128, 4, 4)

extern "C" __global__ __launch_bounds__(1024) void hbr_head_sum_f32(HeadSumArgs a) { head_sum<F32>(a); }
extern "C" __global__ __launch_bounds__(1024) void hbr_head_sum_bf16(HeadSumArgs a) { head_sum<Bf16>(a); }
extern "C" __global__ __launch_bounds__(256) void hbr_head_parts_f32(HeadPartsArgs a) { head_parts<F32, 3>(a); }
extern "C" __global__ __launch_bounds__(256) void hbr_head_parts_bf16(HeadPartsArgs a) { head_parts<Bf16, 1>(a); }

// A row's tiles joined: a.wide rows a workgroup (a power of two, 64 at most),
// a lane of a wave for each, the wave's other lanes and the 16 waves shares of
// the class tiles, in order within a lane, over the lanes and over the waves.
extern "C" __global__ __launch_bounds__(1024) void hbr_head_finish(HeadFinishArgs a) {
    constexpr uint32_t kWaves = 16;
    __shared__ float top_of[kWaves][kWave], sum_of[kWaves][kWave];
    __shared__ int32_t best_of[kWaves][kWave];
    const uint32_t lane = lane_id(), wave = threadIdx.x / kWave, in = lane & (a.wide - 1);
    const uint64_t r = (uint64_t)blockIdx.x * a.wide + in;
    const uint32_t lanes = kWave / a.wide, share = (a.tiles + kWaves * lanes - 1) / (kWaves * lanes);
    const uint32_t first = (wave * lanes + lane / a.wide) * share, end = min(a.tiles, first + share);
    float top = -INFINITY, sum = 0.0f;
    int32_t best = 0x7fffffff;
    auto join = [&](float m, float s, int32_t b) {
        const float both = fmaxf(top, m), shift = shift_of(both);
        sum = sum * exp_of(top - shift) + s * exp_of(m - shift);
        best = m > top ? b : m == top ? min(best, b) : best;
        top = both;
    };
    constexpr uint32_t kAhead = 8;
    if (r < a.rows)
        for (uint32_t t0 = first; t0 < end; t0 += kAhead) {
            float m[kAhead], s[kAhead];
            int32_t b[kAhead];
#pragma unroll
            for (uint32_t u = 0; u < kAhead; u++) {
                const uint64_t at = (t0 + u) * a.rows + r;
                const bool in = t0 + u < end;
                m[u] = in ? a.part_max[at] : 0.0f;
                s[u] = in ? a.part_sum[at] : 0.0f;
                b[u] = in && a.part_best ? a.part_best[at] : 0;
            }
#pragma unroll
            for (uint32_t u = 0; u < kAhead; u++)
                if (t0 + u < end) join(m[u], s[u], b[u]);
        }
    for (uint32_t d = a.wide; d < (uint32_t)kWave; d <<= 1)
        join(__shfl_down(top, d, kWave), __shfl_down(sum, d, kWave), __shfl_down(best, d, kWave));
    top_of[wave][lane] = top;
    sum_of[wave][lane] = sum;
    best_of[wave][lane] = best;
    __syncthreads();
    if (wave != 0 || lane >= a.wide || r >= a.rows) return;
    for (uint32_t w = 1; w < kWaves; w++) join(top_of[w][lane], sum_of[w][lane], best_of[w][lane]);
    const int32_t y = a.labels ? a.labels[r] : -1;
    // a label that is no class: neither a loss nor a gradient
    const bool no_class = y >= 0 && (uint64_t)y >= a.classes;
    const float shift = shift_of(top), more2 = no_class ? NAN : __builtin_amdgcn_logf(sum), more = more2 * kLn2;
    a.lse2[r] = __builtin_fmaf(shift, kLog2e, more2);
    if (a.lse) a.lse[r] = shift + more;
    if (a.best) a.best[r] = best == 0x7fffffff ? 0 : best;  // a row of NaN has none
    if (!a.loss) return;
    if (!a.labels) {
        a.loss[r] = (shift - top) + more;
        return;
    }
    const float by = a.weight ? a.weight[r] : 1.0f;
    a.loss[r] = y < 0 ? 0.0f : no_class ? NAN : by * ((shift - a.label_margin[r]) + more);
}
