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
// id: the adapter of the thread's row of the tile, before: of the row before it
// (none: below 0).
template <typename Tile, typename E>
__device__ __forceinline__ void linear_adapters(const LinearArgs &a, char *lds, Tile &t, int32_t id, int32_t before_id) {
    using T = typename E::type;
    constexpr int kParts = sizeof(T) == 4 ? 3 : 1, kPairs = kParts == 3 ? 6 : 1;
    constexpr uint32_t kM = Tile::kM, kNone = 0xffffu, kWaves = Tile::kThreads / kWave;
    // A step is 32 products, in f32 16 of all three parts; its operands lie in
    // front of the slots.
    constexpr uint32_t kStep = kParts == 1 ? 32 : 16, kRow = kStep * 2, kPart = kM * kRow;
    int32_t *slot_id = reinterpret_cast<int32_t *>(lds + 2 * kParts * kPart);    // [kM] a slot's adapter
    uint16_t *slot_of = reinterpret_cast<uint16_t *>(slot_id + kM);              // [kM] a row's slot
    uint16_t *joined = slot_of + kM;                                             // [kM] a slot's place among the joined
    uint32_t *counts = reinterpret_cast<uint32_t *>(joined + kM);                // [kWaves]
    static_assert(2 * kParts * kPart + kM * 8 + kWaves * 4 <= (uint32_t)Tile::kLds && kM <= (uint32_t)Tile::kThreads, "all fits the stages");
    const uint32_t m = threadIdx.x, lane = lane_id(), wave = threadIdx.x / kWave;
    const bool starts = id >= 0 && (m == 0 || before_id != id);
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
    const bool eights = a.rank % 8 == 0;
    const bool wide = eights && a.up_stride % 8 == 0 && reinterpret_cast<uint64_t>(a.up) % 16 == 0;
    // pieces of eight products of a row: of the rows' low values, and of the
    // outputs' second factors. Every load is made, from within its array, and
    // what does not count is zeroed.
    constexpr uint32_t kIn = kStep / 8;  // pieces of a row
    constexpr int kPieces = kM * kIn / Tile::kThreads;
    static_assert(Tile::kM == Tile::kN && kM * kIn % Tile::kThreads == 0, "as many pieces of each a thread");
    // a piece's place: the rows that LDS serves at once meet different banks
    auto place = [&](uint32_t row, uint32_t piece) { return row * kRow + (piece ^ ((row >> (kIn == 4 ? 2 : 3)) & (kIn - 1))) * 16; };
    auto put = [&](uint32_t to, const float (&v)[8]) {
        Vec<uint16_t, 8> out[kParts];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if constexpr (kParts == 1) {
                out[0].v[j] = to_bf16(v[j]);
            } else {
                uint16_t p[3];
                split3(v[j], p);
#pragma unroll
                for (int q = 0; q < kParts; q++) out[q].v[j] = p[q];
            }
        }
#pragma unroll
        for (int q = 0; q < kParts; q++) *reinterpret_cast<Vec<uint16_t, 8> *>(lds + q * kPart + to) = out[q];
    };
    for (uint32_t k0 = 0; k0 < all; k0 += kStep) {
        float low[kPieces][8], up[kPieces][8];
#pragma unroll
        for (int q = 0; q < kPieces; q++) {
            const uint32_t at = q * Tile::kThreads + threadIdx.x, row = at / kIn, k = k0 + at % kIn * 8;
            const uint32_t own = slot_of[row];
            const float *lows = a.low + (uint64_t)(min(t.m0 + row, a.p.m - 1)) * a.rank;
            const uint64_t out = min(t.n0 + row, a.p.n - 1);
            const T *ups = static_cast<const T *>(a.up);
            const uint32_t kc = min(k, all - 1);
            uint32_t s = kc / a.rank, rho = kc - s * a.rank;
            if (eights) {  // (a piece is one slot's)
                rho &= ~7u;
                const Vec<float, 4> l0 = *reinterpret_cast<const Vec<float, 4> *>(lows + rho),
                                    l1 = *reinterpret_cast<const Vec<float, 4> *>(lows + rho + 4);
                const T *from = ups + ((uint64_t)slot_id[s] * a.p.n + out) * a.up_stride + rho;
                Vec<T, 8> x;
                if (wide) {
                    x = *reinterpret_cast<const Vec<T, 8> *>(from);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; j++) x.v[j] = from[j];
                }
                const bool some = k < all, mine = some && s == own;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    low[q][j] = mine ? j < 4 ? l0.v[j % 4] : l1.v[j % 4] : 0.0f;
                    up[q][j] = some ? E::up(x.v[j]) : 0.0f;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const bool some = k + j < all;
                    const float l = lows[rho], u = E::up(ups[((uint64_t)slot_id[s] * a.p.n + out) * a.up_stride + rho]);
                    low[q][j] = some && s == own ? l : 0.0f;
                    up[q][j] = some ? u : 0.0f;
                    if (++rho == a.rank) rho = 0, s = min(s + 1, slots - 1);
                }
            }
        }
#pragma unroll
        for (int q = 0; q < kPieces; q++) {
            const uint32_t at = q * Tile::kThreads + threadIdx.x, to = place(at / kIn, at % kIn);
            put(to, low[q]);
            put(to + kParts * kPart, up[q]);
        }
        __syncthreads();
#pragma unroll
        for (uint32_t kk = 0; kk < kStep / 16; kk++) {
            const uint32_t piece = kk * 2 + lane / 32;
            auto fragment = [&](uint32_t part, uint32_t row) {
                return *reinterpret_cast<const bf16x8 *>(lds + part * kPart + place(row + lane % 32, piece));
            };
#pragma unroll
            for (int pair = 0; pair < kPairs; pair++) {
                const uint32_t pa = kParts == 1 ? 0 : kPartA >> 2 * pair & 3u, pb = kParts == 1 ? 0 : kPartB >> 2 * pair & 3u;
                bf16x8 fa[Tile::kI], fb[Tile::kJ];
#pragma unroll
                for (int i = 0; i < Tile::kI; i++) fa[i] = fragment(pa, t.wave_m + 32 * i);
#pragma unroll
                for (int j = 0; j < Tile::kJ; j++) fb[j] = fragment(kParts + pb, t.wave_n + 32 * j);
#pragma unroll
                for (int i = 0; i < Tile::kI; i++)
#pragma unroll
                    for (int j = 0; j < Tile::kJ; j++)
                        t.acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[i], fb[j], t.acc[i][j], 0, 0, 0);
                if (kPairs > 1) __builtin_amdgcn_sched_barrier(0);  // one pair's fragments at a time in registers
            }
        }
        __syncthreads();
    }
}

// E: the inputs' type; Part: f32 sums of a share of the steps
template <typename Tile, typename E, bool Part>
__device__ __forceinline__ void linear_y(const LinearArgs &a, char *lds) {
    Tile t;
    head_place(a.p, t);
    const bool adapters = a.low && (!Part || t.split == 0);
    // (loaded here, and waited for behind the products)
    auto adapter = [&](uint32_t in) {
        const uint32_t row = t.m0 + in;
        const int32_t id = adapters && in < Tile::kM && row < a.p.m ? a.ids[row] : -1;
        return id >= 0 && (uint32_t)id < a.adapters ? id : -1;
    };
    const int32_t id = adapter(threadIdx.x), before = threadIdx.x ? adapter(threadIdx.x - 1) : -1;
    head_product<false, false>(a.p, lds, t);
    if (adapters) linear_adapters<Tile, E>(a, lds, t, id, before);
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
// adapters, each adapter once, 32 of those rows of `down` at a time; its four
// waves share the steps. A cell counts where the row's adapter is the column's.
template <typename E, bool Wide>
__device__ __forceinline__ void linear_low(const LinearLowArgs &a) {
    using T = typename E::type;
    using S = Strip<E, Wide>;
    constexpr uint32_t kRows = 16, kCols = 2, kWaves = 4, kAhead = 4;
    __shared__ int32_t slot_id[kRows], slot_of[kRows];
    __shared__ f32x4 part[kWaves][kCols][kWave];
    const uint32_t lane = lane_id(), wave = threadIdx.x / kWave, in = lane % 16, quarter = lane / 16;
    const uint64_t r0 = (uint64_t)blockIdx.x * kRows;
    // every wave finds the slots: the rows' adapters in order of their first rows
    int32_t id = r0 + in < a.n_rows ? a.ids[r0 + in] : -1;
    if (id < 0 || (uint32_t)id >= a.adapters) id = -1;
    uint32_t first = in;
#pragma unroll
    for (int o = kRows - 1; o >= 0; o--)
        if (__shfl(id, o, kWave) == id) first = min(first, (uint32_t)o);
    const uint64_t firsts = __ballot(lane < kRows && id >= 0 && first == in);
    const uint32_t slots = (uint32_t)__popcll(firsts), slot = (uint32_t)__popcll(firsts & ((1ull << first) - 1));
    if (wave == 0 && lane < kRows) {
        slot_of[lane] = id >= 0 ? (int32_t)slot : -1;
        if (id >= 0 && first == lane) slot_id[slot] = id;
    }
    __syncthreads();
    const uint32_t all = slots * a.rank;
    const T *x = static_cast<const T *>(a.x) + min(r0 + in, (uint64_t)a.n_rows - 1) * a.x_stride;
    for (uint32_t v0 = blockIdx.y * kCols * 16; v0 < all; v0 += gridDim.y * kCols * 16) {
        const T *down[kCols];
#pragma unroll
        for (uint32_t q = 0; q < kCols; q++) {
            const uint32_t v = min(v0 + q * 16 + in, all - 1), s = v / a.rank;
            down[q] = static_cast<const T *>(a.down) + ((uint64_t)slot_id[s] * a.rank + (v - s * a.rank)) * a.down_stride;
        }
        f32x4 acc[kCols] = {};
        for (uint32_t c0 = wave * kAhead * S::kStep; c0 < a.dim; c0 += kWaves * kAhead * S::kStep) {
            Vec<T, S::kV> fx[kAhead], fd[kAhead][kCols];
#pragma unroll
            for (uint32_t k = 0; k < kAhead; k++) {
                const uint32_t c = c0 + k * S::kStep + quarter * S::kV;
                fx[k] = S::load(x, c, a.dim);
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
                const T *up = static_cast<const T *>(a.up) + ((uint64_t)id * a.outs + o0 + o) * a.up_stride;
                const float *low = a.low + (uint64_t)r * a.rank;
                float more = 0.0f;
#pragma unroll 4
                for (uint32_t rho = 0; rho < a.rank; rho++) more = __builtin_fmaf(low[rho], E::up(up[rho]), more);
                s += more;
            }
        }
        static_cast<T *>(a.out)[(uint64_t)r * a.out_stride + o0 + o] = E::down(s + bias);
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

// waves: a SIMD's, at least
#define HBR_LINEAR(name, Tile, waves, ...)                                               \
    extern "C" __global__ __launch_bounds__(Tile::kThreads, waves) void name(LinearArgs a) { \
        __shared__ __align__(1024) char lds[Tile::kLds];                                 \
        __VA_ARGS__(a, lds);                                                             \
    }
#define HBR_LINEARS(suffix, Tile, waves)                                                 \
    HBR_LINEAR(hbr_linear_y_f32_##suffix, Tile, waves, linear_y<Tile, F32, false>)       \
    HBR_LINEAR(hbr_linear_y_bf16_##suffix, Tile, waves, linear_y<Tile, Bf16, false>)     \
    HBR_LINEAR(hbr_linear_y_part_f32_##suffix, Tile, waves, linear_y<Tile, F32, true>)   \
    HBR_LINEAR(hbr_linear_y_part_bf16_##suffix, Tile, waves, linear_y<Tile, Bf16, true>) \
    HBR_LINEAR(hbr_linear_dx_f32_##suffix, Tile, waves, linear_d<Tile, F32, false, false>) \
    HBR_LINEAR(hbr_linear_dx_bf16_##suffix, Tile, waves, linear_d<Tile, Bf16, false, false>) \
    HBR_LINEAR(hbr_linear_dx_part_##suffix, Tile, waves, linear_d<Tile, F32, false, true>) \
    HBR_LINEAR(hbr_linear_dw_f32_##suffix, Tile, waves, linear_d<Tile, F32, true, false>) \
    HBR_LINEAR(hbr_linear_dw_bf16_##suffix, Tile, waves, linear_d<Tile, Bf16, true, false>) \
    HBR_LINEAR(hbr_linear_dw_part_##suffix, Tile, waves, linear_d<Tile, F32, true, true>)
using Tile256 = HeadTile<8>;
using Tile128 = HeadTile<4>;
using Tile128Deep = HeadTile<4, 8>;
HBR_LINEARS(256, Tile256, 2)
HBR_LINEARS(128, Tile128, 4)
HBR_LINEARS(128_deep, Tile128Deep, 1)

extern "C" __global__ __launch_bounds__(256) void hbr_linear_join_f32(LinearJoinArgs a) { linear_join<F32>(a); }
extern "C" __global__ __launch_bounds__(256) void hbr_linear_join_bf16(LinearJoinArgs a) { linear_join<Bf16>(a); }
#define HBR_STRIPS(t, E, v, Wide)                                                                                                   \
    extern "C" __global__ __launch_bounds__(256) void hbr_linear_low_##t##_##v(LinearLowArgs a) { linear_low<E, Wide>(a); }         \
    extern "C" __global__ __launch_bounds__(256) void hbr_linear_few_##t##_##v##_16(LinearFewArgs a) { linear_few<E, 1, Wide>(a); } \
    extern "C" __global__ __launch_bounds__(256) void hbr_linear_few_##t##_##v##_32(LinearFewArgs a) { linear_few<E, 2, Wide>(a); } \
    extern "C" __global__ __launch_bounds__(256) void hbr_linear_few_##t##_##v##_64(LinearFewArgs a) { linear_few<E, 4, Wide>(a); }
HBR_STRIPS(f32, F32, 1, false)
HBR_STRIPS(f32, F32, 4, true)
HBR_STRIPS(bf16, Bf16, 1, false)
HBR_STRIPS(bf16, Bf16, 8, true)
extern "C" __global__ __launch_bounds__(256) void hbr_lay_codes(LayCodesArgs a) { lay_codes(a); }
extern "C" __global__ __launch_bounds__(256) void hbr_column_sum_f32(ColumnSumArgs a) { column_sum<F32>(a); }
extern "C" __global__ __launch_bounds__(256) void hbr_column_sum_bf16(ColumnSumArgs a) { column_sum<Bf16>(a); }
