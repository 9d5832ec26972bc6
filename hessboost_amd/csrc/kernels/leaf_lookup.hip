// Leaf vectors: a table looked up by each row's ids, scaled by column and
// summed, and the table's gradient.
#include "elements.h"

namespace hbr {

// The table row of an id of column t; table_rows when it adds nothing (a
// negative id, or one that leads out of the column's rows). With offsets
// column t holds the rows from offset[t] up to the next column's, the last
// up to the table's end.
__device__ __forceinline__ uint64_t table_row(int32_t id, const int32_t *offset, uint32_t t, uint32_t columns,
                                              uint64_t table_rows) {
    int64_t row = id, end = (int64_t)table_rows;
    if (offset) {
        row += offset[t];
        if (t + 1 < columns) end = min(end, (int64_t)offset[t + 1]);
    }
    return id < 0 || row < 0 || row >= end ? table_rows : (uint64_t)row;
}

__device__ __forceinline__ uint32_t nowhere() { return 0x80000000u; }  // past every buffer: reads as zero

// A workgroup takes rows_per_block rows and places their ids in LDS as the
// byte offsets of their table rows, kPlaces of them and kPlaceColumns columns
// at a time; a thread then holds one
// vector of one row's sum and walks the columns in order, eight look-ups in
// flight. What an id costs (its check, its address) is paid once and not by
// every vector of its row, and an id that adds nothing reads past the
// buffer's end, as zeros. Far: tables of 2 GiB and more hold row numbers
// there, and the addresses are made in 64 bits.
//
// Bound by the vectors that the L2 gives to the CUs and by their unpacking
// (two instructions an element, 65 us of the following): 200,003 rows x 100 ids
// of 64 bf16 out of 12,700 rows take 112 us, 22.8 TB/s of vectors (143 with a
// branch around each scale and a check in 64 bits of each id); the ids alone
// are 16 us of HBM. 32 rows x 100 ids of 32 f32: 10 us, latency.
constexpr uint32_t kPlaces = 4096, kPlaceColumns = 1024;
template <typename E, int V, bool Far>
__device__ __forceinline__ void leaf_embed(const EmbedArgs &a) {
    using T = typename E::type;
    constexpr uint32_t kAhead = 8;
    // f32 sums eight columns by themselves first: a sum of 100 in order is off
    // by 1.7e-7 of it, so by 0.9e-7. A bf16 result's own rounding is 2^-8.
    constexpr bool kEights = sizeof(T) == 4;
    __shared__ __align__(16) uint32_t place[kPlaces];
    __shared__ __align__(16) float scale[kPlaceColumns];
    __shared__ uint32_t first[kPlaceColumns], end[kPlaceColumns];  // the columns' table rows
    const uint64_t blocks = (a.n_rows + a.rows_per_block - 1) / a.rows_per_block;
    const uint32_t cells = a.rows_per_block * a.vecs, wide = a.columns_per_pass;
    const uint32_t inverse = 0xffffffffu / wide + 1;  // q / wide = q inverse / 2^32 for q < kPlaces
    const uint32_t row_bytes = (uint32_t)(a.table_stride * sizeof(T));
    __amdgpu_buffer_rsrc_t table = __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(a.table), 0, 0x7fffffff, 0x00020000);
    for (uint64_t b = blockIdx.x; b < blocks; b += gridDim.x) {
        const uint64_t r0 = b * a.rows_per_block;
        const uint32_t rows = (uint32_t)min((uint64_t)a.rows_per_block, a.n_rows - r0);
        for (uint32_t i0 = 0; i0 < cells; i0 += 256) {
            const uint32_t i = i0 + threadIdx.x, in = i / a.vecs, c = i % a.vecs * V;
            const bool live = i < cells && in < rows;
            float acc[V] = {};
            for (uint32_t t0 = 0; t0 < a.columns; t0 += wide) {
                if (t0 || i0 || b != blockIdx.x) __syncthreads();
                for (uint32_t q = threadIdx.x; q < wide; q += 256) {
                    const uint32_t t = t0 + q;
                    const bool is = t < a.columns;
                    scale[q] = !is ? 0.0f : a.scale ? a.scale[t] : 1.0f;
                    first[q] = is && a.offset ? (uint32_t)a.offset[t] : 0;
                    int64_t to = is ? (int64_t)a.table_rows : 0;
                    if (a.offset && t + 1 < a.columns) to = max((int64_t)0, min(to, (int64_t)a.offset[t + 1]));
                    end[q] = (uint32_t)to;
                }
                __syncthreads();
                for (uint32_t q = threadIdx.x; q < wide * a.rows_per_block; q += 256) {
                    // a row below the table's is 2^31 or more here, and past
                    // every end; one beyond 2^31 - 1 stays so
                    const uint32_t row = __umulhi(q, inverse), t = q - row * wide;
                    const int32_t id = a.ids[(r0 + min(row, rows - 1)) * a.ids_stride + min(t0 + t, a.columns - 1)];
                    const uint32_t v = (uint32_t)id + first[t];
                    place[q] = id < 0 || v >= end[t] ? nowhere() : Far ? v : v * row_bytes;
                }
                __syncthreads();
                if (!live) continue;
                const uint32_t here = min(wide, (a.columns - t0 + kAhead - 1) / kAhead * kAhead);
                for (uint32_t t = 0; t < here; t += kAhead) {
                    uint32_t at[kAhead];
                    float by[kAhead];
                    Vec<T, V> v[kAhead];
#pragma unroll
                    for (uint32_t j = 0; j < kAhead; j++) {
                        at[j] = place[in * wide + t + j];
                        by[j] = scale[t + j];
                    }
#pragma unroll
                    for (uint32_t j = 0; j < kAhead; j++) {
                        if constexpr (Far) {
                            if (at[j] != nowhere())
                                v[j] = *reinterpret_cast<const Vec<T, V> *>(static_cast<const T *>(a.table) +
                                                                             at[j] * a.table_stride + c);
                            else
                                v[j] = Vec<T, V>{};
                        } else {
                            v[j] = buffer_vec<T, V>(table, at[j] + c * (uint32_t)sizeof(T));
                        }
                    }
                    float part[V];
#pragma unroll
                    for (int k = 0; k < V; k++) part[k] = kEights ? 0.0f : acc[k];
#pragma unroll
                    for (uint32_t j = 0; j < kAhead; j++) {
                        const float s = at[j] == nowhere() ? 0.0f : by[j];  // whatever the column's scale
#pragma unroll
                        for (int k = 0; k < V; k++) part[k] = __builtin_fmaf(s, E::up(v[j].v[k]), part[k]);
                    }
#pragma unroll
                    for (int k = 0; k < V; k++) acc[k] = kEights ? acc[k] + part[k] : part[k];
                }
            }
            if (!live) continue;
            Vec<T, V> out;
#pragma unroll
            for (int k = 0; k < V; k++) out.v[k] = E::down(acc[k]);
            *reinterpret_cast<Vec<T, V> *>(static_cast<T *>(a.out) + (r0 + in) * a.out_stride + c) = out;
        }
    }
}

// ---- the gradient, a column at a time ----------------------------------------------------

// A workgroup takes one column, one block of rows and one slice of the
// vectors. Its ids are sorted in LDS, in order within a key: a wave holds
// consecutive rows, a lane's rank among the wave's rows of its
// key is a count of matching ballots behind the wave's count so far, and the
// counts of (key, wave) are joined by one scan. The waves then sum even
// shares of the sorted rows as lookup_sum does; a key that reaches over
// shares is joined from LDS. Keys are taken kColumnKeys at a time.
//
// No id is written to memory, and the rows of dout that a block gathers stay
// in the L2 of the XCD that has the block. Bound by instructions (the VALU is
// busy 57% of the time: ranks, and two an element summed) and the gathers:
// 200,003 x 100 ids of 64 bf16 into 12,700 rows 288 us, and 9 to join the
// blocks' sums, 8.9 TB/s of vectors; 4,000 x 20 ids of 16 f32 15 and 4 us.
constexpr uint32_t kColumnThreads = 1024, kColumnWaves = kColumnThreads / kWave;
constexpr uint32_t kColumnSteps = kColumnBlock / kColumnThreads;

template <typename E, int V>
__device__ __forceinline__ void lookup_columns(const LookupColumnArgs &a) {
    using T = typename E::type;
    __shared__ uint32_t count[kColumnWaves][kColumnKeys];  // then the shares' edges
    __shared__ uint16_t list[kColumnBlock];
    __shared__ uint32_t start[kColumnKeys + 1];
    __shared__ uint32_t wave_total[kColumnWaves];
    float(*edge)[2][kColumnSlice] = reinterpret_cast<float(*)[2][kColumnSlice]>(&count[0][0]);
    static_assert(sizeof(float) * 2 * kColumnSlice <= sizeof(uint32_t) * kColumnKeys, "a wave's edges fit its counts");
    // a block's columns and slices on one XCD, one block after the other
    const uint32_t each = a.columns * a.slices;
    uint32_t block = blockIdx.x / each, in = blockIdx.x % each;
    if (a.blocks % 8 == 0) {
        in = blockIdx.x / 8;
        block = in / each * 8 + blockIdx.x % 8;
        in %= each;
    }
    const uint32_t t = in / a.slices, slice = in % a.slices;
    const uint64_t r0 = (uint64_t)block * a.block_rows;
    const uint32_t m = r0 < a.n_rows ? (uint32_t)min((uint64_t)a.block_rows, a.n_rows - r0) : 0;
    // the column's table rows; the first column's begin with the table
    int64_t lo = 0, hi = (int64_t)a.table_rows, off = 0;
    if (a.offset) {
        off = a.offset[t];
        if (t) lo = max(off, (int64_t)0);
        if (t + 1 < a.columns) hi = min(hi, (int64_t)a.offset[t + 1]);
    }
    const float scale = a.scale ? a.scale[t] : 1.0f;
    // the slice's vectors on the lanes of a group
    const uint32_t v0 = slice * a.slice_vecs, vecs = min(a.slice_vecs, a.vecs - v0);
    uint32_t wide = 1;
    while (wide < vecs) wide <<= 1;
    const uint32_t groups = kWave / wide, group = lane_id() / wide, c = lane_id() & (wide - 1);
    const bool live = c < vecs;
    // a block's rows lie within 2 GiB
    __amdgpu_buffer_rsrc_t dout = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<T *>(static_cast<const T *>(a.dout) + r0 * a.dout_stride), 0, 0x7fffffff, 0x00020000);
    __amdgpu_buffer_rsrc_t ids = __builtin_amdgcn_make_buffer_rsrc(const_cast<int32_t *>(a.ids + r0 * a.ids_stride + t), 0,
                                                                   0x7fffffff, 0x00020000);
    const uint32_t dout_stride = (uint32_t)(a.dout_stride * sizeof(T)), ids_stride = (uint32_t)(a.ids_stride * 4);
    const uint32_t dout_at = (v0 + c) * (uint32_t)(V * sizeof(T));
    auto write = [&](uint64_t row, const float(&acc)[V], float by) {
        if (a.blocks == 1) {
            Vec<T, V> out;
#pragma unroll
            for (int k = 0; k < V; k++) out.v[k] = E::down(by * acc[k]);
            *reinterpret_cast<Vec<T, V> *>(static_cast<T *>(a.dtable) + row * a.dtable_stride + (v0 + c) * V) = out;
        } else {
            Vec<float, V> out;
#pragma unroll
            for (int k = 0; k < V; k++) out.v[k] = by * acc[k];
            *reinterpret_cast<Vec<float, V> *>(a.part + ((uint64_t)block * a.table_rows + row) * a.part_stride + (v0 + c) * V) = out;
        }
    };
    for (int64_t k0 = lo; k0 < hi; k0 += kColumnKeys) {
        // made anew each round: what a compiler would keep of them over the
        // rounds does not fit the registers
        uint32_t thread = threadIdx.x;
        asm volatile("" : "+v"(thread));
        const uint32_t lane = thread % kWave, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(thread / kWave));
        const uint32_t keys = (uint32_t)min((int64_t)kColumnKeys, hi - k0);
        for (uint32_t k = lane; k < keys; k += kWave) count[wave][k] = 0;  // its own: before its own counts
        const uint32_t wave_rows = (a.block_rows + kColumnThreads - 1) / kColumnThreads * kWave;
        uint32_t held[kColumnSteps];  // the key, and the rank in the upper half
        uint32_t bits = 0;
        while ((1u << bits) < keys) bits++;
#pragma unroll
        for (uint32_t j = 0; j < kColumnSteps; j++) {
            const uint32_t i = wave * wave_rows + j * kWave + lane;
            held[j] = 0xffffffffu;
            if (j * kWave < wave_rows && i < m) held[j] = __builtin_amdgcn_raw_buffer_load_b32(ids, i * ids_stride, 0, 0);
        }
#pragma unroll
        for (uint32_t j = 0; j < kColumnSteps; j++) {
            const int64_t key = off + (int32_t)held[j] - k0;
            held[j] = (int32_t)held[j] >= 0 && key >= 0 && key < keys ? (uint32_t)key : 0xffffffffu;
        }
#pragma unroll
        for (uint32_t j = 0; j < kColumnSteps; j++) {
            if (j * kWave >= wave_rows) continue;
            const bool ok = held[j] != 0xffffffffu;
            const uint32_t key = ok ? held[j] : 0;
            uint64_t same = __ballot(ok);
#pragma unroll 1
            for (uint32_t bit = 0; bit < bits; bit++) {
                const uint64_t set = __ballot(ok && ((key >> bit) & 1u));
                same &= (key >> bit) & 1u ? set : ~set;
            }
            const uint64_t below = same & ((1ull << lane) - 1);
            volatile uint32_t *mine = &count[wave][key];
            const uint32_t before = *mine;
            __builtin_amdgcn_wave_barrier();
            if (ok && below == 0) *mine = before + (uint32_t)__popcll(same);
            __builtin_amdgcn_wave_barrier();
            if (ok) held[j] = key | (before + (uint32_t)__popcll(below)) << 16;
        }
        __syncthreads();
        // each key's total over the waves, their scan, and the waves' places
        uint32_t total = 0;
        if (thread < keys)
#pragma unroll 8
            for (uint32_t w = 0; w < kColumnWaves; w++) total += count[w][thread];
        uint32_t upto = total;
#pragma unroll 1
        for (uint32_t d = 1; d < (uint32_t)kWave; d <<= 1) {
            const uint32_t other = __shfl_up(upto, d, kWave);
            if (lane >= d) upto += other;
        }
        if (lane == kWave - 1) wave_total[wave] = upto;
        __syncthreads();
        uint32_t at = upto - total, all = 0;
#pragma unroll 1
        for (uint32_t w = 0; w < kColumnWaves; w++) {
            if (w == wave) at += all;
            all += wave_total[w];
        }
        if (thread < kColumnKeys) start[thread] = at;
        if (thread < keys) {
#pragma unroll 1
            for (uint32_t w = 0; w < kColumnWaves; w += 8) {
                uint32_t n[8];
#pragma unroll
                for (uint32_t u = 0; u < 8; u++) n[u] = count[w + u][thread];
#pragma unroll
                for (uint32_t u = 0; u < 8; u++) {
                    count[w + u][thread] = at;
                    at += n[u];
                }
            }
        }
        if (thread == 0) start[kColumnKeys] = all;
        __syncthreads();
#pragma unroll
        for (uint32_t j = 0; j < kColumnSteps; j++)
            if (held[j] != 0xffffffffu)
                list[count[wave][held[j] & 0xffffu] + (held[j] >> 16)] =
                    (uint16_t)(wave * wave_rows + j * kWave + lane);
        __syncthreads();
        const uint32_t a0 = (uint32_t)((uint64_t)all * wave / kColumnWaves), a1 = (uint32_t)((uint64_t)all * (wave + 1) / kColumnWaves);
        uint32_t key = 0;
        if (a0 < a1) {  // the key of the share's first row: the last that begins at or before it
            uint32_t low = 0, high = keys;
            while (high - low > 1) {
                const uint32_t mid = (low + high) / 2;
                if (start[mid] <= a0) low = mid;
                else high = mid;
            }
            key = low;
        }
        uint32_t tail = kColumnKeys;  // the key that goes on past the share, if it began in it
        for (uint32_t i = a0; i < a1; key++) {
            const uint32_t s = start[key], end = start[key + 1], e = min(end, a1);
            if (s == end) continue;
            float acc[V] = {};
            if (live) {
                constexpr uint32_t kAhead = 4;
                for (uint32_t j = i + group; j < e; j += kAhead * groups) {
                    Vec<T, V> v[kAhead];
#pragma unroll
                    for (uint32_t u = 0; u < kAhead; u++) {
                        const uint32_t p = j + u * groups;
                        v[u] = buffer_vec<T, V>(dout, p < e ? list[p] * dout_stride + dout_at : nowhere());
                    }
#pragma unroll
                    for (uint32_t u = 0; u < kAhead; u++)
#pragma unroll
                        for (int k = 0; k < V; k++) acc[k] += E::up(v[u].v[k]);
                }
            }
            for (uint32_t d = wide; d < (uint32_t)kWave; d <<= 1)
#pragma unroll
                for (int k = 0; k < V; k++) acc[k] += __shfl_xor(acc[k], d, kWave);
            if (group == 0 && live) {
                if (s >= a0 && end <= a1) {
                    write((uint64_t)(k0 + key), acc, scale);
                } else {
#pragma unroll
                    for (int k = 0; k < V; k++) edge[wave][s < a0 ? 0 : 1][c * V + k] = acc[k];
                }
            }
            if (s >= a0 && end > a1) tail = key;
            i = e;
        }
        __syncthreads();
        if (tail < kColumnKeys && group == 0 && live) {
            float acc[V];
#pragma unroll
            for (int k = 0; k < V; k++) acc[k] = edge[wave][1][c * V + k];
#pragma unroll 1
            for (uint32_t w = wave + 1; w < kColumnWaves; w++) {
                const uint32_t b0 = (uint32_t)((uint64_t)all * w / kColumnWaves), b1 = (uint32_t)((uint64_t)all * (w + 1) / kColumnWaves);
                if (b0 >= start[tail + 1]) break;
                if (b0 == b1) continue;
#pragma unroll
                for (int k = 0; k < V; k++) acc[k] += edge[w][0][c * V + k];
            }
            write((uint64_t)(k0 + tail), acc, scale);
        }
        // rows that nothing leads to
        for (uint32_t k = thread / wide; k < keys; k += kColumnThreads / wide) {
            if (start[k] != start[k + 1] || !live) continue;
            const float none[V] = {};
            write((uint64_t)(k0 + k), none, 1.0f);  // zeros, whatever the scale
        }
        __syncthreads();
    }
}

// The blocks' sums of each table row, in order.
template <typename E, int V>
__device__ __forceinline__ void lookup_join(const LookupColumnArgs &a) {
    using T = typename E::type;
    const uint64_t cells = a.table_rows * a.vecs;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < cells; i += (uint64_t)gridDim.x * 256) {
        const uint64_t row = i / a.vecs;
        const uint32_t c = (uint32_t)(i - row * a.vecs) * V;
        const float *p = a.part + row * a.part_stride + c;
        float acc[V] = {};
        for (uint32_t b = 0; b < a.blocks; b++, p += a.table_rows * a.part_stride) {
            const Vec<float, V> v = *reinterpret_cast<const Vec<float, V> *>(p);
#pragma unroll
            for (int k = 0; k < V; k++) acc[k] += v.v[k];
        }
        Vec<T, V> out;
#pragma unroll
        for (int k = 0; k < V; k++) out.v[k] = E::down(acc[k]);
        *reinterpret_cast<Vec<T, V> *>(static_cast<T *>(a.dtable) + row * a.dtable_stride + c) = out;
    }
}

// ---- entries sorted by table row ---------------------------------------------------

// Entry i's key in this pass's input; the first pass makes it from the ids.
__device__ __forceinline__ uint32_t sort_key(const LookupSortArgs &a, uint32_t i) {
    if (a.keys_in) return a.keys_in[i];
    const uint32_t r = i / a.columns, t = i - r * a.columns;
    return (uint32_t)table_row(a.ids[(uint64_t)r * a.ids_stride + t], a.offset, t, a.columns, a.table_rows);
}

}  // namespace hbr

using namespace hbr;

#define HBR_EMBED(suffix, E, V)                                                                               \
    extern "C" __global__ __launch_bounds__(256) void hbr_leaf_embed_##suffix(EmbedArgs a) {                  \
        leaf_embed<E, V, false>(a);                                                                           \
    }                                                                                                         \
    extern "C" __global__ __launch_bounds__(256) void hbr_leaf_embed_far_##suffix(EmbedArgs a) {              \
        leaf_embed<E, V, true>(a);                                                                            \
    }                                                                                                         \
    extern "C" __global__ __launch_bounds__(kColumnThreads, 8) void hbr_lookup_columns_##suffix(LookupColumnArgs a) { \
        lookup_columns<E, V>(a);                                                                              \
    }                                                                                                         \
    extern "C" __global__ __launch_bounds__(256) void hbr_lookup_join_##suffix(LookupColumnArgs a) {          \
        lookup_join<E, V>(a);                                                                                 \
    }
HBR_EMBED(f32_4, F32, 4)
HBR_EMBED(f32_2, F32, 2)
HBR_EMBED(f32_1, F32, 1)
HBR_EMBED(bf16_8, Bf16, 8)
HBR_EMBED(bf16_4, Bf16, 4)
HBR_EMBED(bf16_2, Bf16, 2)
HBR_EMBED(bf16_1, Bf16, 1)

namespace hbr {

// A tile's entries counted by the pass's digit (integer counts: any order).
template <uint32_t Steps>
__device__ __forceinline__ void sort_count(const LookupSortArgs &a) {
    __shared__ uint32_t count[kSortDigits];
    for (uint32_t d = threadIdx.x; d < kSortDigits; d += 256) count[d] = 0;
    __syncthreads();
    const uint32_t base = blockIdx.x * (Steps * 256);
#pragma unroll
    for (uint32_t j = 0; j < Steps; j++) {
        const uint32_t i = base + j * 256 + threadIdx.x;
        if (i < a.n) atomicAdd(&count[(sort_key(a, i) >> a.shift) & (kSortDigits - 1)], 1u);
    }
    __syncthreads();
    for (uint32_t d = threadIdx.x; d < kSortDigits; d += 256) a.hist[(uint64_t)d * a.tiles + blockIdx.x] = count[d];
}

// A tile's entries to their places, in order within a digit: wave w holds the
// tile's w-th quarter, 64 entries a step; a lane's rank is the lanes below it
// with its digit (a ballot a bit), behind the wave's earlier steps.
template <uint32_t Steps>
__device__ __forceinline__ void sort_scatter(const LookupSortArgs &a) {
    constexpr uint32_t kWaves = 256 / kWave, kEach = kSortDigits / 256;
    __shared__ uint32_t count[kWaves][kSortDigits];
    const uint32_t lane = lane_id(), wave = threadIdx.x / kWave;
    for (uint32_t i = threadIdx.x; i < kWaves * kSortDigits; i += 256) (&count[0][0])[i] = 0;
    // where the digits of this thread begin, over all tiles and for this one
    uint32_t total[kEach], sum = 0, all;
#pragma unroll
    for (uint32_t q = 0; q < kEach; q++) {
        total[q] = a.total[threadIdx.x * kEach + q];
        sum += total[q];
    }
    uint32_t digit_at = block_exclusive_scan<256>(sum, &all);
    const uint32_t base = blockIdx.x * (Steps * 256) + wave * (Steps * kWave);
    uint32_t key[Steps], rank[Steps];
#pragma unroll
    for (uint32_t j = 0; j < Steps; j++) {
        const uint32_t i = base + j * kWave + lane;
        key[j] = i < a.n ? sort_key(a, i) : 0;
    }
#pragma unroll
    for (uint32_t j = 0; j < Steps; j++) {
        const bool in = base + j * kWave + lane < a.n;
        const uint32_t digit = (key[j] >> a.shift) & (kSortDigits - 1);
        uint64_t same = __ballot(in);
#pragma unroll
        for (uint32_t bit = 0; bit < kSortBits; bit++) {
            const uint64_t set = __ballot(in && ((digit >> bit) & 1u));
            same &= (digit >> bit) & 1u ? set : ~set;
        }
        const uint64_t below = same & ((1ull << lane) - 1);
        // the wave's own counts: its LDS accesses keep their order
        volatile uint32_t *mine = &count[wave][digit];
        const uint32_t before = *mine;
        rank[j] = before + (uint32_t)__popcll(below);
        __builtin_amdgcn_wave_barrier();
        if (in && below == 0) *mine = before + (uint32_t)__popcll(same);
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
#pragma unroll
    for (uint32_t q = 0; q < kEach; q++) {
        const uint32_t d = threadIdx.x * kEach + q;
        uint32_t at = digit_at + a.hist[(uint64_t)d * a.tiles + blockIdx.x];
        digit_at += total[q];
        for (uint32_t w = 0; w < kWaves; w++) {
            const uint32_t c = count[w][d];
            count[w][d] = at;
            at += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (uint32_t j = 0; j < Steps; j++) {
        const uint32_t i = base + j * kWave + lane;
        if (i >= a.n) continue;
        const uint32_t p = count[wave][(key[j] >> a.shift) & (kSortDigits - 1)] + rank[j];
        a.keys_out[p] = key[j];
        a.vals_out[p] = a.vals_in ? a.vals_in[i] : i;
    }
}

}  // namespace hbr

extern "C" __global__ __launch_bounds__(256) void hbr_sort_count_2(LookupSortArgs a) { sort_count<2>(a); }
extern "C" __global__ __launch_bounds__(256) void hbr_sort_count_16(LookupSortArgs a) { sort_count<16>(a); }
extern "C" __global__ __launch_bounds__(256) void hbr_sort_scatter_2(LookupSortArgs a) { sort_scatter<2>(a); }
extern "C" __global__ __launch_bounds__(256) void hbr_sort_scatter_16(LookupSortArgs a) { sort_scatter<16>(a); }

// One workgroup a digit: its tiles' counts to places, and the digit's total.
extern "C" __global__ __launch_bounds__(256) void hbr_sort_scan(LookupSortArgs a) {
    uint32_t *h = a.hist + (uint64_t)blockIdx.x * a.tiles;
    uint32_t run = 0;
    for (uint32_t t0 = 0; t0 < a.tiles; t0 += 256) {
        const uint32_t t = t0 + threadIdx.x;
        const uint32_t v = t < a.tiles ? h[t] : 0;
        uint32_t all;
        const uint32_t at = block_exclusive_scan<256>(v, &all);
        if (t < a.tiles) h[t] = run + at;
        run += all;
    }
    if (threadIdx.x == 0) a.total[blockIdx.x] = run;
}

// Few entries, sorted in one workgroup: (key, entry) pairs are all different,
// so that any sort gives their one order (bitonic). The whole gradient of 1,024
// ids of 64 f32 takes 30 us so and 34 with two passes of three launches, of
// 1,500 37 and 34.
extern "C" __global__ __launch_bounds__(1024) void hbr_sort_small(LookupSortArgs a) {
    __shared__ uint64_t pair[kSortSmall];
    uint32_t size = 64;
    while (size < a.n) size <<= 1;
    for (uint32_t i = threadIdx.x; i < size; i += 1024)
        pair[i] = i < a.n ? (uint64_t)sort_key(a, i) << 32 | i : ~0ull;
    for (uint32_t k = 2; k <= size; k <<= 1)
        for (uint32_t d = k / 2; d; d >>= 1) {
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < size / 2; i += 1024) {
                const uint32_t low = i / d * 2 * d + i % d, high = low + d;
                const uint64_t x = pair[low], y = pair[high];
                if ((x > y) == ((low & k) == 0)) pair[low] = y, pair[high] = x;
            }
        }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < a.n; i += 1024) {
        a.keys_out[i] = (uint32_t)(pair[i] >> 32);
        a.vals_out[i] = (uint32_t)pair[i];
    }
}

namespace hbr {

// A chunk of the sorted entries a group of lanes, a vector of the rows a lane:
// eight entries' rows in flight, added up run by run of equal keys. A run that
// the chunk holds whole is its table row's sum and is written at once, one
// that reaches the chunk's start or end leaves its part in f32. One pass over
// dout's rows and the written rows of the table, bound by HBM: 65,536 ids of
// 1,024 bf16 into 131,072 rows 60 us (134 MB read and about 70 written, 3.4
// TB/s), 40 for the zeros of the other rows (5 TB/s), 27 for the sort.
template <typename E, int V>
__device__ __forceinline__ void lookup_sum(const LookupSumArgs &a) {
    using T = typename E::type;
    constexpr uint32_t kAhead = 8, kNone = 0xffffffffu;
    const uint32_t groups = 256 / a.wide, c = blockIdx.y * a.wide + (threadIdx.x & (a.wide - 1));
    const uint32_t chunk = blockIdx.x * groups + threadIdx.x / a.wide;
    if (chunk >= a.chunks || c >= a.vecs) return;  // a chunk has an entry at least
    const uint32_t c0 = chunk * a.chunk, c1 = min(c0 + a.chunk, a.n);
    const uint32_t before = c0 ? a.keys[c0 - 1] : kNone, behind = c1 < a.n ? a.keys[c1] : kNone;
    const T *dout = static_cast<const T *>(a.dout) + c * V;
    uint32_t run = kNone, first = c0;  // the run's key, and where it begins in the chunk
    float acc[V] = {};
    auto flush = [&](uint32_t end) {
        if (run >= a.table_rows) return;  // none, or the ids that add nothing
        if ((first > c0 || run != before) && (end < c1 || run != behind)) {
            Vec<T, V> out;
#pragma unroll
            for (int k = 0; k < V; k++) out.v[k] = E::down(acc[k]);
            *reinterpret_cast<Vec<T, V> *>(static_cast<T *>(a.dtable) + run * a.dtable_stride + c * V) = out;
        } else {
            float *p = a.part + ((uint64_t)chunk * 2 + (first == c0 ? 0 : 1)) * a.dim + c * V;
#pragma unroll
            for (int k = 0; k < V; k++) p[k] = acc[k];
        }
    };
    // Loads without conditions, so that none waits for another: past the
    // chunk its last entry's again, and for an id that adds nothing (behind
    // every other, in a run that is not written) a row like any.
    uint32_t key[kAhead], next_key[kAhead], next_val[kAhead];
    auto entries = [&](uint32_t at) {  // the eight from `at` on, one round ahead of their rows
#pragma unroll
        for (uint32_t u = 0; u < kAhead; u++) {
            next_key[u] = a.keys[min(at + u, c1 - 1)];
            next_val[u] = a.vals[min(at + u, c1 - 1)];
        }
    };
    entries(c0);
    for (uint32_t i0 = c0; i0 < c1; i0 += kAhead) {
        float s[kAhead];
        Vec<T, V> v[kAhead];
#pragma unroll
        for (uint32_t u = 0; u < kAhead; u++) {
            key[u] = next_key[u];
            const uint32_t r = a.columns == 1 ? next_val[u] : next_val[u] / a.columns;
            s[u] = a.scale ? a.scale[next_val[u] - r * a.columns] : 1.0f;
            v[u] = *reinterpret_cast<const Vec<T, V> *>(dout + r * a.dout_stride);
        }
        entries(i0 + kAhead);
#pragma unroll
        for (uint32_t u = 0; u < kAhead; u++) {
            if (i0 + u >= c1) break;
            if (key[u] != run) {
                flush(i0 + u);
                run = key[u];
                first = i0 + u;
#pragma unroll
                for (int k = 0; k < V; k++) acc[k] = 0.0f;
            }
#pragma unroll
            for (int k = 0; k < V; k++) acc[k] = __builtin_fmaf(s[u], E::up(v[u].v[k]), acc[k]);
        }
    }
    flush(c1);
}

// The first entry whose key is not below `key`.
__device__ __forceinline__ uint32_t first_entry(const LookupSumArgs &a, uint64_t key) {
    uint32_t low = 0, high = a.n;
    while (low < high) {
        const uint32_t mid = low + (high - low) / 2;
        if (a.keys[mid] < key) low = mid + 1;
        else high = mid;
    }
    return low;
}

// The table rows that no chunk wrote. The first blocks write zeros where no
// entry is: a wave finds where the entries of 64 rows begin, a search a lane,
// and has the ends of 63. The others join the parts of runs that reach over
// chunks, in order: a group of lanes a chunk (and 64 vectors), for the run
// that begins in it and goes on behind it.
template <typename E, int V>
__device__ __forceinline__ void lookup_finish(const LookupSumArgs &a) {
    using T = typename E::type;
    const uint32_t lane = lane_id(), c0 = lane & (a.wide - 1), groups = kWave / a.wide;
    T *dtable = static_cast<T *>(a.dtable);
    if (blockIdx.x < a.row_blocks) {
        if (blockIdx.y) return;
        const uint64_t r0 = ((uint64_t)blockIdx.x * 4 + threadIdx.x / kWave) * (kWave - 1);
        if (r0 >= a.table_rows) return;
        const uint32_t at = first_entry(a, r0 + lane);
        const uint32_t rows = (uint32_t)min((uint64_t)(kWave - 1), a.table_rows - r0);
        const Vec<T, V> none{};
        for (uint32_t j0 = 0; j0 < rows; j0 += groups) {
            const uint32_t j = j0 + lane / a.wide;
            const uint32_t s = __shfl(at, min(j, 63u), kWave), e = __shfl(at, min(j + 1, 63u), kWave);
            if (j >= rows || s < e) continue;
            for (uint32_t c = c0; c < a.vecs; c += a.wide)
                *reinterpret_cast<Vec<T, V> *>(dtable + (r0 + j) * a.dtable_stride + c * V) = none;
        }
        return;
    }
    const uint32_t chunk = ((blockIdx.x - a.row_blocks) * 4 + threadIdx.x / kWave) * groups + lane / a.wide;
    if (chunk + 1 >= a.chunks) return;  // nothing goes on behind the last
    const uint32_t last = (chunk + 1) * a.chunk;  // the chunk is whole, another follows
    const uint32_t key = a.keys[last - 1];
    if (key >= a.table_rows || a.keys[last] != key) return;
    const uint32_t start = first_entry(a, key), to = (first_entry(a, (uint64_t)key + 1) - 1) / a.chunk;
    if (start < chunk * a.chunk) return;  // it began before
    const uint32_t slot = start != chunk * a.chunk ? 1 : 0, c = blockIdx.y * a.wide + c0;
    if (c >= a.vecs) return;
    float acc[V];
    const float *p = a.part + ((uint64_t)chunk * 2 + slot) * a.dim + c * V;
#pragma unroll
    for (int k = 0; k < V; k++) acc[k] = p[k];
#pragma unroll 8
    for (uint32_t q = chunk + 1; q <= to; q++) {
        p = a.part + (uint64_t)q * 2 * a.dim + c * V;
#pragma unroll
        for (int k = 0; k < V; k++) acc[k] += p[k];
    }
    Vec<T, V> out;
#pragma unroll
    for (int k = 0; k < V; k++) out.v[k] = E::down(acc[k]);
    *reinterpret_cast<Vec<T, V> *>(dtable + key * a.dtable_stride + c * V) = out;
}

}  // namespace hbr

#define HBR_LOOKUP(suffix, E, V)                                                                             \
    extern "C" __global__ __launch_bounds__(256) void hbr_lookup_sum_##suffix(LookupSumArgs a) {             \
        lookup_sum<E, V>(a);                                                                                 \
    }                                                                                                        \
    extern "C" __global__ __launch_bounds__(256) void hbr_lookup_finish_##suffix(LookupSumArgs a) {          \
        lookup_finish<E, V>(a);                                                                              \
    }
HBR_LOOKUP(f32_4, F32, 4)
HBR_LOOKUP(f32_2, F32, 2)
HBR_LOOKUP(f32_1, F32, 1)
HBR_LOOKUP(bf16_8, Bf16, 8)
HBR_LOOKUP(bf16_4, Bf16, 4)
HBR_LOOKUP(bf16_2, Bf16, 2)
HBR_LOOKUP(bf16_1, Bf16, 1)
