// Leaf vectors: a table looked up by each row's ids, scaled by column and
// summed, and the table's gradient.
#include "common.h"

namespace hbr {

__device__ __forceinline__ float bf16_f32(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }

// To nearest, ties to even; a NaN stays one.
__device__ __forceinline__ uint16_t f32_bf16(float f) {
    const uint32_t u = __float_as_uint(f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40u);
    return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}

struct F32 {
    using type = float;
    static __device__ __forceinline__ float up(float v) { return v; }
    static __device__ __forceinline__ float down(float v) { return v; }
};
struct Bf16 {
    using type = uint16_t;
    static __device__ __forceinline__ float up(uint16_t v) { return bf16_f32(v); }
    static __device__ __forceinline__ uint16_t down(float v) { return f32_bf16(v); }
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
    T v[V];
};

// The table row of an id of column t; at or past table_rows when it adds
// nothing (a negative id, or one that leads out of the table).
__device__ __forceinline__ uint64_t table_row(int32_t id, const int32_t *offset, uint32_t t, uint64_t table_rows) {
    const int64_t row = (int64_t)id + (offset ? offset[t] : 0);
    return id < 0 || row < 0 || (uint64_t)row >= table_rows ? table_rows : (uint64_t)row;
}

// A thread holds one vector of one row's sum and walks the columns in order,
// kAhead look-ups in flight.
template <typename E, int V>
__device__ __forceinline__ void leaf_embed(const EmbedArgs &a) {
    using T = typename E::type;
    constexpr uint32_t kAhead = 8;
    const uint64_t blocks = (a.n_rows + a.rows_per_block - 1) / a.rows_per_block;
    const uint32_t cells = a.rows_per_block * a.vecs;
    for (uint64_t b = blockIdx.x; b < blocks; b += gridDim.x) {
        for (uint32_t i = threadIdx.x; i < cells; i += 256) {
            const uint64_t r = b * a.rows_per_block + i / a.vecs;
            const uint32_t c = i % a.vecs * V;
            if (r >= a.n_rows) break;
            const int32_t *ids = a.ids + r * a.ids_stride;
            const T *table = static_cast<const T *>(a.table) + c;
            float acc[V] = {};
            for (uint32_t t0 = 0; t0 < a.columns; t0 += kAhead) {
                uint64_t row[kAhead];
                Vec<T, V> v[kAhead];
#pragma unroll
                for (uint32_t j = 0; j < kAhead; j++)
                    row[j] = t0 + j < a.columns ? table_row(ids[t0 + j], a.offset, t0 + j, a.table_rows) : a.table_rows;
#pragma unroll
                for (uint32_t j = 0; j < kAhead; j++)
                    if (row[j] < a.table_rows)
                        v[j] = *reinterpret_cast<const Vec<T, V> *>(table + row[j] * a.table_stride);
#pragma unroll
                for (uint32_t j = 0; j < kAhead; j++) {
                    if (row[j] >= a.table_rows) continue;
                    const float s = a.scale ? a.scale[t0 + j] : 1.0f;
#pragma unroll
                    for (int k = 0; k < V; k++) acc[k] = __builtin_fmaf(s, E::up(v[j].v[k]), acc[k]);
                }
            }
            Vec<T, V> out;
#pragma unroll
            for (int k = 0; k < V; k++) out.v[k] = E::down(acc[k]);
            *reinterpret_cast<Vec<T, V> *>(static_cast<T *>(a.out) + r * a.out_stride + c) = out;
        }
    }
}

// ---- entries sorted by table row ---------------------------------------------------

// Entry i's key in this pass's input; the first pass makes it from the ids.
__device__ __forceinline__ uint32_t sort_key(const LookupSortArgs &a, uint32_t i) {
    if (a.keys_in) return a.keys_in[i];
    const uint32_t r = i / a.columns, t = i - r * a.columns;
    return (uint32_t)table_row(a.ids[(uint64_t)r * a.ids_stride + t], a.offset, t, a.table_rows);
}

}  // namespace hbr

using namespace hbr;

#define HBR_EMBED(name, E, V) \
    extern "C" __global__ __launch_bounds__(256) void name(EmbedArgs a) { leaf_embed<E, V>(a); }
HBR_EMBED(hbr_leaf_embed_f32_4, F32, 4)
HBR_EMBED(hbr_leaf_embed_f32_2, F32, 2)
HBR_EMBED(hbr_leaf_embed_f32_1, F32, 1)
HBR_EMBED(hbr_leaf_embed_bf16_8, Bf16, 8)
HBR_EMBED(hbr_leaf_embed_bf16_4, Bf16, 4)
HBR_EMBED(hbr_leaf_embed_bf16_2, Bf16, 2)
HBR_EMBED(hbr_leaf_embed_bf16_1, Bf16, 1)

// A tile's entries counted by the pass's digit (integer counts: any order).
extern "C" __global__ __launch_bounds__(256) void hbr_sort_count(LookupSortArgs a) {
    __shared__ uint32_t count[kSortDigits];
    count[threadIdx.x] = 0;
    __syncthreads();
    const uint32_t base = blockIdx.x * kSortTile;
    for (uint32_t j = 0; j < kSortTile / 256; j++) {
        const uint32_t i = base + j * 256 + threadIdx.x;
        if (i < a.n) atomicAdd(&count[(sort_key(a, i) >> a.shift) & (kSortDigits - 1)], 1u);
    }
    __syncthreads();
    a.hist[(uint64_t)threadIdx.x * a.tiles + blockIdx.x] = count[threadIdx.x];
}

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

// A tile's entries to their places, in order within a digit: wave w holds the
// tile's w-th quarter, 64 entries a step; a lane's rank is the lanes below it
// with its digit (eight ballots), behind the wave's earlier steps.
extern "C" __global__ __launch_bounds__(256) void hbr_sort_scatter(LookupSortArgs a) {
    constexpr uint32_t kWaves = 256 / kWave, kSteps = kSortTile / 256;
    __shared__ uint32_t count[kWaves][kSortDigits];
    const uint32_t lane = lane_id(), wave = threadIdx.x / kWave, d = threadIdx.x;
    for (uint32_t w = 0; w < kWaves; w++) count[w][d] = 0;
    uint32_t all;
    const uint32_t digit_at = block_exclusive_scan<256>(a.total[d], &all) + a.hist[(uint64_t)d * a.tiles + blockIdx.x];
    __syncthreads();
    const uint32_t base = blockIdx.x * kSortTile + wave * (kSortTile / kWaves);
    uint32_t key[kSteps], rank[kSteps];
#pragma unroll
    for (uint32_t j = 0; j < kSteps; j++) {
        const uint32_t i = base + j * kWave + lane;
        const bool in = i < a.n;
        key[j] = in ? sort_key(a, i) : 0;
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
    uint32_t at = digit_at;
    for (uint32_t w = 0; w < kWaves; w++) {
        const uint32_t c = count[w][d];
        count[w][d] = at;
        at += c;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t j = 0; j < kSteps; j++) {
        const uint32_t i = base + j * kWave + lane;
        if (i >= a.n) continue;
        const uint32_t p = count[wave][(key[j] >> a.shift) & (kSortDigits - 1)] + rank[j];
        a.keys_out[p] = key[j];
        a.vals_out[p] = a.vals_in ? a.vals_in[i] : i;
    }
}

// Where each table row's entries begin (the first entry whose key is not below it).
extern "C" __global__ __launch_bounds__(256) void hbr_lookup_starts(LookupSumArgs a) {
    for (uint64_t v = (uint64_t)blockIdx.x * 256 + threadIdx.x; v <= a.table_rows; v += (uint64_t)gridDim.x * 256) {
        uint32_t lo = 0, hi = a.n;
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (a.keys[mid] < v) lo = mid + 1;
            else hi = mid;
        }
        a.start[v] = lo;
    }
}

namespace hbr {

// One wave a chunk of the sorted entries. A run of equal keys is summed by
// the wave's lane groups (each a row's vectors wide, every group an entry of
// its own) and folded over the groups; a run inside the chunk is a table
// row's whole sum and is written at once, one that reaches the chunk's start
// or end leaves its part in f32.
template <typename E, int V>
__device__ __forceinline__ void lookup_sum(const LookupSumArgs &a) {
    using T = typename E::type;
    const uint32_t lane = lane_id(), wave = threadIdx.x / kWave;
    const uint32_t chunk = blockIdx.x * (256 / kWave) + wave;
    if (chunk >= a.chunks) return;
    const uint32_t valid = a.start[a.table_rows];
    const uint32_t c0 = chunk * a.chunk;
    const uint32_t c1 = min(c0 + a.chunk, valid);
    uint32_t wide = 1;  // lanes a row: the power of two that covers its vectors, at most the wave
    while (wide < a.vecs && wide < (uint32_t)kWave) wide <<= 1;
    const uint32_t groups = kWave / wide, group = lane / wide, in_group = lane & (wide - 1);
    for (uint32_t i = c0; i < c1;) {
        const uint32_t key = a.keys[i];
        const uint32_t first = a.start[key], end = a.start[key + 1];
        const uint32_t e = min(end, c1);
        const bool whole = first >= c0 && end <= c0 + a.chunk;
        for (uint32_t c = in_group; c - in_group < a.vecs; c += wide) {
            float acc[V] = {};
            if (c < a.vecs) {
                for (uint32_t j = i + group; j < e; j += groups) {
                    const uint32_t entry = a.vals[j];
                    const uint32_t r = entry / a.columns, t = entry - r * a.columns;
                    const float s = a.scale ? a.scale[t] : 1.0f;
                    const Vec<T, V> v = *reinterpret_cast<const Vec<T, V> *>(static_cast<const T *>(a.dout) +
                                                                             r * a.dout_stride + c * V);
#pragma unroll
                    for (int k = 0; k < V; k++) acc[k] = __builtin_fmaf(s, E::up(v.v[k]), acc[k]);
                }
            }
            for (uint32_t d = wide; d < (uint32_t)kWave; d <<= 1)
#pragma unroll
                for (int k = 0; k < V; k++) acc[k] += __shfl_xor(acc[k], d, kWave);
            if (group == 0 && c < a.vecs) {
                if (whole) {
                    Vec<T, V> out;
#pragma unroll
                    for (int k = 0; k < V; k++) out.v[k] = E::down(acc[k]);
                    *reinterpret_cast<Vec<T, V> *>(static_cast<T *>(a.dtable) + key * a.dtable_stride + c * V) = out;
                } else {
                    float *p = a.part + ((uint64_t)chunk * 2 + (i == c0 ? 0 : 1)) * a.dim + c * V;
#pragma unroll
                    for (int k = 0; k < V; k++) p[k] = acc[k];
                }
            }
        }
        i = e;
    }
}

// The table rows that no chunk wrote: zeros where no entry is, the parts in
// order where the entries lie in several chunks.
template <typename E, int V>
__device__ __forceinline__ void lookup_finish(const LookupSumArgs &a) {
    using T = typename E::type;
    const uint64_t cells = a.table_rows * a.vecs;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < cells; i += (uint64_t)gridDim.x * 256) {
        const uint64_t v = i / a.vecs;
        const uint32_t c = (uint32_t)(i - v * a.vecs) * V;
        const uint32_t s = a.start[v], e = a.start[v + 1];
        float acc[V] = {};
        if (s < e) {
            const uint32_t first = s / a.chunk, last = (e - 1) / a.chunk;
            if (first == last) continue;
            for (uint32_t q = first; q <= last; q++) {
                const float *p = a.part + ((uint64_t)q * 2 + (q == first && s != q * a.chunk ? 1 : 0)) * a.dim + c;
#pragma unroll
                for (int k = 0; k < V; k++) acc[k] += p[k];
            }
        }
        Vec<T, V> out;
#pragma unroll
        for (int k = 0; k < V; k++) out.v[k] = E::down(acc[k]);
        *reinterpret_cast<Vec<T, V> *>(static_cast<T *>(a.dtable) + v * a.dtable_stride + c) = out;
    }
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
