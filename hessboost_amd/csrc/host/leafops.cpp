#include "leafops.h"

#include <algorithm>
#include <cmath>
#include <string>
#include <vector>

#include "../abi.h"

namespace hbr {

namespace {

constexpr uint32_t kWaveLanes = 64;

uint64_t up(uint64_t v, uint64_t to) { return (v + to - 1) / to * to; }

// A workspace handed out from its start, 256 bytes apart. Without memory it
// only counts. An array may have more room than the call at hand uses.
struct Arena {
    char *base;
    uint64_t used = 0;
    explicit Arena(void *p) : base(static_cast<char *>(p)) {}
    template <typename T>
    T *take(uint64_t n, uint64_t used_of_it = 0) {
        if (used_of_it > n) fail(kRefused, "a workspace has no room for the plan");
        T *p = base ? reinterpret_cast<T *>(base + used) : nullptr;
        used += up(n * sizeof(T), 256);
        return p;
    }
};

// The caller's stream, with its device current while the call runs and the
// thread's own device current again behind it.
class Queue {
public:
    Queue(int ordinal, void *stream) : stream_(static_cast<hipStream_t>(stream)) {
        if (hipGetDevice(&before_) != hipSuccess) before_ = -1;
        try {
            device_ = &device(ordinal);
            hipDevice_t of = ordinal;
            if (stream_) HBR_HIP(hipStreamGetDevice(stream_, &of));
            if (of != ordinal) fail(kInvalid, "the stream is not one of device " + std::to_string(ordinal));
        } catch (...) {
            restore();
            throw;
        }
    }
    ~Queue() { restore(); }
    Queue(const Queue &) = delete;
    Queue &operator=(const Queue &) = delete;
    template <typename Args>
    void launch(const char *kernel, dim3 grid, dim3 block, const Args &args, uint32_t lds_bytes = 0) {
        if ((uint64_t)grid.x * block.x > 0xffffffffull) fail(kRefused, std::string(kernel) + ": more than 2^32 - 1 threads");
        device_->launch_on(stream_, kernel, grid, block, args, lds_bytes);
    }

private:
    void restore() {
        if (before_ >= 0) (void)hipSetDevice(before_);
    }
    int before_ = -1;
    Device *device_ = nullptr;
    hipStream_t stream_;
};

uint64_t size_of(uint32_t dtype, const char *what) {
    if (dtype == HBR_F32) return 4;
    if (dtype == HBR_BF16) return 2;
    fail(kInvalid, std::string(what) + ": the type is neither HBR_F32 nor HBR_BF16");
}

void check_workspace(const void *p, uint64_t have, uint64_t need, const char *what) {
    if (need == 0) return;
    if (!p || have < need)
        fail(kInvalid, std::string(what) + ": the workspace holds " + std::to_string(p ? have : 0) + " bytes of " +
                           std::to_string(need));
    if (reinterpret_cast<uint64_t>(p) % 16)
        fail(kInvalid, std::string(what) + ": the workspace is not aligned to 16 bytes");
}

void check_aligned(const void *p, uint64_t size, const char *what) {
    if (reinterpret_cast<uint64_t>(p) % size)
        fail(kInvalid, std::string(what) + ": an array is not aligned to its elements");
}

// An array's bytes: rows of `width`, `stride` apart.
struct Extent {
    uint64_t begin, rows, width, stride;
    Extent(const void *p, uint64_t n) : Extent(p, 1, n, n) {}
    Extent(const void *p, uint64_t n_rows, uint64_t row, uint64_t step)
        : begin(reinterpret_cast<uint64_t>(p)), rows(p && row ? n_rows : 0), width(row), stride(n_rows > 1 ? step : row) {}
    uint64_t end() const { return begin + (rows - 1) * stride + width; }
};

// Whether two arrays share a byte. Rows of one stride may lie between each
// other's; of two arrays with gaps of different strides it is not found out.
bool overlap(const Extent &a, const Extent &b) {
    if (!a.rows || !b.rows || a.begin >= b.end() || b.begin >= a.end()) return false;
    if (a.stride == b.stride) {
        const uint64_t by = b.begin >= a.begin ? (b.begin - a.begin) % a.stride
                                               : (a.stride - (a.begin - b.begin) % a.stride) % a.stride;
        return by < a.width || by + b.width > a.stride;
    }
    const bool a_whole = a.width == a.stride;
    if (!a_whole && b.width != b.stride) return false;
    const Extent &whole = a_whole ? a : b, &rows = a_whole ? b : a;
    // the first of the rows that ends behind the whole array's begin
    const uint64_t first = rows.begin + rows.width > whole.begin ? 0 : (whole.begin - rows.begin - rows.width) / rows.stride + 1;
    return first < rows.rows && rows.begin + first * rows.stride < whole.end();
}

void check_apart(std::initializer_list<Extent> outputs, std::initializer_list<Extent> inputs, const Extent &workspace, const char *what) {
    for (const auto &list : {outputs, inputs})
        for (const Extent &a : list)
            if (overlap(a, workspace)) fail(kInvalid, std::string(what) + ": an array lies in the memory for the call's own use");
    for (auto o = outputs.begin(); o != outputs.end(); o++) {
        for (auto other = outputs.begin(); other != o; other++)
            if (overlap(*o, *other)) fail(kInvalid, std::string(what) + ": two outputs overlap");
        for (const Extent &i : inputs)
            if (overlap(*o, i)) fail(kInvalid, std::string(what) + ": an output overlaps an input");
    }
}

// The widest vector (elements, at most 16 bytes) that divides every row
// length, stride and address.
uint32_t vector_width(uint64_t size, std::initializer_list<uint64_t> lengths, std::initializer_list<const void *> ptrs) {
    uint32_t v = (uint32_t)(16 / size);
    for (; v > 1; v /= 2) {
        bool ok = true;
        for (uint64_t n : lengths) ok = ok && n % v == 0;
        for (const void *p : ptrs) ok = ok && reinterpret_cast<uint64_t>(p) % (v * size) == 0;
        if (ok) break;
    }
    return v;
}

// Vectors and inputs are shorter, so that offsets within one fit 32 bits and
// grids over their elements a launch.
constexpr uint64_t kDimLimit = 1u << 20;

const char *name_of(uint32_t dtype) { return dtype == HBR_F32 ? "f32" : "bf16"; }

// ---- leaf vectors ------------------------------------------------------------------

void check_lookup(const hbr_lookup &p, const char *what) {
    size_of(p.dtype, what);
    if (p.dim == 0) fail(kInvalid, std::string(what) + ": vectors of no elements");
    if (p.dim >= kDimLimit) fail(kRefused, std::string(what) + ": vectors of 1,048,576 elements or more");
    if (p.n_rows && p.n_columns && !p.ids) fail(kInvalid, std::string(what) + ": null ids");
    if (p.n_rows > 1 && p.ids_stride < p.n_columns) fail(kInvalid, std::string(what) + ": the rows of ids overlap");
    if (p.table_rows > 1 && p.table_stride < p.dim) fail(kInvalid, std::string(what) + ": the table's rows overlap");
    if (p.n_rows > 1 && p.out_stride < p.dim) fail(kInvalid, std::string(what) + ": the rows' vectors overlap");
    check_aligned(p.ids, 4, what);
    check_aligned(p.offset, 4, what);
    check_aligned(p.scale, 4, what);
    // (the kernels count columns by passes in 32 bits)
    if (p.table_rows > 0x7fffffffull || p.n_rows > 0x7fffffffull || p.n_columns > 0x7fffffffu)
        fail(kRefused, std::string(what) + ": more than 2^31 - 1 rows or columns");
}

// The table (or its gradient), the rows' vectors, and what leads from the one to the other.
void check_lookup_apart(const hbr_lookup &p, const void *table, const void *vectors, bool out, const Extent &workspace, const char *what) {
    const uint64_t size = size_of(p.dtype, what);
    const Extent t(table, p.table_rows, p.dim * size, p.table_stride * size), v(vectors, p.n_rows, p.dim * size, p.out_stride * size);
    check_apart({out ? v : t}, {out ? t : v, Extent(p.ids, p.n_rows, p.n_columns * 4ull, p.ids_stride * 4),
                                Extent(p.offset, p.n_columns * 4ull), Extent(p.scale, p.n_columns * 4ull)}, workspace, what);
}

}  // namespace

void leaf_embedding(int ordinal, void *stream, const hbr_lookup &p, const void *table, void *out) {
    const char *what = "leaf embedding";
    check_lookup(p, what);
    const uint64_t size = size_of(p.dtype, what);
    if (p.n_rows == 0) return;
    if (!out || (!table && p.table_rows)) fail(kInvalid, std::string(what) + ": null argument");
    check_aligned(table, size, what);
    check_aligned(out, size, what);
    check_lookup_apart(p, table, out, true, Extent(nullptr, 0), what);
    Queue queue(ordinal, stream);
    const uint32_t v = vector_width(size, {p.dim, p.table_stride, p.out_stride}, {table, out});
    EmbedArgs a{};
    a.table = table;
    a.ids = p.ids;
    a.offset = p.offset;
    a.scale = p.scale;
    a.out = out;
    a.n_rows = p.n_rows;
    a.table_rows = p.table_rows;
    a.table_stride = p.table_stride;
    a.ids_stride = p.ids_stride;
    a.out_stride = p.out_stride;
    a.columns = p.table_rows ? p.n_columns : 0;
    a.dim = p.dim;
    a.vecs = p.dim / v;
    a.rows_per_block = std::max(1u, 256 / a.vecs);
    a.columns_per_pass = (uint32_t)std::min<uint64_t>(up(std::max(a.columns, 1u), 8), std::min(1024u, 4096 / a.rows_per_block / 8 * 8));
    const uint64_t blocks = (p.n_rows + a.rows_per_block - 1) / a.rows_per_block;
    const bool far = p.table_rows * p.table_stride * size >= (1ull << 31);
    const std::string k = std::string(far ? "hbr_leaf_embed_far_" : "hbr_leaf_embed_") + name_of(p.dtype) + "_" + std::to_string(v);
    queue.launch(k.c_str(), dim3((uint32_t)std::min<uint64_t>(blocks, 1u << 20)), dim3(256), a);
}

namespace {

struct LookupPlan {
    // a column at a time
    bool columns;
    uint32_t blocks, block_rows;
    // by sorting
    uint64_t n;  // entries
    uint32_t tile, tiles, passes, chunk, chunks;
    uint32_t *key[2], *val[2], *hist, *total;
    float *part;
    uint64_t bytes;
};

// A workspace named for some rows serves fewer: what fewer of them split finer
// is counted by the most that any number of rows up to the given takes, here
// the parts of the sort's chunks and tiles.
constexpr uint64_t kSortLargeTiles = 600000;  // entries from which on the sort's tiles are large
uint64_t sort_waves(const hbr_lookup &p) { return (p.dim * (p.dtype == HBR_F32 ? 4 : 2) + 1023) / 1024; }
uint64_t sort_tiles(uint64_t n) {
    const uint64_t small = (std::min(n, kSortLargeTiles - 1) + 511) / 512;
    return n < kSortLargeTiles ? small : std::max(small, (n + 4095) / 4096);
}
uint64_t sort_chunks(const hbr_lookup &p, uint64_t n) {
    uint64_t most = 0;
    for (uint64_t chunk = 16; chunk <= 64; chunk += 8) {  // for each, the most entries that are chunked so
        const uint64_t end = chunk == 64 ? n : std::min(n, ((chunk + 1) * 4096 - 1) / sort_waves(p));
        most = std::max(most, (end + chunk - 1) / chunk);
    }
    return most;
}
// The bytes that sorting takes of the workspace.
uint64_t sort_bytes(const hbr_lookup &p, uint64_t n) {
    return 4 * up(n * 4, 256) + up(kSortDigits * sort_tiles(n) * 4, 256) + up(kSortDigits * 4, 256) +
           up(sort_chunks(p, n) * 2 * p.dim * 4, 256);
}
// The blocks' sums of the columns are held in no more bytes than sorting
// takes, and 16 MiB.
uint64_t columns_limit(const hbr_lookup &p, uint64_t n) { return std::max<uint64_t>(sort_bytes(p, n), 16u << 20); }
uint64_t columns_bytes(const hbr_lookup &p, uint64_t blocks) { return blocks > 1 ? up(blocks * p.table_rows * up(p.dim, 4) * 4, 256) : 0; }
uint64_t columns_least(const hbr_lookup &p) { return (p.n_rows + kColumnBlock - 1) / kColumnBlock; }
// (rounded up to whole XCDs)
uint64_t columns_most(const hbr_lookup &p, uint64_t n) {
    return 7 + std::max(columns_least(p), std::min({n / (8 * p.table_rows), (p.n_rows + 511) / 512, (uint64_t)4096}));
}

uint64_t lookup_ids(const hbr_lookup &p) {
    if (p.n_columns && p.n_rows > 0x7fffffffull / p.n_columns)
        fail(kRefused, "leaf embedding gradient: more than 2^31 - 1 ids");
    return p.n_rows * p.n_columns;
}

// A slice's vectors of v elements, a lane each at most.
uint32_t slice_vectors(uint32_t v) { return std::min<uint32_t>(kColumnSlice / v, kWaveLanes); }

// by_column: columns may be summed one at a time (they have table rows of their
// own, and strides that allow it). v: the vectors' elements.
LookupPlan lookup_plan(const hbr_lookup &p, void *workspace, bool by_column, uint32_t v) {
    LookupPlan q{};
    q.n = lookup_ids(p);
    Arena w(workspace);
    uint32_t bits = 1;  // keys run from 0 to table_rows
    while (bits < 32 && (p.table_rows >> bits)) bits++;
    q.passes = (bits + kSortBits - 1) / kSortBits;
    // Columns of their own table rows are summed a column at a time, in blocks
    // of rows, or all of the ids are sorted: what takes less time. In us, beside
    // the vectors' bytes (5 TB/s):
    //   a workgroup (512 run at once) 5 ns a row and round of keys, 100 ns a key,
    //   and the joins of the blocks' sums 1.75 ps each;
    //   the sort 18 a pass, and 25 ps an id and pass.
    // Both sides: 200,003 x 100 ids of 64 bf16, 127 rows a column, take 0.30 ms by
    // columns, with 511 rows a column 0.49 against 1.43 by sorting, with 1,000
    // 0.94 against 1.49; 100,000 x 10 ids and 512 rows a column 89 us against 104,
    // with 1,024 164 against 105; 10,000 x 20 and 512 77 against 55; 130 x 100 and 127
    // 26 against 44; 20,000 ids of 256 f32 into 500 rows 46 against 28, 2,000 ids 30
    // against 38.
    const uint64_t slices = (p.dim / v + slice_vectors(v) - 1) / slice_vectors(v);
    constexpr uint64_t kGroups = (1u << 22) - 1;  // workgroups of 1,024 that make a launch
    if (by_column && q.n && p.table_rows && p.n_columns * slices <= 1u << 18) {
        const uint64_t least = columns_least(p), most = columns_most(p, q.n), limit = columns_limit(p, q.n);
        const double keys = std::ceil((double)p.table_rows / p.n_columns), key_rounds = std::ceil(keys / kColumnKeys);
        uint64_t blocks = 0;
        double best = 0.0;
        for (uint64_t b = least; b <= most && b * p.n_columns * slices <= kGroups && columns_bytes(p, b) <= limit;
             b = b < 4 ? b + 1 : b / 8 * 8 + 8) {  // whole XCDs
            if (b > 4 && b % 8) continue;
            // (whole rounds where they are few; later ones overlap)
            const double groups = (double)(b * p.n_columns * slices) / 512;
            const double rounds = groups <= 2.0 ? std::ceil(groups) : groups + 0.5;
            const double cost = 8.0 + rounds * (5e-3 * (double)((p.n_rows + b - 1) / b) * key_rounds + 0.1 * keys) +
                                (b > 1 ? 5.0 + 1.75e-6 * (double)(b * p.table_rows * p.dim) : 0.0);
            if (!blocks || cost < best) best = cost, blocks = b;
        }
        const double passes = q.n <= kSortSmall ? 1.0 : q.passes;
        q.columns = blocks && best <= 4.0 + passes * (18.0 + 25e-6 * (double)q.n);
        if (q.columns) {
            q.blocks = (uint32_t)blocks;
            q.block_rows = (uint32_t)((p.n_rows + blocks - 1) / blocks);
            if (blocks > 1) q.part = w.take<float>(blocks * p.table_rows * up(p.dim, 4));
            q.bytes = w.used;
            return q;
        }
    }
    // small tiles where large ones would be too few for the device (524,288
    // entries of 16 bf16 105 us against 111, 700,000 ones 118 against 114)
    q.tile = q.n < kSortLargeTiles ? 512 : 4096;
    q.tiles = (uint32_t)((q.n + q.tile - 1) / q.tile);
    // 16 to 64 entries a chunk, for about 4,096 waves of 16-byte vectors: of
    // 20,000 ids of 256 bf16 42 us with 16, 48 with 32, 62 with 64; of 1,000,000
    // of 64 191 with 64 and 194 with 16 (a frequent id's parts are more)
    q.chunk = (uint32_t)std::min<uint64_t>(64, std::max<uint64_t>(16, up(q.n * sort_waves(p) / 4096, 8)));
    q.chunks = (uint32_t)((q.n + q.chunk - 1) / q.chunk);
    for (int b = 0; b < 2; b++) {
        q.key[b] = w.take<uint32_t>(q.n);
        q.val[b] = w.take<uint32_t>(q.n);
    }
    q.hist = w.take<uint32_t>(kSortDigits * sort_tiles(q.n), (uint64_t)kSortDigits * q.tiles);
    q.total = w.take<uint32_t>(kSortDigits);
    q.part = w.take<float>(sort_chunks(p, q.n) * 2 * p.dim, (uint64_t)q.chunks * 2 * p.dim);
    q.bytes = w.used;
    return q;
}

}  // namespace

uint64_t leaf_embedding_grad_workspace(const hbr_lookup &p) {
    hbr_lookup q = p;
    q.ids = reinterpret_cast<const int32_t *>(16);  // sizes alone count
    q.offset = nullptr;
    q.scale = nullptr;
    check_lookup(q, "leaf embedding gradient");
    // whatever the arrays allow, and of any number of rows up to the given
    const uint64_t n = lookup_ids(p);
    if (n == 0 || p.table_rows == 0) return sort_bytes(p, n);
    return std::max(sort_bytes(p, n), std::min(columns_limit(p, n), columns_bytes(p, columns_most(p, n))));
}

void leaf_embedding_grad(int ordinal, void *stream, const hbr_lookup &p, const void *dout, void *dtable,
                         void *workspace, uint64_t workspace_bytes) {
    const char *what = "leaf embedding gradient";
    check_lookup(p, what);
    const uint64_t size = size_of(p.dtype, what);
    if (p.table_rows == 0) return;
    if (!dtable || (!dout && p.n_rows)) fail(kInvalid, std::string(what) + ": null argument");
    check_aligned(dout, size, what);
    check_aligned(dtable, size, what);
    // (a block's rows lie within 2 GiB of dout and of the ids)
    const bool by_column = (p.n_columns == 1 || p.offset) && std::max(p.out_stride, p.ids_stride) < 32768;
    const uint32_t v = vector_width(size, {p.dim, p.table_stride, p.out_stride}, {dout, dtable});
    const LookupPlan q = lookup_plan(p, workspace, by_column, v);
    check_workspace(workspace, workspace_bytes, q.bytes, what);
    check_lookup_apart(p, dtable, dout, false, Extent(workspace, q.bytes), what);
    Queue queue(ordinal, stream);
    const std::string suffix = std::string(name_of(p.dtype)) + "_" + std::to_string(v);
    auto blocks = [](uint64_t threads) { return dim3((uint32_t)std::min<uint64_t>((threads + 255) / 256, 1u << 16)); };
    if (q.columns) {
        LookupColumnArgs a{};
        a.ids = p.ids;
        a.offset = p.offset;
        a.scale = p.scale;
        a.dout = dout;
        a.dtable = dtable;
        a.part = q.part;
        a.ids_stride = p.ids_stride;
        a.dout_stride = p.out_stride;
        a.dtable_stride = p.table_stride;
        a.part_stride = up(p.dim, 4);
        a.table_rows = p.table_rows;
        a.n_rows = p.n_rows;
        a.columns = p.n_columns;
        a.vecs = p.dim / v;
        a.block_rows = q.block_rows;
        a.blocks = q.blocks;
        a.slice_vecs = slice_vectors(v);
        a.slices = (a.vecs + a.slice_vecs - 1) / a.slice_vecs;
        queue.launch(("hbr_lookup_columns_" + suffix).c_str(), dim3(q.blocks * a.columns * a.slices), dim3(1024), a);
        if (q.blocks > 1) queue.launch(("hbr_lookup_join_" + suffix).c_str(), blocks(p.table_rows * a.vecs), dim3(256), a);
        return;
    }
    int from = 0;
    const std::string steps = q.tile == 512 ? "_2" : "_16";
    const bool small = q.n <= kSortSmall;
    for (uint32_t pass = 0; pass < (small ? 1 : q.passes) && q.n; pass++) {
        LookupSortArgs a{};
        a.ids = p.ids;
        a.offset = p.offset;
        a.ids_stride = p.ids_stride;
        a.table_rows = p.table_rows;
        a.columns = p.n_columns;
        a.n = (uint32_t)q.n;
        a.tiles = q.tiles;
        a.shift = pass * kSortBits;
        a.keys_in = pass ? q.key[from] : nullptr;
        a.vals_in = pass ? q.val[from] : nullptr;
        a.keys_out = q.key[from ^ 1];
        a.vals_out = q.val[from ^ 1];
        a.hist = q.hist;
        a.total = q.total;
        from ^= 1;
        if (small) {
            queue.launch("hbr_sort_small", dim3(1), dim3(1024), a);
            break;
        }
        queue.launch(("hbr_sort_count" + steps).c_str(), dim3(q.tiles), dim3(256), a);
        queue.launch("hbr_sort_scan", dim3(kSortDigits), dim3(256), a);
        queue.launch(("hbr_sort_scatter" + steps).c_str(), dim3(q.tiles), dim3(256), a);
    }
    LookupSumArgs a{};
    a.keys = q.key[from];
    a.vals = q.val[from];
    a.dout = dout;
    a.scale = p.scale;
    a.dtable = dtable;
    a.part = q.part;
    a.table_rows = p.table_rows;
    a.dout_stride = p.out_stride;
    a.dtable_stride = p.table_stride;
    a.n = (uint32_t)q.n;
    a.columns = p.n_columns;
    a.dim = p.dim;
    a.vecs = p.dim / v;
    a.wide = 1;
    while (a.wide < a.vecs && a.wide < kWaveLanes) a.wide *= 2;
    a.chunk = q.chunk;
    a.chunks = q.chunks;
    const uint32_t groups = 256 / a.wide, slices = (a.vecs + a.wide - 1) / a.wide;
    queue.launch(("hbr_lookup_sum_" + suffix).c_str(), dim3((q.chunks + groups - 1) / groups, slices), dim3(256), a);
    a.row_blocks = (uint32_t)((p.table_rows + 4 * 63 - 1) / (4 * 63));
    queue.launch(("hbr_lookup_finish_" + suffix).c_str(), dim3(a.row_blocks + (q.chunks + groups - 1) / groups, slices), dim3(256), a);
}

// ---- the softmax head ------------------------------------------------------------------

namespace {

// The scores' gradients of one piece of the classes are held at a time, in at
// most about this many bytes.
constexpr uint64_t kPieceBytes = 1ull << 30;
// Bytes from one chunk of 32 bf16 columns to the next. An odd multiple of
// 2 KiB: the chunks of a tile, whose steps of 32 rows are 2 KiB each, then
// begin in different halves of the L2's channels.
constexpr uint64_t kChunkStep = 2048;
uint64_t chunk_bytes(uint64_t rows) { return ((rows * 64 + 2 * kChunkStep - 1) / (2 * kChunkStep) * 2 + 1) * kChunkStep; }

// From this many rows on, w is laid out in chunks too (and h in a call that
// only scores): 2,048 rows scored against 32,768 classes of 512 bf16 take 105 us
// with the operands in place and 108 laid out, 4,096 rows 194 and 187; with
// the gradients 336 and 346, 642 and 635.
constexpr uint64_t kLayRows = 4096;

uint64_t tiles(uint64_t n, uint64_t of) { return (n + of - 1) / of; }

// Scores alone over short inputs are made by rows too from this many on (and
// from kLayRows rows): their partial results are held for a few shares of the
// classes then, and not for every tile of 128 (200,000 rows, 20,000 classes of
// 64 bf16: 115 MB against 407, and 1.12 ms against 1.78; 4,096 and 1,000 16.8 us
// against 15.8, 200,000 and 70 41 against 48; in f32 17.8 us against 20.6 and 67
// against 72).
constexpr uint64_t kNarrowScores = 1u << 23;

// A product's tiles, and how many of them fill 256 CUs (of the small ones twice
// as many run at once, at hardly more rate).
struct HeadTiling {
    uint64_t tile, threads, slots;
    const char *name;
};
constexpr HeadTiling kTile256{256, 512, 256, "_256"}, kTile128{128, 256, 512, "_128"};

// Shares of a product's steps: where its tiles are fewer than the device
// runs at once, enough of them to fill it, of 16 steps at least.
uint32_t head_splits(const HeadTiling &t, uint64_t m, uint64_t n, uint64_t k, uint64_t segments) {
    const uint64_t all = tiles(m, t.tile) * tiles(n, t.tile), steps = tiles(k, kHeadK) * segments;
    return (uint32_t)std::max<uint64_t>(1, std::min(t.slots / std::max<uint64_t>(all, 1), steps / 16));
}

// The tiles of a product with the gradients: those that take less time, in us:
// a step of 256 large tiles is one (1.1 PFLOP/s), one of 512 small ones 0.54,
// and shares' sums are read once more at 4.5 TB/s. Both at their best:
// 16,384 x 131,072 x 1,024 products of bf16 take 3.9 ms with large tiles and
// 4.2 with small ones, 8,191 x 32,768 x 512 ones 0.29 and 0.32, 3,229 x 2,810 x
// 335 ones of f32 with their sums 70 us and 60. (The scores and pairs keep the
// small ones: four workgroups on a CU hide each other's exponentials and
// stores. 16,384 x 32,768 pairs of 1,024 take 1.34 ms against 1.35 with large
// ones, 4,096 x 5,003 ones of 256 in f32 84 us against 119.)
const HeadTiling &head_tiling(uint64_t m, uint64_t n, uint64_t k, uint64_t segments) {
    const uint64_t steps = tiles(k, kHeadK) * segments;
    auto cost = [&](const HeadTiling &t, double step) {
        const uint64_t shares = head_splits(t, m, n, k, segments);
        return (double)(tiles(tiles(m, t.tile) * tiles(n, t.tile) * shares, t.slots) * tiles(steps, shares)) * step +
               (shares > 1 ? (double)(shares * m * n) * 4.0 / 4.5e6 : 0.0);
    };
    return cost(kTile256, 1.0) <= cost(kTile128, 0.54) ? kTile256 : kTile128;
}

struct HeadPlan {
    bool few;  // few classes: their own kernels, and the products' shares of the rows
    uint32_t score_blocks, shares;
    uint64_t g_stride;
    uint64_t parts, segments, chunks;
    bool lay;     // h and w are laid out in chunks whatever their rows
    bool narrow;  // short inputs: no pairs are stored, and the scores are made by rows
    uint64_t piece, pieces;
    const HeadTiling *by_h, *by_w;  // the tiles of the products with the gradients
    uint32_t splits_h, splits_w, splits_z;  // splits_z: of the classes, for the scores over short inputs
    bool sum_h;  // dh is summed from f32 parts
    float *part_max, *part_sum, *label_margin, *lse2, *part_db, *dh, *dw;
    int32_t *part_best;
    char *h, *w, *g;
    uint32_t *keep;
    uint64_t bytes;
};

// What the products can read in place: bf16 rows of whole 16-byte pieces,
// near enough to each other for a tile's 32-bit offsets.
bool head_in_place(const void *p, uint64_t stride, const hbr_softmax &a) {
    return a.dtype == HBR_BF16 && a.dim % 8 == 0 && stride % 8 == 0 && stride < (1u << 22) &&
           reinterpret_cast<uint64_t>(p) % 16 == 0;
}

// Every array has room for what any number of rows up to n takes (fewer rows
// may be shared out finer, or taken in fewer pieces), and the arrays of a call
// with gradients hold those of one without: a workspace serves smaller calls.
HeadPlan head_plan(uint64_t n, uint64_t classes, uint64_t dim, uint32_t dtype, bool gradient, void *workspace) {
    size_of(dtype, "softmax head");
    if (classes == 0 || dim == 0) fail(kInvalid, "softmax head: no classes, or inputs of no elements");
    if (classes > 0x7fffffffull || n > 0x7fffffffull) fail(kRefused, "softmax head: more than 2^31 - 1 rows or classes");
    if (dim >= kDimLimit) fail(kRefused, "softmax head: inputs of 1,048,576 elements or more");
    HeadPlan q{};
    q.parts = dtype == HBR_F32 ? 3 : 1;
    q.segments = dtype == HBR_F32 ? 6 : 1;
    q.chunks = tiles(dim, 32);
    const bool short_inputs = dim <= (dtype == HBR_F32 ? kNarrowDimF32 : kNarrowDim);
    q.narrow = short_inputs && (gradient || (n >= kLayRows && n * classes >= kNarrowScores));
    q.lay = dtype == HBR_F32 || n >= kLayRows || q.narrow;
    // shares of the walked side, for about 1,024 workgroups, or 512 of the
    // longest inputs, whose registers let fewer run at once (30,497 x 13,116
    // scores of 20 in f32 1.01 ms, 1.26 with 512; 16,384 x 8,192 of 64 533 us, 545
    // with 1,024), of four steps or more, in f32, whose steps are longer, of two
    // (2,000 x 3,000 scores of 64: bf16 59 us, 69 with eight and 64 with two; f32 83,
    // 138 with eight and 94 with four)
    const uint64_t groups = dim > (dtype == HBR_F32 ? 32 : 64) ? 512 : 1024;
    auto shares = [&](uint64_t held, uint64_t walked) {
        return (uint32_t)std::max<uint64_t>(1, std::min(groups / std::max<uint64_t>(1, tiles(held, 128)), tiles(walked, dtype == HBR_F32 ? 128 : 256)));
    };
    q.splits_z = shares(n, classes);
    // rows times their shares of `walked`, at most (a tile of 128 rows a workgroup)
    const uint64_t shared_rows = std::max(n, std::min(groups * 128, n * tiles(classes, dtype == HBR_F32 ? 128 : 256)));
    Arena w(workspace);
    q.few = classes <= kFewClasses;
    if (q.few) {
        // groups of 32 rows, evenly: at most 2,048 waves of scores (of 100,000
        // rows of 64 bf16 and 48 classes 51 us, 58 with 4,096) and of products
        // (200,003 rows of 50 f32 and ten classes 69 us, 84 with 1,024, 72 with 4,096)
        const uint64_t groups = std::max<uint64_t>(1, tiles(n, 32)), cols = tiles(dim, 32);
        q.score_blocks = (uint32_t)tiles(tiles(groups, tiles(groups, 2048)), 4);
        q.shares = (uint32_t)tiles(groups, tiles(groups, std::max<uint64_t>(1, 2048 / cols)));
        q.g_stride = up(classes, 16);
        if (gradient) {
            q.g = w.take<char>(n * q.g_stride * (dtype == HBR_F32 ? 4 : 2));
            q.keep = w.take<uint32_t>(groups);
            q.part_db = w.take<float>(tiles(std::min<uint64_t>(groups, 2048), 4) * 4 * classes, q.score_blocks * 4ull * classes);
            q.dw = w.take<float>(std::min(groups, std::max<uint64_t>(1, 2048 / cols)) * classes * dim, q.shares * classes * dim);
        }
        q.bytes = w.used;
        return q;
    }
    // of the rows whose scores are made in tiles, at most
    const uint64_t tiled = short_inputs ? std::min(n, std::max(kLayRows - 1, (kNarrowScores - 1) / classes)) : n;
    const uint64_t parts = std::max(tiled * tiles(classes, kTile128.tile), short_inputs ? shared_rows : 0);
    const uint64_t parts_used = (q.narrow ? q.splits_z : tiles(classes, kTile128.tile)) * n;
    q.part_max = w.take<float>(parts, parts_used);
    q.part_sum = w.take<float>(parts, parts_used);
    q.part_best = w.take<int32_t>(parts, parts_used);
    q.label_margin = w.take<float>(n);
    q.lse2 = w.take<float>(n);
    q.h = w.take<char>(q.parts * q.chunks * chunk_bytes(n));
    q.w = w.take<char>(q.parts * q.chunks * chunk_bytes(classes));
    if (gradient && q.narrow) {
        q.splits_h = q.splits_z;
        q.splits_w = shares(classes, n);
        q.dh = w.take<float>(shared_rows * dim, q.splits_h * n * dim);
        q.dw = w.take<float>(q.splits_w * classes * dim);
        q.part_db = w.take<float>(q.splits_w * classes);
    } else if (gradient) {
        // the pieces as even as whole tiles allow
        const uint64_t row_bytes = std::max<uint64_t>(n, 1) * 2 * q.parts;
        q.pieces = tiles(classes, std::max<uint64_t>(256, kPieceBytes / row_bytes / 256 * 256));
        q.piece = up(tiles(classes, q.pieces), 256);
        q.pieces = tiles(classes, q.piece);
        q.by_h = &head_tiling(n, dim, q.piece, q.segments);
        q.by_w = &head_tiling(q.piece, dim, n, q.segments);
        q.splits_h = head_splits(*q.by_h, n, dim, q.piece, q.segments);
        q.splits_w = head_splits(*q.by_w, q.piece, dim, n, q.segments);
        q.sum_h = q.splits_h > 1 || q.pieces > 1;
        // The pairs: all classes at once, or one piece of at most kPieceBytes
        // beside what the chunks' steps add to the fewest rows taken in pieces,
        // or of 256 classes.
        const uint64_t all = up(classes, 256), per = kPieceBytes / (2 * q.parts), row_tiles = tiles(n, kTile128.tile);
        q.g = w.take<char>(q.parts * std::min(all / 32 * chunk_bytes(n),
                                              std::max(8 * chunk_bytes(n), 2 * per + all / 32 * 3 * kChunkStep)),
                           q.parts * (q.piece / 32) * chunk_bytes(n));
        q.part_db = w.take<float>(std::min(row_tiles * all, std::max(row_tiles * 256, per / 128 + all)),
                                  row_tiles * q.piece);
        // the shares of a product: as many of its rows as fill the device once,
        // of 16 steps each at least
        const uint64_t fill = 65536 / tiles(dim, kTile256.tile);
        static_assert(kTile256.slots * 256 == 65536 && kTile128.slots * 128 == 65536, "rows of a launch's tiles");
        auto split = [&](uint64_t m, uint64_t k) {
            const uint64_t most = tiles(k, kHeadK) * q.segments / 16;
            return most > 1 ? std::min(fill, m * most) : 0;
        };
        const uint64_t sum_rows = std::max(split(n, all), q.pieces > 1 ? n : 0);
        q.dh = w.take<float>(sum_rows * dim, q.sum_h ? q.splits_h * n * dim : 0);
        q.dw = w.take<float>(split(all, n) * dim, q.splits_w > 1 ? q.splits_w * q.piece * dim : 0);
    }
    q.bytes = w.used;
    return q;
}

}  // namespace

uint64_t softmax_head_workspace(uint64_t n_rows, uint32_t n_classes, uint32_t dim, uint32_t dtype, bool gradient) {
    return head_plan(n_rows, n_classes, dim, dtype, gradient, nullptr).bytes;
}

void softmax_head(int ordinal, void *stream, const hbr_softmax &p, void *workspace, uint64_t workspace_bytes) {
    const char *what = "softmax head";
    const bool gradient = p.dh || p.dw || p.db;
    const uint64_t size = size_of(p.dtype, what), n = p.n_rows, classes = p.n_classes, dim = p.dim;
    const HeadPlan q = head_plan(n, classes, dim, p.dtype, gradient, workspace);
    if (!p.w || (n && !p.h)) fail(kInvalid, std::string(what) + ": null inputs or weights");
    if (gradient && !p.labels && n) fail(kInvalid, std::string(what) + ": gradients need labels");
    if ((n > 1 && p.h_stride < dim) || (classes > 1 && p.w_stride < dim) || (p.dh && n > 1 && p.dh_stride < dim) ||
        (p.dw && classes > 1 && p.dw_stride < dim))
        fail(kInvalid, std::string(what) + ": rows overlap");
    // (a single row's stride counts nothing, and may be less than the row: the
    // products' tiles tell the rows behind it by their place alone)
    const uint64_t dh_stride = n > 1 ? p.dh_stride : dim, dw_stride = classes > 1 ? p.dw_stride : dim;
    if ((p.dh && dh_stride >= (1u << 21)) || (p.dw && dw_stride >= (1u << 21)))
        fail(kRefused, std::string(what) + ": gradients whose rows lie 2,097,152 elements or more apart");
    if (!q.few && std::max(tiles(n, 128) * tiles(classes, 128), q.narrow ? tiles(n, 128) * q.splits_z : 0) >= 1u << 24)
        fail(kRefused, std::string(what) + ": 2^24 tiles of 128 rows and 128 classes or more");
    for (const void *x : {p.h, p.w, (const void *)p.dh, (const void *)p.dw}) check_aligned(x, size, what);
    for (const void *x : {(const void *)p.bias, (const void *)p.labels, (const void *)p.weight, (const void *)p.loss,
                          (const void *)p.lse, (const void *)p.best, (const void *)p.db})
        check_aligned(x, 4, what);
    check_workspace(workspace, workspace_bytes, q.bytes, what);
    check_apart({{p.loss, n * 4}, {p.lse, n * 4}, {p.best, n * 4}, {p.db, classes * 4},
                 {p.dh, n, dim * size, dh_stride * size}, {p.dw, classes, dim * size, dw_stride * size}},
                {{p.h, n, dim * size, p.h_stride * size}, {p.w, classes, dim * size, p.w_stride * size},
                 {p.bias, classes * 4}, {p.labels, n * 4}, {p.weight, n * 4}}, Extent(workspace, q.bytes), what);
    Queue queue(ordinal, stream);
    const std::string suffix = name_of(p.dtype);
    const dim3 threads(256);
    auto cells = [](uint64_t n) { return dim3((uint32_t)std::min<uint64_t>((n + 255) / 256, 1u << 16)); };
    auto sum = [&](const char *kernel, const float *part, uint64_t parts, uint64_t part_stride, void *dst, uint64_t rows,
                   uint64_t cols, uint64_t dst_stride) {
        HeadSumArgs a{};
        a.scale = p.grad_scale;
        a.part = part;
        a.parts = (uint32_t)parts;
        a.part_stride = part_stride;
        a.dst = dst;
        a.rows = rows;
        a.cols = cols;
        a.dst_stride = dst_stride;
        // few cells of many parts: a workgroup's waves share the parts
        a.shares = 1;
        while (a.shares < 16 && parts >= 8 * a.shares && rows * cols * a.shares < 64 * 2048) a.shares *= 4;
        const uint32_t waves = a.shares == 16 ? 16 : 4;
        const uint64_t each = waves / a.shares * 64;
        queue.launch(kernel, dim3((uint32_t)std::min<uint64_t>(tiles(rows * cols, each), 1u << 16)), dim3(waves * 64), a);
    };
    const std::string sum_kernel = "hbr_head_sum_" + suffix;
    if (n == 0) {  // sums over no rows
        if (p.dw) sum(sum_kernel.c_str(), nullptr, 0, 0, p.dw, classes, dim, dw_stride);
        if (p.db) sum("hbr_head_sum_f32", nullptr, 0, 0, p.db, 1, classes, classes);
        return;
    }
    if (q.few) {
        FewArgs f{};
        f.h = p.h;
        f.w = p.w;
        f.h_stride = p.h_stride;
        f.w_stride = p.w_stride;
        f.rows = n;
        f.classes = (uint32_t)classes;
        f.dim = (uint32_t)dim;
        f.bias = p.bias;
        f.labels = p.labels;
        f.weight = p.weight;
        f.loss = p.loss;
        f.lse = p.lse;
        f.best = p.best;
        f.scale = p.grad_scale;
        f.chunks = q.shares;
        f.g = q.g;
        f.g_stride = q.g_stride;
        f.keep = q.keep;
        f.part_db = q.part_db;
        f.part_dw = q.dw;
        f.dh = p.dh;
        f.dh_stride = dh_stride;
        f.col_tiles = (uint32_t)tiles(dim, 32);
        f.dw = p.dw != nullptr;
        const std::string few = suffix + (classes > 32 ? "_2" : "_1");
        queue.launch(("hbr_few_scores_" + few).c_str(), dim3(q.score_blocks), threads, f);
        if (!gradient) return;
        if (p.dh || p.dw)
            queue.launch(("hbr_few_products_" + few).c_str(), dim3((uint32_t)tiles((uint64_t)q.shares * f.col_tiles, 4)), threads, f);
        if (p.dw || p.db) {
            FewSumsArgs a{};
            a.part_dw = p.dw ? q.dw : nullptr;
            a.part_db = p.db ? q.part_db : nullptr;
            a.dw = p.dw;
            a.db = p.db;
            a.dw_stride = dw_stride;
            a.shares = q.shares;
            a.waves = q.score_blocks * 4;
            a.classes = (uint32_t)classes;
            a.dim = (uint32_t)dim;
            a.scale = p.grad_scale;
            a.dw_blocks = p.dw ? (uint32_t)tiles(classes * dim, 16) : 0;
            queue.launch(("hbr_few_sums_" + suffix).c_str(), dim3(a.dw_blocks + (p.db ? (uint32_t)tiles(classes, 16) : 0)), dim3(1024), a);
        }
        return;
    }
    // the operands of the products
    struct Laid {
        const char *p;
        uint64_t row, chunk, part;
        uint32_t cols;
    };
    auto lay = [&](const void *src, uint64_t stride, uint64_t rows, char *to, bool always, const int32_t *labels) -> Laid {
        if (rows == 1) stride = up(dim, 8);
        if (!always && head_in_place(src, stride, p))
            return {static_cast<const char *>(src), stride * 2, 64, 0, (uint32_t)dim};
        HeadPartsArgs a{};
        a.src = src;
        a.labels = labels;
        a.dst = reinterpret_cast<uint16_t *>(to);
        a.rows = rows;
        a.src_stride = stride;
        a.chunk = chunk_bytes(rows) / 2;
        a.part = q.chunks * a.chunk;
        a.cols = (uint32_t)dim;
        a.chunks = (uint32_t)q.chunks;
        queue.launch(("hbr_head_parts_" + suffix).c_str(), cells(rows * q.chunks * 4), threads, a);
        return {static_cast<const char *>(to), 64, a.chunk * 2, a.part * 2, (uint32_t)(q.chunks * 32)};
    };
    const bool by_rows = p.dw || p.db || q.narrow;  // rows that take no part are read with the others
    const Laid h = lay(p.h, p.h_stride, n, q.h, q.lay || by_rows, by_rows ? p.labels : nullptr);
    const Laid w = lay(p.w, p.w_stride, classes, q.w, q.lay, nullptr);
    auto set_a = [](HeadArgs &a, const Laid &o) { a.a = o.p, a.a_row = o.row, a.a_chunk = o.chunk, a.a_part = o.part; };
    auto set_b = [](HeadArgs &a, const Laid &o) { a.b = o.p, a.b_row = o.row, a.b_chunk = o.chunk, a.b_part = o.part; };
    auto product = [&](const std::string &kernel, const HeadTiling &t, HeadArgs a) {
        a.m_tiles = (uint32_t)tiles(a.m, t.tile);
        a.n_tiles = (uint32_t)tiles(a.n, t.tile);
        a.segments = (uint32_t)q.segments;
        queue.launch((kernel + t.name).c_str(), dim3(a.m_tiles * a.n_tiles * a.splits), dim3((uint32_t)t.threads), a);
    };
    HeadArgs z{};
    set_a(z, w);
    set_b(z, h);
    z.m = (uint32_t)classes;
    z.n = (uint32_t)n;
    z.k = std::min(h.cols, w.cols);
    z.check = z.k % kHeadK != 0;
    z.splits = 1;
    z.bias = p.bias;
    z.labels = p.labels;
    z.part_max = q.part_max;
    z.part_sum = q.part_sum;
    z.part_best = p.best ? q.part_best : nullptr;
    z.label_margin = q.label_margin;
    auto walk = [&](const char *kernel, bool rows, uint32_t splits, float *part) {
        const Laid &x = rows ? h : w, &y = rows ? w : h;
        NarrowArgs a{};
        a.x = x.p;
        a.y = y.p;
        a.x_chunk = x.chunk;
        a.y_chunk = y.chunk;
        a.x_part = x.part;
        a.y_part = y.part;
        a.nx = (uint32_t)(rows ? n : classes);
        a.ny = (uint32_t)(rows ? classes : n);
        a.x_tiles = (uint32_t)tiles(a.nx, 128);
        a.splits = splits;
        a.bias = p.bias;
        a.labels = p.labels;
        a.weight = p.weight;
        a.lse2 = q.lse2;
        a.part = part;
        a.part_db = rows ? nullptr : q.part_db;
        a.part_max = q.part_max;
        a.part_sum = q.part_sum;
        a.part_best = p.best ? q.part_best : nullptr;
        a.label_margin = q.label_margin;
        a.dim = (uint32_t)dim;
        queue.launch((kernel + suffix + "_" + std::to_string(q.chunks)).c_str(), dim3(a.x_tiles * a.splits), threads, a);
    };
    if (q.narrow) walk("hbr_head_narrow_scores_", true, q.splits_z, nullptr);
    else product("hbr_head_scores", kTile128, z);
    HeadFinishArgs f{};
    f.part_max = q.part_max;
    f.part_sum = q.part_sum;
    f.part_best = z.part_best;
    f.label_margin = q.label_margin;
    f.labels = p.labels;
    f.weight = p.weight;
    f.lse2 = q.lse2;
    f.lse = p.lse;
    f.loss = p.loss;
    f.best = p.best;
    f.rows = n;
    f.classes = classes;
    f.tiles = (uint32_t)(q.narrow ? q.splits_z : tiles(classes, kTile128.tile));
    // fewer rows a workgroup where they would not fill the device and a lane
    // would have more than eight tiles
    f.wide = 64;
    while (f.wide > 1 && tiles(n, f.wide) < 256 && f.tiles > 8 * 16 * (64 / f.wide)) f.wide /= 4;
    queue.launch("hbr_head_finish", dim3((uint32_t)tiles(n, f.wide)), dim3(1024), f);
    if (!gradient) return;
    if (q.narrow) {
        if (p.dh) {
            walk("hbr_head_narrow_dh_", true, q.splits_h, q.dh);
            sum(sum_kernel.c_str(), q.dh, q.splits_h, n * dim, p.dh, n, dim, dh_stride);
        }
        if (p.dw || p.db) walk("hbr_head_narrow_dw_", false, q.splits_w, q.dw);
        if (p.dw) sum(sum_kernel.c_str(), q.dw, q.splits_w, classes * dim, p.dw, classes, dim, dw_stride);
        if (p.db) sum("hbr_head_sum_f32", q.part_db, q.splits_w, classes, p.db, 1, classes, classes);
        return;
    }
    for (uint64_t k0 = 0; k0 < classes; k0 += q.piece) {
        const uint64_t kc = std::min(q.piece, classes - k0);
        Laid wk = w;  // w from class k0 on, and its scores' gradients
        wk.p += k0 * w.row;
        const Laid pairs{static_cast<const char *>(q.g), 64, chunk_bytes(n), chunk_bytes(n) * (q.piece / 32), (uint32_t)q.piece};
        HeadArgs g{};
        set_a(g, h);
        set_b(g, wk);
        g.m = (uint32_t)n;
        g.n = (uint32_t)kc;
        g.k = z.k;
        g.check = z.check;
        g.splits = 1;
        g.bias = p.bias ? p.bias + k0 : nullptr;
        g.labels = p.labels;
        g.lse2 = q.lse2;
        g.weight = p.weight;
        g.first = k0;
        g.g = q.g;
        g.g_stride = q.piece;
        g.g_chunk = pairs.chunk / 2;
        g.g_part = pairs.part / 2;
        g.part_db = q.part_db;
        product("hbr_head_pairs_" + suffix, kTile128, g);
        if (p.db) sum("hbr_head_sum_f32", q.part_db, tiles(n, kTile128.tile), q.piece, p.db + k0, 1, kc, kc);
        if (p.dw) {
            HeadArgs c{};
            set_a(c, pairs);
            set_b(c, h);
            c.m = (uint32_t)up(kc, 32);
            c.rows = (uint32_t)kc;
            c.n = (uint32_t)dim;
            c.k = (uint32_t)n;
            c.splits = q.splits_w;
            c.scale = q.splits_w == 1 ? p.grad_scale : 1.0f;  // else the sum's
            char *to = static_cast<char *>(p.dw) + k0 * dw_stride * size;
            const bool direct = q.splits_w == 1;
            c.c = direct ? (void *)to : q.dw;
            c.c_stride = direct ? dw_stride : dim;
            c.c_split = q.piece * dim;
            product(direct && p.dtype == HBR_BF16 ? "hbr_head_dw_bf16" : "hbr_head_dw_part", *q.by_w, c);
            if (!direct) sum(sum_kernel.c_str(), q.dw, q.splits_w, q.piece * dim, to, kc, dim, dw_stride);
        }
        if (p.dh) {
            HeadArgs c{};
            set_a(c, pairs);
            set_b(c, wk);
            c.m = c.rows = (uint32_t)n;
            c.n = (uint32_t)dim;
            c.k = (uint32_t)kc;
            c.splits = q.splits_h;
            c.scale = q.sum_h ? 1.0f : p.grad_scale;
            c.c = q.sum_h ? q.dh : p.dh;
            c.c_stride = q.sum_h ? dim : dh_stride;
            c.c_split = n * dim;
            c.accumulate = k0 != 0;
            product(!q.sum_h && p.dtype == HBR_BF16 ? "hbr_head_dh_bf16" : "hbr_head_dh_part", *q.by_h, c);
        }
    }
    if (p.dh && q.sum_h) sum(sum_kernel.c_str(), q.dh, q.splits_h, n * dim, p.dh, n, dim, dh_stride);
}

// ---- clipping ----------------------------------------------------------------------------

namespace {

// The launches of one pass over the tensors: kClipTensors of them at a time.
uint64_t clip_launches(uint64_t n) { return (n + kClipTensors - 1) / kClipTensors; }

// No output may lie over another tensor or output, or over its own tensor but
// in place: a tensor given twice would be scaled twice, or once. The norm lies
// in none.
void check_apart(const hbr_tensor *tensors, uint64_t n, const float *norm, const char *what) {
    struct Span {
        uint64_t begin, end;
        bool written;
    };
    std::vector<Span> spans;
    spans.reserve(n + 1);
    if (norm) spans.push_back({reinterpret_cast<uint64_t>(norm), reinterpret_cast<uint64_t>(norm) + sizeof(float), true});
    for (uint64_t i = 0; i < n; i++) {
        const hbr_tensor &t = tensors[i];
        const uint64_t bytes = t.len * size_of(t.dtype, what), in = reinterpret_cast<uint64_t>(t.data),
                       out = reinterpret_cast<uint64_t>(t.out);
        if (!bytes) continue;
        spans.push_back({out, out + bytes, true});
        if (in != out) spans.push_back({in, in + bytes, false});
    }
    std::sort(spans.begin(), spans.end(), [](const Span &a, const Span &b) { return a.begin < b.begin; });
    uint64_t all = 0, written = 0;  // where the spans so far end
    for (const Span &s : spans) {
        if (s.begin < (s.written ? all : written)) fail(kInvalid, std::string(what) + ": an output overlaps another tensor");
        all = std::max(all, s.end);
        if (s.written) written = std::max(written, s.end);
    }
}

}  // namespace

uint64_t clip_gradients_workspace(uint64_t n_tensors) {
    if (n_tensors > (1u << 20)) fail(kRefused, "clip gradients: more than 1,048,576 tensors");
    return clip_launches(n_tensors) * kClipBlocks * sizeof(double);
}

void clip_gradients(int ordinal, void *stream, const hbr_tensor *tensors, uint64_t n, double max_norm, float *norm,
                    void *workspace, uint64_t workspace_bytes) {
    const char *what = "clip gradients";
    if (n && !tensors) fail(kInvalid, std::string(what) + ": null tensors");
    if (!(max_norm >= 0.0)) fail(kInvalid, std::string(what) + ": the largest norm is negative or no number");
    check_aligned(norm, 4, what);
    check_workspace(workspace, workspace_bytes, clip_gradients_workspace(n), what);
    uint64_t blocks = 0;  // of a launch
    for (uint64_t i = 0; i < n; i++) {
        const uint64_t size = size_of(tensors[i].dtype, what);
        if (tensors[i].len && (!tensors[i].data || !tensors[i].out)) fail(kInvalid, std::string(what) + ": null tensor");
        if (tensors[i].len > (1ull << 42)) fail(kRefused, std::string(what) + ": a tensor of more than 2^42 elements");
        check_aligned(tensors[i].data, size, what);
        check_aligned(tensors[i].out, size, what);
        blocks = (i % kClipTensors ? blocks : 0) + (tensors[i].len + kClipElems - 1) / kClipElems;
        if (blocks > 0x7fffffffull) fail(kRefused, std::string(what) + ": too many elements");
    }
    check_apart(tensors, n, norm, what);
    const Extent room(workspace, clip_gradients_workspace(n));
    for (uint64_t i = 0; i < n; i++)
        for (const void *x : {tensors[i].data, (const void *)tensors[i].out})
            if (overlap(room, Extent(x, tensors[i].len * size_of(tensors[i].dtype, what))))
                fail(kInvalid, std::string(what) + ": a tensor lies in the memory for the call's own use");
    if (overlap(room, Extent(norm, sizeof(float)))) fail(kInvalid, std::string(what) + ": the norm lies in the memory for the call's own use");
    Queue queue(ordinal, stream);
    const uint64_t launches = std::max<uint64_t>(1, clip_launches(n));
    auto fill = [&](uint64_t l, ClipArgs &a) {
        a = ClipArgs{};
        uint64_t block = 0;
        for (uint64_t i = l * kClipTensors; i < std::min(n, (l + 1) * kClipTensors); i++) {
            if (tensors[i].len == 0) continue;
            ClipTensor &t = a.t[a.tensors++];
            t.data = tensors[i].data;
            t.out = tensors[i].out;
            t.len = tensors[i].len;
            t.dtype = tensors[i].dtype;
            t.block = (uint32_t)block;
            block += (t.len + kClipElems - 1) / kClipElems;
        }
        a.blocks = (uint32_t)block;
        a.part = static_cast<double *>(workspace);
        a.norm = norm;
        a.max_norm = max_norm;
    };
    ClipArgs a;
    uint32_t parts = 0;
    for (uint64_t l = 0; l < launches; l++) {
        fill(l, a);
        a.first_part = parts;
        const uint32_t groups = std::min(a.blocks, kClipBlocks);
        if (groups) queue.launch("hbr_clip_norm", dim3(groups), dim3(256), a);
        parts += groups;
    }
    for (uint64_t l = 0; l < launches; l++) {
        fill(l, a);
        a.parts = parts;
        a.first_part = (uint32_t)l;  // the first launch gives the norm
        const uint32_t groups = std::min(a.blocks, kClipBlocks);
        if (groups || l == 0) queue.launch("hbr_clip_scale", dim3(std::max(groups, 1u)), dim3(256), a);
    }
}

}  // namespace hbr
