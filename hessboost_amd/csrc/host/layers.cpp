#include "layers.h"

#include "opcalls.h"

namespace hbr {

namespace {

constexpr uint64_t kRowsLimit = 0x7fffffffull;

void check_rows(uint64_t n, uint64_t dim, const char *what) {
    if (dim == 0) fail(kInvalid, std::string(what) + ": rows of no elements");
    if (dim >= kDimLimit) fail(kRefused, std::string(what) + ": rows of 1,048,576 elements or more");
    if (n > kRowsLimit) fail(kRefused, std::string(what) + ": more than 2^31 - 1 rows");
}

// An array of rows, as its checks and its kernels see it.
struct Rows {
    const void *p;
    uint64_t n, width, stride, size;  // size: of an element
    Rows(const void *ptr, uint64_t rows, uint64_t cols, uint64_t step, uint64_t bytes, const char *what)
        : p(ptr), n(rows), width(cols), stride(rows > 1 ? step : cols), size(bytes) {
        if (!p) return;
        if (stride < width) fail(kInvalid, std::string(what) + ": rows overlap");
        check_aligned(p, size, what);
    }
    Extent extent() const { return {p, n, width * size, stride * size}; }
    bool is(const Rows &o) const { return p && p == o.p && stride == o.stride && size == o.size; }
};

// The widest vector that every array's rows are made of.
uint32_t rows_vector(uint64_t size, uint64_t dim, std::initializer_list<const Rows *> all) {
    uint32_t v = (uint32_t)(16 / size);
    for (; v > 1; v /= 2) {
        bool ok = dim % v == 0;
        for (const Rows *r : all)
            ok = ok && (!r->p || ((r->n <= 1 || r->stride % v == 0) && reinterpret_cast<uint64_t>(r->p) % (v * r->size) == 0));
        if (ok) break;
    }
    return v;
}

// The rows' kernels take vectors of 16 bytes wherever they lie and let a row's
// last one reach back (65,537 rows of 1,023 bf16: norm 203 us and its gradient
// 183, element by element 542 and 444), and rows shorter than a vector element
// by element.
uint32_t row_vector(uint64_t size, uint64_t dim) { return dim >= 16 / size ? (uint32_t)(16 / size) : 1; }
// Rows of f32 that are whole vectors of 8 bytes only take those up to `most`
// columns, and beyond vectors of 16 that reach back (67,000,000 elements, us, 8
// bytes and 16): norm 310 columns 120 and 142, 510 115 and 127, 514 207 and 120,
// 2,046 135 and 119; gradient 50 162 and 221, 510 176 and 183, 2,046 151 and 247,
// 2,050 272 and 230, 3,582 206 and 184.
constexpr uint64_t kNormNarrow = 512, kNormGradNarrow = 2048;
uint32_t norm_vector(uint64_t size, uint64_t dim, uint64_t most) {
    return size == 4 && dim % 4 == 2 && dim <= most ? 2 : row_vector(size, dim);
}

uint64_t scales_of(uint64_t dim) { return tiles(dim, kPackBlock); }

uint32_t power_of_two(uint64_t n) {
    uint32_t p = 1;
    while (p < n) p *= 2;
    return p;
}

// A row's lanes and its vectors a lane: a wave or less of a workgroup of 256,
// else the whole of one; 0 vectors where the registers hold no row. `most`
// vectors a lane: what 128 registers hold of the kernel's arrays.
struct RowPlan {
    uint32_t lanes, held, threads;
    uint64_t per() const { return threads / lanes; }  // rows a workgroup
    std::string name() const { return "_" + std::to_string(held); }
};
RowPlan row_plan(uint64_t vecs, uint32_t v, uint32_t most, bool codes) {
    const uint64_t least = std::max<uint64_t>(vecs, codes ? kPackBlock / v : 1);
    if (least <= kWaveLanes) return {power_of_two(least), 1, 256};
    for (uint32_t held = 2; held <= most; held *= 2)
        if (vecs <= kWaveLanes * held) return {kWaveLanes, held, 256};
    for (uint32_t threads = most == 2 ? 128 : 256; threads <= 1024; threads *= 2)
        if (vecs <= threads * 2) return {threads, 2, threads};
    return {1024, 0, 1024};
}

// (rows of other than whole vectors have kernels of their own)
std::string rows_kernel(const char *name, uint32_t dtype, uint32_t v, uint64_t dim) {
    return std::string(name) + "_" + name_of(dtype) + "_" + std::to_string(v) + (dim % v ? "r" : "");
}

std::string kernel_of(const char *name, uint32_t dtype, uint32_t v) {
    return std::string(name) + "_" + name_of(dtype) + "_" + std::to_string(v);
}

void check_packed(const uint8_t *codes, const uint8_t *scales, const char *what) {
    if (!codes != !scales) fail(kInvalid, std::string(what) + ": codes and scales go together");
}

}  // namespace

// ---- the norm ----------------------------------------------------------------------

void rms_norm(int ordinal, void *stream, const hbr_norm &p) {
    const char *what = "rms norm";
    const uint64_t size = size_of(p.dtype, what), n = p.n_rows, dim = p.dim;
    check_rows(n, dim, what);
    check_packed(p.codes, p.scales, what);
    if (!(p.eps >= 0.0f)) fail(kInvalid, std::string(what) + ": eps is negative or no number");
    if (n == 0) return;
    if (!p.x) fail(kInvalid, std::string(what) + ": null argument");
    const Rows x(p.x, n, dim, p.x_stride, size, what), residual(p.residual, n, dim, p.residual_stride, size, what),
        out(p.out, n, dim, p.out_stride, size, what), total(p.total, n, dim, p.total_stride, size, what),
        codes(p.codes, n, dim, p.codes_stride, 1, what), scales(p.scales, n, scales_of(dim), p.scales_stride, 1, what);
    check_aligned(p.weight, 4, what);
    check_aligned(p.inv, 4, what);
    // (a row is read before it is written, so an output may be an input itself)
    auto apart = [&](const Rows &in) { return in.is(out) || in.is(total) ? Extent(nullptr, 0) : in.extent(); };
    check_apart({out.extent(), total.extent(), codes.extent(), scales.extent(), {p.inv, n * 4}},
                {apart(x), apart(residual), {p.weight, dim * 4}}, Extent(nullptr, 0), what);
    Queue queue(ordinal, stream);
    const uint32_t v = norm_vector(size, dim, kNormNarrow);
    const RowPlan q = row_plan(tiles(dim, v), v, v == 8 ? 2 : 4, p.codes != nullptr);
    NormArgs a{};
    a.x = p.x;
    a.residual = p.residual;
    a.weight = p.weight;
    a.out = p.out;
    a.total = p.total;
    a.inv = p.inv;
    a.codes = p.codes;
    a.scales = p.scales;
    a.x_stride = x.stride;
    a.residual_stride = residual.stride;
    a.out_stride = out.stride;
    a.total_stride = total.stride;
    a.codes_stride = codes.stride;
    a.scales_stride = scales.stride;
    a.n_rows = n;
    a.dim = p.dim;
    a.vecs = (uint32_t)tiles(dim, v);
    a.lanes = q.lanes;
    a.eps = p.eps;
    a.mean = 1.0f / (float)p.dim;
    a.normed = p.normed;
    queue.launch((rows_kernel("hbr_rms_norm", p.dtype, v, dim) + q.name()).c_str(),
                 dim3((uint32_t)std::min<uint64_t>(tiles(n, q.per()), 2048 * 256 / q.threads)), dim3(q.threads), a);
}

namespace {

// Workgroups of the gradient at most: their sums of the weights' gradient are
// held in the workspace, 4 MiB of them where that leaves 512 workgroups, and read
// once more (200,003 rows of 50: 2,048 of them 31.7 us, 1,024 38.3; 65,537 rows of
// 1,024: 119 and 110).
uint64_t norm_grad_blocks(uint64_t dim) {
    const uint64_t by_sums = std::max<uint64_t>(512, std::min<uint64_t>(2048, (1u << 20) / dim));
    return std::max<uint64_t>(1, std::min<uint64_t>(by_sums, (1u << 22) / dim));
}

}  // namespace

uint64_t rms_norm_grad_workspace(uint64_t n, uint32_t dim, uint32_t dtype) {
    size_of(dtype, "rms norm gradient");
    check_rows(n, dim, "rms norm gradient");
    return up(std::min(n, norm_grad_blocks(dim)) * dim * sizeof(float), 256);
}

void rms_norm_grad(int ordinal, void *stream, const hbr_norm_grad &p, void *workspace, uint64_t workspace_bytes) {
    const char *what = "rms norm gradient";
    const uint64_t size = size_of(p.dtype, what), n = p.n_rows, dim = p.dim;
    check_rows(n, dim, what);
    check_packed(p.codes, p.scales, what);
    if (n && (!p.x == !p.codes)) fail(kInvalid, std::string(what) + ": the rows, or the normed rows in 8 bits, are needed");
    if (n && p.codes && !p.inv) fail(kInvalid, std::string(what) + ": rows in 8 bits need inv");
    if (n && !p.dout) fail(kInvalid, std::string(what) + ": null argument");
    if (!p.inv && !(p.eps >= 0.0f)) fail(kInvalid, std::string(what) + ": eps is negative or no number");
    const Rows dout(p.dout, n, dim, p.dout_stride, size, what), x(p.x, n, dim, p.x_stride, size, what),
        codes(p.codes, n, dim, p.codes_stride, 1, what), scales(p.scales, n, scales_of(dim), p.scales_stride, 1, what),
        dtotal(p.dtotal, n, dim, p.dtotal_stride, size, what), dx(p.dx, n, dim, p.dx_stride, size, what);
    for (const void *f : {(const void *)p.inv, (const void *)p.weight, (const void *)p.dweight}) check_aligned(f, 4, what);
    const uint64_t need = p.dweight ? rms_norm_grad_workspace(n, p.dim, p.dtype) : 0;
    check_workspace(workspace, workspace_bytes, need, what);
    auto apart = [&](const Rows &in) { return in.is(dx) ? Extent(nullptr, 0) : in.extent(); };
    check_apart({dx.extent(), {p.dweight, dim * 4}},
                {apart(dout), apart(dtotal), x.extent(), codes.extent(), scales.extent(), {p.inv, n * 4}, {p.weight, dim * 4}},
                Extent(need ? workspace : nullptr, need), what);
    if (!p.dx && !p.dweight) return;
    Queue queue(ordinal, stream);
    uint64_t blocks = 0;
    if (n) {
        const uint32_t v = norm_vector(size, dim, kNormGradNarrow);
        // Two vectors a lane. Four of f32 take 150 registers, which leave a SIMD three
        // waves: 65,429 rows of 1,024 177 us (153 held to 128 registers, ten of them
        // put away), 129,844 of 516 197, 216,129 of 310 212; by two on twice the lanes
        // 147, 168 and 194. Rows that reach back take 206 to 273 us of four and 226 to
        // 256 of two (515 to 1,023 columns, 67,000,000 elements).
        const RowPlan q = row_plan(tiles(dim, v), v, 2, false);
        blocks = std::min(tiles(n, q.per()), norm_grad_blocks(dim));
        NormGradArgs a{};
        a.dout = p.dout;
        a.x = p.x;
        a.dtotal = p.dtotal;
        a.codes = p.codes;
        a.scales = p.scales;
        a.inv = p.inv;
        a.weight = p.weight;
        a.dx = p.dx;
        a.part = p.dweight ? static_cast<float *>(workspace) : nullptr;
        a.dout_stride = dout.stride;
        a.x_stride = x.stride;
        a.dtotal_stride = dtotal.stride;
        a.codes_stride = codes.stride;
        a.scales_stride = scales.stride;
        a.dx_stride = dx.stride;
        a.n_rows = n;
        a.dim = p.dim;
        a.vecs = (uint32_t)tiles(dim, v);
        a.lanes = q.lanes;
        a.eps = p.eps;
        a.mean = 1.0f / (float)p.dim;
        queue.launch((rows_kernel("hbr_rms_norm_grad", p.dtype, v, dim) + q.name()).c_str(), dim3((uint32_t)blocks),
                     dim3(q.threads), a);
    }
    if (!p.dweight) return;
    ColumnJoinArgs j{};
    j.part = static_cast<const float *>(workspace);
    j.dst = p.dweight;
    j.parts = (uint32_t)blocks;
    j.cols = p.dim;
    queue.launch("hbr_column_join", dim3((uint32_t)tiles(dim, 16)), dim3(1024), j);
}

// ---- rows in 8 bits -------------------------------------------------------------------

namespace {

void packed(int ordinal, void *stream, const hbr_packed &p, const void *x, const uint8_t *codes, const uint8_t *scales,
            const float *weight, bool pack, const char *what) {
    const uint64_t size = size_of(p.dtype, what), n = p.n_rows, dim = p.dim;
    check_rows(n, dim, what);
    if (n == 0) return;
    if (!x || !codes || !scales) fail(kInvalid, std::string(what) + ": null argument");
    const Rows rx(x, n, dim, p.x_stride, size, what), rc(codes, n, dim, p.codes_stride, 1, what),
        rs(scales, n, scales_of(dim), p.scales_stride, 1, what), rw(weight, 1, dim, dim, 4, what);
    if (pack) check_apart({rc.extent(), rs.extent()}, {rx.extent()}, Extent(nullptr, 0), what);
    else check_apart({rx.extent()}, {rc.extent(), rs.extent(), rw.extent()}, Extent(nullptr, 0), what);
    Queue queue(ordinal, stream);
    const uint32_t v = row_vector(size, dim);
    PackArgs a{};
    a.x = const_cast<void *>(x);
    a.codes = const_cast<uint8_t *>(codes);
    a.scales = const_cast<uint8_t *>(scales);
    a.weight = weight;
    a.x_stride = rx.stride;
    a.codes_stride = rc.stride;
    a.scales_stride = rs.stride;
    a.n_rows = n;
    a.dim = p.dim;
    a.vecs = (uint32_t)tiles(dim, v);
    a.lanes = power_of_two(std::min<uint64_t>(kWaveLanes, std::max(a.vecs, kPackBlock / v)));
    a.each = 8;
    queue.launch(rows_kernel(pack ? "hbr_pack" : "hbr_unpack", p.dtype, v, dim).c_str(),
                 dim3((uint32_t)std::min<uint64_t>(tiles(n, 256 / a.lanes), 1u << 16), (uint32_t)tiles(up(a.vecs, 32), a.lanes * a.each)),
                 dim3(256), a);
}

}  // namespace

void pack_rows(int ordinal, void *stream, const hbr_packed &p, const void *x, uint8_t *codes, uint8_t *scales) {
    packed(ordinal, stream, p, x, codes, scales, nullptr, true, "pack rows");
}

void unpack_rows(int ordinal, void *stream, const hbr_packed &p, const uint8_t *codes, const uint8_t *scales, const float *weight,
                 void *x) {
    packed(ordinal, stream, p, x, codes, scales, weight, false, "unpack rows");
}

// ---- projections -------------------------------------------------------------------------

namespace {

// A projection's tiles: four waves, a workgroup a CU or two, 64 products a step.
constexpr HeadTiling kLarge{256, 256, 256, "_256"}, kSmall{128, 256, 512, "_128"};
constexpr uint64_t kStepK = 64;

// A product's tiles (m: columns, n: rows of the result) and the shares of its steps.
struct Product {
    const HeadTiling *t;
    uint64_t m_tiles, n_tiles, splits;
    uint64_t groups() const { return m_tiles * n_tiles * splits; }
    // Tiles that do not fill the device have a CU each, and its LDS for more
    // steps in flight.
    std::string name() const { return std::string(t->name) + (t == &kSmall && groups() <= 256 ? "_deep" : ""); }
};
constexpr uint64_t kLeastSteps = 2;  // of a share

uint64_t steps_of(uint64_t k, uint64_t segments) { return tiles(k, kStepK) * segments; }

// The tiles and shares that take least by what a step and a tile's end take, in us
// (bf16 rows of 1,024 to 4,096, the call's 6 in the ends): 4,096 x 4,096 results in
// large tiles 1.48 a step and 15 besides, 8,192 x 4,096 in two rounds 1.50 and 20;
// in small ones 2,048 x 2,048 0.52 and 7, 2,048 x 4,096, two a CU, 0.94 and 6. The
// shares' sums are written and read once more: 512 x 512 results of 4,096 take 36.5
// in small tiles, 24, 17, 16 and 19 in 2, 4, 8 and 16 shares of them, and 82, 30 and
// 23 in large tiles and 4 and 16 shares; 1,024 x 1,024 ones 37, 27, 24 and 27.
Product product_plan(uint64_t m, uint64_t n, uint64_t k, uint64_t segments) {
    const uint64_t steps = steps_of(k, segments);
    Product best{};
    double least = 0.0;
    for (const HeadTiling *t : {&kLarge, &kSmall}) {
        const uint64_t mt = tiles(m, t->tile), nt = tiles(n, t->tile), all = mt * nt;
        const uint64_t most = std::max<uint64_t>(1, std::min(t->slots / std::max<uint64_t>(all, 1), steps / kLeastSteps));
        for (uint64_t s = 1; s <= most; s++) {
            const uint64_t groups = all * s, each = tiles(steps, s);
            const double step = t == &kLarge ? 1.4 : groups <= 256 ? 0.5 : 0.9, more = t == &kLarge ? 9.0 : 4.0;
            const double cost = (double)tiles(groups, t->slots) * ((double)each * step + more) +
                                (s > 1 ? 4.0 + (double)(groups * t->tile * t->tile) * 4.0 / 4.5e6 : 0.0);
            if (!best.t || cost < least) best = {t, mt, nt, s}, least = cost;
        }
    }
    return best;
}

// The f32 sums of its shares, for any number of rows up to those given: no more
// tiles than run at once, nor than shares of the least steps make.
uint64_t part_cells(uint64_t m, uint64_t n, uint64_t k, uint64_t segments) {
    const uint64_t most = steps_of(k, segments) / kLeastSteps;
    uint64_t cells = 0;
    if (most > 1)
        for (const HeadTiling *t : {&kLarge, &kSmall})
            cells = std::max(cells, std::min(t->slots, most * tiles(m, t->tile) * tiles(n, t->tile)) * t->tile * t->tile);
    return cells;
}
uint64_t part_used(const Product &p) { return p.splits > 1 ? p.groups() * p.t->tile * p.t->tile : 0; }

// Chunks of 64 columns: twice the head's.
uint64_t chunk_step(uint64_t rows) { return chunk_bytes(2 * rows); }
uint64_t laid_bytes(uint64_t rows, uint64_t cols, uint64_t parts) { return parts * tiles(cols, kStepK) * chunk_step(rows); }

// A call's operands: in place, or laid out, all of them in one launch.
struct Operands {
    uint32_t dtype;
    LayArgs args{};
    explicit Operands(uint32_t type) : dtype(type) {}
    Laid add(const Rows &r, void *to) {
        if (head_in_place(r.p, r.n > 1 ? r.stride : up(r.width, 8), r.width, dtype))
            return {static_cast<const char *>(r.p), r.stride * 2, kStepK * 2, 0, (uint32_t)r.width};
        return lay(r, nullptr, dtype == HBR_F32 ? kLayF32 : kLayBf16, to);
    }
    Laid add(const Rows &codes, const Rows &scales, void *to) { return lay(codes, &scales, kLayCodes, to); }
    uint32_t blocks() const {
        uint32_t n = 0;
        for (uint32_t i = 0; i < args.arrays; i++) n += args.of[i].blocks;
        return n;
    }
    void launch(Queue &queue) const {
        if (blocks()) queue.launch("hbr_lay", dim3(blocks()), dim3(256), args);
    }

private:
    Laid lay(const Rows &r, const Rows *scales, uint32_t kind, void *to) {
        LayArray &a = args.of[args.arrays++];
        a.src = r.p;
        a.dst = static_cast<uint16_t *>(to);
        a.rows = r.n;
        a.stride = r.stride;
        if (scales) a.scales = static_cast<const uint8_t *>(scales->p), a.scales_stride = scales->stride;
        a.chunk = chunk_step(r.n) / 2;
        a.cols = (uint32_t)r.width;
        a.chunks = (uint32_t)tiles(r.width, kStepK);
        a.part = a.chunks * a.chunk;
        a.kind = kind;
        a.blocks = (uint32_t)std::min<uint64_t>(tiles(r.n * a.chunks * 8, 256), 1u << 16);
        return {static_cast<const char *>(to), kStepK * 2, a.chunk * 2, kind == kLayF32 ? a.part * 2 : 0, a.chunks * (uint32_t)kStepK};
    }
};

// The parts' products of two f32 operands, or of one whose rows are in 8 bits.
void set_segments(HeadArgs &a, uint64_t segments) {
    a.segments = (uint32_t)segments;
    if (segments == 6) a.a_order = kPartA, a.b_order = kPartB;
    if (segments == 3) a.b_order = kPartsByOne;
}

void set_product(LinearArgs &a, const Product &p, float *part) {
    a.p.m_tiles = (uint32_t)p.m_tiles;
    a.p.n_tiles = (uint32_t)p.n_tiles;
    a.p.splits = (uint32_t)p.splits;
    a.large = p.t == &kLarge;
    a.part = p.splits > 1 ? part : nullptr;
}

void run_product(Queue &queue, const std::string &name, const Product &p, const LinearArgs &a) {
    // (a workgroup of the large tiles takes several)
    const uint64_t groups = p.t == &kLarge ? std::min(p.groups(), kLarge.slots) : p.groups();
    queue.launch((name + p.name()).c_str(), dim3((uint32_t)groups), dim3((uint32_t)p.t->threads), a);
}

// What is joined behind products: shares (a workgroup takes four columns of
// every thread's rows of a tile), and db.
struct Joins {
    LinearPairArgs args{};
    uint32_t products = 0;
    void add(const Product &p, const LinearArgs &a) {
        if (p.splits == 1) return;
        args.of[products] = a;
        args.groups[products++] = (uint32_t)(p.m_tiles * p.n_tiles * (p.t->tile * p.t->tile / p.t->threads / 4));
    }
    void launch(Queue &queue, const std::string &type) const {
        const uint32_t groups = args.groups[0] + args.groups[1] + (args.db ? (uint32_t)tiles(args.outs, 16) : 0);
        if (groups) queue.launch(("hbr_linear_joins_" + type).c_str(), dim3(groups), dim3(256), args);
    }
};

void check_product(uint64_t n, uint64_t outs, uint64_t dim, uint32_t dtype, const char *what) {
    size_of(dtype, what);
    check_rows(n, dim, what);
    if (outs == 0) fail(kInvalid, std::string(what) + ": no outputs");
    if (outs >= kDimLimit) fail(kRefused, std::string(what) + ": 1,048,576 outputs or more");
}

// Tiles of 128 that a launch takes.
void check_tiles(uint64_t m, uint64_t n, const char *what) {
    if (tiles(m, 128) * tiles(n, 128) >= 1u << 22) fail(kRefused, std::string(what) + ": 2^22 tiles of 128 x 128 or more");
}

// Whether w is read straight into the matrix instructions' registers: up to 64
// rows, which are read again with every 16 outputs. In f32 always (32 rows,
// 4,096 x 4,096: 29 us, 60 in tiles of three parts); in bf16 while those reads
// take less than the tiles' stages and shares (64 rows: 1,024 x 4,096 7.4 us,
// 11.9 in tiles, 4,096 x 8,192 38.7 and 20.9; 32 rows 25.2 and 20.2). Of 40 cases
// each of 1 to 64 rows, 512 to 8,192 columns and 1,024 to 16,384 outputs that is the
// slower way in seven of bf16 and three of f32, most of them long rows by few outputs,
// whose workgroups leave CUs idle (32 rows of 8,192 by 1,024 bf16 23.1 us and 14.6, 64
// of f32 74.8 and 43.0).
bool few_rows(uint64_t n, uint64_t outs, uint64_t dim, uint32_t dtype) {
    return n <= 64 && (dtype == HBR_F32 || n <= 16 || tiles(n, 16) * outs * dim * 2 <= 48u << 20);
}

struct LinearPlan {
    bool few;
    char *x, *w;
    float *low, *part;
    uint16_t *slot_of;
    int32_t *slot_id;
    uint32_t *slots;
    Product product;
    uint64_t segments, bytes;
};
LinearPlan linear_plan(uint64_t n, uint64_t outs, uint64_t dim, uint64_t rank, uint32_t dtype, void *workspace) {
    LinearPlan q{};
    const uint64_t parts = dtype == HBR_F32 ? 3 : 1;
    Arena w(workspace);
    // (a number of rows is few with every smaller one: room for more serves them)
    q.few = few_rows(n, outs, dim, dtype);
    if (q.few) {
        q.low = w.take<float>(n * rank);
        q.bytes = w.used;
        return q;
    }
    q.segments = dtype == HBR_F32 ? 6 : 1;
    q.product = product_plan(outs, n, dim, q.segments);
    q.x = w.take<char>(laid_bytes(n, dim, parts));
    q.w = w.take<char>(laid_bytes(outs, dim, parts));
    q.low = w.take<float>(n * rank);
    if (rank) {
        q.slot_of = w.take<uint16_t>(n);
        q.slot_id = w.take<int32_t>(up(n, kLarge.tile));
        q.slots = w.take<uint32_t>(tiles(n, kSmall.tile));
    }
    q.part = w.take<float>(part_cells(outs, n, dim, q.segments), part_used(q.product));
    q.bytes = w.used;
    return q;
}

}  // namespace

uint64_t linear_workspace(uint64_t n, uint32_t outs, uint32_t dim, uint32_t rank, uint32_t dtype) {
    check_product(n, outs, dim, dtype, "linear");
    if (rank >= kDimLimit) fail(kRefused, "linear: adapters of rank 1,048,576 or more");
    check_tiles(n, outs, "linear");
    return linear_plan(n, outs, dim, rank, dtype, nullptr).bytes;
}

void linear(int ordinal, void *stream, const hbr_linear_args &p, void *workspace, uint64_t workspace_bytes) {
    const char *what = "linear";
    const uint64_t n = p.n_rows, outs = p.n_outs, dim = p.dim;
    check_product(n, outs, dim, p.dtype, what);
    const uint64_t size = size_of(p.dtype, what), rank = p.n_adapters ? p.rank : 0;
    if (rank >= kDimLimit) fail(kRefused, std::string(what) + ": adapters of rank 1,048,576 or more");
    if (p.n_adapters > 0x7fffffffu) fail(kRefused, std::string(what) + ": more than 2^31 - 1 adapters");
    check_tiles(n, outs, what);
    if (rank && n >= 1u << 27) fail(kRefused, std::string(what) + ": adapters of 2^27 rows or more");
    if (n == 0) return;
    if (!p.x || !p.w || !p.out) fail(kInvalid, std::string(what) + ": null argument");
    if (rank && (!p.down || !p.up || !p.ids)) fail(kInvalid, std::string(what) + ": adapters need down, up and ids");
    const Rows x(p.x, n, dim, p.x_stride, size, what), w(p.w, outs, dim, p.w_stride, size, what),
        out(p.out, n, outs, p.out_stride, size, what),
        down(rank ? p.down : nullptr, p.n_adapters * rank, dim, p.down_stride, size, what),
        up_rows(rank ? p.up : nullptr, p.n_adapters * outs, rank, p.up_stride, size, what);
    for (const void *f : {(const void *)p.bias, (const void *)p.ids, (const void *)p.scale}) check_aligned(f, 4, what);
    const LinearPlan q = linear_plan(n, outs, dim, rank, p.dtype, workspace);
    check_workspace(workspace, workspace_bytes, q.bytes, what);
    check_apart({out.extent()},
                {x.extent(), w.extent(), down.extent(), up_rows.extent(), {p.bias, outs * 4}, {rank ? p.ids : nullptr, n * 4},
                 {rank ? p.scale : nullptr, p.n_adapters * 4ull}}, Extent(workspace, q.bytes), what);
    Queue queue(ordinal, stream);
    const std::string type = name_of(p.dtype);
    // rows of whole 16 bytes, or element by element
    auto strips = [&](const char *name, std::initializer_list<const Rows *> all) {
        const uint32_t v = rows_vector(size, dim, all);
        return kernel_of(name, p.dtype, v == 16 / size ? v : 1);
    };
    const bool few = q.few;
    LinearArgs a{};
    Operands operands(p.dtype);
    if (!few) {
        set_a(a.p, operands.add(w, q.w));
        set_b(a.p, operands.add(x, q.x));
    }
    if (rank) {
        LinearLowArgs l{};
        l.x = p.x;
        l.down = p.down;
        l.ids = p.ids;
        l.scale = p.scale;
        l.low = q.low;
        l.x_stride = x.stride;
        l.down_stride = down.stride;
        l.n_rows = (uint32_t)n;
        l.dim = p.dim;
        l.rank = p.rank;
        l.adapters = p.n_adapters;
        // 16 rows a workgroup; of few of them several for the adapters' ranks
        const uint64_t groups = tiles(n, 16), most = tiles(std::min<uint64_t>(n, 16) * rank, 32);
        l.groups = (uint32_t)groups;
        l.shares = (uint32_t)std::max<uint64_t>(1, std::min(most, 256 / groups));
        if (!few && q.product.splits == 1) {
            l.tile = (uint32_t)q.product.t->tile;
            l.tiles = (uint32_t)q.product.n_tiles;
        }
        l.slot_of = q.slot_of;
        l.slot_id = q.slot_id;
        l.slots = q.slots;
        l.lay = operands.args;
        queue.launch((strips("hbr_linear_low", {&x, &down}) + (few ? "_16" : "")).c_str(),
                     dim3(l.groups * l.shares + l.tiles + operands.blocks()), dim3(few ? 1024 : 256), l);
    } else {
        operands.launch(queue);
    }
    if (few) {
        LinearFewArgs f{};
        f.x = p.x;
        f.w = p.w;
        f.bias = p.bias;
        f.out = p.out;
        f.low = rank ? q.low : nullptr;
        f.up = p.up;
        f.ids = p.ids;
        f.x_stride = x.stride;
        f.w_stride = w.stride;
        f.out_stride = out.stride;
        f.up_stride = up_rows.stride;
        f.n_rows = (uint32_t)n;
        f.dim = p.dim;
        f.outs = p.n_outs;
        f.rank = p.rank;
        f.adapters = p.n_adapters;
        queue.launch((strips("hbr_linear_few", {&x, &w}) + (n <= 16 ? "_16" : n <= 32 ? "_32" : "_64")).c_str(), dim3((uint32_t)tiles(outs, 16)),
                     dim3(256), f);
        return;
    }
    a.p.m = a.cols = p.n_outs;
    a.p.n = a.rows = (uint32_t)n;
    a.p.k = p.dim;
    set_segments(a.p, q.segments);
    set_product(a, q.product, q.part);
    a.out = p.out;
    a.out_stride = out.stride;
    a.bias = p.bias;
    a.low = rank ? q.low : nullptr;
    a.up = p.up;
    a.ids = p.ids;
    a.slot_of = q.slot_of;
    a.slot_id = q.slot_id;
    a.slots = q.slots;
    a.up_stride = up_rows.stride;
    a.rank = p.rank;
    a.adapters = p.n_adapters;
    run_product(queue, a.part ? "hbr_linear_y_part" : (rank ? "hbr_linear_ya_" : "hbr_linear_y_") + type, q.product, a);
    Joins joins;
    joins.add(q.product, a);
    joins.launch(queue, type);
}

namespace {

// Shares of the rows whose sums make db, at most.
uint64_t column_shares(uint64_t outs) { return std::max<uint64_t>(1, 2048 / tiles(outs, 256)); }

struct LinearGradPlan {
    char *dout, *w, *x;
    float *part_x, *part_w, *part_b;
    uint64_t segments_x, segments_w, bytes;
    Product by_x, by_w;
};
// held: the rows are in 8 bits, one part whatever the type
LinearGradPlan linear_grad_plan(uint64_t n, uint64_t outs, uint64_t dim, uint32_t dtype, bool held, void *workspace) {
    LinearGradPlan q{};
    const uint64_t parts = dtype == HBR_F32 ? 3 : 1, segments = dtype == HBR_F32 ? 6 : 1;
    q.segments_x = segments;
    q.segments_w = dtype == HBR_F32 && held ? 3 : segments;
    q.by_x = product_plan(dim, n, outs, q.segments_x);
    q.by_w = product_plan(dim, outs, n, q.segments_w);
    Arena w(workspace);
    q.dout = w.take<char>(laid_bytes(n, outs, parts));
    q.w = w.take<char>(laid_bytes(outs, dim, parts));
    q.x = w.take<char>(laid_bytes(n, dim, parts));
    q.part_x = w.take<float>(part_cells(dim, n, outs, segments), part_used(q.by_x));
    q.part_w = w.take<float>(part_cells(dim, outs, n, segments), part_used(q.by_w));
    // db: sums of the rows' shares, or of the products' shares and tiles of columns
    // (those that run at once, by a tile's rows; or every tile's)
    q.part_b = w.take<float>(std::max({column_shares(outs) * outs, (uint64_t)65536, tiles(dim, kSmall.tile) * outs}),
                             std::max(column_shares(outs), q.by_w.splits * q.by_w.m_tiles) * outs);
    static_assert(kLarge.slots * 256 == 65536 && kSmall.slots * 128 == 65536, "rows of the tiles that run at once");
    q.bytes = w.used;
    return q;
}

}  // namespace

uint64_t linear_grad_workspace(uint64_t n, uint32_t outs, uint32_t dim, uint32_t dtype) {
    check_product(n, outs, dim, dtype, "linear gradient");
    check_tiles(n, dim, "linear gradient");
    check_tiles(outs, dim, "linear gradient");
    return linear_grad_plan(n, outs, dim, dtype, false, nullptr).bytes;
}

void linear_grad(int ordinal, void *stream, const hbr_linear_grad_args &p, void *workspace, uint64_t workspace_bytes) {
    const char *what = "linear gradient";
    const uint64_t n = p.n_rows, outs = p.n_outs, dim = p.dim;
    check_product(n, outs, dim, p.dtype, what);
    check_tiles(n, dim, what);
    check_tiles(outs, dim, what);
    check_packed(p.codes, p.scales, what);
    const uint64_t size = size_of(p.dtype, what);
    if (n && !p.dout) fail(kInvalid, std::string(what) + ": null argument");
    if (p.dx && n && !p.w) fail(kInvalid, std::string(what) + ": dx needs w");
    if (p.dw && n && (!p.x == !p.codes)) fail(kInvalid, std::string(what) + ": dw needs the rows, as they are or in 8 bits");
    const Rows dout(p.dout, n, outs, p.dout_stride, size, what), w(p.w, outs, dim, p.w_stride, size, what),
        x(p.x, n, dim, p.x_stride, size, what), codes(p.codes, n, dim, p.codes_stride, 1, what),
        scales(p.scales, n, scales_of(dim), p.scales_stride, 1, what), dx(p.dx, n, dim, p.dx_stride, size, what),
        dw(p.dw, outs, dim, p.dw_stride, size, what);
    check_aligned(p.weight, 4, what);
    check_aligned(p.db, 4, what);
    const bool held = p.codes != nullptr;
    const LinearGradPlan q = linear_grad_plan(n, outs, dim, p.dtype, held, workspace);
    check_workspace(workspace, workspace_bytes, q.bytes, what);
    check_apart({dx.extent(), dw.extent(), {p.db, outs * 4}},
                {dout.extent(), w.extent(), x.extent(), codes.extent(), scales.extent(), {p.weight, dim * 4}},
                Extent(workspace, q.bytes), what);
    if (!p.dw && !p.db && (!p.dx || n == 0)) return;
    Queue queue(ordinal, stream);
    const std::string type = name_of(p.dtype);
    if (n == 0) {  // sums over no rows
        if (p.dw) sum_parts(queue, p.dtype, 1.0f, nullptr, 0, 0, p.dw, outs, dim, dw.stride);
        if (p.db) sum_parts(queue, HBR_F32, 1.0f, nullptr, 0, 0, p.db, 1, outs, outs);
        return;
    }
    uint64_t sums = 0;  // of db
    Joins joins;
    if (p.db && !p.dw) {
        ColumnSumArgs a{};
        a.x = p.dout;
        a.part = q.part_b;
        a.rows = n;
        a.x_stride = dout.stride;
        a.cols = p.n_outs;
        a.shares = (uint32_t)std::min(column_shares(outs), tiles(n, 32));
        sums = a.shares;
        queue.launch(("hbr_column_sum_" + type).c_str(), dim3((uint32_t)tiles(outs, 256) * a.shares), dim3(256), a);
    }
    if (p.dx || p.dw) {
        LinearArgs x_args{}, w_args{};
        Operands operands(p.dtype);
        const Laid by = operands.add(dout, q.dout);
        if (p.dx) set_a(x_args.p, operands.add(w, q.w));
        if (p.dw) set_a(w_args.p, held ? operands.add(codes, scales, q.x) : operands.add(x, q.x));
        operands.launch(queue);
        // (a transposed operand's columns are read in eights: in place there are
        // whole ones, laid out zeros stand behind them)
        if (p.dx) {
            LinearArgs &a = x_args;
            set_b(a.p, by);
            a.p.m = (uint32_t)up(dim, 8);
            a.p.n = a.rows = (uint32_t)n;
            a.cols = p.dim;
            a.p.k = p.n_outs;
            set_segments(a.p, q.segments_x);
            set_product(a, q.by_x, q.part_x);
            a.out = p.dx;
            a.out_stride = dx.stride;
        }
        if (p.dw) {
            LinearArgs &a = w_args;
            set_b(a.p, by);
            a.p.m = (uint32_t)up(dim, 8);
            a.p.n = (uint32_t)up(outs, 8);
            a.cols = p.dim;
            a.rows = p.n_outs;
            a.p.k = (uint32_t)n;
            set_segments(a.p, q.segments_w);
            set_product(a, q.by_w, q.part_w);
            a.out = p.dw;
            a.out_stride = dw.stride;
            a.weight = p.weight;
            a.part_b = p.db ? q.part_b : nullptr;
            if (p.db) sums = q.by_w.splits * q.by_w.m_tiles;
        }
        // both in one launch where both have small tiles that run at once (4,001 x
        // 250 x 333 in f32: 26 us in two launches)
        if (p.dx && p.dw && q.by_x.t == &kSmall && q.by_w.t == &kSmall && q.by_x.groups() + q.by_w.groups() <= kSmall.slots) {
            LinearPairArgs pair{};
            pair.of[0] = x_args;
            pair.of[1] = w_args;
            pair.groups[0] = (uint32_t)q.by_x.groups();
            pair.groups[1] = (uint32_t)q.by_w.groups();
            queue.launch(("hbr_linear_pair_" + type).c_str(), dim3(pair.groups[0] + pair.groups[1]), dim3(256), pair);
        } else {
            if (p.dx) run_product(queue, "hbr_linear_dx_" + type, q.by_x, x_args);
            if (p.dw) run_product(queue, "hbr_linear_dw_" + type, q.by_w, w_args);
        }
        if (p.dx) joins.add(q.by_x, x_args);
        if (p.dw) joins.add(q.by_w, w_args);
    }
    joins.args.part_b = q.part_b;
    joins.args.db = p.db;
    joins.args.b_parts = (uint32_t)sums;
    joins.args.outs = p.n_outs;
    joins.launch(queue, type);
}

}  // namespace hbr
