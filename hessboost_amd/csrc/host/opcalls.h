// What the operators' host code shares: checks of arrays, workspaces, the
// caller's stream, and the tiles of the products.
#pragma once
#include <algorithm>
#include <cstdint>
#include <initializer_list>
#include <string>

#include "../abi.h"
#include "hessboost_rocm.h"
#include "runtime.h"

namespace hbr {

constexpr uint32_t kWaveLanes = 64;

inline uint64_t up(uint64_t v, uint64_t to) { return (v + to - 1) / to * to; }

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

inline uint64_t size_of(uint32_t dtype, const char *what) {
    if (dtype == HBR_F32) return 4;
    if (dtype == HBR_BF16) return 2;
    fail(kInvalid, std::string(what) + ": the type is neither HBR_F32 nor HBR_BF16");
}

inline void check_workspace(const void *p, uint64_t have, uint64_t need, const char *what) {
    if (need == 0) return;
    if (!p || have < need)
        fail(kInvalid, std::string(what) + ": the workspace holds " + std::to_string(p ? have : 0) + " bytes of " +
                           std::to_string(need));
    if (reinterpret_cast<uint64_t>(p) % 16)
        fail(kInvalid, std::string(what) + ": the workspace is not aligned to 16 bytes");
}

inline void check_aligned(const void *p, uint64_t size, const char *what) {
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
inline bool overlap(const Extent &a, const Extent &b) {
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

inline void check_apart(std::initializer_list<Extent> outputs, std::initializer_list<Extent> inputs, const Extent &workspace, const char *what) {
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

// Vectors and inputs are shorter, so that offsets within one fit 32 bits and
// grids over their elements a launch.
constexpr uint64_t kDimLimit = 1u << 20;

inline const char *name_of(uint32_t dtype) { return dtype == HBR_F32 ? "f32" : "bf16"; }

// ---- products ------------------------------------------------------------------

inline uint64_t tiles(uint64_t n, uint64_t of) { return (n + of - 1) / of; }

// Bytes from one chunk of 32 bf16 columns to the next. An odd multiple of
// 2 KiB: the chunks of a tile, whose steps of 32 rows are 2 KiB each, then
// begin in different halves of the L2's channels.
constexpr uint64_t kChunkStep = 2048;
inline uint64_t chunk_bytes(uint64_t rows) { return ((rows * 64 + 2 * kChunkStep - 1) / (2 * kChunkStep) * 2 + 1) * kChunkStep; }

// What the products can read in place: bf16 rows of whole 16-byte pieces,
// near enough to each other for a tile's 32-bit offsets.
inline bool head_in_place(const void *p, uint64_t stride, uint64_t dim, uint32_t dtype) {
    return dtype == HBR_BF16 && dim % 8 == 0 && stride % 8 == 0 && stride < (1u << 22) &&
           reinterpret_cast<uint64_t>(p) % 16 == 0;
}

// An operand of a product, in place or laid out in chunks of 32 columns.
struct Laid {
    const char *p;
    uint64_t row, chunk, part;
    uint32_t cols;
};
inline void set_a(HeadArgs &a, const Laid &o) { a.a = o.p, a.a_row = o.row, a.a_chunk = o.chunk, a.a_part = o.part; }
inline void set_b(HeadArgs &a, const Laid &o) { a.b = o.p, a.b_row = o.row, a.b_chunk = o.chunk, a.b_part = o.part; }

// dst = scale times the sum of the parts.
inline void sum_parts(Queue &queue, uint32_t dtype, float scale, const float *part, uint64_t parts, uint64_t part_stride, void *dst,
                      uint64_t rows, uint64_t cols, uint64_t dst_stride) {
    HeadSumArgs a{};
    a.scale = scale;
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
    queue.launch(dtype == HBR_F32 ? "hbr_head_sum_f32" : "hbr_head_sum_bf16",
                 dim3((uint32_t)std::min<uint64_t>(tiles(rows * cols, each), 1u << 16)), dim3(waves * 64), a);
}

// A product's tiles, and how many of them fill 256 CUs (of the small ones twice
// as many run at once, at hardly more rate).
struct HeadTiling {
    uint64_t tile, threads, slots;
    const char *name;
};

}  // namespace hbr
