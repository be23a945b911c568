// The operators whose parameters are chosen row by row behind the C ABI: checks of arguments, choice of kernels, launches.
// Their device code is in row_groups.h and typed_products.h (compiled per element type from typed_products.hip).
#include "oeq_amd.h"
#include "oeq_error.h"

#include "row_groups.h"
#include "typed_products_launch.h"

#include <algorithm>
#include <climits>
#include <cmath>

using oeq_internal::fail;

namespace {

int element_bytes(int type) {
    return type == OEQ_FLOAT32 ? 4 : type == OEQ_FLOAT16 || type == OEQ_BFLOAT16 ? 2 : 0;
}

bool aligned(const void* p, int to = 16) { return ((uintptr_t)p & (to - 1)) == 0; }
// Whether rows with these strides, in elements of some bytes, all begin at multiples of 16 bytes.
bool aligned(const void* p, int bytes, std::initializer_list<int64_t> strides) {
    for (int64_t s : strides)
        if (s * bytes % 16) return false;
    return aligned(p);
}

int64_t divide_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Blocks of 256 threads in a launch: threads are counted in 32 bits.
constexpr int64_t kMostBlocks = (1 << 24) - 1;
// Rows (times parts) and types: slots and places are counted in 32 bits.
constexpr int64_t kMostRows = 1 << 29, kMostTypes = 1 << 23;

// Elements between rows of sums' operands: their bytes are counted in 32 bits.
constexpr int64_t kMostStride = INT_MAX / 4;

int check_index(const char* who, int64_t rows, int64_t parts, int64_t types) {
    if (rows < 0 || parts < 1 || types < 0 || types > kMostTypes || rows > kMostRows / parts)
        return fail(OEQ_ERR_INVALID, "%s: %lld rows of %lld parts, %lld types", who, (long long)rows, (long long)parts,
                    (long long)types);
    return OEQ_OK;
}

// Passes over the bits of keys 0 .. types.
int passes_of(int64_t types) {
    int passes = 1;
    while (types >> (passes * row_groups::kBits)) ++passes;
    return passes;
}

// Rows of a block in a pass.
int span_of(int64_t rows) {
    const int64_t least = row_groups::kThreads, even = divide_up(rows, row_groups::kMostBlocks);
    return (int)std::max(least, divide_up(even, row_groups::kThreads) * row_groups::kThreads);
}

// Lanes next to each other that share a row of that many vectors: a power of two.
int lanes_across(int64_t vectors) {
    int lanes = 1;
    while (lanes < 256 && lanes < vectors) lanes *= 2;
    return lanes;
}

template <typename T, int V>
int launch_lookup(int64_t rows, int64_t types, int64_t channels, const int64_t* type_of_row, const void* table,
                  int64_t table_row, float scale, void* out, hipStream_t s) {
    const int across = lanes_across(channels / V), each = 256 / across * row_groups::kLookups;
    const int64_t blocks = divide_up(rows, each);
    for (int64_t first = 0; first < blocks; first += kMostBlocks) {
        const int64_t row = first * each;
        row_groups::lookup<T, V><<<(unsigned)std::min(kMostBlocks, blocks - first), 256, 0, s>>>(
            (const T*)table, table_row, type_of_row + row, rows - row, (int)types, (int)channels, across, scale,
            (T*)out + row * channels);
        HIP_TRY(hipGetLastError());
    }
    return OEQ_OK;
}

template <typename T, int V>
int launch_sum(const row_groups::Sums& g, hipStream_t s) {
    const int64_t vectors = g.channels / V;
    const int across = lanes_across(vectors);
    const unsigned chunks = g.n > row_groups::kChunk ? (unsigned)divide_up(g.n, row_groups::kChunk) : 0;
    const unsigned blocks = (unsigned)divide_up(g.count, 256 / across * row_groups::kTypes);
    row_groups::sum_types<T, V><<<dim3(blocks + chunks, (unsigned)divide_up(vectors, across)), 256, 0, s>>>(g, across, (int)blocks);
    HIP_TRY(hipGetLastError());
    if (chunks) {
        const int few = std::min(across, 16);
        row_groups::join_chunks<T, V><<<dim3(chunks, (unsigned)divide_up(vectors, few)), 256, 0, s>>>(g, few);
        HIP_TRY(hipGetLastError());
    }
    return OEQ_OK;
}

int check_rows(const char* who, const oeq_typed_rows* a, bool thin_result) {
    if (!a) return fail(OEQ_ERR_INVALID, "%s: NULL description", who);
    if (!element_bytes(a->type)) return fail(OEQ_ERR_INVALID, "%s: element type %d", who, a->type);
    if (int rc = check_index(who, a->rows, a->parts, a->types)) return rc;
    if (a->inner < 0 || a->outer < 0 || a->inner > INT_MAX - 256 || a->outer > INT_MAX - 256)
        return fail(OEQ_ERR_INVALID, "%s: %lld inner and %lld outer channels", who, (long long)a->inner, (long long)a->outer);
    if (a->rank < 0 || a->rank > INT_MAX - 8 || (a->rank && (a->parts != 1 || thin_result)))
        return fail(OEQ_ERR_INVALID, "%s: a thin product of rank %d", who, a->rank);
    for (int64_t s : {a->x_row_stride, a->x_part_stride, a->w_type_stride, a->w_row_stride, a->up_type_stride, a->up_outer_stride,
                      a->up_rank_stride})
        if (s < 0) return fail(OEQ_ERR_INVALID, "%s: a stride of %lld elements", who, (long long)s);
    if (a->bias && a->shared) return fail(OEQ_ERR_INVALID, "%s: a bias beside shared weights", who);
    if (a->rows == 0 || a->outer == 0) return OEQ_OK;
    if ((a->inner && (!a->x || ((a->types || a->shared) && !a->w))) || !a->type_of_row)
        return fail(OEQ_ERR_INVALID, "%s: NULL buffer", who);
    if (oeq_typed_needs_index(a) && (!a->order || !a->ptr)) return fail(OEQ_ERR_INVALID, "%s: NULL buffer", who);
    if (a->rank && a->types && (!a->thin || !a->up)) return fail(OEQ_ERR_INVALID, "%s: NULL buffer", who);
    const int bytes = element_bytes(a->type);
    if (!aligned(a->x, bytes) || !aligned(a->w, bytes) || !aligned(a->bias, bytes) || !aligned(a->up, bytes) || !aligned(a->thin))
        return fail(OEQ_ERR_INVALID, "%s: unaligned buffer", who);
    return OEQ_OK;
}

typed_products::Args rows_args(const oeq_typed_rows& a) {
    typed_products::Args g = {};
    g.x = a.x, g.w = a.w, g.bias = a.bias, g.up = a.up, g.thin = a.rank ? a.thin : nullptr;
    g.order = a.order, g.ptr = a.ptr, g.type_of_row = a.type_of_row;
    g.x_row = a.x_row_stride, g.x_part = a.x_part_stride, g.w_type = a.shared ? 0 : a.w_type_stride, g.w_row = a.w_row_stride;
    g.bias_type = a.outer, g.out_row = a.outer;
    g.up_type = a.up_type_stride, g.up_col = a.up_outer_stride, g.up_rank = a.up_rank_stride;
    g.rows = (int)a.rows, g.types = (int)a.types, g.parts = (int)a.parts;
    g.inner = (int)a.inner, g.outer = (int)a.outer, g.rank = a.rank, g.thin_row = (int)oeq_thin_stride(a.rank);
    g.shared = a.shared != 0;
    return g;
}

int launch_rows(const char* who, const oeq_typed_rows& a, const typed_products::Args& g, bool wide, void* stream) {
    const int bytes = element_bytes(a.type), e = 16 / bytes;
    const bool direct = aligned(a.x, bytes, {a.x_row_stride, a.x_part_stride}) &&
                        aligned(a.w, bytes, {a.shared ? 0 : a.w_type_stride, a.w_row_stride}) && a.inner % e == 0 &&
                        (!a.across || a.outer % e == 0);
    const auto s = (hipStream_t)stream;
    const hipError_t status = a.type == OEQ_FLOAT32 ? typed_products::Launch<float>::rows(g, a.across != 0, wide, direct, s)
                          : a.type == OEQ_FLOAT16 ? typed_products::Launch<_Float16>::rows(g, a.across != 0, wide, direct, s)
                                                  : typed_products::Launch<__bf16>::rows(g, a.across != 0, wide, direct, s);
    if (status == hipErrorInvalidConfiguration)
        return fail(OEQ_ERR_INVALID, "%s: %lld rows of %lld parts and %lld columns are too many for a launch", who,
                    (long long)a.rows, (long long)a.parts, (long long)a.outer);
    HIP_TRY(status);
    return OEQ_OK;
}

// How a sum over rows is cut: columns of a tile, and the rows that a block sums up before their sums pass through memory. How many
// rows a type has is on the device; a cut costs only types that have more rows than one block's.
struct Cut {
    int tile;
    int64_t chunk, shares;
    Cut(const oeq_typed_sum& a, bool direct) {
        using namespace typed_products;
        constexpr int64_t kBlocks = 1024, kLeast = 256, kShort = 1024, kMostBytes = (int64_t)1 << 29;
        const auto tiles = [&](int to) {
            return std::min(divide_up(a.a_columns, a.thin == 1 ? kThinTile : to) * divide_up(a.b_columns, a.thin == 2 ? kThinTile : to),
                            (int64_t)1 << 30);
        };
        const int64_t rows = a.rows * a.parts;
        shares = 0;
        // (through registers small tiles only, whose loads on their way fit beside the sums)
        tile = a.thin || (direct && (a.types * tiles(kSumTile) >= kBlocks || rows / kLeast * tiles(kSumTile) >= kBlocks)) ? kSumTile
                                                                                                                     : kSmallSumTile;
        if (!a.thin && direct && a.parts == 1 && a.type != OEQ_FLOAT32 && a.types * tiles(kLargeSumTile) >= 256) tile = kLargeSumTile;
        chunk = rows + 1;
        // Every type's tiles fill the card, or large ones of all types together several times over, or sums are so short that they end
        // before a second launch has begun (whose grid has room for so many types). A cut costs what is even and saves what is not: 16 411
        // rows, 32 matrices of 1024 x 2048, 144 .. 163 us of sums uncut; with shares of 4096 rows, of which these types need one each, 177
        // (128 blocks more have no rows, but shift the others' places on the XCDs) and 6 for the launch that joins nothing. With 9 800 of the
        // rows of one type 318 uncut, 203 and 43 cut. Uncut is the choice for types that are used evenly.
        if (tiles(tile) >= 256 || (tile == kLargeSumTile && a.types * tiles(tile) >= kBlocks) || rows <= kShort || a.types > 65535) return;
        if (tile == kLargeSumTile || a.types * tiles(tile) >= kBlocks) {
            // All types' tiles together fill it: cut only what would go on when the others have ended. 20 000 rows, 89 types
            // of which one has 12 400, 512 x 512, float32: 208 us, 851 without.
            chunk = tile == kLargeSumTile ? 4096 : 2048;
        } else {
            chunk = std::max(kLeast, divide_up(rows * tiles(tile), kBlocks * 64) * 64);
        }
        const int64_t bytes = 2 * a.a_columns * a.b_columns * (int64_t)sizeof(float);  // (of 256 tiles at most)
        chunk = std::max(chunk, divide_up(rows * bytes / kMostBytes + 1, 64) * 64);
        shares = rows > chunk ? 2 * (rows / chunk + 1) : 0;
    }
};

bool direct_sum(const oeq_typed_sum& a) {
    const int a_bytes = a.thin == 1 ? 4 : element_bytes(a.type), b_bytes = a.thin == 2 ? 4 : element_bytes(a.type);
    return aligned(a.a, a_bytes, {a.a_row_stride, a.a_part_stride, a.a_columns}) &&
           aligned(a.b, b_bytes, {a.b_row_stride, a.b_part_stride, a.b_columns});
}

}  // namespace

extern "C" {

size_t oeq_group_rows_workspace_bytes(int64_t rows, int64_t types) {
    if (rows <= row_groups::kOneBlock || types < 0) return 0;
    const int passes = passes_of(types);
    // digits' counts; keys and numbers on their way, twice where there is a pass between two others
    const int64_t buffers = passes == 1 ? 0 : passes == 2 ? 3 : 4;
    return (size_t)(divide_up(rows, span_of(rows)) * row_groups::kDigits + buffers * rows) * sizeof(int);
}

int oeq_group_rows(int64_t rows, int64_t types, const int64_t* type_of_row, int32_t* order, int32_t* ptr, void* workspace,
                   size_t workspace_bytes, void* stream) {
    const char* who = "oeq_group_rows";
    if (int rc = check_index(who, rows, 1, types)) return rc;
    if (!ptr || (rows && (!type_of_row || !order))) return fail(OEQ_ERR_INVALID, "%s: NULL buffer", who);
    const size_t need = oeq_group_rows_workspace_bytes(rows, types);
    if (need && (!workspace || workspace_bytes < need)) return fail(OEQ_ERR_INVALID, "%s: workspace too small", who);
    const auto s = (hipStream_t)stream;
    const int passes = passes_of(types), n = (int)rows;
    if (rows <= row_groups::kOneBlock) {
        row_groups::sort_in_block<<<1, row_groups::kThreads, 0, s>>>(type_of_row, n, (int)types, passes, order, ptr);
        HIP_TRY(hipGetLastError());
        return OEQ_OK;
    }
    const int span = span_of(rows), blocks = (int)divide_up(rows, span);
    int* counts = (int*)workspace;
    int* buffer[4];
    for (int i = 0; i < 4; ++i) buffer[i] = counts + blocks * row_groups::kDigits + i * rows;
    // pass p reads keys and numbers of the pass before; the last one's numbers are the order
    row_groups::Source from = {type_of_row, nullptr, nullptr, (int)types};
    for (int p = 0; p < passes; ++p) {
        const bool last = p + 1 == passes;
        int* keys = passes == 1 ? nullptr : buffer[passes == 2 ? (p ? 2 : 0) : (p % 2 ? 2 : 0)];
        int* numbers = last ? order : buffer[p % 2 ? 3 : 1];
        row_groups::count_digits<<<blocks, row_groups::kThreads, 0, s>>>(from, n, span, p * row_groups::kBits, counts);
        HIP_TRY(hipGetLastError());
        row_groups::place_rows<<<blocks, row_groups::kThreads, 0, s>>>(from, n, span, p * row_groups::kBits, counts, blocks, keys,
                                                                     numbers, passes == 1 ? ptr : nullptr, (int)types);
        HIP_TRY(hipGetLastError());
        from = {nullptr, keys, numbers, (int)types};
    }
    if (passes > 1) {
        row_groups::find_types<<<(unsigned)divide_up(types + 1, 256), 256, 0, s>>>(from.keys, n, (int)types, ptr);
        HIP_TRY(hipGetLastError());
    }
    return OEQ_OK;
}

int oeq_type_lookup(int type, int64_t rows, int64_t types, int64_t channels, const int64_t* type_of_row, const void* table,
                    int64_t table_row_stride, double scale, void* out, void* stream) {
    const char* who = "oeq_type_lookup";
    const int bytes = element_bytes(type);
    if (!bytes) return fail(OEQ_ERR_INVALID, "%s: element type %d", who, type);
    if (rows < 0 || types < 0 || types > INT_MAX || channels < 0 || channels > INT_MAX - 1024 || table_row_stride < 0)
        return fail(OEQ_ERR_INVALID, "%s: %lld rows, %lld types of %lld channels", who, (long long)rows, (long long)types,
                    (long long)channels);
    if (rows == 0 || channels == 0) return OEQ_OK;
    if (!type_of_row || !out || (types && !table)) return fail(OEQ_ERR_INVALID, "%s: NULL buffer", who);
    if (!aligned(table, bytes) || !aligned(out, bytes)) return fail(OEQ_ERR_INVALID, "%s: unaligned buffer", who);
    const bool vec = aligned(table, bytes, {table_row_stride, channels}) && aligned(out);
    const auto s = (hipStream_t)stream;
#define OEQ_LOOKUP(T, V) launch_lookup<T, V>(rows, types, channels, type_of_row, table, table_row_stride, (float)scale, out, s)
    switch (type) {
        case OEQ_FLOAT32: return vec ? OEQ_LOOKUP(float, 4) : OEQ_LOOKUP(float, 1);
        case OEQ_FLOAT16: return vec ? OEQ_LOOKUP(_Float16, 8) : OEQ_LOOKUP(_Float16, 1);
        default: return vec ? OEQ_LOOKUP(__bf16, 8) : OEQ_LOOKUP(__bf16, 1);
    }
#undef OEQ_LOOKUP
}

size_t oeq_type_sum_workspace_bytes(int64_t rows, int64_t, int64_t channels) {
    if (rows <= row_groups::kChunk || channels <= 0) return 0;
    return (size_t)divide_up(rows, row_groups::kChunk) * 2 * channels * sizeof(float);
}

int oeq_type_sum(int type, int64_t rows, int64_t parts, int64_t types, int64_t channels, const int64_t* type_of_row,
                 const int32_t* order, const int32_t* ptr, const void* x, int64_t row_stride, int64_t part_stride, double scale,
                 void* out, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "oeq_type_sum";
    const int bytes = element_bytes(type);
    if (!bytes) return fail(OEQ_ERR_INVALID, "%s: element type %d", who, type);
    if (int rc = check_index(who, rows, parts, types)) return rc;
    if (types + divide_up(rows, row_groups::kChunk) > kMostBlocks)
        return fail(OEQ_ERR_INVALID, "%s: %lld rows of %lld types are too many for a launch", who, (long long)rows, (long long)types);
    if (channels < 0 || channels > (1 << 19) || row_stride < 0 || part_stride < 0)
        return fail(OEQ_ERR_INVALID, "%s: %lld channels, strides of %lld and %lld elements", who, (long long)channels,
                    (long long)row_stride, (long long)part_stride);
    if (types == 0 || channels == 0) return OEQ_OK;
    if (!out || !ptr || (rows && (!x || !order || !type_of_row))) return fail(OEQ_ERR_INVALID, "%s: NULL buffer", who);
    if (!aligned(x, bytes) || !aligned(out, bytes)) return fail(OEQ_ERR_INVALID, "%s: unaligned buffer", who);
    const size_t need = oeq_type_sum_workspace_bytes(rows, types, channels);
    if (need && (!workspace || workspace_bytes < need)) return fail(OEQ_ERR_INVALID, "%s: workspace too small", who);
    row_groups::Sums g = {};
    g.rows = x, g.row = row_stride, g.part = part_stride, g.out = out, g.types = type_of_row, g.order = order, g.ptr = ptr;
    g.partial = (float*)workspace, g.count = (int)types, g.n = (int)rows, g.parts = (int)parts, g.channels = (int)channels;
    g.scale = (float)scale;
    const bool vec = aligned(x, bytes, {row_stride, part_stride, channels}) && aligned(out);
    const auto s = (hipStream_t)stream;
    switch (type) {
        case OEQ_FLOAT32: return vec ? launch_sum<float, 4>(g, s) : launch_sum<float, 1>(g, s);
        case OEQ_FLOAT16: return vec ? launch_sum<_Float16, 8>(g, s) : launch_sum<_Float16, 1>(g, s);
        default: return vec ? launch_sum<__bf16, 8>(g, s) : launch_sum<__bf16, 1>(g, s);
    }
}

int oeq_typed_needs_index(const oeq_typed_rows* a) {
    if (!a || a->rows <= 0 || a->parts < 1 || a->rows > kMostRows / a->parts) return 1;
    typed_products::Args g = {};
    g.rows = (int)a->rows, g.parts = (int)a->parts, g.shared = a->shared;
    return !typed_products::few(g, a->across != 0);
}

int oeq_typed_product(const oeq_typed_rows* a, void* out, void* stream) {
    const char* who = "oeq_typed_product";
    if (int rc = check_rows(who, a, false)) return rc;
    if (a->rows == 0 || a->outer == 0) return OEQ_OK;
    if (!out) return fail(OEQ_ERR_INVALID, "%s: NULL buffer", who);
    if (!aligned(out)) return fail(OEQ_ERR_INVALID, "%s: unaligned buffer", who);
    typed_products::Args g = rows_args(*a);
    g.out = out;
    return launch_rows(who, *a, g, false, stream);
}

int64_t oeq_thin_stride(int64_t rank) { return (rank + 7) / 8 * 8; }

int oeq_typed_thin_product(const oeq_typed_rows* a, const float* scale, float* out, void* stream) {
    const char* who = "oeq_typed_thin_product";
    if (int rc = check_rows(who, a, true)) return rc;
    if (a->rows == 0 || a->outer == 0) return OEQ_OK;
    if (a->parts != 1 || a->shared || a->bias) return fail(OEQ_ERR_INVALID, "%s: parts, shared weights or a bias", who);
    if (!out) return fail(OEQ_ERR_INVALID, "%s: NULL buffer", who);
    if (!aligned(out)) return fail(OEQ_ERR_INVALID, "%s: unaligned buffer", who);
    typed_products::Args g = rows_args(*a);
    g.out = out, g.scale = scale, g.out_row = oeq_thin_stride(a->outer);
    return launch_rows(who, *a, g, true, stream);
}

size_t oeq_typed_sum_workspace_bytes(const oeq_typed_sum* a) {
    if (!a || !element_bytes(a->type) || a->rows <= 0 || a->parts < 1 || a->types <= 0 || a->a_columns <= 0 || a->b_columns <= 0) return 0;
    return (size_t)Cut(*a, direct_sum(*a)).shares * a->a_columns * a->b_columns * sizeof(float);
}

int oeq_typed_sum_products(const oeq_typed_sum* a, void* out, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "oeq_typed_sum_products";
    if (!a) return fail(OEQ_ERR_INVALID, "%s: NULL description", who);
    if (!element_bytes(a->type)) return fail(OEQ_ERR_INVALID, "%s: element type %d", who, a->type);
    if (int rc = check_index(who, a->rows, a->parts, a->types)) return rc;
    if (a->a_columns < 0 || a->b_columns < 0 || a->a_columns > INT_MAX - 256 || a->b_columns > INT_MAX - 256)
        return fail(OEQ_ERR_INVALID, "%s: %lld and %lld columns", who, (long long)a->a_columns, (long long)a->b_columns);
    if (a->thin < 0 || a->thin > 2) return fail(OEQ_ERR_INVALID, "%s: thin operand %d", who, a->thin);
    // (the kernel of mixed operands is built for rows of one part: it would look places times parts up in the index)
    if (a->thin && a->parts != 1) return fail(OEQ_ERR_INVALID, "%s: a thin operand of %lld parts", who, (long long)a->parts);
    for (int64_t s : {a->a_row_stride, a->a_part_stride, a->b_row_stride, a->b_part_stride})
        if (s < 0 || s > kMostStride) return fail(OEQ_ERR_INVALID, "%s: a stride of %lld elements", who, (long long)s);
    if (a->types == 0 || a->a_columns == 0 || a->b_columns == 0) return OEQ_OK;
    if (!out || !a->ptr || (a->rows && (!a->a || !a->b || !a->order))) return fail(OEQ_ERR_INVALID, "%s: NULL buffer", who);
    const int a_bytes = a->thin == 1 ? 4 : element_bytes(a->type), b_bytes = a->thin == 2 ? 4 : element_bytes(a->type);
    if (!aligned(a->a, a_bytes) || !aligned(a->b, b_bytes) || !aligned(out, element_bytes(a->type)))
        return fail(OEQ_ERR_INVALID, "%s: unaligned buffer", who);
    const size_t need = oeq_typed_sum_workspace_bytes(a);
    if (need && (!workspace || workspace_bytes < need)) return fail(OEQ_ERR_INVALID, "%s: workspace too small", who);
    typed_products::SumArgs g = {};
    g.a = a->a, g.b = a->b, g.out = out, g.partial = need ? (float*)workspace : nullptr;
    g.order = a->order, g.ptr = a->ptr;
    g.a_row = a->a_row_stride, g.a_part = a->a_part_stride, g.b_row = a->b_row_stride, g.b_part = a->b_part_stride;
    g.rows = (int)a->rows, g.types = (int)a->types, g.parts = (int)a->parts;
    g.a_columns = (int)a->a_columns, g.b_columns = (int)a->b_columns;
    const int64_t rows = a->rows * a->parts;
    const bool direct = direct_sum(*a);
    const Cut cut(*a, direct);
    g.tile = cut.tile, g.chunk = (int)cut.chunk;
    g.slots = (int)(rows / g.chunk + a->types);
    const auto thin = (typed_products::Thin)a->thin;
    const auto s = (hipStream_t)stream;
    const hipError_t status = a->type == OEQ_FLOAT32 ? typed_products::Launch<float>::sums(g, thin, direct, s)
                         : a->type == OEQ_FLOAT16 ? typed_products::Launch<_Float16>::sums(g, thin, direct, s)
                                                  : typed_products::Launch<__bf16>::sums(g, thin, direct, s);
    if (status == hipErrorInvalidConfiguration)
        return fail(OEQ_ERR_INVALID, "%s: %lld by %lld columns of %lld types are too many for a launch", who,
                    (long long)a->a_columns, (long long)a->b_columns, (long long)a->types);
    HIP_TRY(status);
    return OEQ_OK;
}

}  // extern "C"
