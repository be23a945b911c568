// Device code of matrix products whose weights are chosen row by row (typed_products.hip has the launches).
//
// Rows x_i of type t become y_i = x_i W_t^T (+ b_t), and for a gradient g of y
//
//   dx_i = g_i W_t,   dW_t = sum_{i of type t} g_i^T x_i,   db_t = sum g_i.
//
// Rows are taken by type through an index (row_groups.h), so that a tile of them has one matrix; nothing is gathered or
// padded in memory. The number of rows of a type is known to the device alone: a launch has a slot for every BM rows
// and one more for every type, type t owns the slots from floor(begin_t / BM) + t on, which are as many as it can need
// (floor(b / m) - floor(a / m) + 1 is never less than ceil((b - a) / m)), and a block whose slot is past its type's rows ends.
// A row can have several parts (the components of an irrep), which share its type: they count as rows here.
//
// Products run on the 32x32 matrix instructions, sums in 32 bits. Tiles of both operands go from memory to LDS 128 bytes of
// the summation at a time, into one of two buffers while the products read the other; there is one barrier a step. Nothing is
// rounded to fewer bits but the results, and what lies between two thin products, which keeps 16 bits or more (row_products; a sum of
// few rows or of float operands keeps all). Long sums of floats are added up in parts, kSpan steps each.
//
// What bounds them and what they reach, bf16 if nothing else is said: large products the matrix units and the card's power, 8 192 rows
// of one 8192 x 8192 matrix 953 us, 1.15 PFLOP/s (1.13 to 1.26 for the library's product there, which has neither types nor
// rows in another order; gradient of x 912, of the weights 983), float32 4096 x 4096 2.06 ms, 134 TFLOP/s of 154. Of shorter sums the beginning and end of a tile
// take a share, some 12 us of a tile of 256 x 256 where all compute units write at a time: 32 768 rows, 16 matrices of
// 2048 x 5632 800 us, 0.95 PFLOP/s. (Blocks that stay for several tiles took 820.) Few rows: memory, 64 rows of 64 types,
// 2048 x 2048, 69 us, 4.9 TB/s of the matrices that are read.
#ifndef OEQ_TYPED_PRODUCTS_H
#define OEQ_TYPED_PRODUCTS_H

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

namespace typed_products {

// Rows and parts of x and the rows of w are strided, their elements contiguous; strides in elements.
struct Args {
    const void *x, *w, *bias, *up;
    const float *thin, *scale;  // thin: [rows, thin_row]; scale: of each type
    void* out;                  // [rows, parts, out_row]
    const int *order, *ptr;
    const int64_t* type_of_row;
    int64_t x_row, x_part, w_type, w_row, bias_type, up_type, up_col, up_rank, out_row;
    int rows, types, parts, inner, outer, rank, thin_row;
    int slots, tiles;  // of rows, of columns
    int shared;        // rows without a type have w too
};

// Sums of products over rows: out[t] = sum a_i^T b_i, [types, a columns, b columns].
struct SumArgs {
    const void *a, *b;
    void* out;
    float* partial;  // [shares, a columns, b columns]
    const int *order, *ptr;
    int64_t a_row, a_part, b_row, b_part;
    int rows, types, parts, a_columns, b_columns;
    int chunk;  // rows (with their parts) that a block sums up
    int tile;   // columns of a block
    int slots, a_tiles, b_tiles;
};

typedef float float4_t __attribute__((ext_vector_type(4)));
typedef float float8_t __attribute__((ext_vector_type(8)));
typedef float float16_t __attribute__((ext_vector_type(16)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf8_t __attribute__((ext_vector_type(8)));
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef unsigned uint4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(1))) const void* gptr_t;
typedef __attribute__((address_space(3))) void* lptr_t;
typedef __attribute__((address_space(3))) short4_t* ltr_t;

// A fragment: 16 bytes of a row, the operand of a product over twice as many elements (one half in either half of a wave).
template <typename T>
struct Types;
template <>
struct Types<float> {
    typedef float4_t frag;
    typedef float4_t quad;
};
template <>
struct Types<_Float16> {
    typedef half8_t frag;
    typedef half4_t quad;
};
template <>
struct Types<__bf16> {
    typedef bf8_t frag;
    typedef bf4_t quad;
};

__device__ __forceinline__ float16_t mma(float4_t a, float4_t b, float16_t c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ float16_t mma(float8_t a, float8_t b, float16_t c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ float16_t mma(half8_t a, half8_t b, float16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float16_t mma(bf8_t a, bf8_t b, float16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// ---------------------------------------------------------------------------
// slots
// ---------------------------------------------------------------------------

// Blocks go to the eight XCDs in turn, each with a cache of its own: an XCD takes 32 neighbouring tiles, one for each of its
// compute units, then the 32 that follow those of the other seven. (Longer runs leave some XCDs with the slots that have no rows: 8 192
// rows, 8192 x 8192, bf16: 1 028 us with an eighth of all tiles to each XCD, 953 so.)
__device__ __forceinline__ int tile_of_block(int block, int blocks) {
    constexpr int kRun = 32;
    if (block >= blocks / (8 * kRun) * (8 * kRun)) return block;
    const int xcd = block & 7, turn = block >> 3;
    return (turn / kRun * 8 + xcd) * kRun + turn % kRun;
}

struct Range {
    int type, lo, hi;  // places of the index times parts
};

// Where type t's rows begin (t = types: the rows without one).
__device__ __forceinline__ int begin_of(const int* ptr, int t, int rows, int parts) { return min(max(ptr[t], 0), rows) * parts; }

// The type that owns a slot of `each` rows, among `types` (and the rows without a type, if `rest`), and the slot's rows.
__device__ __forceinline__ Range rows_of_slot(const int* ptr, int slot, int each, int types, bool rest, int rows, int parts) {
    const int lane = threadIdx.x & 63;
    Range r;
    int begin;
    if (types < 64) {  // every type's beginning in a lane
        const int mine = begin_of(ptr, min(lane, types), rows, parts);
        const bool early = lane == 0 || (lane < types + rest && mine / each + lane <= slot);
        r.type = __builtin_amdgcn_readfirstlane(63 - __builtin_clzll(__ballot(early)));
        begin = __builtin_amdgcn_readlane(mine, r.type);
        r.hi = r.type < types ? __builtin_amdgcn_readlane(mine, r.type + 1) : rows * parts;
    } else {
        int t = 0, n = types + rest;
        while (n > 1) {  // 64 candidates at a time; the first of them always begins early enough
            const int step = (n + 63) >> 6;
            const int at = lane * step;
            const bool early = lane == 0 || (at < n && begin_of(ptr, t + at, rows, parts) / each + t + at <= slot);
            const int last = 63 - __builtin_clzll(__ballot(early));
            t += last * step;
            n = min(step, n - last * step);
        }
        r.type = __builtin_amdgcn_readfirstlane(t);
        begin = begin_of(ptr, r.type, rows, parts);
        r.hi = r.type < types ? begin_of(ptr, r.type + 1, rows, parts) : rows * parts;
    }
    const int64_t lo = begin + (int64_t)(slot - begin / each - r.type) * each;
    r.lo = lo < r.hi ? (int)lo : r.hi;
    return r;
}

// Place of the index -> row and part. (An index that was not made here is kept inside the rows.)
struct Place {
    int row, part;
    __device__ __forceinline__ Place(const int* order, int at, int parts, int rows) {
        const int i = parts == 1 ? at : at / parts;
        part = at - i * parts;
        row = order ? order[i] : i;
        if ((unsigned)row >= (unsigned)rows) row = 0;
    }
};

// ---------------------------------------------------------------------------
// tiles in LDS
// ---------------------------------------------------------------------------

__device__ const uint4_t kZeros = {0, 0, 0, 0};

// ROWS rows of CH chunks of 16 bytes; chunk c of row r lies at place c ^ swizzle(r) of the row. LDS has 64 banks, 256 bytes.
// A 16-byte read meets them with one chunk of 16 consecutive rows, a transposing read with four neighbouring chunks of four
// rows that begin at a multiple of four: either way the 16 have to lie in different places modulo 16. Four-byte
// reads of float columns have 32 columns of two rows that lie four apart: the rows' places have to differ in the half.
template <typename T, int CH, int ROWS, int WAVES>
struct Tile {
    static constexpr int kRowBytes = CH * 16, kBytes = ROWS * kRowBytes, kElements = 16 / (int)sizeof(T);
    static constexpr int kRowsPer = 64 / CH, kEach = kBytes / 1024 / WAVES;
    static_assert(CH >= 8 && CH <= 64 && kEach * 1024 * WAVES == kBytes, "the waves share a tile");

    // After this many of a lane's requests the same chunk comes again.
    static constexpr int kPeriod = CH > 8 && sizeof(T) == 4 ? 8 : 16, kApart = WAVES * kRowsPer;
    static constexpr int kColumns = kApart >= kPeriod ? 1 : kEach < kPeriod / kApart ? kEach : kPeriod / kApart;
    static __device__ __forceinline__ int swizzle(int r) {
        if constexpr (CH == 8) return (r >> 1 & 1) << 2 | (r >> 2 & 3);
        else if constexpr (sizeof(T) == 4) return (r >> 2 & 1) << 3;
        else return (r & 3) << 2 | (r >> 2 & 3);
    }
    // What a lane of a wave brings with its i-th request: 1 KB for the wave.
    static __device__ __forceinline__ int row(int i, int wave, int lane) { return (i * WAVES + wave) * kRowsPer + lane / CH; }
    static __device__ __forceinline__ int chunk(int i, int wave, int lane) { return (lane % CH) ^ swizzle(row(i, wave, lane)); }
    static __device__ __forceinline__ void request(char* lds, const char* from, int i, int wave) {
        __builtin_amdgcn_global_load_lds((gptr_t)from, (lptr_t)(lds + (i * WAVES + wave) * 1024), 16, 0, 0);
    }
    static __device__ __forceinline__ void put(char* lds, uint4_t x, int i, int wave, int lane) {
        *(uint4_t*)(lds + (i * WAVES + wave) * 1024 + lane * 16) = x;
    }

    // 16 bytes of row r: fragment f of it.
    static __device__ __forceinline__ typename Types<T>::frag along(const char* lds, int r, int f, int half) {
        return *(const typename Types<T>::frag*)(lds + r * kRowBytes + (((2 * f + half) ^ swizzle(r)) << 4));
    }
    // The rows 2 E f + E half .. + E of column `first` + lane % 32.
    static __device__ __forceinline__ typename Types<T>::frag down(const char* lds, int f, int first, int lane) {
        typename Types<T>::frag x;
        if constexpr (sizeof(T) == 2) {
            // a transposing read gives each of 16 lanes four rows of its column out of the 4 x 16 block whose rows the lanes
            // address by quarters
            const int l = lane & 15, c = (first >> 3) + 2 * ((lane >> 4) & 1) + ((l & 3) >> 1);
            union {
                short4_t q[2];
                typename Types<T>::frag f;
            } u;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const int r = 16 * f + 8 * (lane >> 5) + 4 * g + (l >> 2);
                u.q[g] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ltr_t)(lds + r * kRowBytes + ((c ^ swizzle(r)) << 4) + ((l & 1) << 3)));
            }
            x = u.f;
        } else {
            const int d = first + (lane & 31);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = 8 * f + 4 * (lane >> 5) + j;
                x[j] = *(const float*)(lds + r * kRowBytes + (((d >> 2) ^ swizzle(r)) << 4) + ((d & 3) << 2));
            }
        }
        return x;
    }
};

typedef uint4_t anywhere2_t __attribute__((aligned(2)));
typedef uint4_t anywhere4_t __attribute__((aligned(4)));

// 16 bytes from anywhere in memory, of which `left` elements are there; zeros for the others. (Pointers are told to be global
// ones: next to kZeros the compiler takes them for any, and such loads are waited for all at once.)
template <typename T>
__device__ __forceinline__ uint4_t fetch(const char* from, int left) {
    constexpr int E = 16 / (int)sizeof(T);
    typedef typename std::conditional<sizeof(T) == 2, anywhere2_t, anywhere4_t>::type anywhere_t;
    if (left >= E) return *(__attribute__((address_space(1))) const anywhere_t*)from;
    union {
        uint4_t v;
        T e[E];
    } u;
    u.v = uint4_t{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < E; ++j)
        if (j < left) u.e[j] = ((__attribute__((address_space(1))) const T*)from)[j];
    return u.v;
}

// Quarters of a step's products, between which the next step's operands are requested: early enough to be there in time.
// 8 192 rows, 8192 x 8192, bf16, us: 1 1 064, 2 1 028, 4 1 135.
constexpr int kEarly = 2;

// Steps whose products of floats are summed up by themselves (512 terms) before they join the total: one chain's error grows with its
// length. Root mean square errors relative to the results: 300 rows, sums of 3 392 terms 1.0e-6 in one chain, 4.0e-7 so (a library product
// 5.1e-7); 4096 x 4096 x 4096 1.1e-6 and 4.1e-7, in 1 147 us and 1 149.
constexpr int kSpan = 16;

// What this wave requested is in LDS; then the same for the others, and all are done with the other buffer.
__device__ __forceinline__ void arrived() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// ---------------------------------------------------------------------------
// products of rows
// ---------------------------------------------------------------------------

// A float u beside operands of 16 bits is hi + lo. Its products with weights that are not finite are those of hi alone (the weights of lo
// are 0 there: lo inf would be NaN, or an infinity of the other sign), so hi is not 0 where u is not: then the smallest there is.
template <typename T>
__device__ __forceinline__ T upper_part(float u) {
    union {
        T t;
        unsigned short bits;
    } hi;
    hi.t = (T)u;
    if (!(hi.bits & 0x7fff) && u != 0.0f) hi.bits |= 1;
    if constexpr (!std::is_same<T, _Float16>::value)  // (where u is past what 8 bits hold: the largest there is)
        if ((hi.bits & 0x7fff) == 0x7f80 && fabsf(u) < INFINITY) --hi.bits;
    return hi.t;
}
template <typename T>
__device__ __forceinline__ uint4_t finite_or_zero(uint4_t x) {
    constexpr unsigned short kExponent = std::is_same<T, _Float16>::value ? 0x7c00 : 0x7f80;
    union {
        uint4_t v;
        unsigned short e[8];
    } y;
    y.v = x;
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if ((y.e[j] & kExponent) == kExponent) y.e[j] = 0;
    return y.v;
}

// A tile of BM rows and BN columns. ACROSS: the weights' rows run along the columns (w[k, n]), else along the summation
// (w[n, k]). DIRECT: everything is aligned to 16 bytes and goes straight to LDS; else through registers, by elements where a
// row ends. The result is transposed in registers: lane l has row l % 32, register r column 8 (r / 4) + 4 (l / 32) + r % 4.
template <typename T, typename O, bool ACROSS, bool DIRECT, bool THIN, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void row_products(Args g) {
    constexpr int WAVES = WM * WN, BK = 128 / (int)sizeof(T), E = 16 / (int)sizeof(T);
    constexpr int TM = BM / WM / 32, TN = BN / WN / 32;
    typedef Tile<T, 8, BM, WAVES> X;
    typedef Tile<T, ACROSS ? BN * (int)sizeof(T) / 16 : 8, ACROSS ? BK : BN, WAVES> W;
    __shared__ __align__(1024) char x0[X::kBytes], x1[X::kBytes], w0[W::kBytes], w1[W::kBytes];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
    // neighbours in a run: eight slots, column by column
    const int id = tile_of_block(blockIdx.x, g.slots * g.tiles);
    const int group = id / (8 * g.tiles), in_group = id - group * 8 * g.tiles, size = min(8, g.slots - group * 8);
    const int slot = group * 8 + in_group % size, n0 = in_group / size * BN;
    const Range rows = rows_of_slot(g.ptr, slot, BM, g.types, true, g.rows, g.parts);
    if (rows.lo >= rows.hi) return;
    const int m0 = rows.lo;
    const bool typed = rows.type < g.types;
    const int steps = typed || g.shared ? (g.inner + BK - 1) / BK : 0;

    // where this lane's chunks of the tiles come from
    const char* xs[X::kEach];
    const char* ws[W::kEach];
    int w_left[W::kEach];  // elements of w from there on to the end of its row (ACROSS)
    if (steps) {
        const T* w = (const T*)g.w + (typed ? rows.type : 0) * g.w_type;
#pragma unroll
        for (int i = 0; i < X::kEach; ++i) {
            const int at = m0 + X::row(i, wave, lane);
            const Place p(g.order, at < rows.hi ? at : m0, g.parts, g.rows);
            xs[i] = (const char*)((const T*)g.x + p.row * g.x_row + p.part * g.x_part) + X::chunk(i, wave, lane) * 16;
        }
#pragma unroll
        for (int i = 0; i < W::kEach; ++i) {
            const int r = W::row(i, wave, lane), c = W::chunk(i, wave, lane) * E;
            if constexpr (ACROSS) {
                const bool in = n0 + c < g.outer;
                w_left[i] = in ? g.outer - n0 - c : 0;
                ws[i] = (const char*)(w + r * g.w_row + (in ? n0 + c : 0));
            } else {
                ws[i] = (const char*)(w + (int64_t)min(n0 + r, g.outer - 1) * g.w_row + c);
            }
        }
    }
    const int64_t w_step = ACROSS ? BK * g.w_row * (int64_t)sizeof(T) : 128;
    uint4_t x_reg[DIRECT ? 1 : X::kEach], w_reg[DIRECT ? 1 : W::kEach];

    // Requests the tiles of step k, a quarter at a time between the products. (Past the last step zeros come, which nobody reads.)
    auto request_x = [&](char* xt, int k, int i) __attribute__((always_inline)) {
        const int left = g.inner - k * BK - X::chunk(i, wave, lane) * E;
        if constexpr (DIRECT)
            X::request(xt, left <= 0 ? (const char*)&kZeros : xs[i], i, wave);
        else
            x_reg[i] = fetch<T>(xs[i], left);
        xs[i] += 128;
    };
    auto request_w = [&](char* wt, int k, int i) __attribute__((always_inline)) {
        if constexpr (ACROSS) {
            const bool in = k * BK + W::row(i, wave, lane) < g.inner;
            if constexpr (DIRECT)
                W::request(wt, !in ? (const char*)&kZeros : ws[i], i, wave);
            else
                w_reg[i] = fetch<T>(ws[i], in ? w_left[i] : 0);
        } else {
            const int left = g.inner - k * BK - W::chunk(i, wave, lane) * E;
            if constexpr (DIRECT)
                W::request(wt, left <= 0 ? (const char*)&kZeros : ws[i], i, wave);
            else
                w_reg[i] = fetch<T>(ws[i], left);
        }
        ws[i] += w_step;
    };
    auto request = [&](char* xt, char* wt, int k, int quarter) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < X::kEach; ++i)
            if (i % 4 == quarter) request_x(xt, k, i);
#pragma unroll
        for (int i = 0; i < W::kEach; ++i)
            if (i % 4 == quarter) request_w(wt, k, i);
    };
    auto request_all = [&](char* xt, char* wt, int k) __attribute__((always_inline)) {
#pragma unroll
        for (int quarter = 0; quarter < 4; ++quarter) request(xt, wt, k, quarter);
    };
    auto put = [&](char* xt, char* wt) __attribute__((always_inline)) {
        if constexpr (!DIRECT) {
#pragma unroll
            for (int i = 0; i < X::kEach; ++i) X::put(xt, x_reg[i], i, wave, lane);
#pragma unroll
            for (int i = 0; i < W::kEach; ++i) W::put(wt, w_reg[i], i, wave, lane);
        }
    };

    const int wm = wave % WM * (BM / WM), wn = wave / WM * (BN / WN);
    float16_t acc[TM][TN];
#pragma unroll
    for (int m = 0; m < TM; ++m)
#pragma unroll
        for (int n = 0; n < TN; ++n) acc[m][n] = 0.0f;

    // The fragments of a quarter are read while the products of the quarter before are computed: those of w into other registers,
    // those of x each when the last product with it has been issued. (The barriers keep the compiler from moving reads down to
    // where they are waited for.)
    auto products = [&](const char* xt, const char* wt, auto between) __attribute__((always_inline)) {
        typename Types<T>::frag a[2][TN], b[TM];
        auto read_w = [&](int f) __attribute__((always_inline)) {
#pragma unroll
            for (int n = 0; n < TN; ++n)
                a[f & 1][n] = ACROSS ? W::down(wt, f, wn + 32 * n, lane) : W::along(wt, wn + 32 * n + (lane & 31), f, half);
        };
        auto read_x = [&](int f, int m) __attribute__((always_inline)) { b[m] = X::along(xt, wm + 32 * m + (lane & 31), f, half); };
        read_w(0);
#pragma unroll
        for (int m = 0; m < TM; ++m) read_x(0, m);
#pragma unroll
        for (int f = 0; f < 4; ++f) {
            if (f < 3) read_w(f + 1);
            between(f);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int m = 0; m < TM; ++m) {
#pragma unroll
                for (int n = 0; n < TN; ++n) acc[m][n] = mma(a[f & 1][n], b[m], acc[m][n]);
                if (f < 3) read_x(f + 1, m);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    auto step = [&](char* xt, char* wt, char* xn, char* wn_, int k) __attribute__((always_inline)) {
        arrived();
        products(xt, wt, [&](int f) __attribute__((always_inline)) {
            if (f < kEarly)
#pragma unroll
                for (int quarter = f * 4 / kEarly; quarter < (f + 1) * 4 / kEarly; ++quarter) request(xn, wn_, k + 1, quarter);
        });
        put(xn, wn_);
    };
    if (steps) request_all(x0, w0, 0);
    if constexpr (THIN) {
        // The thin product first, from the other buffer. Its rows are float; as operands beside 16 bits they have two parts, u =
        // hi + lo, next to each other along the summation: 16 bits of u or more, when what it adds to is rounded to 8 or 11.
        if (typed && g.rank) {
            constexpr int PARTS = sizeof(T) == 2 ? 2 : 1;
            const int width = g.thin_row;
            float* lift = (float*)w1;  // (done with before w1 is filled)
            float down[TM];
            float up_by[X::kEach];
            if constexpr (std::is_same<T, _Float16>::value) {
                // A power of two for each row, which brings its largest element near the end of float16's range: parts of 11 bits each
                // whatever the size of u, and what is small beside the largest keeps 16 bits down to 2^-24 of it.
                for (int r = tid; r < BM; r += 64 * WAVES) {
                    const int at = min(m0 + r, rows.hi - 1);
                    const float* u = g.thin + (int64_t)Place(g.order, at, 1, g.rows).row * width;
                    float most = 0;
                    for (int k = 0; k < width; k += 4) {
                        const float4_t v = *(const float4_t*)(u + k);
#pragma unroll
                        for (int j = 0; j < 4; ++j) most = fmaxf(most, fabsf(v[j]) < INFINITY ? fabsf(v[j]) : 0.0f);
                    }
                    // the largest that is finite, most, times 2^e is between 2^14 and 2^15; infinities and NaN stay what they are
                    const int e = most > 0 ? 15 - __builtin_amdgcn_frexp_expf(most) : 0;
                    lift[r] = __builtin_amdgcn_ldexpf(1.0f, min(e, 126));
                }
                __syncthreads();
#pragma unroll
                for (int m = 0; m < TM; ++m) down[m] = 1.0f / lift[wm + 32 * m + (lane & 31)];
#pragma unroll
                for (int i = 0; i < X::kEach; ++i) up_by[i] = lift[X::row(i, wave, lane)];
                __syncthreads();
            }
            const T* up = (const T*)g.up + rows.type * g.up_type;
            for (int k0 = 0; k0 < PARTS * width; k0 += BK) {
#pragma unroll
                for (int i = 0; i < X::kEach; ++i) {
                    const int at = min(m0 + X::row(i, wave, lane), rows.hi - 1), kk = k0 + X::chunk(i, wave, lane) * E;
                    const bool low = kk >= width;
                    union {
                        uint4_t v;
                        T e[E];
                    } y;
                    y.v = uint4_t{0, 0, 0, 0};
                    if (kk < PARTS * width) {
                        const float* u = g.thin + (int64_t)Place(g.order, at, 1, g.rows).row * width + (low ? kk - width : kk);
#pragma unroll
                        for (int j = 0; j < E; ++j) {
                            const float v = std::is_same<T, _Float16>::value ? u[j] * up_by[i] : u[j];
                            if constexpr (PARTS == 2) {
                                const T hi = upper_part<T>(v);
                                y.e[j] = !low ? hi : (T)(fabsf((float)hi) < INFINITY ? v - (float)hi : 0.0f);
                            } else {
                                y.e[j] = v;
                            }
                        }
                    }
                    X::put(x1, y.v, i, wave, lane);
                }
#pragma unroll
                for (int i = 0; i < W::kEach; ++i) {
                    const int r = W::row(i, wave, lane), c = W::chunk(i, wave, lane) * E;
                    union {
                        uint4_t v;
                        T e[E];
                    } y;
                    y.v = uint4_t{0, 0, 0, 0};
                    if constexpr (ACROSS) {
                        const int k = k0 + r >= width ? k0 + r - width : k0 + r;
                        const int left = k0 + r < PARTS * width && k < g.rank ? g.outer - n0 - c : 0;
                        const T* from = up + k * g.up_rank + (n0 + c) * g.up_col;
                        if (g.up_col == 1)
                            y.v = fetch<T>((const char*)from, left);
                        else
#pragma unroll
                            for (int j = 0; j < E; ++j)
                                if (j < left) y.e[j] = from[j * g.up_col];
                        if (PARTS == 2 && k0 + r >= width) y.v = finite_or_zero<T>(y.v);
                    } else {
                        const int kk = k0 + c, k = kk >= width ? kk - width : kk;
                        const int left = kk < PARTS * width ? g.rank - k : 0;
                        const T* from = up + min(n0 + r, g.outer - 1) * g.up_col + k * g.up_rank;
                        if (g.up_rank == 1)
                            y.v = fetch<T>((const char*)from, left);
                        else
#pragma unroll
                            for (int j = 0; j < E; ++j)
                                if (j < left) y.e[j] = from[j * g.up_rank];
                        if (PARTS == 2 && kk >= width) y.v = finite_or_zero<T>(y.v);
                    }
                    W::put(w1, y.v, i, wave, lane);
                }
                __syncthreads();
                products(x1, w1, [](int) {});
                __syncthreads();
            }
            if constexpr (std::is_same<T, _Float16>::value)
#pragma unroll
                for (int m = 0; m < TM; ++m)
#pragma unroll
                    for (int n = 0; n < TN; ++n) acc[m][n] *= down[m];
        }
    }
    if (steps) put(x0, w0);
    if constexpr (sizeof(T) == 4) {
        float16_t total[TM][TN];
#pragma unroll
        for (int m = 0; m < TM; ++m)
#pragma unroll
            for (int n = 0; n < TN; ++n) total[m][n] = 0.0f;
        for (int k0 = 0; k0 < steps; k0 += kSpan) {
            const int end = min(k0 + kSpan, steps);
            for (int k = k0; k < end; k += 2) {
                step(x0, w0, x1, w1, k);
                if (k + 1 < end) step(x1, w1, x0, w0, k + 1);
            }
#pragma unroll
            for (int m = 0; m < TM; ++m)
#pragma unroll
                for (int n = 0; n < TN; ++n) total[m][n] += acc[m][n], acc[m][n] = 0.0f;
        }
#pragma unroll
        for (int m = 0; m < TM; ++m)
#pragma unroll
            for (int n = 0; n < TN; ++n) acc[m][n] += total[m][n];
    } else {
        for (int k = 0; k < steps; k += 2) {
            step(x0, w0, x1, w1, k);
            if (k + 1 < steps) step(x1, w1, x0, w0, k + 1);
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the zeros)

    // Results pass through LDS, a wave's 32 rows at a time, so that rows are written in pieces of up to 128 bytes. (From the
    // registers, four columns of 32 rows at a time, a tile of 256 x 256 took 4 us to write.)
    constexpr int SLAB = 128 / (int)sizeof(O) < 32 * TN ? 128 / (int)sizeof(O) : 32 * TN, CHUNKS = SLAB * (int)sizeof(O) / 16;
    constexpr int EO = 16 / (int)sizeof(O), ROWS = 64 / CHUNKS;
    constexpr bool FITS = WAVES * 32 * SLAB * (int)sizeof(O) <= X::kBytes;
    __shared__ __align__(16) char results[FITS ? 16 : WAVES * 32 * SLAB * (int)sizeof(O)];
    char* slab = (FITS ? x0 : results) + wave * 32 * SLAB * (int)sizeof(O);
    const auto place = [&](int r, int c) { return slab + r * SLAB * (int)sizeof(O) + ((c ^ (r & (CHUNKS - 1))) << 4); };
    float by = 1.0f;
    if (g.scale) by = typed ? g.scale[rows.type] : 0.0f;
    O* out = (O*)g.out;
    const bool whole = g.out_row % EO == 0 && ((uintptr_t)out & 15) == 0;
    const T* bias = g.bias && typed ? (const T*)g.bias + rows.type * g.bias_type : nullptr;
    __syncthreads();  // (all are done with x0)
#pragma unroll
    for (int m = 0; m < TM; ++m) {
        const int first = m0 + wm + 32 * m;
        int64_t to = 0;
        if (first < rows.hi) {
            const Place p(g.order, min(first + (lane & 31), rows.hi - 1), g.parts, g.rows);
            to = ((int64_t)p.row * g.parts + p.part) * g.out_row;
        }
#pragma unroll
        for (int s = 0; s < 32 * TN / SLAB; ++s) {
            const int col0 = n0 + wn + s * SLAB;
#pragma unroll
            for (int n = 0; n < SLAB / 32; ++n)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int c = 32 * n + 8 * q + 4 * half;  // of the slab
                    typename Types<O>::quad y;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float v = acc[m][s * (SLAB / 32) + n][4 * q + j] * by;
                        const bool in = col0 + c + j < g.outer;
                        if (bias && in) v += (float)bias[col0 + c + j];
                        y[j] = (O)(in ? v : 0.0f);
                    }
                    *(typename Types<O>::quad*)(place(lane & 31, c / EO) + c % EO * (int)sizeof(O)) = y;
                }
#pragma unroll
            for (int i = 0; i < 32 / ROWS; ++i) {
                const int r = i * ROWS + lane / CHUNKS, c = lane % CHUNKS, col = col0 + c * EO;
                const int64_t at = __shfl(to, r) + col;
                const uint4_t y = *(const uint4_t*)place(r, c);
                if (first + r >= rows.hi || col >= g.out_row) continue;
                if (whole) {
                    *(uint4_t*)(out + at) = y;
                } else {
                    union {
                        uint4_t v;
                        O e[EO];
                    } u;
                    u.v = y;
#pragma unroll
                    for (int j = 0; j < EO; ++j)
                        if (col + j < g.out_row) out[at + j] = u.e[j];
                }
            }
        }
    }
}

// ---------------------------------------------------------------------------
// products of few rows
// ---------------------------------------------------------------------------

// Up to 64 rows, as in serving, where each matrix that has a row is read once and nothing else takes time: bound by memory.
// A block has 16 columns and the rows of one type (of all types, where w is shared); its waves share the summation in turns of
// 128 bytes of a row, straight from memory to registers, and are added up through LDS. No index: a wave holds the types of 64
// rows in its lanes, and the block of the first row of a type takes all of them.
template <typename T>
struct Few;  // products on the 16x16 matrix instructions: lane l has row l % 16, register r column 4 (l / 16) + r
template <>
struct Few<float> {
    static __device__ __forceinline__ float4_t mma(float4_t a, float4_t b, float4_t c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
        return c;
    }
};
template <>
struct Few<_Float16> {
    static __device__ __forceinline__ float4_t mma(half8_t a, half8_t b, float4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Few<__bf16> {
    static __device__ __forceinline__ float4_t mma(bf8_t a, bf8_t b, float4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};

constexpr int kFewRows = 64, kFewWaves = 4;

// acc[m][n] += products of 16 x rows and 16 w rows for this wave's turns of the summation: 128 bytes of each row, from memory to a
// part of LDS that is the wave's own (no barrier), two turns ahead of the products. rows(r) is where row r begins: first the x rows,
// 16 X of them, then those of w. (Straight to registers a request has 16 bytes of 16 rows, lanes next to each other in different rows:
// 27 accesses to the cache where 8 rows of 128 bytes take 8; 48 requests beside 4096 x 4096, bf16: 21 us, so 14.)
template <typename T, bool DIRECT, int X, int W, typename Rows>
__device__ __forceinline__ void sum_turns(float4_t (&acc)[X][W], char* stage0, char* stage1, char* stage2, const Rows& rows, int inner,
                                          int wave, int lane) {
    constexpr int E = 16 / (int)sizeof(T), BK = 128 / (int)sizeof(T), REQUESTS = 2 * (X + W);
    typedef Tile<T, 8, 16 * (X + W), 1> L;
    static_assert(L::kEach == REQUESTS, "1 KB a request");
    const int steps = (inner + BK - 1) / BK;
    if (wave >= steps) return;
    const char* from[REQUESTS];
#pragma unroll
    for (int i = 0; i < REQUESTS; ++i) from[i] = (const char*)rows(L::row(i, 0, lane)) + L::chunk(i, 0, lane) * 16;
    const auto request = [&](char* to, int step) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < REQUESTS; ++i) {
            const int left = inner - step * BK - L::chunk(i, 0, lane) * E;
            const char* at = from[i] + (int64_t)step * 128;
            if constexpr (DIRECT)
                L::request(to, left <= 0 ? (const char*)&kZeros : at, i, 0);
            else
                L::put(to, fetch<T>(at, left), i, 0, lane);
        }
    };
    // (floats: three turns by themselves, then they join the total, as in row_products)
    constexpr bool SPLIT = sizeof(T) == 4;
    float4_t part[X][W];
    const auto products = [&](const char* from_) __attribute__((always_inline)) {
        auto& into = [&]() -> auto& {
            if constexpr (SPLIT) return part;
            else return acc;
        }();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            typename Types<T>::frag a[W], b[X];
            const auto read = [&](int r) __attribute__((always_inline)) {
                return *(const typename Types<T>::frag*)(from_ + r * 128 + (((4 * h + (lane >> 4)) ^ L::swizzle(r)) << 4));
            };
#pragma unroll
            for (int m = 0; m < X; ++m) b[m] = read(16 * m + (lane & 15));
#pragma unroll
            for (int n = 0; n < W; ++n) a[n] = read(16 * (X + n) + (lane & 15));
#pragma unroll
            for (int m = 0; m < X; ++m)
#pragma unroll
                for (int n = 0; n < W; ++n) into[m][n] = Few<T>::mma(a[n], b[m], into[m][n]);
        }
    };
    const auto step = [&](const char* now, char* next, int k) __attribute__((always_inline)) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // what was read from `next` has come
        request(next, k + 2 * kFewWaves);
        if constexpr (DIRECT) {  // vmcnt(2 REQUESTS), as a builtin that the compiler counts with
            __builtin_amdgcn_s_waitcnt((2 * REQUESTS & 15) | 0xf70 | (2 * REQUESTS >> 4) << 14);
            asm volatile("" ::: "memory");
        }
        products(now);
    };
    // (No branch around a request: the compiler would not know how many are on their way, and wait for all. Past the last step
    // zeros come, which nobody needs.)
    request(stage0, wave);
    request(stage1, wave + kFewWaves);
    for (int k = wave; k < steps; k += 3 * kFewWaves) {
        if constexpr (SPLIT)
#pragma unroll
            for (int m = 0; m < X; ++m)
#pragma unroll
                for (int n = 0; n < W; ++n) part[m][n] = 0.0f;
        step(stage0, stage2, k);
        step(stage1, stage0, k + kFewWaves);
        step(stage2, stage1, k + 2 * kFewWaves);
        if constexpr (SPLIT)
#pragma unroll
            for (int m = 0; m < X; ++m)
#pragma unroll
                for (int n = 0; n < W; ++n) acc[m][n] += part[m][n];
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// MT: tiles of 16 rows at a time. blockIdx.x: columns; blockIdx.y: rows, of which the first of a type stands for all; with shared
// weights: every 16 MT rows.
template <typename T, typename O, bool DIRECT, int MT>
__global__ __launch_bounds__(64 * kFewWaves) void few_products(Args g) {
    constexpr int E = 16 / (int)sizeof(T), STAGE = 16 * (MT + 1) * 128;
    __shared__ int members[kFewRows];
    __shared__ __align__(1024) char stage0[kFewWaves * STAGE], stage1[kFewWaves * STAGE], stage2[kFewWaves * STAGE];
    typedef float Sums[kFewWaves][16 * MT][17];
    static_assert(sizeof(Sums) <= sizeof(stage0), "the sums lie where the operands did");
    Sums& sums = *(Sums*)stage0;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n0 = blockIdx.x * 16, total = g.rows * g.parts;
    int type = g.types, count;
    if (g.shared) {
        const int first = blockIdx.y * 16 * MT;
        count = min(16 * MT, total - first);
        if (tid < count) members[tid] = first + tid;
    } else {
        const auto type_of = [&](int at) {
            const int64_t t = g.type_of_row[g.parts == 1 ? at : at / g.parts];
            return t >= 0 && t < g.types ? (int)t : g.types;
        };
        const int mine = lane < total ? type_of(lane) : -1;
        type = __builtin_amdgcn_readlane(mine, blockIdx.y);
        const uint64_t same = __ballot(mine == type);
        if (__builtin_ctzll(same) != (int)blockIdx.y) return;
        count = __popcll(same);
        if (wave == 0 && mine == type) members[__popcll(same & ((1ull << lane) - 1))] = lane;
    }
    __syncthreads();
    const bool typed = type < g.types;
    const T* w = (const T*)g.w + (typed ? type : 0) * g.w_type;
    const float by = g.scale ? (typed ? g.scale[type] : 0.0f) : 1.0f;
    for (int first = 0; first < count; first += 16 * MT) {
        const int here = min(16 * MT, count - first);
        float4_t acc[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[m] = 0.0f;
        const auto sum_up = [&](auto tiles) __attribute__((always_inline)) {
            constexpr int TILES = decltype(tiles)::value;
            const auto rows = [&](int r) {
                if (r >= 16 * TILES) return w + min(n0 + r - 16 * TILES, g.outer - 1) * g.w_row;
                const int at = members[first + min(r, here - 1)], row = g.parts == 1 ? at : at / g.parts;
                return (const T*)g.x + row * g.x_row + (at - row * g.parts) * g.x_part;
            };
            float4_t part[TILES][1];
#pragma unroll
            for (int m = 0; m < TILES; ++m) part[m][0] = 0.0f;
            sum_turns<T, DIRECT, TILES, 1>(part, stage0 + wave * STAGE, stage1 + wave * STAGE, stage2 + wave * STAGE, rows, g.inner, wave, lane);
#pragma unroll
            for (int m = 0; m < TILES; ++m) acc[m] = part[m][0];
        };
        if (typed || g.shared) {
            const int tiles = (here + 15) / 16;
            if (tiles == 1) sum_up(std::integral_constant<int, 1>());
            if constexpr (MT >= 2)
                if (tiles == 2) sum_up(std::integral_constant<int, 2>());
            if constexpr (MT >= 3)
                if (tiles == 3) sum_up(std::integral_constant<int, 3>());
            if constexpr (MT >= 4)
                if (tiles == 4) sum_up(std::integral_constant<int, 4>());
        }
        __syncthreads();
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r) sums[wave][16 * m + (lane & 15)][4 * (lane >> 4) + r] = acc[m][r];
        __syncthreads();
        for (int i = tid; i < 16 * here; i += 64 * kFewWaves) {
            const int r = i / 16, col = n0 + i % 16;
            if (col >= g.out_row) continue;
            float sum = 0;
#pragma unroll
            for (int v = 0; v < kFewWaves; ++v) sum += sums[v][r][i % 16];
            sum *= by;
            const int at = members[first + r];
            if (col >= g.outer) sum = 0;
            else if (g.bias && typed) sum += (float)((const T*)g.bias)[type * g.bias_type + col];
            if (col < g.outer && g.thin) {
                const int64_t t = g.type_of_row[at];
                if (t >= 0 && t < g.types) {
                    const float* u = g.thin + (int64_t)at * g.thin_row;
                    const T* v = (const T*)g.up + t * g.up_type + col * g.up_col;
                    if (g.up_rank == 1) {
#pragma unroll 2
                        for (int k = 0; k < g.rank; k += E) {
                            union {
                                uint4_t v;
                                T e[E];
                            } y;
                            y.v = fetch<T>((const char*)(v + k), g.rank - k);
#pragma unroll
                            for (int j = 0; j < E; j += 4) {  // (thin rows are filled up with zeros)
                                const float4_t z = *(const float4_t*)(u + k + j);
#pragma unroll
                                for (int i = 0; i < 4; ++i) sum += z[i] * (float)y.e[j + i];
                            }
                        }
                    } else {
                        for (int k = 0; k < g.rank; ++k) sum += u[k] * (float)v[k * g.up_rank];
                    }
                }
            }
            ((O*)g.out)[(int64_t)at * g.out_row + col] = (O)sum;
        }
        __syncthreads();  // (the sums lie where the next rows' operands go)
    }
}

// ---------------------------------------------------------------------------
// thin products
// ---------------------------------------------------------------------------

// Many rows, few columns, a long summation: bound by reading the rows. A block has 32 rows of a type and 16 NT columns; its
// waves share the summation as those of few_products do.
constexpr int kThinRows = 32;

template <typename T, bool DIRECT, int NT>
__global__ __launch_bounds__(64 * kFewWaves) void thin_products(Args g) {
    constexpr int MT = kThinRows / 16, STAGE = 16 * (MT + NT) * 128;
    __shared__ __align__(1024) char stage0[kFewWaves * STAGE], stage1[kFewWaves * STAGE], stage2[kFewWaves * STAGE];
    typedef float Sums[kFewWaves][kThinRows][16 * NT + 1];
    static_assert(sizeof(Sums) <= sizeof(stage0), "the sums lie where the operands did");
    Sums& sums = *(Sums*)stage0;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Range range = rows_of_slot(g.ptr, blockIdx.x, kThinRows, g.types, true, g.rows, 1);
    if (range.lo >= range.hi) return;
    const int n0 = blockIdx.y * 16 * NT, count = min(kThinRows, range.hi - range.lo);
    const bool typed = range.type < g.types;
    float4_t acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[m][n] = 0.0f;
    if (typed) {
        const T* w = (const T*)g.w + range.type * g.w_type;
        const auto rows = [&](int r) {
            if (r >= kThinRows) return w + min(n0 + r - kThinRows, g.outer - 1) * g.w_row;
            return (const T*)g.x + Place(g.order, range.lo + min(r, count - 1), 1, g.rows).row * g.x_row;
        };
        sum_turns<T, DIRECT, MT, NT>(acc, stage0 + wave * STAGE, stage1 + wave * STAGE, stage2 + wave * STAGE, rows, g.inner, wave, lane);
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) sums[wave][16 * m + (lane & 15)][16 * n + 4 * (lane >> 4) + r] = acc[m][n][r];
    __syncthreads();
    const float by = typed ? (g.scale ? g.scale[range.type] : 1.0f) : 0.0f;
    for (int i = tid; i < 16 * NT * count; i += 64 * kFewWaves) {
        const int r = i / (16 * NT), c = i % (16 * NT);
        if (n0 + c >= g.out_row) continue;
        float sum = 0;
#pragma unroll
        for (int v = 0; v < kFewWaves; ++v) sum += sums[v][r][c];
        const int row = Place(g.order, range.lo + r, 1, g.rows).row;
        ((float*)g.out)[(int64_t)row * g.out_row + n0 + c] = n0 + c < g.outer ? sum * by : 0.0f;
    }
}

// ---------------------------------------------------------------------------
// sums of products over rows
// ---------------------------------------------------------------------------

// Operands of which one is float and the other is not are multiplied as floats.
template <typename T, bool WIDE>
__device__ __forceinline__ auto widened(typename Types<T>::frag x) {
    if constexpr (sizeof(T) == 2 && WIDE)
        return __builtin_convertvector(x, float8_t);
    else
        return x;
}

// Where the share of a slot lies, of a type that has more than one: such a type has more than `chunk` rows, so of the shares that begin in
// a stretch of that many rows one at most is its type's first, and one at most is not.
__device__ __forceinline__ int64_t share_of(int lo, int chunk, bool first) { return 2 * (int64_t)(lo / chunk) + first; }

// A tile of BM columns of a and BN columns of b, summed over the rows of a slot. BK rows at a time; rows past the end are zeros.
// PARTS: rows have more than one. (A kernel of its own: branches inside the loop send the sums through other registers and back.)
template <typename A, typename B, typename O, bool DIRECT, bool PARTS, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void sum_products(SumArgs g) {
    constexpr int WAVES = WM * WN, BK = sizeof(A) + sizeof(B) == 4 ? 64 : 32;
    constexpr bool MIXED = sizeof(A) != sizeof(B);
    constexpr int EA = 16 / (int)sizeof(A), EB = 16 / (int)sizeof(B);
    constexpr int TM = BM / WM / 32, TN = BN / WN / 32;
    typedef Tile<A, BM * (int)sizeof(A) / 16, BK, WAVES> TA;
    typedef Tile<B, BN * (int)sizeof(B) / 16, BK, WAVES> TB;
    __shared__ __align__(1024) char a0[TA::kBytes], a1[TA::kBytes], b0[TB::kBytes], b1[TB::kBytes];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // slot by slot; in a slot neighbours are eight tiles of a, column by column of b
    const int id = tile_of_block(blockIdx.x, g.slots * g.a_tiles * g.b_tiles);
    const int slot = id / (g.a_tiles * g.b_tiles), tile = id - slot * g.a_tiles * g.b_tiles;
    const int group = tile / (8 * g.b_tiles), in_group = tile - group * 8 * g.b_tiles, high = min(8, g.a_tiles - group * 8);
    const int m0 = (group * 8 + in_group % high) * BM, n0 = in_group / high * BN;
    const Range rows = rows_of_slot(g.ptr, slot, g.chunk, g.types, false, g.rows, g.parts);
    const int begin = begin_of(g.ptr, rows.type, g.rows, g.parts);
    const bool whole = rows.hi - begin <= g.chunk;  // the type has no other slot
    if (rows.lo >= rows.hi && !(whole && rows.type + begin / g.chunk == slot)) return;
    const int end = min(rows.hi, rows.hi - rows.lo > g.chunk ? rows.lo + g.chunk : rows.hi);
    const int steps = (end - rows.lo + BK - 1) / BK;

    // Requests of an operand: the rows of a step are looked up one step ahead, their numbers have come when the step before
    // has its operands. Lanes keep their columns.
    uint4_t a_reg[DIRECT ? 1 : TA::kEach], b_reg[DIRECT ? 1 : TB::kEach];
    constexpr bool SAME = TA::kRowsPer == TB::kRowsPer && TA::kEach == TB::kEach;
    int a_row[TA::kEach], b_row[SAME ? 1 : TB::kEach];
    constexpr int CA = TA::kColumns, CB = TB::kColumns;
    int a_left[CA], b_left[CB];  // elements from a lane's columns on
    const char *a_from[CA], *b_from[CB];
#pragma unroll
    for (int i = 0; i < CA; ++i) {
        const int column = m0 + TA::chunk(i, wave, lane) * EA;
        a_left[i] = max(g.a_columns - column, 0);
        a_from[i] = (const char*)((const A*)g.a + (a_left[i] ? column : 0));
    }
#pragma unroll
    for (int i = 0; i < CB; ++i) {
        const int column = n0 + TB::chunk(i, wave, lane) * EB;
        b_left[i] = max(g.b_columns - column, 0);
        b_from[i] = (const char*)((const B*)g.b + (b_left[i] ? column : 0));
    }
    const unsigned a_stride = (unsigned)g.a_row * (unsigned)sizeof(A), b_stride = (unsigned)g.b_row * (unsigned)sizeof(B);
    const auto look_up = [&](int k) __attribute__((always_inline)) {
        const auto row_at = [&](int at) { return g.order[PARTS ? min(at, end - 1) / g.parts : min(at, end - 1)]; };
#pragma unroll
        for (int i = 0; i < TA::kEach; ++i) a_row[i] = row_at(rows.lo + k * BK + TA::row(i, wave, lane));
        if constexpr (!SAME)
#pragma unroll
            for (int i = 0; i < TB::kEach; ++i) b_row[i] = row_at(rows.lo + k * BK + TB::row(i, wave, lane));
    };
    const auto place = [&](const char* from, int row, unsigned stride, int j, int64_t part) __attribute__((always_inline)) {
        row = (unsigned)row < (unsigned)g.rows ? row : 0;  // (an index that was not made here)
        const char* p = from + (uint64_t)(unsigned)row * stride;
        return PARTS ? p + min(j, end - 1) % g.parts * part : p;
    };
    auto request = [&](char* at, char* bt, int k, int quarter) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < TA::kEach; ++i) {
            if (i % 4 != quarter) continue;
            const int j = rows.lo + k * BK + TA::row(i, wave, lane);
            const char* from = place(a_from[i % CA], a_row[i], a_stride, j, g.a_part * (int64_t)sizeof(A));
            if constexpr (DIRECT)
                TA::request(at, j < end ? from : (const char*)&kZeros, i, wave);
            else
                a_reg[i] = fetch<A>(from, j < end ? a_left[i % CA] : 0);
        }
#pragma unroll
        for (int i = 0; i < TB::kEach; ++i) {
            if (i % 4 != quarter) continue;
            const int j = rows.lo + k * BK + TB::row(i, wave, lane);
            const char* from = place(b_from[i % CB], SAME ? a_row[i] : b_row[i], b_stride, j, g.b_part * (int64_t)sizeof(B));
            if constexpr (DIRECT)
                TB::request(bt, j < end ? from : (const char*)&kZeros, i, wave);
            else
                b_reg[i] = fetch<B>(from, j < end ? b_left[i % CB] : 0);
        }
    };
    auto put = [&](char* at, char* bt) __attribute__((always_inline)) {
        if constexpr (!DIRECT) {
#pragma unroll
            for (int i = 0; i < TA::kEach; ++i) TA::put(at, a_reg[i], i, wave, lane);
#pragma unroll
            for (int i = 0; i < TB::kEach; ++i) TB::put(bt, b_reg[i], i, wave, lane);
        }
    };

    const int wm = wave % WM * (BM / WM), wn = wave / WM * (BN / WN);
    float16_t acc[TM][TN];
#pragma unroll
    for (int m = 0; m < TM; ++m)
#pragma unroll
        for (int n = 0; n < TN; ++n) acc[m][n] = 0.0f;

    // A fragment of floats has 8 of the rows that one of 16 bits has: 8 f + 4 half .. + 4 (16 f + 8 half .. + 8); where
    // both meet, two reads of four rows make the longer one.
    auto a_frag = [&](const char* at, int f, int first) __attribute__((always_inline)) {
        if constexpr (MIXED && sizeof(A) == 4) {
            float8_t x;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int r = 16 * f + 8 * (lane >> 5) + j, d = first + (lane & 31);
                x[j] = *(const float*)(at + r * TA::kRowBytes + (((d >> 2) ^ TA::swizzle(r)) << 4) + ((d & 3) << 2));
            }
            return x;
        } else {
            return widened<A, MIXED>(TA::down(at, f, first, lane));
        }
    };
    auto b_frag = [&](const char* bt, int f, int first) __attribute__((always_inline)) {
        if constexpr (MIXED && sizeof(B) == 4) {
            float8_t x;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int r = 16 * f + 8 * (lane >> 5) + j, d = first + (lane & 31);
                x[j] = *(const float*)(bt + r * TB::kRowBytes + (((d >> 2) ^ TB::swizzle(r)) << 4) + ((d & 3) << 2));
            }
            return x;
        } else {
            return widened<B, MIXED>(TB::down(bt, f, first, lane));
        }
    };
    constexpr int FRAGS = sizeof(A) == 4 && sizeof(B) == 4 ? BK / 8 : BK / 16;
    // As in row_products: fragments one ahead, requests between.
    auto products = [&](const char* at, const char* bt, auto between) __attribute__((always_inline)) {
        decltype(a_frag(at, 0, 0)) a[TM];
        decltype(b_frag(bt, 0, 0)) b[2][TN];
        auto read_b = [&](int f) __attribute__((always_inline)) {
#pragma unroll
            for (int n = 0; n < TN; ++n) b[f & 1][n] = b_frag(bt, f, wn + 32 * n);
        };
        read_b(0);
#pragma unroll
        for (int m = 0; m < TM; ++m) a[m] = a_frag(at, 0, wm + 32 * m);
#pragma unroll
        for (int f = 0; f < FRAGS; ++f) {
            if (f + 1 < FRAGS) read_b(f + 1);
            between(f);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int m = 0; m < TM; ++m) {
#pragma unroll
                for (int n = 0; n < TN; ++n) acc[m][n] = mma(a[m], b[f & 1][n], acc[m][n]);
                if (f + 1 < FRAGS) a[m] = a_frag(at, f + 1, wm + 32 * m);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    // (Past the last step zeros are requested, and the last row is looked up again.)
    auto step = [&](char* at, char* bt, char* an, char* bn, int k) __attribute__((always_inline)) {
        arrived();
        products(at, bt, [&](int f) __attribute__((always_inline)) {
            if (f < kEarly)
#pragma unroll
                for (int quarter = f * 4 / kEarly; quarter < (f + 1) * 4 / kEarly; ++quarter) request(an, bn, k + 1, quarter);
            if (f == kEarly - 1) look_up(k + 2);
        });
        put(an, bn);
    };
    if (steps > 0) {
        look_up(0);
#pragma unroll
        for (int quarter = 0; quarter < 4; ++quarter) request(a0, b0, 0, quarter);
        look_up(1);
        put(a0, b0);
    }
    if constexpr (sizeof(A) == 4 && sizeof(B) == 4) {
        float16_t total[TM][TN];
#pragma unroll
        for (int m = 0; m < TM; ++m)
#pragma unroll
            for (int n = 0; n < TN; ++n) total[m][n] = 0.0f;
        for (int k0 = 0; k0 < steps; k0 += kSpan) {
            const int last = min(k0 + kSpan, steps);
            for (int k = k0; k < last; k += 2) {
                step(a0, b0, a1, b1, k);
                if (k + 1 < last) step(a1, b1, a0, b0, k + 1);
            }
#pragma unroll
            for (int m = 0; m < TM; ++m)
#pragma unroll
                for (int n = 0; n < TN; ++n) total[m][n] += acc[m][n], acc[m][n] = 0.0f;
        }
#pragma unroll
        for (int m = 0; m < TM; ++m)
#pragma unroll
            for (int n = 0; n < TN; ++n) acc[m][n] = total[m][n];
    } else {
        for (int k = 0; k < steps; k += 2) {
            step(a0, b0, a1, b1, k);
            if (k + 1 < steps) step(a1, b1, a0, b0, k + 1);
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

    // lane l has column l % 32 of b, register r row 8 (r / 4) + 4 (l / 32) + r % 4 (the lane counted again: kept over the loop it
    // would leave no registers for the sums)
    const int l = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0));
    const int64_t size = (int64_t)g.a_columns * g.b_columns;
    O* out = (O*)g.out + rows.type * size;
    float* partial = g.partial + share_of(rows.lo, g.chunk, rows.lo == begin) * size;
#pragma unroll
    for (int m = 0; m < TM; ++m)
#pragma unroll
        for (int n = 0; n < TN; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int i = m0 + wm + 32 * m + 8 * (r / 4) + 4 * (l >> 5) + r % 4, j = n0 + wn + 32 * n + (l & 31);
                if (i >= g.a_columns || j >= g.b_columns) continue;
                const int64_t at = (int64_t)i * g.b_columns + j;
                if (whole)
                    out[at] = (O)acc[m][n][r];
                else
                    partial[at] = acc[m][n][r];
            }
}

// The slots of a type, where it has more than one: 16 lanes with V columns each, and 16 groups with every sixteenth slot.
template <typename O, int V>
__global__ __launch_bounds__(256) void join_slots(SumArgs g) {
    typedef float vec __attribute__((ext_vector_type(V)));
    typedef O result __attribute__((ext_vector_type(V)));
    __shared__ vec lds[16][16];
    const int t = blockIdx.y, lane = threadIdx.x & 15, group = threadIdx.x >> 4;
    const int begin = begin_of(g.ptr, t, g.rows, g.parts), n = begin_of(g.ptr, t + 1, g.rows, g.parts) - begin;
    if (n <= g.chunk) return;
    const int64_t size = (int64_t)g.a_columns * g.b_columns;
    const float* from = g.partial;
    const int slots = (n - 1) / g.chunk + 1;
    for (int64_t block = blockIdx.x; block * 16 * V < size; block += gridDim.x) {
        const int64_t i = (block * 16 + lane) * V;
        vec sum = 0.0f;
        if (i < size)
#pragma unroll 4
            for (int s = group; s < slots; s += 16) sum += *(const vec*)(from + share_of(begin + s * g.chunk, g.chunk, s == 0) * size + i);
        lds[group][lane] = sum;
        __syncthreads();
        if (group == 0 && i < size) {
            sum = lds[0][lane];
            for (int k = 1; k < min(slots, 16); ++k) sum += lds[k][lane];
            *(result*)((O*)g.out + t * size + i) = __builtin_convertvector(sum, result);
        }
        __syncthreads();
    }
}

}  // namespace typed_products
#endif
