// Kernels of typed_products.h for one element type (OEQ_PRODUCT_TYPE; one object file each, compiled side by side) and their
// launches.
#include "typed_products.h"
#include "typed_products_launch.h"

#include <algorithm>
#include <cmath>

namespace typed_products {
namespace {

typedef OEQ_PRODUCT_TYPE T;

int64_t divide_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Threads along the first dimension of a launch are counted in 32 bits.
bool too_many(int64_t blocks, int threads) { return blocks * threads > UINT32_MAX; }

template <typename O, bool ACROSS, bool DIRECT, bool THIN, int BM, int BN, int WM, int WN>
hipError_t rows_by(Args a, hipStream_t stream) {
    a.slots = (int)((int64_t)a.rows * a.parts / BM + a.types + 1);
    a.tiles = (int)divide_up(a.out_row, BN);
    const int64_t blocks = (int64_t)a.slots * a.tiles;
    if (too_many(blocks, 64 * WM * WN)) return hipErrorInvalidConfiguration;
    row_products<T, O, ACROSS, DIRECT, THIN, BM, BN, WM, WN><<<(unsigned)blocks, 64 * WM * WN, 0, stream>>>(a);
    return hipGetLastError();
}

template <typename O, bool DIRECT, int MT>
hipError_t few_by(const Args& a, hipStream_t stream) {
    const int64_t rows = (int64_t)a.rows * a.parts, columns = divide_up(a.out_row, 16);
    if (too_many(columns, 64 * kFewWaves)) return hipErrorInvalidConfiguration;
    few_products<T, O, DIRECT, MT><<<dim3((unsigned)columns, (unsigned)(a.shared ? divide_up(rows, 16 * MT) : rows)), 64 * kFewWaves, 0,
                                     stream>>>(a);
    return hipGetLastError();
}

template <bool DIRECT, int NT>
hipError_t thin_by(const Args& a, hipStream_t stream) {
    const int64_t slots = a.rows / kThinRows + a.types + 1, tiles = divide_up(a.out_row, 16 * NT);
    if (slots > (1 << 23) - 1 || tiles > 65535) return hipErrorInvalidConfiguration;
    thin_products<T, DIRECT, NT><<<dim3((unsigned)slots, (unsigned)tiles), 64 * kFewWaves, 0, stream>>>(a);
    return hipGetLastError();
}

template <typename O, bool ACROSS, bool DIRECT>
hipError_t rows_of_size(const Args& a, bool thin_result, hipStream_t stream) {
    if constexpr (!ACROSS) {
        if (few(a, false)) {
            // As many rows at a time as a type has about twice: with more, fewer blocks fit a compute unit, with fewer a type's
            // matrix is read again. 64 rows of 64 types, 2048 x 2048, bf16: 103 us for 64 rows at a time, 69 for 16.
            const int64_t all = (int64_t)a.rows * a.parts, at_a_time = a.shared ? all : 2 * divide_up(all, std::max(1, std::min(a.types, a.rows)));
            return at_a_time <= 16 ? few_by<O, DIRECT, 1>(a, stream) : at_a_time <= 32 ? few_by<O, DIRECT, 2>(a, stream)
                   : at_a_time <= 48 ? few_by<O, DIRECT, 3>(a, stream) : few_by<O, DIRECT, 4>(a, stream);
        }
    }
    if constexpr (std::is_same<O, float>::value && !ACROSS)
        if (thin_result) return a.outer <= 16 ? thin_by<DIRECT, 1>(a, stream) : a.outer <= 32 ? thin_by<DIRECT, 2>(a, stream) : thin_by<DIRECT, 4>(a, stream);
    // Tiles by an estimate, in us, of what measured tiles take: a block's beginning and end, and steps that last as long as one
    // alone or as all blocks of a compute unit together. (Half a tile of each type's rows is left over; compute units hold four
    // tiles of 64, two of 128, one of 256.) bf16, us with tiles of 64 / 128 / 256: 1 000 rows, 4 matrices of 1024 x 1024 10 / 16 / 31,
    // 8 000 34 / 39 / 36, 16 000 63 / 48 / 68; 4 001 rows, 16 of 2048 x 2048 70 / 68 / 60, one of 4096 x 4096 207 / 148 / 125;
    // float32: 5 000 rows, 5 of 512 x 512 36 / 43, 20 000 rows, 10 of 128 x 128 14 / 18.
    constexpr bool SHORT = sizeof(T) == 2;
    constexpr int64_t BK = 128 / (int)sizeof(T);
    const int64_t rows = (int64_t)a.rows * a.parts;
    const double steps = (double)(divide_up(a.inner, BK) + divide_up((SHORT ? 2 : 1) * (int64_t)(a.rank ? a.thin_row : 0), BK));
    const auto takes = [&](int64_t tile, int at_once, double ends, double alone, double together) {
        const int64_t blocks = (rows / tile + std::min<int64_t>(a.types, rows) / 2 + 1) * divide_up(a.out_row, tile);
        const double mean = blocks / 256.0, each = mean < 1 ? mean : (mean + std::ceil(mean)) / 2;  // (of a compute unit)
        return ends * std::max(1.0, each / at_once) + steps * std::max(alone, each * together);
    };
    const double small = takes(64, 4, 6, SHORT ? 0.5 : 0.7, SHORT ? 0.22 : 0.5), middle = takes(128, 2, 6, SHORT ? 0.7 : 2, SHORT ? 0.62 : 1.95);
    constexpr bool MAY_BE_THIN = std::is_same<O, T>::value;
    if constexpr (DIRECT && SHORT)
        if (takes(256, 1, 12, 1.37, 1.95) < std::min(small, middle)) {
            if constexpr (MAY_BE_THIN)
                if (a.rank) return rows_by<O, ACROSS, DIRECT, true, 256, 256, 2, 4>(a, stream);
            return rows_by<O, ACROSS, DIRECT, false, 256, 256, 2, 4>(a, stream);
        }
    if (small < middle) {
        if constexpr (MAY_BE_THIN)
            if (a.rank) return rows_by<O, ACROSS, DIRECT, true, 64, 64, 2, 2>(a, stream);
        return rows_by<O, ACROSS, DIRECT, false, 64, 64, 2, 2>(a, stream);
    }
    if constexpr (MAY_BE_THIN)
        if (a.rank) return rows_by<O, ACROSS, DIRECT, true, 128, 128, 2, 2>(a, stream);
    return rows_by<O, ACROSS, DIRECT, false, 128, 128, 2, 2>(a, stream);
}

template <typename A, typename B, typename O, bool DIRECT, int BM, int BN, int WM, int WN>
hipError_t sums_by(SumArgs g, hipStream_t stream) {
    g.a_tiles = (int)divide_up(g.a_columns, BM), g.b_tiles = (int)divide_up(g.b_columns, BN);
    const int64_t blocks = (int64_t)g.slots * g.a_tiles * g.b_tiles;
    if (too_many(blocks, 64 * WM * WN)) return hipErrorInvalidConfiguration;
    if constexpr (sizeof(A) == sizeof(B) && BM < kLargeSumTile) {
        if (g.parts > 1)
            sum_products<A, B, O, DIRECT, true, BM, BN, WM, WN><<<(unsigned)blocks, 64 * WM * WN, 0, stream>>>(g);
        else
            sum_products<A, B, O, DIRECT, false, BM, BN, WM, WN><<<(unsigned)blocks, 64 * WM * WN, 0, stream>>>(g);
    } else {
        sum_products<A, B, O, DIRECT, false, BM, BN, WM, WN><<<(unsigned)blocks, 64 * WM * WN, 0, stream>>>(g);
    }
    if (g.partial) {
        const int64_t size = (int64_t)g.a_columns * g.b_columns;
        // (most blocks are of types with nothing to join)
        const int64_t most = std::max(32, (1 << 14) / g.types);
        const auto grid = [&](int each) { return dim3((unsigned)std::min(divide_up(size, 16 * each), most), (unsigned)g.types); };
        if (size % 4 == 0 && ((uintptr_t)g.out & 15) == 0)
            join_slots<O, 4><<<grid(4), 256, 0, stream>>>(g);
        else
            join_slots<O, 1><<<grid(1), 256, 0, stream>>>(g);
    }
    return hipGetLastError();
}

template <bool DIRECT>
hipError_t sums_of(const SumArgs& g, Thin thin, hipStream_t stream) {
    if (thin == kFirst) return sums_by<float, T, T, DIRECT, kThinTile, kSumTile, 1, 4>(g, stream);
    if (thin == kSecond) return sums_by<T, float, T, DIRECT, kSumTile, kThinTile, 4, 1>(g, stream);
    if constexpr (DIRECT && sizeof(T) == 2)
        if (g.tile == kLargeSumTile) return sums_by<T, T, T, true, kLargeSumTile, kLargeSumTile, 2, 4>(g, stream);
    if constexpr (DIRECT)
        if (g.tile == kSumTile) return sums_by<T, T, T, true, kSumTile, kSumTile, 2, 2>(g, stream);
    return sums_by<T, T, T, DIRECT, kSmallSumTile, kSmallSumTile, 2, 2>(g, stream);
}

}  // namespace

template <>
hipError_t Launch<T>::rows(Args a, bool across, bool wide, bool direct, hipStream_t stream) {
    if (wide)
        return across ? (direct ? rows_of_size<float, true, true>(a, true, stream) : rows_of_size<float, true, false>(a, true, stream))
                      : (direct ? rows_of_size<float, false, true>(a, true, stream) : rows_of_size<float, false, false>(a, true, stream));
    return across ? (direct ? rows_of_size<T, true, true>(a, false, stream) : rows_of_size<T, true, false>(a, false, stream))
                  : (direct ? rows_of_size<T, false, true>(a, false, stream) : rows_of_size<T, false, false>(a, false, stream));
}

template <>
hipError_t Launch<T>::sums(SumArgs a, Thin thin, bool direct, hipStream_t stream) {
    return direct ? sums_of<true>(a, thin, stream) : sums_of<false>(a, thin, stream);
}

}  // namespace typed_products
