// Kernels of typed_products.h for one element type (OEQ_PRODUCT_TYPE; one object file each, compiled side by side) and their
// launches.
#include "typed_products.h"
#include "typed_products_launch.h"

#include <algorithm>

namespace typed_products {
namespace {

typedef OEQ_PRODUCT_TYPE T;

int64_t divide_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

template <typename O, bool ACROSS, bool DIRECT, int BM, int BN, int WM, int WN>
hipError_t rows_by(Args a, hipStream_t stream) {
    a.slots = (int)((int64_t)a.rows * a.parts / BM + a.types + 1);
    a.tiles = (int)divide_up(a.out_row, BN);
    const int64_t blocks = (int64_t)a.slots * a.tiles;
    if (blocks > (1 << 24) - 1) return hipErrorInvalidConfiguration;
    row_products<T, O, ACROSS, DIRECT, BM, BN, WM, WN><<<(unsigned)blocks, 64 * WM * WN, 0, stream>>>(a);
    return hipGetLastError();
}

template <typename O, bool DIRECT, int MT>
hipError_t few_by(const Args& a, hipStream_t stream) {
    const int64_t rows = (int64_t)a.rows * a.parts;
    few_products<T, O, DIRECT, MT><<<dim3((unsigned)divide_up(a.out_row, 16), (unsigned)(a.shared ? divide_up(rows, 16 * MT) : rows)),
                                     64 * kFewWaves, 0, stream>>>(a);
    return hipGetLastError();
}

template <typename O, bool ACROSS, bool DIRECT>
hipError_t rows_of_size(const Args& a, hipStream_t stream) {
    if constexpr (!ACROSS) {
        const int64_t rows = (int64_t)a.rows * a.parts;
        if (few(a, false)) return rows <= 16 ? few_by<O, DIRECT, 1>(a, stream) : rows <= 32 ? few_by<O, DIRECT, 2>(a, stream) : few_by<O, DIRECT, 4>(a, stream);
    }
    if (a.out_row <= 64) return rows_by<O, ACROSS, DIRECT, 64, 64, 2, 2>(a, stream);
    return rows_by<O, ACROSS, DIRECT, 128, 128, 2, 2>(a, stream);
}

template <typename A, typename B, typename O, bool DIRECT, int BM, int BN, int WM, int WN>
hipError_t sums_by(SumArgs g, hipStream_t stream) {
    g.a_tiles = (int)divide_up(g.a_columns, BM), g.b_tiles = (int)divide_up(g.b_columns, BN);
    const int64_t blocks = (int64_t)g.slots * g.a_tiles * g.b_tiles;
    if (blocks > (1 << 24) - 1) return hipErrorInvalidConfiguration;
    sum_products<A, B, O, DIRECT, BM, BN, WM, WN><<<(unsigned)blocks, 64 * WM * WN, 0, stream>>>(g);
    if (g.partial) {
        const int64_t size = (int64_t)g.a_columns * g.b_columns;
        const dim3 grid((unsigned)std::min<int64_t>(divide_up(size, 256), 4096), (unsigned)g.types);
        join_slots<O><<<grid, 256, 0, stream>>>(g);
    }
    return hipGetLastError();
}

template <bool DIRECT>
hipError_t sums_of(const SumArgs& g, Thin thin, hipStream_t stream) {
    if (thin == kFirst) return sums_by<float, T, T, DIRECT, kThinTile, kSumTile, 1, 4>(g, stream);
    if (thin == kSecond) return sums_by<T, float, T, DIRECT, kSumTile, kThinTile, 4, 1>(g, stream);
    // (through registers: smaller tiles, whose loads on their way fit beside the sums)
    return sums_by<T, T, T, DIRECT, DIRECT ? kSumTile : 64, DIRECT ? kSumTile : 64, 2, 2>(g, stream);
}

}  // namespace

template <>
hipError_t Launch<T>::rows(Args a, bool across, bool wide, bool direct, hipStream_t stream) {
    if (wide)
        return across ? (direct ? rows_of_size<float, true, true>(a, stream) : rows_of_size<float, true, false>(a, stream))
                      : (direct ? rows_of_size<float, false, true>(a, stream) : rows_of_size<float, false, false>(a, stream));
    return across ? (direct ? rows_of_size<T, true, true>(a, stream) : rows_of_size<T, true, false>(a, stream))
                  : (direct ? rows_of_size<T, false, true>(a, stream) : rows_of_size<T, false, false>(a, stream));
}

template <>
hipError_t Launch<T>::sums(SumArgs a, Thin thin, bool direct, hipStream_t stream) {
    return direct ? sums_of<true>(a, thin, stream) : sums_of<false>(a, thin, stream);
}

}  // namespace typed_products
