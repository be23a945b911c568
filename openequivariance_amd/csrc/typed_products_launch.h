// The launches that typed_products.hip defines for each element type.
#ifndef OEQ_TYPED_PRODUCTS_LAUNCH_H
#define OEQ_TYPED_PRODUCTS_LAUNCH_H

#include "typed_products.h"

namespace typed_products {

// Whether the form for few rows, which needs no index, takes a product: rows in the lanes of a wave, or, where all share the
// weights, as many as are faster so. bf16, adapters of rank 16 beside 4096 x 4096, us with it / with tiles: 64 rows 22 / 44, 128 41 / 50, 192
// 54 / 47.
inline bool few(const Args& a, bool across) { return !across && (int64_t)a.rows * a.parts <= (a.shared ? 2 * kFewRows : kFewRows); }

enum Thin { kNeither, kFirst, kSecond };  // which operand of a sum of products is float beside elements of 16 bits

template <typename T>
struct Launch {
    // across: the weights' rows run along the columns. wide: the result is float. direct: see row_products.
    static hipError_t rows(Args a, bool across, bool wide, bool direct, hipStream_t stream);
    static hipError_t sums(SumArgs a, Thin thin, bool direct, hipStream_t stream);
};

// Columns of a tile of sum_products of which there are few (float operands of a thin product), else.
constexpr int kThinTile = 32, kSumTile = 128, kSmallSumTile = 64, kLargeSumTile = 256;

}  // namespace typed_products
#endif
