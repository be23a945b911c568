// The launches that packed_attention.hip defines for each element type.
#ifndef OEQ_PACKED_ATTENTION_LAUNCH_H
#define OEQ_PACKED_ATTENTION_LAUNCH_H

#include "packed_attention.h"

namespace packed_attention {

template <typename T>
struct Launch {
    static hipError_t forward(const Args& a, hipStream_t stream);
    static hipError_t backward(const Args& a, int key_tiles, hipStream_t stream);
};

// Rows of a tile of queries and of keys.
constexpr int kQueryTile = 128, kKeyTile = 64;

}  // namespace packed_attention
#endif
