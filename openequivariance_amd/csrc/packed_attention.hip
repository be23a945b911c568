// Kernels of packed_attention.h for one element type (OEQ_ATTENTION_TYPE; one object file each, compiled side by side) and
// their launches.
#include "packed_attention.h"
#include "packed_attention_launch.h"

namespace packed_attention {
namespace {

template <int DP>
struct Kernels {
    typedef OEQ_ATTENTION_TYPE T;
    static hipError_t forward_rows(const Args& a, hipStream_t stream) {
        if (a.split == 2)
            forward<T, DP, 2><<<(unsigned)(a.tiles * a.hq), 256, 0, stream>>>(a);
        else
            forward<T, DP, 1><<<(unsigned)(a.tiles * a.hq), 256, 0, stream>>>(a);
        return hipGetLastError();
    }
    static hipError_t forward_shares(const Args& a, hipStream_t stream) {
        const unsigned stacks = (unsigned)(a.hq / a.hk + 31) / 32;
        forward_few<T, DP><<<(unsigned)a.nq * a.hk * stacks * a.parts, 64 * Few<T, DP>::kWaves, 0, stream>>>(a);
        if (a.parts > 1) join<T, DP><<<(unsigned)a.nq * a.hq, 256, 0, stream>>>(a);
        return hipGetLastError();
    }
    // Whether blocks of keys' gradients fit a compute unit twice, but are faster alone: 249 registers a lane, or 400.
    static constexpr bool kAlone = sizeof(T) == 2 && DP == 96;
    static hipError_t gradients(const Args& a, int key_tiles, hipStream_t stream) {
        if (a.tiles && a.split == 2)
            query_gradient<T, DP, 2><<<(unsigned)(a.tiles * a.hq), 256, 0, stream>>>(a);
        else if (a.tiles)
            query_gradient<T, DP, 1><<<(unsigned)(a.tiles * a.hq), 256, 0, stream>>>(a);
        Args b = a;
        b.tiles = key_tiles;
        const unsigned blocks = (unsigned)(key_tiles * a.hk);
        if (!blocks) return hipGetLastError();
        if constexpr (sizeof(T) * DP > 256) {
            // Sums of values' and keys' gradients together do not fit the registers beside rows of 512 bytes (580 bytes of
            // scratch memory a lane): one after the other, with the scores computed twice. 8 segments of 1 000 rows, 8 / 2
            // heads of 128, causal: gradients 1 893 us together, 1 183 apart; elsewhere together is faster (heads of 64: 737
            // and 859, bf16 of 128 in 9 packed sequences: 393 and 580).
            key_gradient<T, DP, 2, 2><<<blocks, 256, 0, stream>>>(b);
            key_gradient<T, DP, 1, 2><<<blocks, 256, 0, stream>>>(b);
        } else if (blocks < 256) {
            // Fewer blocks than compute units: half as many keys to a block and half as long a walk. Gradients together, us, with
            // 64 / 32 keys: 56 blocks, float32 heads of 64 226 / 145; 126, float32 of 64 416 / 268; 252, bf16
            // of 128 159 / 161; 504 217 / 278. All of them run at once, so they need no order (which is of tiles of 64 keys).
            b.tiles = (a.nk + 31) / 32, b.k_order = nullptr;
            key_gradient<T, DP, 3, 1, kAlone ? 1 : key_blocks_per_unit<T, DP, 3>()><<<(unsigned)(b.tiles * a.hk), 256, 0, stream>>>(b);
        } else {
            if constexpr (kAlone)
                if (a.causal && blocks <= 512) {
                    // Two blocks share a compute unit, or one has it alone and all registers, where the longest of few
                    // uneven walks decides. bf16, 16 heads of 96, gradients, shared / alone: causal, 284 blocks 485 / 431 us,
                    // 376 169 / 155, 500 556 / 492, 628 1 372 / 1 431, 2 000 170 / 215; not causal, 500 blocks 1 524 / 1 687.
                    key_gradient<T, DP, 3, 2, 1><<<blocks, 256, 0, stream>>>(b);
                    return hipGetLastError();
                }
            key_gradient<T, DP, 3, 2><<<blocks, 256, 0, stream>>>(b);
        }
        return hipGetLastError();
    }
};

}  // namespace

// Heads of 72 to 96 elements leave out a quarter of the products of 128: bf16, 16 / 4 heads of 96, two segments of 4 000
// rows, causal, forward 134 us, not 152, gradients 490, not 559; float32, 8 heads of 96, 4 000 rows 249 and 949, not 309 and 1 196.
#define OEQ_BY_HEAD(call) \
    (a.d <= 32   ? Kernels<32>::call \
     : a.d <= 64 ? Kernels<64>::call \
     : a.d <= 96 ? Kernels<96>::call : Kernels<128>::call)

template <>
hipError_t Launch<OEQ_ATTENTION_TYPE>::forward(const Args& a, hipStream_t stream) {
    if (a.parts)
        return a.d <= 32   ? Kernels<32>::forward_shares(a, stream)
               : a.d <= 64 ? Kernels<64>::forward_shares(a, stream)
                           : Kernels<128>::forward_shares(a, stream);
    return OEQ_BY_HEAD(forward_rows(a, stream));
}

template <>
hipError_t Launch<OEQ_ATTENTION_TYPE>::backward(const Args& a, int key_tiles, hipStream_t stream) {
    return OEQ_BY_HEAD(gradients(a, key_tiles, stream));
}

}  // namespace packed_attention
