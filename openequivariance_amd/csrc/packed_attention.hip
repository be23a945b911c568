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
        forward<T, DP><<<(unsigned)(a.tiles * a.hq), 256, 0, stream>>>(a);
        return hipGetLastError();
    }
    static hipError_t forward_shares(const Args& a, hipStream_t stream) {
        const unsigned stacks = (unsigned)(a.hq / a.hk + 31) / 32;
        forward_few<T, DP><<<(unsigned)a.nq * a.hk * stacks * a.parts, 64 * Few<T, DP>::kWaves, 0, stream>>>(a);
        if (a.parts > 1) join<T, DP><<<(unsigned)a.nq * a.hq, 256, 0, stream>>>(a);
        return hipGetLastError();
    }
    static hipError_t gradients(const Args& a, int key_tiles, hipStream_t stream) {
        if (a.tiles) query_gradient<T, DP><<<(unsigned)(a.tiles * a.hq), 256, 0, stream>>>(a);
        Args b = a;
        b.tiles = key_tiles;
        if (key_tiles) key_gradient<T, DP><<<(unsigned)(key_tiles * a.hk), 256, 0, stream>>>(b);
        return hipGetLastError();
    }
};

}  // namespace

#define OEQ_BY_HEAD(call) (a.d <= 32 ? Kernels<32>::call : a.d <= 64 ? Kernels<64>::call : Kernels<128>::call)

template <>
hipError_t Launch<OEQ_ATTENTION_TYPE>::forward(const Args& a, hipStream_t stream) {
    return a.parts ? OEQ_BY_HEAD(forward_shares(a, stream)) : OEQ_BY_HEAD(forward_rows(a, stream));
}

template <>
hipError_t Launch<OEQ_ATTENTION_TYPE>::backward(const Args& a, int key_tiles, hipStream_t stream) {
    return OEQ_BY_HEAD(gradients(a, key_tiles, stream));
}

}  // namespace packed_attention
