// Device code of the norm of queries and keys and their rotation by position.
//
// A head x of d elements becomes y = w x / sqrt(mean(x^2) + eps) (or stays, without w), and of y the first r elements
// turn in pairs: (u, v) -> (u c - v s, v c + u s) with cosine and sine from the row of a table that the node's position
// names. Pairs are elements i and i + r / 2, or 2 i and 2 i + 1 (interleaved).
//
// A head belongs to 8 (a power of two up to 16) neighbouring lanes with eight elements each, chosen so that both partners
// of a pair are in one lane: two quads that lie r / 2 apart, or one behind the other where pairs are neighbours or past
// the r turned elements. So the only thing that passes between lanes is the sum of squares. A block has one row or several
// and its groups of lanes walk the row's heads, kHeads of them requested at a time, with the row's cosines and sines in
// registers. The kernels are bound by memory: every head is read once and written once. 16 411 rows of 32 and 8 heads of 128,
// bf16, 168 MB: forward 68 us for two times that, 4.9 TB/s, gradient 119 for three times, 4.2, and 5 for the weights' sums (a copy of
// 4 GiB 4.7). (Both kinds' heads requested before either is computed: 78 and 155 us, for the registers; one head at a time in
// the gradient 149; fewer registers by scratch memory 250 to 630.) A batch of 64 rows takes 5 us, about
// a launch.
#ifndef OEQ_QK_ROTARY_H
#define OEQ_QK_ROTARY_H

#include <hip/hip_runtime.h>

#include <cstdint>

namespace qk_rotary {

struct Args {
    const void *q, *k, *v, *q_weight, *k_weight, *q_grad, *k_grad;
    void *q_out, *k_out, *v_out;  // outputs, caches or gradients
    const int64_t *positions, *slots;
    const float* table;
    float* partial;  // sums of the weights' gradients: [blocks, 2, 8 lanes]
    int groups;      // groups of lanes to a row: a power of two
    int64_t q_row, q_head, k_row, k_head, v_row, v_head;
    int64_t gq_row, gq_head, gk_row, gk_head;       // strides of the outputs' gradients
    int64_t ko_row, ko_head, vo_row, vo_head;       // strides of k_out, v_out
    int64_t table_rows, slots_end;
    int64_t rows;
    int q_heads, k_heads, d, rotary, interleaved;
    float eps, per_d;  // and 1 / d
};

template <typename T>
struct Quad {
    typedef T type __attribute__((ext_vector_type(4)));
};
typedef float float4_t __attribute__((ext_vector_type(4)));

// Where a lane's two quads begin.
struct Where {
    int a, b;
    bool turned;
    __device__ __forceinline__ Where(const Args& g, int i) {
        turned = i < g.rotary / 8;
        const bool apart = turned && !g.interleaved;
        a = apart ? 4 * i : 8 * i;
        b = apart ? g.rotary / 2 + 4 * i : 8 * i + 4;
    }
};

struct Eight {
    float u[4], v[4];  // the two quads
};

// As they are in memory: the conversion waits for the load, so it comes when others have been requested.
template <typename T>
struct Raw {
    typename Quad<T>::type a, b;
    __device__ __forceinline__ Raw() {}
    __device__ __forceinline__ Raw(const T* row, Where w)
        : a(*(const typename Quad<T>::type*)(row + w.a)), b(*(const typename Quad<T>::type*)(row + w.b)) {}
    __device__ __forceinline__ Eight wide() const {
        Eight x;
#pragma unroll
        for (int j = 0; j < 4; ++j) x.u[j] = (float)a[j], x.v[j] = (float)b[j];
        return x;
    }
};

template <typename T>
__device__ __forceinline__ void store(T* row, Where w, const Eight& x) {
    float4_t a, b;
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = x.u[j], b[j] = x.v[j];
    *(typename Quad<T>::type*)(row + w.a) = __builtin_convertvector(a, typename Quad<T>::type);
    *(typename Quad<T>::type*)(row + w.b) = __builtin_convertvector(b, typename Quad<T>::type);
}

// The angles of a lane's pairs in a row. (A position that the table does not have gives NaN.)
struct Angle {
    float4_t c, s;
    __device__ __forceinline__ Angle(const Args& g, int64_t row, int i, bool turned) {
        c = 1.0f, s = 0.0f;
        if (!turned) return;
        const int64_t at = g.positions[row];
        const bool known = at >= 0 && at < g.table_rows;
        if (known) {
            c = *(const float4_t*)(g.table + at * g.rotary + 4 * i);
            s = *(const float4_t*)(g.table + at * g.rotary + g.rotary / 2 + 4 * i);
        } else {
            c = NAN, s = NAN;
        }
    }
};

// Turns the lane's four pairs, or back.
__device__ __forceinline__ void turn(Eight& x, const Args& g, const Angle& angle, float sign) {
    const float4_t &c = angle.c, &s = angle.s;
    if (g.interleaved) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float a = x.u[2 * j], b = x.u[2 * j + 1], p = x.v[2 * j], q = x.v[2 * j + 1];
            x.u[2 * j] = a * c[j] - sign * b * s[j];
            x.u[2 * j + 1] = b * c[j] + sign * a * s[j];
            x.v[2 * j] = p * c[2 + j] - sign * q * s[2 + j];
            x.v[2 * j + 1] = q * c[2 + j] + sign * p * s[2 + j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float a = x.u[j], b = x.v[j];
            x.u[j] = a * c[j] - sign * b * s[j];
            x.v[j] = b * c[j] + sign * a * s[j];
        }
    }
}

// The sum over the lanes of a head, in the vector unit: with the neighbour, the next pair, and by mirrors of eight and of
// sixteen lanes the other quad and the other eight.
template <int LANES>
__device__ __forceinline__ float head_sum(float x) {
#define OEQ_ADD_DPP(control) \
    x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), control, 0xf, 0xf, true))
    if (LANES > 1) OEQ_ADD_DPP(0xb1);    // quad_perm 1 0 3 2
    if (LANES > 2) OEQ_ADD_DPP(0x4e);    // quad_perm 2 3 0 1
    if (LANES > 4) OEQ_ADD_DPP(0x141);   // row_half_mirror
    if (LANES > 8) OEQ_ADD_DPP(0x140);   // row_mirror
#undef OEQ_ADD_DPP
    return x;
}

__device__ __forceinline__ float squares(const Eight& x) {
    float s = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) s = fmaf(x.u[j], x.u[j], fmaf(x.v[j], x.v[j], s));
    return s;
}

constexpr int kHeads = 2;  // requested at a time

// Which part of a block's rows and heads a thread has. Lanes without elements, heads and rows past the last read what the
// last ones do and store nothing.
template <int LANES>
struct Place {
    int64_t mine, row;
    int i, first;
    bool holds, live;
    __device__ __forceinline__ Place(const Args& g, int64_t top) {
        const int lane = threadIdx.x & (LANES - 1);
        first = threadIdx.x / LANES & (g.groups - 1);
        mine = top + threadIdx.x / (LANES * g.groups);
        row = min(mine, g.rows - 1);
        holds = 8 * lane < g.d;
        live = holds && mine < g.rows;
        i = holds ? lane : 0;
    }
};

// The heads of one kind in a row: normed by `weight` (if there is one), turned, stored.
template <typename T, int LANES, bool TURNS>
__device__ __forceinline__ void heads_forward(const Args& g, const Place<LANES>& at, Where w, const Angle& angle, const T* from,
                                              int64_t from_head, T* to, int64_t to_head, int heads, const T* weight, bool live) {
    Eight y;
    if (weight) y = Raw<T>(weight, w).wide();
    for (int base = at.first; base < heads; base += kHeads * g.groups) {
        Raw<T> raw[kHeads];
#pragma unroll
        for (int n = 0; n < kHeads; ++n) raw[n] = Raw<T>(from + min(base + n * g.groups, heads - 1) * from_head, w);
#pragma unroll
        for (int n = 0; n < kHeads; ++n) {
            const int h = base + n * g.groups;
            Eight x = raw[n].wide();
            if (weight) {
                const float by = __builtin_amdgcn_rsqf(head_sum<LANES>(at.holds ? squares(x) : 0.0f) * g.per_d + g.eps);
#pragma unroll
                for (int j = 0; j < 4; ++j) x.u[j] *= by * y.u[j], x.v[j] *= by * y.v[j];
            }
            if (TURNS && w.turned) turn(x, g, angle, 1.0f);
            if (live && h < heads) store<T>(to + h * to_head, w, x);
        }
    }
}

// APPEND: keys go to the row of the cache that slots[] names, values as they are beside them; rows that the cache does not
// have are left out.
template <typename T, int LANES, bool APPEND>
__global__ __launch_bounds__(256) void forward(Args g) {
    const int each = 256 / (LANES * g.groups);
    for (int64_t top = (int64_t)blockIdx.x * each; top < g.rows; top += (int64_t)gridDim.x * each) {
        const Place<LANES> at(g, top);
        const Where w(g, at.i);
        const Angle angle(g, at.row, at.i, w.turned);
        int64_t to = at.row;
        bool live = at.live;
        if (APPEND) {
            to = g.slots[at.row];
            live = live && to >= 0 && to < g.slots_end;
        }
        heads_forward<T, LANES, true>(g, at, w, angle, (const T*)g.q + at.row * g.q_row, g.q_head,
                                      (T*)g.q_out + at.row * g.q_heads * g.d, g.d, g.q_heads, (const T*)g.q_weight, at.live);
        heads_forward<T, LANES, true>(g, at, w, angle, (const T*)g.k + at.row * g.k_row, g.k_head, (T*)g.k_out + to * g.ko_row,
                                      g.ko_head, g.k_heads, (const T*)g.k_weight, live);
        if (APPEND)
            heads_forward<T, LANES, false>(g, at, w, angle, (const T*)g.v + at.row * g.v_row, g.v_head, (T*)g.v_out + to * g.vo_row,
                                           g.vo_head, g.k_heads, nullptr, live);
    }
}

// The gradients of one kind of heads in a row: gradients turned back, gy; with n = x / rms, dx = (gy w - n mean(gy w n)) / rms
// and dw = sum gy n.
template <typename T, int LANES>
__device__ __forceinline__ void heads_backward(const Args& g, const Place<LANES>& at, Where w, const Angle& angle, const T* grad,
                                               int64_t grad_head, const T* from, int64_t from_head, T* to, int heads,
                                               const T* weight, const Eight& wt, Eight& dw) {
    for (int base = at.first; base < heads; base += kHeads * g.groups) {
        Raw<T> rx[kHeads], ry[kHeads];
#pragma unroll
        for (int n = 0; n < kHeads; ++n) {
            const int h = min(base + n * g.groups, heads - 1);
            ry[n] = Raw<T>(grad + h * grad_head, w);
            if (weight) rx[n] = Raw<T>(from + h * from_head, w);
        }
#pragma unroll
        for (int n = 0; n < kHeads; ++n) {
            const int h = base + n * g.groups;
            const bool live = at.live && h < heads;
            Eight y = ry[n].wide();
            if (w.turned) turn(y, g, angle, -1.0f);
            if (weight) {
                Eight x = rx[n].wide(), z;
                const float by = __builtin_amdgcn_rsqf(head_sum<LANES>(at.holds ? squares(x) : 0.0f) * g.per_d + g.eps);
                float along = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    x.u[j] *= by, x.v[j] *= by;
                    z.u[j] = y.u[j] * wt.u[j], z.v[j] = y.v[j] * wt.v[j];
                    along = fmaf(z.u[j], x.u[j], fmaf(z.v[j], x.v[j], along));
                }
                along = head_sum<LANES>(at.holds ? along : 0.0f) * g.per_d;
                if (live) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        dw.u[j] = fmaf(y.u[j], x.u[j], dw.u[j]), dw.v[j] = fmaf(y.v[j], x.v[j], dw.v[j]);
                        y.u[j] = by * (z.u[j] - x.u[j] * along);
                        y.v[j] = by * (z.v[j] - x.v[j] * along);
                    }
                }
            }
            if (live) store<T>(to + h * g.d, w, y);
        }
    }
}

// Blocks walk rows at the distance of the grid; their sums of dw go, one row a block, to `partial`, which weight_gradient adds
// up in order.
template <typename T, int LANES>
__global__ __launch_bounds__(256) void backward(Args g) {
    __shared__ float sums[2][256][8];
    const int each = 256 / (LANES * g.groups);
    Eight dq = {}, dk = {}, wq = {}, wk = {};
    {
        const Place<LANES> at(g, 0);
        const Where w(g, at.i);
        if (g.q_weight) wq = Raw<T>((const T*)g.q_weight, w).wide();
        if (g.k_weight) wk = Raw<T>((const T*)g.k_weight, w).wide();
    }
    for (int64_t top = (int64_t)blockIdx.x * each; top < g.rows; top += (int64_t)gridDim.x * each) {
        const Place<LANES> at(g, top);
        const Where w(g, at.i);
        const Angle angle(g, at.row, at.i, w.turned);
        heads_backward<T, LANES>(g, at, w, angle, (const T*)g.q_grad + at.row * g.gq_row, g.gq_head,
                                 (const T*)g.q + at.row * g.q_row, g.q_head, (T*)g.q_out + at.row * g.q_heads * g.d, g.q_heads,
                                 (const T*)g.q_weight, wq, dq);
        heads_backward<T, LANES>(g, at, w, angle, (const T*)g.k_grad + at.row * g.gk_row, g.gk_head,
                                 (const T*)g.k + at.row * g.k_row, g.k_head, (T*)g.k_out + at.row * g.k_heads * g.d, g.k_heads,
                                 (const T*)g.k_weight, wk, dk);
    }
    if (!g.partial) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        sums[0][threadIdx.x][j] = dq.u[j], sums[0][threadIdx.x][4 + j] = dq.v[j];
        sums[1][threadIdx.x][j] = dk.u[j], sums[1][threadIdx.x][4 + j] = dk.v[j];
    }
    __syncthreads();
    constexpr int kColumns = 8 * LANES;  // (up to 128: with both weights one column to a thread)
    for (int at = threadIdx.x; at < 2 * kColumns; at += 256) {
        const int which = at / kColumns, column = at % kColumns;
        float s = 0;
        for (int n = 0; n < 256 / LANES; ++n) s += sums[which][n * LANES + column / 8][column % 8];
        g.partial[((int64_t)blockIdx.x * 2 + which) * kColumns + column] = s;
    }
}

// Adds up the blocks' rows for 16 columns, in order within each of 64 parts and then over the parts.
template <typename T>
__global__ __launch_bounds__(1024) void weight_gradient(Args g, int lanes, int blocks, T* dq, T* dk) {
    __shared__ float sums[64][16];
    const int columns = 8 * lanes, at = blockIdx.x * 16 + (threadIdx.x & 15), part = threadIdx.x >> 4;
    float s = 0;
#pragma unroll 8
    for (int n = part; n < blocks; n += 64) s += g.partial[(int64_t)n * 2 * columns + at];
    sums[part][threadIdx.x & 15] = s;
    __syncthreads();
    if (part) return;
    s = 0;
#pragma unroll
    for (int n = 0; n < 64; ++n) s += sums[n][threadIdx.x];
    const int which = at / columns, column = at % columns;
    T* out = which ? dk : dq;
    if (!out || 8 * (column / 8) >= g.d) return;
    const Where w(g, column / 8);
    out[(column % 8 < 4 ? w.a : w.b) + column % 4] = (T)s;
}

}  // namespace qk_rotary
#endif
