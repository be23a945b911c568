// Device code of the norm of queries and keys and their rotation by position.
//
// A head x of d elements becomes y = w x / sqrt(mean(x^2) + eps) (or stays, without w), and of y the first r elements
// turn in pairs: (u, v) -> (u c - v s, v c + u s) with cosine and sine from the row of a table that the node's position
// names. Pairs are elements i and i + r / 2, or 2 i and 2 i + 1 (interleaved).
//
// A head belongs to 8 (a power of two up to 16) neighbouring lanes with eight elements each, chosen so that both partners
// of a pair are in one lane: two quads that lie r / 2 apart, or one behind the other where pairs are neighbours or past
// the r turned elements. So the only thing that passes between lanes is the sum of squares. The kernels are bound by
// memory: every head is read once and written once, the table's rows come from L2.
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
    int64_t q_row, q_head, k_row, k_head, v_row, v_head;
    int64_t gq_row, gq_head, gk_row, gk_head;       // strides of the outputs' gradients
    int64_t ko_row, ko_head, vo_row, vo_head;       // strides of k_out, v_out
    int64_t table_rows, slots_end;
    int64_t units;  // heads of all rows
    int q_heads, k_heads, d, rotary, interleaved, lanes;
    float eps;
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

template <typename T>
__device__ __forceinline__ Eight load(const T* row, Where w) {
    const auto a = *(const typename Quad<T>::type*)(row + w.a), b = *(const typename Quad<T>::type*)(row + w.b);
    Eight x;
#pragma unroll
    for (int j = 0; j < 4; ++j) x.u[j] = (float)a[j], x.v[j] = (float)b[j];
    return x;
}

template <typename T>
__device__ __forceinline__ void store(T* row, Where w, const Eight& x) {
    float4_t a, b;
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = x.u[j], b[j] = x.v[j];
    *(typename Quad<T>::type*)(row + w.a) = __builtin_convertvector(a, typename Quad<T>::type);
    *(typename Quad<T>::type*)(row + w.b) = __builtin_convertvector(b, typename Quad<T>::type);
}

// Turns the lane's four pairs by the angles of the row, or back.
__device__ __forceinline__ void turn(Eight& x, const Args& g, const float* table, int i, bool inside, float sign) {
    float4_t c = NAN, s = NAN;  // (a position that the table does not have)
    if (inside) {
        c = *(const float4_t*)(table + 4 * i);
        s = *(const float4_t*)(table + g.rotary / 2 + 4 * i);
    }
    if (g.interleaved) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float* p = j < 2 ? x.u + 2 * j : x.v + 2 * j - 4;
            const float a = p[0], b = p[1];
            p[0] = a * c[j] - sign * b * s[j];
            p[1] = b * c[j] + sign * a * s[j];
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

// The sum over the lanes of a head.
__device__ __forceinline__ float head_sum(float x, int lanes) {
    for (int m = 1; m < lanes; m <<= 1) x += __shfl_xor(x, m);
    return x;
}

__device__ __forceinline__ float squares(const Eight& x) {
    float s = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) s = fmaf(x.u[j], x.u[j], fmaf(x.v[j], x.v[j], s));
    return s;
}

// One head to a group of lanes. APPEND: keys go to the row of the cache that slots[] names, values as they are beside
// them; rows that the cache does not have are left out.
template <typename T, bool APPEND>
__global__ __launch_bounds__(256) void forward(Args g) {
    const int64_t unit = ((int64_t)blockIdx.x * 256 + threadIdx.x) / g.lanes;
    const int i = threadIdx.x & (g.lanes - 1), heads = g.q_heads + (APPEND ? 2 : 1) * g.k_heads;
    const bool live = unit < g.units && 8 * i < g.d;
    const int64_t row = min(unit, g.units - 1) / heads;
    const int h = (int)(min(unit, g.units - 1) - row * heads);
    const bool is_q = h < g.q_heads, is_v = h >= g.q_heads + g.k_heads;
    const int kh = is_q ? 0 : h - g.q_heads - (is_v ? g.k_heads : 0);
    const T* from = is_q ? (const T*)g.q + row * g.q_row + h * g.q_head
                         : is_v ? (const T*)g.v + row * g.v_row + kh * g.v_head : (const T*)g.k + row * g.k_row + kh * g.k_head;
    const T* weight = (const T*)(is_q ? g.q_weight : is_v ? nullptr : g.k_weight);
    Where w(g, i);
    Eight x = {};
    if (live) x = load<T>(from, w);
    const float mean = head_sum(squares(x), g.lanes) / g.d;
    if (!live) return;
    if (weight) {
        const float by = 1.0f / sqrtf(mean + g.eps);
        const Eight y = load<T>(weight, w);
#pragma unroll
        for (int j = 0; j < 4; ++j) x.u[j] *= by * y.u[j], x.v[j] *= by * y.v[j];
    }
    if (w.turned && !is_v) {
        const int64_t at = g.positions[row];
        turn(x, g, g.table + at * g.rotary, i, at >= 0 && at < g.table_rows, 1.0f);
    }
    if (is_q) {
        store<T>((T*)g.q_out + (row * g.q_heads + h) * g.d, w, x);
        return;
    }
    int64_t to = row;
    if (APPEND) {
        to = g.slots[row];
        if (to < 0 || to >= g.slots_end) return;
    }
    store<T>(is_v ? (T*)g.v_out + to * g.vo_row + kh * g.vo_head : (T*)g.k_out + to * g.ko_row + kh * g.ko_head, w, x);
}

// Gradients: turned back, gy = w-weighted; with n = x / rms, dx = (gy w - n mean(gy w n)) / rms, dw = sum gy n. A group of
// lanes walks heads at the distance of the grid; its sums of dw go, per block, to a row of `partial`, which
// weight_gradient adds up in order.
template <typename T>
__global__ __launch_bounds__(256) void backward(Args g) {
    __shared__ float sums[2][256][8];
    const int i = threadIdx.x & (g.lanes - 1), heads = g.q_heads + g.k_heads;
    const bool holds = 8 * i < g.d;
    Where w(g, i);
    Eight dq = {}, dk = {}, wq = {}, wk = {};
    if (holds && g.q_weight) wq = load<T>((const T*)g.q_weight, w);
    if (holds && g.k_weight) wk = load<T>((const T*)g.k_weight, w);
    const int64_t first = ((int64_t)blockIdx.x * 256 + threadIdx.x) / g.lanes, step = (int64_t)gridDim.x * 256 / g.lanes;
    for (int64_t base = first - threadIdx.x / g.lanes; base < g.units; base += step) {
        const int64_t unit = base + threadIdx.x / g.lanes, row = min(unit, g.units - 1) / heads;
        const bool live = holds && unit < g.units;
        const int h = (int)(min(unit, g.units - 1) - row * heads);
        const bool is_q = h < g.q_heads, normed = is_q ? g.q_weight != nullptr : g.k_weight != nullptr;
        const int kh = h - g.q_heads;
        Eight x = {}, y = {};
        if (live) {
            y = load<T>(is_q ? (const T*)g.q_grad + row * g.gq_row + h * g.gq_head
                             : (const T*)g.k_grad + row * g.gk_row + kh * g.gk_head, w);
            if (normed)
                x = load<T>(is_q ? (const T*)g.q + row * g.q_row + h * g.q_head
                                 : (const T*)g.k + row * g.k_row + kh * g.k_head, w);
            if (w.turned) {
                const int64_t at = g.positions[row];
                turn(y, g, g.table + at * g.rotary, i, at >= 0 && at < g.table_rows, -1.0f);
            }
        }
        const float by = 1.0f / sqrtf(head_sum(squares(x), g.lanes) / g.d + g.eps);
        float along = 0;
        const Eight& wt = is_q ? wq : wk;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x.u[j] *= by, x.v[j] *= by;
            along = fmaf(y.u[j] * wt.u[j], x.u[j], fmaf(y.v[j] * wt.v[j], x.v[j], along));
        }
        along = head_sum(along, g.lanes) / g.d;
        if (!live) continue;
        if (normed) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float du = y.u[j] * x.u[j], dv = y.v[j] * x.v[j];
                if (is_q) dq.u[j] += du, dq.v[j] += dv;
                else dk.u[j] += du, dk.v[j] += dv;
                y.u[j] = by * (y.u[j] * wt.u[j] - x.u[j] * along);
                y.v[j] = by * (y.v[j] * wt.v[j] - x.v[j] * along);
            }
        }
        store<T>(is_q ? (T*)g.q_out + (row * g.q_heads + h) * g.d : (T*)g.k_out + (row * g.k_heads + kh) * g.d, w, y);
    }
    if (!g.partial) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        sums[0][threadIdx.x][j] = dq.u[j], sums[0][threadIdx.x][4 + j] = dq.v[j];
        sums[1][threadIdx.x][j] = dk.u[j], sums[1][threadIdx.x][4 + j] = dk.v[j];
    }
    __syncthreads();
    const int columns = 8 * g.lanes;  // (up to 128: with both weights one column to a thread)
    for (int at = threadIdx.x; at < 2 * columns; at += 256) {
        const int which = at / columns, column = at % columns;
        float s = 0;
        for (int n = 0; n < 256 / g.lanes; ++n) s += sums[which][n * g.lanes + column / 8][column % 8];
        g.partial[((int64_t)blockIdx.x * 2 + which) * columns + column] = s;
    }
}

// Adds up the blocks' rows, in order within each of 16 parts and then over the parts.
template <typename T>
__global__ __launch_bounds__(1024) void weight_gradient(Args g, int blocks, T* dq, T* dk) {
    __shared__ float sums[16][64];
    const int columns = 8 * g.lanes, at = blockIdx.x * 64 + (threadIdx.x & 63), part = threadIdx.x >> 6;
    float s = 0;
    if (at < 2 * columns)
        for (int n = part; n < blocks; n += 16) s += g.partial[(int64_t)n * 2 * columns + at];
    sums[part][threadIdx.x & 63] = s;
    __syncthreads();
    if (part || at >= 2 * columns) return;
    s = 0;
    for (int n = 0; n < 16; ++n) s += sums[n][threadIdx.x];
    const int which = at / columns, column = at % columns;
    T* out = which ? dk : dq;
    if (!out || 8 * (column / 8) >= g.d) return;
    const Where w(g, column / 8);
    out[(column % 8 < 4 ? w.a : w.b) + column % 4] = (T)s;
}

}  // namespace qk_rotary
#endif
