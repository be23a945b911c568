// Device code of attention among the rows of segments (packed_attention.hip has the launches).
//
// Row i of a query segment sees the keys lo(i) <= j < hi(i) of its key segment; with scores s_ij = c q_i.k_j it returns
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(s_ij - lse_i),  lse_i = log sum_j exp(s_ij)
//
// and, for a gradient g of o,  dv_j = sum_i p_ij g_i,  ds_ij = p_ij (g_i.v_j - delta_i) with delta_i = g_i.o_i,
// dq_i = c sum_j ds_ij k_j,  dk_j = c sum_i ds_ij q_i, the last two sums over the query heads that share a key head too.
// Scores, p, ds and all sums are held in 32 bits; where operands have 16, p and ds are rounded to their type as
// operands of the second products (the products themselves are exact in 32 bits), which costs an error of the size of
// the output's own rounding and halves the work of these products, which bound the tiles of rows (p in the form for few queries,
// bound by memory, and in walks of few keys has two parts instead). delta would add a third such error where rows see few keys, were it taken from the rounded
// output: a pass that will be differentiated keeps what the rounding took off beside it (`rest`, 16 bits).
//
// Layout of the products. All of them run on the 32x32 matrix instructions with the *transposed* result in registers:
// S^T = K Q^T puts query i in lane i of either half of a wave and 16 keys in its registers (row 8 (r / 4) + 4 half +
// r % 4 of the tile in register r), so that a row's maximum and sum are sums over a lane's own registers and one
// exchange between the halves. The order in which a product sums over keys is free, so registers of P^T serve as they
// are as the second operand of O^T = V^T P^T if V's rows are read in the order of the registers: no lane ever needs
// another lane's p. V^T comes from LDS through the transposing reads (16 bit) or four-byte reads (32 bit).
// dQ^T = K^T dS^T works the same way, and so do dV^T = G^T P and dK^T = Q^T dS with the keys in the lanes.
//
// Rows are packed without regard to segments: a block takes 128 consecutive rows (64 where there are few blocks, SPLIT: two
// waves to 32 rows, with every other group of 32 keys each), reads the keys from the first that its
// first row sees to the last that its last row sees, and masks by each row's own bounds. Small segments (molecules)
// share a tile that way instead of leaving most of it idle: 512 molecules of 9 to 61 atoms fill 110 tiles.
//
// What a mask hides has no influence, whatever it holds: hidden scores are replaced before the maximum, hidden p and ds
// are set to zero. A product still multiplies that zero with the hidden row, which is no zero if that row holds an
// infinity or NaN; such a product leaves NaN in the sums. So a block with a result that is not finite, for whatever reason,
// walks its tiles a second time (Pass), with the infinities and NaN of the rows that its lanes share taken out of the products
// and counted for each lane by products of their own. Results that were finite stay, and one that is finite now has the
// bits that it has where hidden rows are finite. A causal sequence of 4 000 rows, 8 / 2 heads of 64, bf16: forward 45 us, with an
// infinity among the values 159; gradients 194, with one in the output's gradient 1 040 (fp16 194 and 710). Where all is
// finite it costs a barrier at the end: 512 molecules, float32, training step 132.7 and 133.5 us, large launches within 1 %.
#ifndef OEQ_PACKED_ATTENTION_H
#define OEQ_PACKED_ATTENTION_H

#include <hip/hip_runtime.h>

#include <climits>
#include <cstdint>
#include <type_traits>

namespace packed_attention {

// Rows and heads are strided, a head's elements are contiguous; strides in elements. Gradients and outputs are
// contiguous [rows, heads, d]. lse (log2 of the sum, see below) and delta are [q_heads, stat_stride].
struct Args {
    const void *q, *k, *v, *out, *out_rest, *grad;
    void *o, *rest, *dq, *dk, *dv;
    float *lse, *delta;
    const int64_t *q_ptr, *k_ptr, *k_len;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, g_row, g_head, stat_stride;
    int segments, nq, nk, hq, hk, d, causal, tiles, split;
    float scale_log2;  // c * log2(e): the kernels work with powers of two
    const int *q_order, *k_order;  // tiles by the length of their walks, or NULL
    int parts;  // the form for few queries: shares of a row's keys, and their results
    float* partial;
    float* lifts;  // what the queries' gradient lifted ds by in each tile (see lifted_operands): [q_heads, q_tiles]
    int q_tiles;
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

// A fragment is 16 bytes of a row: E elements, the operand of a product over 2 E elements (E in either half of a wave).
// Powers of two that p and ds carry while they are operands, so that small ones keep their bits (v_exp_f32 knows no
// numbers below 2^-126, and 16-bit floats of eleven bits end at 2^-24, a weight among 10^7 equal ones); they leave the
// sums at the end. In the forward pass p reaches 2^8 before that (its maximum is an older one), in the gradients 1.
// ds of eleven bits has no fixed power of two: its size is that of the output's gradient, which may be anything that the
// caller's scale of the loss makes of it (see lifted_operands).
template <typename T>
struct Types;
template <>
struct Types<float> {
    typedef float4_t frag;
    typedef float4_t quad;
    static constexpr int kForward = 0, kP = 40, kDs = 40;
};
template <>
struct Types<_Float16> {
    typedef half8_t frag;
    typedef half4_t quad;
    static constexpr int kForward = 7, kP = 12, kDs = 60;  // (kDs: before any is seen)
};
template <>
struct Types<__bf16> {
    typedef bf8_t frag;
    typedef bf4_t quad;
    static constexpr int kForward = 0, kP = 40, kDs = 40;
};
template <typename T>
constexpr bool kLifted = Types<T>::kForward > 0;  // elements of eleven bits
template <int N>
constexpr float power = N > 0 ? (float)(1ull << (N > 0 ? N : 0)) : 1.0f / (float)(1ull << (N < 0 ? -N : 0));

// 2^(x + n), pn = 2^n. Where results keep 24 bits the sum would cost some of x's: x is raised only where it is large enough not
// to lose any, else the result is.
template <typename T>
__device__ __forceinline__ float raised(float x, float n, float pn) {
    if constexpr (sizeof(T) == 2) return __builtin_amdgcn_exp2f(x + n);
    const bool low = x < -100.0f;
    return __builtin_amdgcn_exp2f(low ? x + n : x) * (low ? 1.0f : pn);
}

__device__ __forceinline__ float16_t mma(float4_t a, float4_t b, float16_t c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ float16_t mma(half8_t a, half8_t b, float16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float16_t mma(bf8_t a, bf8_t b, float16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// The same quantity of both halves of a wave: lanes l and l + 32.
__device__ __forceinline__ float max_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) x += __shfl_xor(x, m);
    return sum_halves(x);
}
__device__ __forceinline__ int wave_min(int x) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) x = min(x, __shfl_xor(x, m));
    return x;
}
__device__ __forceinline__ float wave_least(float x) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) x = fminf(x, __shfl_xor(x, m));
    return x;
}
__device__ __forceinline__ int wave_max(int x) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) x = max(x, __shfl_xor(x, m));
    return x;
}
__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }
// Its bits without the sign: from 0x7f800000, an infinity, on it is not finite. (Compared as a number in the scalar unit's
// registers where many of them are asked for at a time.)
__device__ __forceinline__ unsigned magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }
// x times a factor that may have come out as zero: an infinity stays one.
__device__ __forceinline__ float scaled(float x, float by) { return finite(x) ? x * by : x; }

// ---------------------------------------------------------------------------
// tiles in LDS
// ---------------------------------------------------------------------------

// Rows of DP elements (96: in places of 128, of which the products leave out the last quarter); 16-byte chunk c of row r
// lies at place c ^ swizzle(r) of the row. LDS has 64 banks, 256 bytes: a
// 16-byte read meets them with the same chunk of 16 consecutive rows, a transposing read with four neighbouring chunks of
// four rows that begin at a multiple of four. Either way the 16 chunks have to lie in different places modulo 16, so the
// rows that share 256 bytes need no swizzle among them, the next bits of the row choose among the groups of four chunks
// and the ones after that within a group. (With the row's bits in order, good for the first kind alone, the forward kernel
// spent 59 % of its clocks in LDS on conflicts.)
template <typename T, int DP, int ROWS, int WAVES = 4>
struct Tile {
    static constexpr int kRowBytes = (DP == 96 ? 128 : DP) * (int)sizeof(T);
    static constexpr int kChunks = kRowBytes / 16;
    static constexpr int kBytes = ROWS * kRowBytes;
    static constexpr int kFrags = DP * (int)sizeof(T) / 32;
    typedef typename Types<T>::frag frag;

    static __device__ __forceinline__ int swizzle(int r) {
        return kChunks >= 16 ? ((r & 3) << 2 | (r >> 2 & 3)) : kChunks == 8 ? ((r >> 1 & 1) << 2 | (r >> 2 & 3)) : (r >> 2 & 3);
    }

    // Where the lanes of a wave find their part of a tile, relative to its first row: 1 KB an instruction. Instructions whose
    // rows lie 16 apart have the same swizzle and are a stride apart (which is added where they are issued: kept in
    // registers, the sums take what the products need). Chunks past the head's end are placed where the reads' own bounds
    // leave them out.
    static constexpr int kRowsPer = 64 / kChunks, kEach = kBytes / 1024 / WAVES;
    static constexpr int kApart = WAVES * kRowsPer, kPlaces = kApart >= 16 ? 1 : kEach < 16 / kApart ? kEach : 16 / kApart;
    struct Places {
        int at[kPlaces];
        __device__ __forceinline__ Places(int row_bytes, int chunks, int wave, int lane) {
            static_assert(kBytes % (1024 * WAVES) == 0, "the waves share a tile");
#pragma unroll
            for (int i = 0; i < kPlaces; ++i) {
                const int r = (i * WAVES + wave) * kRowsPer + lane / kChunks, c = (lane % kChunks) ^ swizzle(r);
                at[i] = c < chunks ? r * row_bytes + c * 16 : INT_MAX;
            }
        }
    };

    // Requests the tile from row `first` on, straight into LDS. `base` is the head's first row. Nothing is read past the
    // last row: bounds go with the request, and what lies outside them arrives as zeros.
    static __device__ __forceinline__ void request(char* lds, const char* base, int row_bytes, const Places& places, int first,
                                                   int rows, int chunks, int wave) {
        const int64_t left = (int64_t)(rows - 1 - first) * row_bytes + chunks * 16;
        const auto from = __builtin_amdgcn_make_buffer_rsrc((void*)(base + (int64_t)first * row_bytes), 0,
                                                            (int)min(left, (int64_t)INT_MAX - 16), 0x00020000);
        int stride = kPlaces * kApart * row_bytes;
        asm volatile("" : "+s"(stride));  // (not to be added up outside the loop)
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lptr_t)(lds + (i * WAVES + wave) * 1024), 16,
                                                     (int)((unsigned)places.at[i % kPlaces] + i / kPlaces * (unsigned)stride), 0, 0, 0);
    }

    // Fragment f of row r: elements (2 f + half) E ... of it.
    static __device__ __forceinline__ frag row(const char* lds, int r, int f, int half) {
        return *(const frag*)(lds + r * kRowBytes + (((2 * f + half) ^ swizzle(r)) << 4));
    }
};

// Fragment of the transposed tile for the summation over its rows: lane l holds column 32 t + l % 32 of the rows that
// registers [E f, E f + E) of a result with these rows belong to; `first` is the result's first row in the tile.
template <typename T, int DP, int ROWS>
__device__ __forceinline__ typename Types<T>::frag column_of(const char* lds, int first, int f, int t, int lane) {
    typedef Tile<T, DP, ROWS> L;
    typename Types<T>::frag x;
    if constexpr (sizeof(T) == 2) {
        // a transposing read gives each of 16 lanes four rows of its column out of the 4 x 16 block whose rows the lanes
        // address by quarters
        const int l = lane & 15, c = 4 * t + 2 * ((lane >> 4) & 1) + ((l & 3) >> 1);
        union {
            short4_t q[2];
            typename Types<T>::frag f;
        } u;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const int r = first + 16 * f + 8 * g + 4 * (lane >> 5) + (l >> 2);
            u.q[g] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (ltr_t)(lds + r * L::kRowBytes + ((c ^ L::swizzle(r)) << 4) + ((l & 1) << 3)));
        }
        x = u.f;
    } else {
        const int d = 32 * t + (lane & 31);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = first + 8 * f + 4 * (lane >> 5) + j;
            x[j] = *(const float*)(lds + r * L::kRowBytes + (((d >> 2) ^ L::swizzle(r)) << 4) + ((d & 3) << 2));
        }
    }
    return x;
}

// Registers [E f, E f + E) of a result as an operand.
template <typename T>
__device__ __forceinline__ typename Types<T>::frag operand(const float16_t& s, int f) {
    typename Types<T>::frag x;
    if constexpr (sizeof(T) == 2) {
        float8_t w;
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = s[8 * f + j];
        x = __builtin_convertvector(w, typename Types<T>::frag);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = s[4 * f + j];
    }
    return x;
}

// What the rounding of an operand of 16 bits took off.
template <typename T>
__device__ __forceinline__ typename Types<T>::frag rest_of(const float16_t& s, typename Types<T>::frag x, int f) {
    float8_t w;
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = s[8 * f + j] - (float)x[j];
    return __builtin_convertvector(w, typename Types<T>::frag);
}

// ds of eleven bits as operands. Every lane carries it at a power of two of its own: 2^kDs until it has seen one, less
// where one would pass 2, so that the largest is about 2^-4. Terms then keep their bits, or are off by 2^-21 of the largest
// seen, whatever the size of the output's gradient, and none overflows (gradients of size 1e-4 at 4 096 keys without that:
// an error of 5 %, not 0.7). `lowered` is called with what changes that power of two. The operands' own bits tell: one of their
// exponents has its highest bit set from 2 on. (Only in the queries' gradient, which 9 sequences, heads of 128, take 219
// us for instead of 204. The keys' one, with one wave to a SIMD, took 450 instead of 390 that way; it goes by what the
// queries' found, one power of two for a block, and takes no longer.)
template <typename T, typename L>
__device__ __forceinline__ void lifted_operands(float16_t& x, typename Types<T>::frag (&d)[2], L lowered) {
#pragma unroll
    for (int f = 0; f < 2; ++f) d[f] = operand<T>(x, f);
    const uint4_t a = __builtin_bit_cast(uint4_t, d[0]), b = __builtin_bit_cast(uint4_t, d[1]);
    const unsigned any = a[0] | a[1] | a[2] | a[3] | b[0] | b[1] | b[2] | b[3];
    if (!__any(any & 0x40004000u)) return;
    float top = 0;
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(x[r]));
    top = max_halves(top);
    const int n = top >= 2.0f && finite(top) ? __builtin_amdgcn_frexp_expf(top) + 3 : 0;  // (an infinity stays)
    const float by = __builtin_amdgcn_ldexpf(1.0f, -n);
    lowered(by);
    x *= by;
#pragma unroll
    for (int f = 0; f < 2; ++f) d[f] = operand<T>(x, f);
}

// Fragments of a lane's row straight from memory; `chunks` of 16 bytes exist.
template <typename T, int FRAGS>
__device__ __forceinline__ void load_row(typename Types<T>::frag (&x)[FRAGS], const char* row, int chunks, int half) {
#pragma unroll
    for (int f = 0; f < FRAGS; ++f) {
        x[f] = 0;
        if (2 * f + half < chunks) x[f] = *(const typename Types<T>::frag*)(row + (2 * f + half) * 16);
    }
}

// A lane's column of a result (the elements 32 t + 8 (r / 4) + 4 half + r % 4 of its row) times `by` to memory, and to
// `rest`, if there is one, what rounding takes off.
template <typename T, int DT>
__device__ __forceinline__ void store_row(T* row, const float16_t (&acc)[DT], float by, int d, int half, T* rest = nullptr) {
#pragma clang fp contract(off)  // (a product is rounded to 32 bits first, here and in store_part)
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int at = 32 * t + 8 * g + 4 * half;
            float4_t w;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = acc[t][4 * g + j] * by;
            const auto x = __builtin_convertvector(w, typename Types<T>::quad);
            if (at < d) *(typename Types<T>::quad*)(row + at) = x;
            if (rest && at < d)
                *(typename Types<T>::quad*)(rest + at) =
                    __builtin_convertvector(w - __builtin_convertvector(x, float4_t), typename Types<T>::quad);
        }
}

// ---------------------------------------------------------------------------
// bounds
// ---------------------------------------------------------------------------

struct Bounds {
    int lo, hi;  // what a row sees: lo <= other < hi
};

__device__ __forceinline__ int clamped(int64_t x, int most) { return (int)(x < 0 ? 0 : x > most ? most : x); }

// The last segment that begins at or before a lane's row (-1: none), out of ascending starts ptr[0 .. segments]. Rows of
// a wave's lanes are near each other: the wave narrows the range for its least row by 64 pivots at a time, then every
// lane looks for its own among the next 64 starts (two or three dependent reads for any number of segments up to 4096).
__device__ __forceinline__ int find_segment(const int64_t* ptr, int segments, int row, int lane) {
    const int least = wave_min(row);
    int base = 0, n = segments + 1;
    while (n > 64) {
        const int step = (n + 63) / 64;
        const bool le = lane * step < n && ptr[base + min(lane * step, n - 1)] <= least;
        const int count = __popcll(__ballot(le));
        const int skip = max(count - 1, 0) * step;
        n = min(step, n - skip);
        base += skip;
    }
    int seg = base - 1;
    for (;;) {
        const int64_t start = ptr[min(base + lane, segments)];
        const int window = min(64, segments + 1 - base);
        const int mine = start > (int64_t)INT_MAX ? INT_MAX : start < (int64_t)INT_MIN ? INT_MIN : (int)start;
        int count = 0;  // how many of the window's starts are at or before the row
#pragma unroll
        for (int step = 32; step >= 1; step >>= 1) {
            const int v = __shfl(mine, count + step - 1);
            if (count + step <= window && v <= row) count += step;
        }
        const int last = __shfl(mine, min(63, window - 1));
        if (count == 63 && window == 64 && last <= row) count = 64;
        if (count > 0) seg = base + count - 1;
        if (window < 64 || !__any(count == 64)) break;
        base += 63;
    }
    return seg;
}

// Keys that query row i sees. Causal: the segments' last rows stand side by side, and a row sees up to its own place.
__device__ __forceinline__ Bounds keys_of(const Args& a, int i, int lane) {
    const int s = find_segment(a.q_ptr, a.segments, i, lane);
    Bounds b = {0, 0};
    if (s >= 0 && s < a.segments) {
        const int q1 = clamped(a.q_ptr[s + 1], a.nq);  // (cut off at the tensor's end, for the diagonal too)
        const int k0 = clamped(a.k_ptr[s], a.nk), k1 = clamped(a.k_ptr[s + 1], a.nk);
        int len = max(k1 - k0, 0);
        if (a.k_len) len = min(len, clamped(a.k_len[s], INT_MAX));
        if (a.causal) len = min(len, max(0, len - (q1 - 1 - i)));
        if (i < q1 && len > 0) b = {k0, k0 + len};
    }
    return b;
}

// Query rows that see key j.
__device__ __forceinline__ Bounds queries_of(const Args& a, int j, int lane) {
    const int s = find_segment(a.k_ptr, a.segments, j, lane);
    Bounds b = {0, 0};
    if (s >= 0 && s < a.segments) {
        const int k0 = clamped(a.k_ptr[s], a.nk), k1 = clamped(a.k_ptr[s + 1], a.nk);
        int len = max(k1 - k0, 0);
        if (a.k_len) len = min(len, clamped(a.k_len[s], INT_MAX));
        const int q0 = clamped(a.q_ptr[s], a.nq), q1 = clamped(a.q_ptr[s + 1], a.nq);
        int first = q0;
        if (a.causal) first = max(q0, q1 - len + (j - k0));
        if (j >= k0 && j < k0 + len && first < q1) b = {first, q1};
    }
    return b;
}

// What a wave needs of its lanes' bounds: the union it walks and the intersection in which nothing is hidden.
struct Walk {
    int lo, hi, full_lo, full_hi;
    __device__ __forceinline__ explicit Walk(Bounds b) {
        const bool any = b.lo < b.hi;
        lo = __builtin_amdgcn_readfirstlane(wave_min(any ? b.lo : INT_MAX));
        hi = __builtin_amdgcn_readfirstlane(wave_max(any ? b.hi : 0));
        full_lo = __builtin_amdgcn_readfirstlane(wave_max(any ? b.lo : INT_MAX));
        full_hi = __builtin_amdgcn_readfirstlane(wave_min(any ? b.hi : 0));
    }
    __device__ __forceinline__ bool needs(int first, int n) const { return first < hi && first + n > lo; }
    __device__ __forceinline__ bool whole(int first, int n) const { return first >= full_lo && first + n <= full_hi; }
};

struct Shared {
    int range[8], bad[2];  // the waves' unions; whether a pass left results that are not finite (any_of_block)
};

// The union over the block's four waves.
__device__ __forceinline__ Bounds block_range(const Walk& w, Shared& shared, int wave, int lane) {
    if (lane == 0) {
        shared.range[2 * wave] = w.lo;
        shared.range[2 * wave + 1] = w.hi;
    }
    if (threadIdx.x < 2) shared.bad[threadIdx.x] = 0;
    __syncthreads();
    Bounds b = {shared.range[0], shared.range[1]};
#pragma unroll
    for (int i = 1; i < 4; ++i) {
        b.lo = min(b.lo, shared.range[2 * i]);
        b.hi = max(b.hi, shared.range[2 * i + 1]);
    }
    b.lo = __builtin_amdgcn_readfirstlane(b.lo);
    b.hi = __builtin_amdgcn_readfirstlane(b.hi);
    return b;
}

// Block -> (tile, head): blocks that an XCD runs (every eighth) share key heads, so that its L2 holds few of them at a
// time; tiles run in the order of `order` (by the length of their walks), or where there is none as they are, causal query
// tiles from the last on.
__device__ __forceinline__ void place(const Args& a, int heads, const int* order, bool reversed, int& tile, int& head) {
    const int id = blockIdx.x, at = id % heads;
    tile = id / heads;
    if (order)
        tile = __builtin_amdgcn_readfirstlane(order[tile]);
    else if (reversed)
        tile = a.tiles - 1 - tile;
    head = heads % 8 == 0 ? (at % 8) * (heads / 8) + at / 8 : at;
}

// Blocks of four waves on a compute unit: 256 registers a lane for two, 512 where a head of 128 four-byte elements needs
// more for its row alone.
template <typename T, int DP>
constexpr int blocks_per_unit() { return sizeof(T) * DP > 256 ? 1 : 2; }

// Small heads go with small segments: there each wave leaves out the groups of 32 keys that none of its rows sees. (512
// molecules of 9 to 61 atoms: a wave's 32 rows see some 90 keys, their block's 128 rows 180.)
template <typename T, int DP>
constexpr bool kSparse = sizeof(T) == 4 && DP == 32;

// A lane's number, or the same hidden from the compiler, which then computes places in LDS anew instead of keeping them in
// registers. In key_gradient: kSparse, 192 registers a lane or 138 (168 with the passes after the first), a wave more to a SIMD: 512 molecules, float32, all
// gradients 139 / 132 us, 2 048 460 / 424, but a segment of 3 000 rows 260 / 266. (bf16 heads of 32, whose products are 8 times as
// fast: 2 048 molecules 185 / 177, a segment of 3 000 rows 64 / 73, so they keep them.)
template <typename X>
__device__ __forceinline__ X anew(X x) {
    asm volatile("" : "+v"(x));
    return x;
}
struct Lane {
    int at, half;
    template <bool ANEW>
    static __device__ __forceinline__ Lane of(int lane, int half) {
        if constexpr (ANEW) lane = anew(lane);
        return {lane, ANEW ? lane >> 5 : half};
    }
};

template <typename T, int DP>
constexpr bool kFenced = sizeof(T) == 2 && DP >= 96;  // key_gradient: one wave to a SIMD, or nearly, see there

template <typename T, int DP, int WHAT>
constexpr int key_blocks_per_unit() { return sizeof(T) * DP >= (WHAT == 3 ? 256 : 384) ? 1 : 2; }

// Keys of a tile: 16 KB, or 8 KB where a block's walk over small segments should have few steps (each waits for its tile).
template <typename T, int DP>
constexpr int tile_rows() { return sizeof(T) == 2 || DP == 32 ? 64 : 32; }

// Everything that was requested so far has come, and the compiler knows: a row that is loaded before a loop would else be
// waited for inside it, at its first use, together with what the loop has requested since.
__device__ __forceinline__ void settle() { __builtin_amdgcn_s_waitcnt(0x0f70); }  // vmcnt(0)

__device__ __forceinline__ void arrived() {
    // what this wave requested is in LDS; then the same for the others, and all are done with the other buffer
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

template <int BYTES>
__device__ __forceinline__ void clear(char* lds) {
    for (int i = threadIdx.x * 16; i < BYTES; i += 256 * 16) *(uint4_t*)(lds + i) = 0;
}

// ---------------------------------------------------------------------------
// results that are not finite (see the beginning)
// ---------------------------------------------------------------------------

template <int DT>
__device__ __forceinline__ bool all_finite(const float16_t (&acc)[DT]) {
    float z = 0;  // 0 x is NaN where x is not finite
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) z = fmaf(acc[t][r], 0.0f, z);
    return z == 0.0f;
}

// Where a careful pass has an element that is not finite and does not know why: its sum may have been too large on the way.
__device__ __forceinline__ bool all_known(const float16_t& acc, unsigned known) {
    unsigned open = 0;
#pragma unroll
    for (int r = 0; r < 16; ++r) open |= (~(magnitude(acc[r]) - 0x7f800000u) >> 31) << r;
    return (open & ~known) == 0;
}

// store_row for 32 columns. `keep`: what is there already and finite stays.
template <typename T>
__device__ __forceinline__ void store_part(T* row, const float16_t& acc, float by, int d, int half, T* rest, bool keep) {
#pragma clang fp contract(off)
    typedef typename Types<T>::quad quad;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int at = 8 * g + 4 * half;
        if (at >= d) break;
        float4_t w;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = acc[4 * g + j] * by;
        quad x = __builtin_convertvector(w, quad), y = __builtin_convertvector(w - __builtin_convertvector(x, float4_t), quad);
        if (keep) {
            const quad was = *(const quad*)(row + at);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (finite((float)was[j])) {
                    x[j] = was[j];
                    if (rest) y[j] = rest[at + j];
                }
        }
        *(quad*)(row + at) = x;
        if (rest) *(quad*)(rest + at) = y;
        __builtin_amdgcn_sched_barrier(0);
    }
}

// Passes of a block over its tiles: the first, a second one if results are not finite, and a third if some are not for a reason
// that the second has not found in the operands: sums may have passed the largest number on the way (in 24 and 8 bits, whose
// range is that of the sums). There p and ds carry no power of two and p never passes 1.
enum Pass { kFirst, kCareful, kCarefulSmall };
template <typename T>
constexpr int kLastPass = kLifted<T> ? kCareful : kCarefulSmall;

// Whether any thread of the block says so. A barrier; every pass has a place of its own.
__device__ __forceinline__ bool any_of_block(bool bad, int& shared) {
    if (__any(bad)) shared = 1;  // (the same from every lane)
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(shared) != 0;
}

// The second and third pass of a block. They take 32 columns of the head at a time, with the scores computed anew for each, so
// that they need hardly more registers than the first. `walk(t, raise, bad)` is a walk for columns 32 t ... that stores the
// results where bad and says whether some of them are not finite for no known reason.
template <typename T, int DT, typename F>
__device__ __forceinline__ void careful_passes(int (&shared)[2], bool bad, F walk) {
    // This is a kernel's last step, and most end here: the program's own end is a jump away, in instructions that would have to
    // be fetched first (6 single rows, 32 / 8 heads of 96, 13.6 us and not 12.9).
    if (__builtin_expect(!any_of_block(bad, shared[0]), 1)) {
        asm volatile("s_endpgm" ::: "memory");
        return;
    }
#pragma unroll 1
    for (int n = kCareful; n <= kLastPass<T> && any_of_block(bad, shared[n - 1]); ++n) {
        bool still = false;
#pragma unroll 1
        for (int t = 0; t < DT; ++t) {
            if (t) __syncthreads();  // (all are done with the last walk's tiles)
            int raise = n == kCareful;
            asm volatile("" : "+s"(raise));  // (one walk for both passes)
            if (walk(t, raise, bad)) still = true;
        }
        bad = still;
    }
}

// acc += columns 32 t ... of the rows at `first`, transposed, times the weights of a result with these rows (in `two` parts or one),
// by the rows' finite elements alone. Returns whether there were others. `known`: a bit for each register whose result is not
// finite for what the operands hold, not for the size of its sum.
template <typename T, int DP, int ROWS>
__device__ __forceinline__ bool finite_product_of(const char* lds, int first, int t, int lane, const float16_t& weights, bool two,
                                                  float16_t& acc, unsigned& known) {
    unsigned left = 0;
#pragma unroll
    for (int r = 0; r < 16; ++r) left = max(left, magnitude(weights[r]));
    const float both = sum_halves(__uint_as_float(left));  // (a product sums over the weights of either half)
    if (both != both) known = ~0u;
    left = 0;
#pragma unroll
    for (int f = 0; f < (int)sizeof(T); ++f) {
        auto x = column_of<T, DP, ROWS>(lds, first, f, t, lane);
#pragma unroll
        for (int j = 0; j < 16 / (int)sizeof(T); ++j) {
            const unsigned size = magnitude((float)x[j]);
            left = max(left, size);
            x[j] = size < 0x7f800000u ? x[j] : (T)0.0f;
        }
        const auto w = operand<T>(weights, f);
        acc = mma(x, w, acc);
        if constexpr (sizeof(T) == 2)
            if (two) acc = mma(x, rest_of<T>(weights, w, f), acc);
        __builtin_amdgcn_sched_barrier(0);
    }
    return kSparse<T, DP> || __any(left >= 0x7f800000u);  // (small heads: a branch around what follows would take registers)
}

// And what the rows' other elements come to in each result whose lane sees them (rows are numbered from `number` on):
// infinities as they are, where weights are above zero (SIGNED), else NaN. A product of 1 where a lane sees a row with 1 for
// each +inf, 2^7 for -inf and 2^14 for NaN counts up to 32 of each exactly.
template <typename T, int DP, int ROWS, bool SIGNED, int BIT = 0>
__device__ __forceinline__ void add_others(const char* lds, int first, int t, int lane, int number, Bounds b, float16_t& acc,
                                           unsigned& known) {
    constexpr int E = 16 / (int)sizeof(T);
    float16_t count = 0.0f;
#pragma unroll
    for (int f = 0; f < 16 / E; ++f) {
        auto x = column_of<T, DP, ROWS>(lds, first, f, t, lane), sees = x;
#pragma unroll
        for (int j = 0; j < E; ++j) {
            const float y = (float)x[j];
            const int r = E * f + j;
            float code = y == INFINITY ? 1.0f : 0.0f;
            code = y == -INFINITY ? 128.0f : code;
            code = y != y ? 16384.0f : code;
            x[j] = (T)code;
            sees[j] = (unsigned)(number + 8 * (r / 4) + 4 * (lane >> 5) + r % 4 - b.lo) < (unsigned)(b.hi - b.lo) ? (T)1.0f : (T)0.0f;
        }
        count = mma(x, sees, count);
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int n = (int)count[r];
        float other = n & 127 ? INFINITY : 0.0f;
        if (n >> 7) other -= INFINITY;
        if (n >> 14 || !SIGNED) other = NAN;
        if (n) acc[r] += other, known |= 1u << (r + BIT);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------
//
// A wave has 32 query rows in registers (128 a block, 64 with SPLIT) and walks keys and values through two LDS buffers, the
// next tile always on its way, with running maximum and sum in the row's lane. Long walks are bound by the matrix units and
// the power they may draw: 7 segments of 500 to 8 192 rows, 32 / 8 heads of 128, bf16, causal, 1.71 ms, 1.03 PFLOP/s of visible
// pairs (a large library product 1.16, both at some 2 GHz); 9 of 200 to 4 001 rows, 16 / 4 heads, 140 us, the longest walk.
// Short ones by a block's chain of waits: 512 molecules, 8 heads of 32, float32, 33 us, of which the matrix units work 13;
// 33 crystals, 6 / 2 heads of 72, fp16, 20 us.
//
// Where a row sees few keys, each weight is a large part of its sum, and so is what its rounding to 16 bits takes off; delta has
// that error too and with it the gradients, whose errors it would raise from 1.41 times those of one rounding (ds has one, the
// result another) to above 1.5. A block that walks no more than kFewKeys keys has p in two parts as the form for few queries has. Forward,
// us, one part / two, bf16: 512 segments of 9 to 61 rows, heads of 32 14.8 / 16.7, 256 of 120, heads of 128 125 / 135, of 32 45 / 54; a
// training step on the 33 crystals 79.3 either way. For walks of up to 2 048 keys it would cost 9 sequences, heads of 128, 649 / 665,
// and take the gradients' errors from 1.44 to 1.41.
constexpr int kFewKeys = 256;

template <typename T, int DP, int SPLIT>  // (heads of 32: without the bound bf16 takes 139 registers, three waves to a SIMD)
__global__ __launch_bounds__(256, (DP == 32 && SPLIT == 1 ? 4 : blocks_per_unit<T, DP>())) void forward(Args a) {
    constexpr int BK = SPLIT == 2 ? 64 : tile_rows<T, DP>(), SUB = SPLIT == 2 || kSparse<T, DP> ? 1 : BK / 32, DT = DP / 32;
    constexpr int PF = sizeof(T) == 2 ? 2 : 4;  // fragments of 32 keys
    typedef Tile<T, DP, BK> L;
    __shared__ __align__(1024) char key0[L::kBytes], key1[L::kBytes], val0[L::kBytes], val1[L::kBytes];
    __shared__ Shared shared;
    __shared__ __align__(16) float4_t swap[SPLIT == 2 ? 512 : 1];
    __shared__ float swap_m[SPLIT == 2 ? 64 : 1], swap_l[SPLIT == 2 ? 64 : 1];
    __shared__ unsigned swap_known[SPLIT == 2 ? 128 : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    int tile, h;
    place(a, a.hq, a.q_order, a.causal, tile, h);
    const int kh = h / (a.hq / a.hk), chunks = a.d * (int)sizeof(T) / 16;
    const int rows = wave % (4 / SPLIT), part = wave / (4 / SPLIT);  // which 32 rows, and which of the groups of keys
    const int row = (tile * (4 / SPLIT) + rows) * 32 + (lane & 31), i = min(row, a.nq - 1);
    typename L::frag q[L::kFrags];
    load_row<T, L::kFrags>(q, (const char*)((const T*)a.q + i * a.q_row + h * a.q_head), chunks, half);
    if (chunks < 2 * L::kFrags) {
        clear<L::kBytes>(key0), clear<L::kBytes>(key1), clear<L::kBytes>(val0), clear<L::kBytes>(val1);
    }
    const Bounds b = keys_of(a, i, lane);
    const Walk walk(b);
    const Bounds all = block_range(walk, shared, wave, lane);
    const char* kbase = (const char*)((const T*)a.k + kh * a.k_head);
    const char* vbase = (const char*)((const T*)a.v + kh * a.v_head);
    const int krow = (int)a.k_row * (int)sizeof(T), vrow = (int)a.v_row * (int)sizeof(T);
    const typename L::Places kplaces(krow, chunks, wave, lane), vplaces(vrow, chunks, wave, lane);
    float m, l;
    unsigned known;
    const float c = a.scale_log2;
    const bool in_parts = sizeof(T) == 2 && all.hi - all.lo <= kFewKeys;
    settle();

    // Sums are scaled to another maximum only where it grew by more than 2^grow: up to 2^8 p fits every type.
    auto pass = [&](auto& acc, auto care, auto two, int t0, float grow) {
        constexpr bool CARE = decltype(care)::value, TWO = decltype(two)::value;
        constexpr int NT = CARE ? 1 : DT;
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t] = 0.0f;
        m = -INFINITY, l = 0, known = 0;
        auto products = [&](const char* kt, const char* vt, int first, int r0) {
            const Lane w = Lane::of<CARE>(lane, half);
            float16_t s[SUB];
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                s[u] = 0.0f;
#pragma unroll
                for (int f = 0; f < L::kFrags; ++f) s[u] = mma(L::row(kt, r0 + 32 * u + (w.at & 31), f, w.half), q[f], s[u]);
            }
            if (!walk.whole(first + r0, 32 * SUB)) {
                const int shift = first + r0 + 4 * half - b.lo;
                const unsigned n = b.hi - b.lo;
#pragma unroll
                for (int u = 0; u < SUB; ++u)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if ((unsigned)(shift + 32 * u + 8 * (r / 4) + r % 4) >= n) s[u][r] = -INFINITY;
            }
            float top = s[0][0];
#pragma unroll
            for (int u = 0; u < SUB; ++u)
#pragma unroll
                for (int r = 0; r < 16; ++r) top = fmaxf(top, s[u][r]);
            top = max_halves(top);
            if (__any((top - m) * c > grow)) {
                const float now = fmaxf(m, top);
                const float by = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - now) * c);
                m = now;
                l *= by;
                if constexpr (CARE) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[0][r] = scaled(acc[0][r], by);
                } else {
#pragma unroll
                    for (int t = 0; t < NT; ++t) acc[t] *= by;
                }
            }
            const float mc = m == -INFINITY ? 0.0f : m * c - Types<T>::kForward;
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    s[u][r] = __builtin_amdgcn_exp2f(fmaf(s[u][r], c, -mc));
                    l += s[u][r];
                }
                if constexpr (CARE) {
                    if (finite_product_of<T, DP, BK>(vt, r0 + 32 * u, t0, w.at, s[u], in_parts, acc[0], known))
                        add_others<T, DP, BK, true>(vt, r0 + 32 * u, t0, w.at, first + r0 + 32 * u, b, acc[0], known);
                } else {
#pragma unroll
                    for (int f = 0; f < PF; ++f) {
                        const auto p = operand<T>(s[u], f);
                        typename L::frag column[TWO ? DT : 1];
#pragma unroll
                        for (int t = 0; t < DT; ++t) {
                            column[TWO ? t : 0] = column_of<T, DP, BK>(vt, r0 + 32 * u, f, t, lane);
                            acc[t] = mma(column[TWO ? t : 0], p, acc[t]);
                        }
                        if constexpr (TWO) {
                            const auto rest = rest_of<T>(s[u], p, f);
#pragma unroll
                            for (int t = 0; t < DT; ++t) acc[t] = mma(column[t], rest, acc[t]);
                        }
                    }
                }
            }
        };
        auto step = [&](char* kt, char* vt, char* kn, char* vn, int first) {
            arrived();
            if (first + BK < all.hi) {
                L::request(kn, kbase, krow, kplaces, first + BK, all.hi, chunks, wave);
                L::request(vn, vbase, vrow, vplaces, first + BK, all.hi, chunks, wave);
            }
            if constexpr (SPLIT == 2) {
                if (walk.needs(first + 32 * part, 32)) products(kt, vt, first, 32 * part);
            } else {
#pragma unroll
                for (int r0 = 0; r0 < BK; r0 += 32 * SUB)
                    if (walk.needs(first + r0, 32 * SUB)) products(kt, vt, first, r0);
            }
        };
        if (all.lo < all.hi) {
            L::request(key0, kbase, krow, kplaces, all.lo, all.hi, chunks, wave);
            L::request(val0, vbase, vrow, vplaces, all.lo, all.hi, chunks, wave);
        }
        for (int first = all.lo; first < all.hi; first += 2 * BK) {
            step(key0, val0, key1, val1, first);
            if (first + BK < all.hi) step(key1, val1, key0, val0, first + BK);
        }
        l = sum_halves(l);
        if constexpr (SPLIT == 2) {
            // the wave with the second groups of keys hands its sums to the one with the first, 32 columns of the head at a time
            if (part && half == 0) swap_m[32 * rows + lane] = m, swap_l[32 * rows + lane] = l;
            if (CARE && part) swap_known[64 * rows + lane] = known;
            __syncthreads();
            if (CARE && !part) known |= swap_known[64 * rows + lane];
            const float other = swap_m[32 * rows + (lane & 31)], top = fmaxf(m, other);
            const float by = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - top) * c);
            const float others = other == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((other - top) * c);
            if (!part) l = l * by + swap_l[32 * rows + (lane & 31)] * others, m = top;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                if (part)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        swap[(rows * 4 + g) * 64 + lane] = float4_t{acc[t][4 * g], acc[t][4 * g + 1], acc[t][4 * g + 2], acc[t][4 * g + 3]};
                __syncthreads();
                if (!part)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float x = acc[t][4 * g + e], y = swap[(rows * 4 + g) * 64 + lane][e];
                            acc[t][4 * g + e] = CARE && !(finite(x) && finite(y)) ? scaled(x, by) + scaled(y, others) : fmaf(x, by, y * others);
                        }
                __syncthreads();
            }
        }
    };
    const bool seen = b.lo < b.hi;
    auto put_sum = [&](int i) {
        if (half == 0) a.lse[h * a.stat_stride + i] = seen ? m * c + (__builtin_amdgcn_logf(l) - Types<T>::kForward) : -INFINITY;
    };
    bool bad = row < a.nq && !part;
    {
        float16_t acc[DT];
        if (in_parts)
            pass(acc, std::false_type(), std::integral_constant<bool, sizeof(T) == 2>(), 0, 8.0f);
        else
            pass(acc, std::false_type(), std::false_type(), 0, 8.0f);
        const float by = seen ? 1.0f / l : 0.0f;
        if (bad) {
            const int64_t at = ((int64_t)i * a.hq + h) * a.d;
            store_row<T, DT>((T*)a.o + at, acc, by, a.d, half, a.rest ? (T*)a.rest + at : nullptr);
            put_sum(i);
        }
        bad = bad && !(all_finite<DT>(acc) && finite(by));
    }
    careful_passes<T, DT>(shared.bad, bad, [&](int t, int raise, bool mine) {
        float16_t acc[1];
        pass(acc, std::true_type(), std::false_type(), t, 8.0f * raise);
        const float by = seen ? 1.0f / l : 0.0f;
        if (mine) {
            const int r = anew(i);
            const int64_t at = ((int64_t)r * a.hq + h) * a.d + 32 * t;
            store_part<T>((T*)a.o + at, acc[0], by, a.d - 32 * t, half, a.rest ? (T*)a.rest + at : nullptr, !raise);
            if (raise) put_sum(r);
        }
        return mine && !all_known(acc[0], known);
    });
}

// ---------------------------------------------------------------------------
// forward, few queries to many keys
// ---------------------------------------------------------------------------
//
// A new token against its cache reads every key and value once and computes next to nothing: the work is to keep reads in
// flight on all compute units. A block has one query row, one key head and one of `parts` equal shares of the row's keys;
// the query heads that share the key head (up to 32) are the columns of the products, so that keys and values are read
// once for all of them. Each wave walks tiles of 32 keys of its own through LDS, the next one always on its way, and
// meets the others only at the end. Rows past the share's end are cut off by the reads' bounds and arrive as zeros. Shares
// of more than one block's row meet in `join`, in the order of the keys. p of 16 bits goes in two parts, itself and what its
// rounding took off, so that nothing but the output is rounded: the second products are done while memory is waited for.
// Bound by memory: a token against 65 537 keys, 32 / 8
// heads of 128, bf16, 60 us with the join (6), 4.5 TB/s of 268 MB where a copy reaches 4.7; 64 tokens against 1 to 4 096 keys
// each, 16 / 4 heads, fp16, 70 us for the same bytes; 7 tokens against up to 60 keys 7 us, about a launch.

template <typename T, int DP>
struct Few {
    typedef Tile<T, DP, 32, 1> L;
    static constexpr int kWaves = 4 * L::kBytes >= 32768 ? 2 : 4;  // (two tiles each of keys and values to a wave)
    static constexpr int kRow = DP + 4;  // floats of a partial result: sums, then the maximum (log2) and the sum of p
    // Where four sums of a wave's column lie once the tiles in LDS are done with: in the first key buffer, the upper half
    // of a 16-bit head in the first value buffer; quads are permuted by column so that columns begin in different banks.
    static __device__ __forceinline__ float4_t* sums(char* key, char* val, int wave, int column, int d) {
        constexpr int kIn = sizeof(T) == 4 ? DP : DP / 2, kQuads = kIn / 4, kMask = kQuads < 8 ? kQuads - 1 : 7;
        char* buffer = d < kIn ? key : val;
        return (float4_t*)(buffer + (((wave * 32 + column) * kQuads + ((d % kIn / 4) ^ (column & kMask))) << 4));
    }
};

constexpr int kMostParts = 256;

struct Share {
    int first, last, count;  // keys of this part; parts that have any
    __device__ __forceinline__ Share(Bounds b, int parts, int part, int grain) {
        const int n = b.hi - b.lo, each = (((n + parts - 1) / parts + grain - 1) / grain) * grain;
        count = n > 0 ? (n + each - 1) / each : 0;
        first = b.lo + (int)min((int64_t)part * each, (int64_t)n);
        last = min(first + each, b.hi);
    }
};

template <typename T, int DP>
__global__ __launch_bounds__((64 * Few<T, DP>::kWaves), (sizeof(T) * DP == 64 ? 4 : 1)) void forward_few(Args a) {
    constexpr int W = Few<T, DP>::kWaves, DT = DP / 32, PF = sizeof(T) == 2 ? 2 : 4, ROW = Few<T, DP>::kRow;
    typedef typename Few<T, DP>::L L;
    __shared__ __align__(1024) char key0[W * L::kBytes], key1[W * L::kBytes], val0[W * L::kBytes], val1[W * L::kBytes];
    __shared__ float top_of[W][32], sum_of[W][32];
    __shared__ int bad[2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int group = a.hq / a.hk, stacks = (group + 31) / 32;
    int id = blockIdx.x;
    const int part = id % a.parts;
    id /= a.parts;
    const int stack = id % stacks;
    id /= stacks;
    const int kh = id % a.hk, i = id / a.hk;
    const int heads = min(32, group - 32 * stack), h0 = kh * group + 32 * stack, column = lane & 31;
    const int chunks = a.d * (int)sizeof(T) / 16;
    const Bounds b = keys_of(a, i, lane);
    const Share mine(Bounds{__builtin_amdgcn_readfirstlane(b.lo), __builtin_amdgcn_readfirstlane(b.hi)}, a.parts, part, 32 * W);
    if (part && mine.first >= mine.last) return;
    char *kt0 = key0 + wave * L::kBytes, *kt1 = key1 + wave * L::kBytes;
    char *vt0 = val0 + wave * L::kBytes, *vt1 = val1 + wave * L::kBytes;
    auto clear_own = [&] {  // (a wave's own part of the buffers: no barrier)
        if (chunks >= L::kChunks) return;
        for (int n = lane * 16; n < L::kBytes; n += 1024)
            *(uint4_t*)(kt0 + n) = 0, *(uint4_t*)(kt1 + n) = 0, *(uint4_t*)(vt0 + n) = 0, *(uint4_t*)(vt1 + n) = 0;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    };
    clear_own();
    const char* kbase = (const char*)((const T*)a.k + kh * a.k_head);
    const char* vbase = (const char*)((const T*)a.v + kh * a.v_head);
    const int krow = (int)a.k_row * (int)sizeof(T), vrow = (int)a.v_row * (int)sizeof(T);
    const typename L::Places kplaces(krow, chunks, 0, lane), vplaces(vrow, chunks, 0, lane);
    auto request = [&](char* kt, char* vt, int first) {
        L::request(kt, kbase, krow, kplaces, first, mine.last, chunks, 0);
        L::request(vt, vbase, vrow, vplaces, first, mine.last, chunks, 0);
    };
    constexpr int kStep = 32 * W, kAhead = 2 * L::kEach;  // (requests of a tile's keys and values)
    const int start = mine.first + 32 * wave;
    if (start < mine.last) request(kt0, vt0, start);
    typename L::frag q[L::kFrags];
    const bool live = column < heads;
    load_row<T, L::kFrags>(q, (const char*)((const T*)a.q + i * a.q_row + (h0 + (live ? column : 0)) * a.q_head),
                           live ? chunks : 0, half);
    float m, l;
    unsigned known;
    const float c = a.scale_log2;

    auto pass = [&](auto& acc, auto care, int t0, float grow) {  // (see forward)
        constexpr bool CARE = decltype(care)::value;
        constexpr int NT = CARE ? 1 : DT;
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t] = 0.0f;
        m = -INFINITY, l = 0, known = 0;
        auto step = [&](char* kt, char* vt, char* kn, char* vn, int first) {
            if (first + kStep < mine.last) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // what was read from there has come
                request(kn, vn, first + kStep);
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kAhead) : "memory");
            } else {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            }
            const Lane w = Lane::of<CARE>(lane, half);
            float16_t s = 0.0f;
#pragma unroll
            for (int f = 0; f < L::kFrags; ++f) s = mma(L::row(kt, w.at & 31, f, w.half), q[f], s);
            if (first + 32 > mine.last) {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (first + 4 * half + 8 * (r / 4) + r % 4 >= mine.last) s[r] = -INFINITY;
            }
            float top = s[0];
#pragma unroll
            for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
            top = max_halves(top);
            if (__any((top - m) * c > grow)) {
                const float now = fmaxf(m, top);
                const float by = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - now) * c);
                m = now;
                l *= by;
                if constexpr (CARE) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[0][r] = scaled(acc[0][r], by);
                } else {
#pragma unroll
                    for (int t = 0; t < NT; ++t) acc[t] *= by;
                }
            }
            const float mc = m == -INFINITY ? 0.0f : m * c - Types<T>::kForward;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, -mc));
                l += s[r];
            }
            if constexpr (!CARE) {
#pragma unroll
                for (int f = 0; f < PF; ++f) {
                    const auto p = operand<T>(s, f);
                    typename L::frag column[DT];
#pragma unroll
                    for (int t = 0; t < DT; ++t) {
                        column[t] = column_of<T, DP, 32>(vt, 0, f, t, lane);
                        acc[t] = mma(column[t], p, acc[t]);
                    }
                    if constexpr (sizeof(T) == 2) {
                        const auto rest = rest_of<T>(s, p, f);
#pragma unroll
                        for (int t = 0; t < DT; ++t) acc[t] = mma(column[t], rest, acc[t]);
                    }
                }
            } else {
                if (finite_product_of<T, DP, 32>(vt, 0, t0, w.at, s, true, acc[0], known))
                    add_others<T, DP, 32, true>(vt, 0, t0, w.at, first, Bounds{mine.first, mine.last}, acc[0], known);
            }
        };
        for (int first = start; first < mine.last; first += 2 * kStep) {
            step(kt0, vt0, kt1, vt1, first);
            if (first + kStep < mine.last) step(kt1, vt1, kt0, vt0, first + kStep);
        }
    };
    // The waves' results, columns 32 t0 ... of the head: sums under the largest maximum, added in order.
    const bool seen = mine.count > 0;
    auto finish = [&](auto& acc, auto care, int t0) {
        constexpr bool CARE = decltype(care)::value;
        constexpr int NT = CARE ? 1 : DT, QUADS = 8 * NT;
        l = sum_halves(l);
        if (half == 0) top_of[wave][column] = m, sum_of[wave][column] = l;
        if (!CARE && threadIdx.x < 2) bad[threadIdx.x] = 0;
        __syncthreads();
        float top = top_of[0][column];
#pragma unroll
        for (int w = 1; w < W; ++w) top = fmaxf(top, top_of[w][column]);
        const float by = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - top) * c);
        if (live)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    float4_t x;
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = CARE ? scaled(acc[t][4 * g + e], by) : acc[t][4 * g + e] * by;
                    *Few<T, DP>::sums(key0, val0, wave, column, 32 * (t0 + t) + 8 * g + 4 * half) = x;
                }
        __syncthreads();
        bool all = true;
        for (int at = threadIdx.x; at < heads * QUADS; at += 64 * W) {
            const int col = at / QUADS, e = 32 * t0 + at % QUADS * 4, h = h0 + col;
            if (e >= a.d) continue;
            float high = top_of[0][col], total = 0;
            float4_t x = 0.0f;
#pragma unroll
            for (int w = 1; w < W; ++w) high = fmaxf(high, top_of[w][col]);
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const float one = top_of[w][col];
                total += one == -INFINITY ? 0.0f * sum_of[w][col] : sum_of[w][col] * __builtin_amdgcn_exp2f((one - high) * c);
                x += *Few<T, DP>::sums(key0, val0, w, col, e);
            }
            all = all && finite(x[0]) && finite(x[1]) && finite(x[2]) && finite(x[3]);
            const float log2_top = high == -INFINITY ? high : high * c - Types<T>::kForward;
            if (mine.count > 1) {
                float* to = a.partial + (((int64_t)i * a.hq + h) * a.parts + part) * ROW;
                *(float4_t*)(to + e) = x;
                if (e == 0) to[DP] = log2_top, to[DP + 1] = total;
                continue;
            }
            const int64_t out = ((int64_t)i * a.hq + h) * a.d + e;
            const float by = seen ? 1.0f / total : 0.0f;
            x *= by;
            const auto y = __builtin_convertvector(x, typename Types<T>::quad);
            *(typename Types<T>::quad*)((T*)a.o + out) = y;
            if (a.rest)
                *(typename Types<T>::quad*)((T*)a.rest + out) =
                    __builtin_convertvector(x - __builtin_convertvector(y, float4_t), typename Types<T>::quad);
            if (e == 0) a.lse[h * a.stat_stride + i] = seen ? log2_top + __builtin_amdgcn_logf(total) : -INFINITY;
        }
        return !all;
    };
    bool open;
    {
        float16_t acc[DT];
        pass(acc, std::false_type(), 0, 8.0f);
        open = finish(acc, std::false_type(), 0);
    }
    careful_passes<T, DT>(bad, open, [&](int t, int raise, bool) {
        float16_t acc[1];
        clear_own();
        if (start < mine.last) request(kt0, vt0, start);
        pass(acc, std::true_type(), t, 8.0f * raise);
        finish(acc, std::true_type(), t);
        return live && !all_known(acc[0], known);
    });
}

// Adds up the shares of one row's head: eight groups of 32 lanes take every eighth share, then in order. A chain of waits: what
// does not depend on the row's bounds (which say how many shares there are; the memory is there for all) is requested
// before them: 32 heads of 128 shares 5.6 us, 9.3 without, 1 024 of 4 shares 5.7 and 5.9.
template <typename T, int DP>
__global__ __launch_bounds__(256) void join(Args a) {
    constexpr int ROW = Few<T, DP>::kRow;
    __shared__ float weight[kMostParts], tops[4], totals[4];
    __shared__ __align__(16) float sums[8][DP];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int h = blockIdx.x % a.hq, i = blockIdx.x / a.hq;
    const float* from = a.partial + ((int64_t)i * a.hq + h) * a.parts * ROW;
    const int e = (threadIdx.x & 31) * 4, n0 = threadIdx.x >> 5;
    constexpr int kAhead = 16;
    float4_t ahead[kAhead];
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
        ahead[n] = 0.0f;
        if (8 * n < a.parts) ahead[n] = *(const float4_t*)(from + (int64_t)min(n0 + 8 * n, a.parts - 1) * ROW + min(e, a.d - 4));
    }
    const float* stats = from + (int64_t)min((int)threadIdx.x, a.parts - 1) * ROW + DP;
    float m = stats[0], l = stats[1];
    const Bounds b = keys_of(a, i, lane);
    const int count = Share(b, a.parts, 0, 32 * Few<T, DP>::kWaves).count;
    if (count <= 1) return;
    if ((int)threadIdx.x >= count) m = -INFINITY, l = 0.0f;
    float top = m;
#pragma unroll
    for (int n = 1; n < 64; n <<= 1) top = fmaxf(top, __shfl_xor(top, n));
    if (lane == 0) tops[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    const float by = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
    weight[threadIdx.x] = by;
    const float total = wave_sum(l * by);
    if (lane == 0) totals[wave] = total;
    __syncthreads();
    if (e < DP) {
        float4_t x = 0.0f;
        auto add = [&](float4_t y, float by) {
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = fmaf(by, y[j], x[j]);
        };
        if (e < a.d) {
#pragma unroll
            for (int n = 0; n < kAhead; ++n)
                if (n0 + 8 * n < count) add(ahead[n], weight[n0 + 8 * n]);
#pragma unroll 8
            for (int n = n0 + 8 * kAhead; n < count; n += 8) add(*(const float4_t*)(from + (int64_t)n * ROW + e), weight[n]);
            if (!(finite(x[0]) && finite(x[1]) && finite(x[2]) && finite(x[3]))) {  // (an infinity under a weight of zero stays one)
                x = 0.0f;
                for (int n = n0; n < count; n += 8)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float y = from[(int64_t)n * ROW + e + j];
                        x[j] = finite(y) ? fmaf(weight[n], y, x[j]) : x[j] + y;
                    }
            }
        }
        *(float4_t*)&sums[n0][e] = x;
    }
    __syncthreads();
    const float all = totals[0] + totals[1] + totals[2] + totals[3];
    if ((int)threadIdx.x < a.d) {
        float x = 0;
#pragma unroll
        for (int n = 0; n < 8; ++n) x += sums[n][threadIdx.x];
        x /= all;
        const int64_t out = ((int64_t)i * a.hq + h) * a.d + threadIdx.x;
        const T y = (T)x;
        ((T*)a.o)[out] = y;
        if (a.rest) ((T*)a.rest)[out] = (T)(x - (float)y);
        if (threadIdx.x == 0) a.lse[h * a.stat_stride + i] = top + __builtin_amdgcn_logf(all);
    }
}

// ---------------------------------------------------------------------------
// gradient of the queries; delta on the way
// ---------------------------------------------------------------------------
//
// As the forward pass, with the output's gradient beside the query and three products for each pair, and bound by the same: in the
// cases there 187 us (9 sequences, 0.87 PFLOP/s of visible pairs), 50 (molecules) and 25 (crystals). Scores are computed again here
// and for the keys' gradient, 14 units of products in all with the forward's 4, where one kernel for both would do 10 + 4 but
// add to dq from many blocks: by atomics, in no fixed order, or through memory.
template <typename T, int DP, int SPLIT>
__global__ __launch_bounds__(256, (blocks_per_unit<T, DP>())) void query_gradient(Args a) {
    constexpr int BK = SPLIT == 2 ? 64 : tile_rows<T, DP>(), SUB = SPLIT == 2 ? 1 : BK / 32, DT = DP / 32;
    constexpr int PF = sizeof(T) == 2 ? 2 : 4;
    typedef Tile<T, DP, BK> L;
    __shared__ __align__(1024) char key0[L::kBytes], key1[L::kBytes], val0[L::kBytes], val1[L::kBytes];
    __shared__ Shared shared;
    __shared__ float least[4];
    __shared__ __align__(16) float4_t swap[SPLIT == 2 ? 512 : 1];
    __shared__ unsigned swap_known[SPLIT == 2 ? 128 : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    int tile, h;
    place(a, a.hq, a.q_order, a.causal, tile, h);
    const int kh = h / (a.hq / a.hk), chunks = a.d * (int)sizeof(T) / 16;
    const int rows = wave % (4 / SPLIT), part = wave / (4 / SPLIT);  // which 32 rows, and which of the groups of keys
    const int row = (tile * (4 / SPLIT) + rows) * 32 + (lane & 31), i = min(row, a.nq - 1);
    if (chunks < 2 * L::kFrags) {
        clear<L::kBytes>(key0), clear<L::kBytes>(key1), clear<L::kBytes>(val0), clear<L::kBytes>(val1);
    }
    const Bounds b = keys_of(a, i, lane);
    const Walk walk(b);
    const Bounds all = block_range(walk, shared, wave, lane);
    const char* kbase = (const char*)((const T*)a.k + kh * a.k_head);
    const char* vbase = (const char*)((const T*)a.v + kh * a.v_head);
    const int krow = (int)a.k_row * (int)sizeof(T), vrow = (int)a.v_row * (int)sizeof(T);
    const typename L::Places kplaces(krow, chunks, wave, lane), vplaces(vrow, chunks, wave, lane);
    auto request_first = [&] {
        if (all.lo >= all.hi) return;
        L::request(key0, kbase, krow, kplaces, all.lo, all.hi, chunks, wave);
        L::request(val0, vbase, vrow, vplaces, all.lo, all.hi, chunks, wave);
    };
    request_first();
    const bool mine = row < a.nq;
    typename L::frag q[L::kFrags], g[L::kFrags];
    load_row<T, L::kFrags>(q, (const char*)((const T*)a.q + i * a.q_row + h * a.q_head), chunks, half);
    load_row<T, L::kFrags>(g, (const char*)((const T*)a.grad + i * a.g_row + h * a.g_head), chunks, half);
    float delta = 0;
    {
        const int64_t at = ((int64_t)i * a.hq + h) * a.d;
        const char *o = (const char*)((const T*)a.out + at), *rest = (const char*)((const T*)a.out_rest + at);
#pragma unroll
        for (int f = 0; f < L::kFrags; ++f) {
            typename L::frag x = 0, y = 0;
            if (2 * f + half < chunks) {
                x = *(const typename L::frag*)(o + (2 * f + half) * 16);
                if (a.out_rest) y = *(const typename L::frag*)(rest + (2 * f + half) * 16);
            }
#pragma unroll
            for (int e = 0; e < 16 / (int)sizeof(T); ++e) delta = fmaf((float)x[e] + (float)y[e], (float)g[f][e], delta);
        }
        delta = sum_halves(delta);
    }
    if (mine && half == 0) a.delta[h * a.stat_stride + i] = delta;
    const float lse = a.lse[h * a.stat_stride + i], c = a.scale_log2;
    settle();

    unsigned known;
    // `times`, 2^up, is what ds is raised by (first). Returns what to multiply the sums by.
    auto pass = [&](auto& acc, auto care, int t0, float up, float times) {
        constexpr bool CARE = decltype(care)::value;
        constexpr int NT = CARE ? 1 : DT;
        float lift = times, low = delta * (kLifted<T> ? lift : 1.0f);
        known = 0;
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t] = 0.0f;
        auto products = [&](const char* kt, const char* vt, int first) {
#pragma unroll
            for (int n = 0; n < SUB; ++n) {
                const int u = SPLIT == 2 ? part : n;
                if ((SPLIT == 2 || kSparse<T, DP>) && !walk.needs(first + 32 * u, 32)) continue;
                constexpr bool kAnew = CARE || (kLifted<T> && DP == 128 && SPLIT == 1);  // (no register is left for the places)
                const Lane l = Lane::of<kAnew>(lane, half);
                float16_t s = 0.0f, x = 0.0f;
#pragma unroll
                for (int f = 0; f < L::kFrags; ++f) s = mma(L::row(kt, 32 * u + (CARE ? l.at & 31 : lane & 31), f, CARE ? l.half : half), q[f], s);
#pragma unroll
                for (int f = 0; f < L::kFrags; ++f) x = mma(L::row(vt, 32 * u + (CARE ? l.at & 31 : lane & 31), f, CARE ? l.half : half), g[f], x);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    if constexpr (kLifted<T>)
                        x[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, -lse)) * fmaf(x[r], lift, -low);
                    else
                        x[r] = raised<T>(fmaf(s[r], c, -lse), up, times) * (x[r] - low);
                }
                if (!(SPLIT == 2 || kSparse<T, DP> ? walk.whole(first + 32 * u, 32) : walk.whole(first, BK))) {
                    const int shift = first + 32 * u + 4 * half - b.lo;
                    const unsigned n = b.hi - b.lo;
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if ((unsigned)(shift + 8 * (r / 4) + r % 4) >= n) x[r] = 0.0f;
                }
                typename L::frag lifted[2];
                if constexpr (kLifted<T>)
                    lifted_operands<T>(x, lifted, [&](float by) {
                        lift *= by, low *= by;
#pragma unroll
                        for (int t = 0; t < NT; ++t) acc[t] *= by;
                    });
                if constexpr (CARE) {
                    if (finite_product_of<T, DP, BK>(kt, 32 * u, t0, l.at, x, false, acc[0], known))
                        add_others<T, DP, BK, false>(kt, 32 * u, t0, l.at, first + 32 * u, b, acc[0], known);
                } else {
#pragma unroll
                    for (int f = 0; f < PF; ++f) {
                        const auto d = kLifted<T> ? lifted[f & 1] : operand<T>(x, f);
#pragma unroll
                        for (int t = 0; t < DT; ++t) acc[t] = mma(column_of<T, DP, BK>(kt, 32 * u, f, t, kAnew ? l.at : lane), d, acc[t]);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);  // (reads of the next 32 keys this early would take registers that are not there)
            }
        };
        auto step = [&](char* kt, char* vt, char* kn, char* vn, int first) {
            arrived();
            if (first + BK < all.hi) {
                L::request(kn, kbase, krow, kplaces, first + BK, all.hi, chunks, wave);
                L::request(vn, vbase, vrow, vplaces, first + BK, all.hi, chunks, wave);
            }
            if (walk.needs(first, BK)) products(kt, vt, first);
        };
        for (int first = all.lo; first < all.hi; first += 2 * BK) {
            step(key0, val0, key1, val1, first);
            if (first + BK < all.hi) step(key1, val1, key0, val0, first + BK);
        }
        if constexpr (kLifted<T> && !CARE) {
            const float mine = wave_least(lift);
            if (lane == 0) least[wave] = mine;
            __syncthreads();
            if (threadIdx.x == 0) a.lifts[(int64_t)h * a.q_tiles + tile] = fminf(fminf(least[0], least[1]), fminf(least[2], least[3]));
        }
        if constexpr (SPLIT == 2) {
            // the wave with the second groups of keys hands its sums to the one with the first, 32 columns of the head at a time
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                acc[t] *= 1.0f / lift;  // (the two may be lifted differently)
                if (CARE && part) swap_known[64 * rows + lane] = known;
                __syncthreads();
                if (part)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        swap[(rows * 4 + g) * 64 + lane] = float4_t{acc[t][4 * g], acc[t][4 * g + 1], acc[t][4 * g + 2], acc[t][4 * g + 3]};
                __syncthreads();
                if (CARE && !part) known |= swap_known[64 * rows + lane];
                if (!part)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[t][4 * g + e] += swap[(rows * 4 + g) * 64 + lane][e];
            }
        }
        return SPLIT == 2 ? 1.0f : 1.0f / lift;
    };
    const float ln2 = 0.6931471805599453f;
    bool bad = mine && !part;
    {
        float16_t acc[DT];
        const float by = pass(acc, std::false_type(), 0, (float)Types<T>::kDs, power<Types<T>::kDs>);
        if (bad) store_row<T, DT>((T*)a.dq + ((int64_t)i * a.hq + h) * a.d, acc, c * ln2 * by, a.d, half);
        bad = bad && !all_finite<DT>(acc);
    }
    careful_passes<T, DT>(shared.bad, bad, [&](int t, int raise, bool which) {
        float16_t acc[1];
        request_first();
        const int up = Types<T>::kDs * raise;
        const float by = pass(acc, std::true_type(), t, (float)up, __builtin_amdgcn_ldexpf(1.0f, up));
        T* dq = (T*)a.dq + ((int64_t)i * a.hq + h) * a.d;
        if (which) store_part<T>(dq + 32 * t, acc[0], c * ln2 * by, a.d - 32 * t, half, nullptr, !raise);
        return which && !all_known(acc[0], known);
    });
}

// ---------------------------------------------------------------------------
// gradients of keys and values
// ---------------------------------------------------------------------------
//
// A block has 64 keys (KEYS = 2 waves' worth) and walks tiles of 64 query rows: of 32 keys one wave takes a tile's first
// half, another the second, and at the end they add up. (With 128 keys a block, one wave for both halves, long walks of
// few blocks decide: a training step on 9 packed sequences took 696 us here, not 480.) Where blocks are too few for the
// compute units they have 32 keys and walk tiles of 128 rows, a wave for each quarter. At a head of 128 a lane holds 128
// sums and 64 elements of its key and value, so there is one wave to a SIMD and nothing else runs while it waits: reads from
// LDS go ahead of their products in batches, with a fence behind each. (Left to itself the compiler puts every read right
// before its product, and the wave waited for 45 % of its clocks.) WHAT: 1 the keys' gradient, 2 the values', 3 both.
// In the cases of the forward kernel 334 us (9 sequences, 0.65 PFLOP/s: the longest walk, matrix units at work for 45 % of the clocks of busy
// compute units, which is what a large library product reaches), 51 (molecules), 36 (crystals).
template <typename T, int DP, int WHAT, int KEYS, int UNIT = key_blocks_per_unit<T, DP, WHAT>()>
__global__ __launch_bounds__(256, UNIT) void key_gradient(Args a) {
    constexpr bool DK = WHAT & 1, DV = WHAT & 2;
    constexpr int GROUPS = 4 / KEYS, BQ = 32 * GROUPS, DT = DP / 32, PF = sizeof(T) == 2 ? 2 : 4;
    typedef Tile<T, DP, BQ> L;
    __shared__ __align__(1024) char que0[L::kBytes], que1[L::kBytes];
    __shared__ __align__(1024) char gra0[L::kBytes], gra1[L::kBytes];
    __shared__ __align__(1024) float sta0[2 * BQ], sta1[2 * BQ];  // lse, then delta, of the tile's rows
    __shared__ __align__(16) float4_t swap[4 - KEYS][4][64];
    __shared__ unsigned swap_known[4 - KEYS][64];
    __shared__ Shared shared;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int keys = wave % KEYS, r0 = 32 * (wave / KEYS);  // which 32 keys, and the wave's first row of a tile
    int tile, kh;
    place(a, a.hk, a.k_order, false, tile, kh);  // (causal: the first keys have the longest walks)
    const int group = a.hq / a.hk, chunks = a.d * (int)sizeof(T) / 16;
    const int row = (tile * KEYS + keys) * 32 + (lane & 31), j = min(row, a.nk - 1);
    typename L::frag k[L::kFrags], v[L::kFrags];
    load_row<T, L::kFrags>(k, (const char*)((const T*)a.k + j * a.k_row + kh * a.k_head), chunks, half);
    if (DK) load_row<T, L::kFrags>(v, (const char*)((const T*)a.v + j * a.v_row + kh * a.v_head), chunks, half);
    if (chunks < 2 * L::kFrags) {
        clear<L::kBytes>(que0), clear<L::kBytes>(que1), clear<L::kBytes>(gra0), clear<L::kBytes>(gra1);
    }
    const Bounds b = queries_of(a, j, lane);
    const Walk walk(b);
    const Bounds all = block_range(walk, shared, wave, lane);
    const int qrow = (int)a.q_row * (int)sizeof(T), grow = (int)a.g_row * (int)sizeof(T);
    const typename L::Places qplaces(qrow, chunks, wave, lane), gplaces(grow, chunks, wave, lane);

    // Tiles of rows are walked from the last on. Causal: blocks of neighbouring keys, which run at the same time on an XCD,
    // see the same last rows and differ in their first, and this way they read the same tiles at the same time.
    const int top = all.lo < all.hi ? all.lo + (all.hi - all.lo - 1) / BQ * BQ : 0, last_head = (kh + 1) * group;
    int next_h = last_head, next_first = top;  // the tile to be requested
    auto request = [&](char* qt, char* gt, float* st) {
        if (next_h == last_head) return;
        L::request(qt, (const char*)((const T*)a.q + next_h * a.q_head), qrow, qplaces, next_first, all.hi, chunks, wave);
        L::request(gt, (const char*)((const T*)a.grad + next_h * a.g_head), grow, gplaces, next_first, all.hi, chunks, wave);
        if (wave < BQ / 32) {
            const int64_t at = min((int64_t)(next_first + 64 * (wave >> 1) + lane), a.stat_stride - 1);
            __builtin_amdgcn_global_load_lds((gptr_t)((wave & 1 ? a.delta : a.lse) + next_h * a.stat_stride + at),
                                             (lptr_t)(st + BQ * (wave & 1) + 64 * (wave >> 1)), 4, 0, 0);
        }
        next_first -= BQ;
        if (next_first < all.lo) next_first = top, ++next_h;
    };
    auto request_first = [&] {
        if (all.lo < all.hi) next_h = kh * group;
        request(que0, gra0, sta0);
    };
    request_first();
    const float c = a.scale_log2;
    // What ds carries over what p does; where it is lifted, as far as the queries' gradient has found that none passes 2^14.
    float ratio = power<Types<T>::kDs - Types<T>::kP>;
    if constexpr (kLifted<T>) {
        float lift = power<Types<T>::kDs>;
        const int each = 128 / a.split, tile0 = all.lo / each, tiles = all.lo < all.hi ? (all.hi - 1) / each - tile0 + 1 : 0;
        for (int n = lane; n < tiles * group; n += 64) lift = fminf(lift, a.lifts[(int64_t)(kh * group + n / tiles) * a.q_tiles + tile0 + n % tiles]);
        ratio = wave_least(lift) * power<13 - Types<T>::kP>;
    }
    settle();

    unsigned known;
    // `times`, 2^up, is what p is raised by. Leaves the sums in the first waves' registers.
    auto pass = [&](auto& dk, auto& dv, auto care, int t0, float up, float times) {
        constexpr bool CARE = decltype(care)::value;
        constexpr int NT = CARE ? 1 : DT;
#pragma unroll
        for (int t = 0; t < NT; ++t) dk[t] = 0.0f, dv[t] = 0.0f;
        known = 0;
        // p and ds from the scores and g.v
        auto weigh = [&](float16_t& s, float16_t& x, const float* st) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float4_t lse = *(const float4_t*)(st + r0 + 8 * g + 4 * half);
                const float4_t delta = *(const float4_t*)(st + BQ + r0 + 8 * g + 4 * half);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = 4 * g + e;
                    s[r] = raised<T>(fmaf(s[r], c, -lse[e]), up, times);
                    if (DK) x[r] = s[r] * fmaf(x[r], ratio, -delta[e] * ratio);
                }
            }
        };
        auto hide = [&](float16_t& s, float16_t& x, int first) {
            if (walk.whole(first + r0, 32)) return;
            const int shift = first + r0 + 4 * half - b.lo;
            const unsigned n = b.hi - b.lo;
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if ((unsigned)(shift + 8 * (r / 4) + r % 4) >= n) s[r] = 0.0f, x[r] = 0.0f;
        };
        const int steps = all.lo < all.hi ? ((all.hi - all.lo - 1) / BQ + 1) * group : 0;
        int first = top;
        auto step = [&](char* qt, char* gt, float* st, char* qn, char* gn, float* sn) {
            arrived();
            request(qn, gn, sn);
            const int now = first;
            first -= BQ;
            if (first < all.lo) first = top;
            if (kSparse<T, DP> && !walk.needs(now + r0, 32)) return;
            float16_t s = 0.0f, x = 0.0f;
            if constexpr (kFenced<T, DP> && WHAT == 3 && !CARE) {
                const Lane l = Lane::of<UNIT == 2>(lane, half);  // (kept, the places would take registers that are not there)
                constexpr int kBatch = L::kFrags / 2;
                typename L::frag rows[2][2 * kBatch], columns[2][2 * DT];
                auto load_rows = [&](int n) {
#pragma unroll
                    for (int f = 0; f < kBatch; ++f) {
                        rows[n][2 * f] = L::row(qt, r0 + (l.at & 31), kBatch * n + f, l.half);
                        rows[n][2 * f + 1] = L::row(gt, r0 + (l.at & 31), kBatch * n + f, l.half);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                };
                auto load_columns = [&](int f) {
#pragma unroll
                    for (int t = 0; t < DT; ++t) {
                        columns[f][2 * t] = column_of<T, DP, BQ>(gt, r0, f, t, l.at);
                        columns[f][2 * t + 1] = column_of<T, DP, BQ>(qt, r0, f, t, l.at);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                };
                load_rows(0);
                load_rows(1);
#pragma unroll
                for (int f = 0; f < L::kFrags; ++f) {
                    s = mma(rows[f / kBatch][2 * (f % kBatch)], k[f], s);
                    x = mma(rows[f / kBatch][2 * (f % kBatch) + 1], v[f], x);
                }
                __builtin_amdgcn_sched_barrier(0);
                load_columns(0);
                weigh(s, x, st);
                hide(s, x, now);
                load_columns(1);
#pragma unroll
                for (int f = 0; f < 2; ++f) {
                    const auto p = operand<T>(s, f), d = operand<T>(x, f);
#pragma unroll
                    for (int t = 0; t < DT; ++t) {
                        dv[t] = mma(columns[f][2 * t], p, dv[t]);
                        dk[t] = mma(columns[f][2 * t + 1], d, dk[t]);
                    }
                }
            } else {
                const Lane l = Lane::of<CARE || kSparse<T, DP>>(lane, half);
#pragma unroll
                for (int f = 0; f < L::kFrags; ++f) s = mma(L::row(qt, r0 + (l.at & 31), f, l.half), k[f], s);
#pragma unroll
                for (int f = 0; f < L::kFrags; ++f)
                    if (DK) x = mma(L::row(gt, r0 + (l.at & 31), f, l.half), v[f], x);
                weigh(s, x, st);
                hide(s, x, now);
                if constexpr (CARE) {
                    __builtin_amdgcn_sched_barrier(0);
                    bool others = DV && finite_product_of<T, DP, BQ>(gt, r0, t0, l.at, s, false, dv[0], known);
                    if (DK && finite_product_of<T, DP, BQ>(qt, r0, t0, l.at, x, false, dk[0], known)) others = true;
                    if (DV && others) add_others<T, DP, BQ, true>(gt, r0, t0, l.at, now + r0, b, dv[0], known);
                    if (DK && others) add_others<T, DP, BQ, false, 16>(qt, r0, t0, l.at, now + r0, b, dk[0], known);
                } else {
#pragma unroll
                    for (int f = 0; f < PF; ++f) {
                        if (DV) {
                            const auto p = operand<T>(s, f);
#pragma unroll
                            for (int t = 0; t < DT; ++t) dv[t] = mma(column_of<T, DP, BQ>(gt, r0, f, t, l.at), p, dv[t]);
                        }
                        if (DK) {
                            const auto d = operand<T>(x, f);
#pragma unroll
                            for (int t = 0; t < DT; ++t) dk[t] = mma(column_of<T, DP, BQ>(qt, r0, f, t, l.at), d, dk[t]);
                        }
                    }
                }
            }
        };
        for (int n = 0; n < steps; n += 2) {
            step(que0, gra0, sta0, que1, gra1, sta1);
            if (n + 1 < steps) step(que1, gra1, sta1, que0, gra0, sta0);
        }
        // the waves with a tile's later rows hand their sums to those with the first ones, 32 columns of the head at a time
#pragma unroll
        for (int t = DK ? 0 : NT; t < (DV ? 2 * NT : NT); ++t) {
            float16_t& x = t < NT ? dk[t] : dv[t - NT];
            if (CARE && r0) swap_known[wave - KEYS][lane] = known;
            __syncthreads();
            if (r0)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    swap[wave - KEYS][g][lane] = float4_t{x[4 * g], x[4 * g + 1], x[4 * g + 2], x[4 * g + 3]};
            __syncthreads();
            if (!r0)
#pragma unroll
                for (int n = 0; n < GROUPS - 1; ++n) {
                    if (CARE) known |= swap_known[n * KEYS + keys][lane];
#pragma unroll
                    for (int g = 0; g < 4; ++g)
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[4 * g + e] += swap[n * KEYS + keys][g][lane][e];
                }
        }
    };
    const float ln2 = 0.6931471805599453f;
    bool bad = row < a.nk && !r0;
    {
        constexpr float by = power<-Types<T>::kP>;
        float16_t dk[DT], dv[DT];
        pass(dk, dv, std::false_type(), 0, (float)Types<T>::kP, power<Types<T>::kP>);
        const int64_t at = ((int64_t)j * a.hk + kh) * a.d;
        if (DK && bad) store_row<T, DT>((T*)a.dk + at, dk, c * (ln2 * by / ratio), a.d, half);
        if (DV && bad) store_row<T, DT>((T*)a.dv + at, dv, by, a.d, half);
        bad = bad && !((!DK || all_finite<DT>(dk)) && (!DV || all_finite<DT>(dv)));
    }
    careful_passes<T, DT>(shared.bad, bad, [&](int t, int raise, bool mine) {
        float16_t dk[1], dv[1];
        request_first();
        const int up = Types<T>::kP * raise;
        pass(dk, dv, std::true_type(), t, (float)up, __builtin_amdgcn_ldexpf(1.0f, up));
        const float by = __builtin_amdgcn_ldexpf(1.0f, -up);
        const int64_t at = ((int64_t)anew(j) * a.hk + kh) * a.d;
        if (DK && mine) store_part<T>((T*)a.dk + at + 32 * t, dk[0], c * (ln2 * by / ratio), a.d - 32 * t, half, nullptr, !raise);
        if (DV && mine) store_part<T>((T*)a.dv + at + 32 * t, dv[0], by, a.d - 32 * t, half, nullptr, !raise);
        return mine && !((!DK || all_known(dk[0], known >> 16)) && (!DV || all_known(dv[0], known)));
    });
}

}  // namespace packed_attention
#endif
