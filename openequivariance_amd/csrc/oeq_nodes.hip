// The operators on the nodes of a batch behind the C ABI: checks of arguments, choice of kernels, launches. Their device
// code is in packed_attention.h (compiled per element type from packed_attention.hip), qk_rotary.h and irrep_dropout.h.
#include "oeq_amd.h"
#include "oeq_error.h"

#include "irrep_dropout.h"
#include "packed_attention_launch.h"
#include "qk_rotary.h"

#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

using oeq_internal::fail;

namespace {

int element_bytes(int type) {
    return type == OEQ_FLOAT32 ? 4 : type == OEQ_FLOAT16 || type == OEQ_BFLOAT16 ? 2 : 0;
}

bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }
bool aligned(int64_t stride, int type) { return stride * element_bytes(type) % 16 == 0; }

// Blocks of 256 threads in a launch: threads are counted in 32 bits.
constexpr int64_t kMostBlocks = (1 << 24) - 1;

// A tile's rows, up to 128, are addressed by 32-bit offsets from its first: 127 strides and a head stay below 2^31.
constexpr int64_t kMostRowBytes = (1 << 24) - 1;

int check_attention(const char* who, const oeq_attention* a) {
    if (!a) return fail(OEQ_ERR_INVALID, "%s: NULL description", who);
    if (!element_bytes(a->type)) return fail(OEQ_ERR_INVALID, "%s: element type %d", who, a->type);
    if (a->segments < 0 || a->q_rows < 0 || a->k_rows < 0 || a->q_rows > INT_MAX - 256 || a->k_rows > INT_MAX - 256)
        return fail(OEQ_ERR_INVALID, "%s: %d segments, %lld query rows, %lld key rows", who, a->segments,
                    (long long)a->q_rows, (long long)a->k_rows);
    if (a->k_heads <= 0 || a->q_heads <= 0 || a->q_heads % a->k_heads)
        return fail(OEQ_ERR_INVALID, "%s: %d query heads for %d key heads", who, a->q_heads, a->k_heads);
    if ((a->q_rows + 63) / 64 > kMostBlocks / a->q_heads || (a->k_rows + 63) / 64 > kMostBlocks / a->k_heads)
        return fail(OEQ_ERR_INVALID, "%s: %lld query rows, %lld key rows", who, (long long)a->q_rows, (long long)a->k_rows);
    if (a->head_dim <= 0 || a->head_dim > 128 || a->head_dim % 8)
        return fail(OEQ_ERR_INVALID, "%s: heads of %d elements (multiples of 8 up to 128)", who, a->head_dim);
    if (!(a->scale > 0) || !std::isfinite(a->scale)) return fail(OEQ_ERR_INVALID, "%s: scale %g", who, a->scale);
    for (int64_t s : {a->q_row_stride, a->q_head_stride, a->k_row_stride, a->k_head_stride, a->v_row_stride, a->v_head_stride})
        if (!aligned(s, a->type)) return fail(OEQ_ERR_INVALID, "%s: a stride of %lld elements", who, (long long)s);
    for (int64_t s : {a->q_row_stride, a->k_row_stride, a->v_row_stride})
        if (s < 0 || s * element_bytes(a->type) > kMostRowBytes)
            return fail(OEQ_ERR_INVALID, "%s: a row stride of %lld elements", who, (long long)s);
    if (a->q_rows && !a->q) return fail(OEQ_ERR_INVALID, "%s: NULL buffer", who);
    if (a->k_rows && (!a->k || !a->v)) return fail(OEQ_ERR_INVALID, "%s: NULL buffer", who);
    if ((a->q_rows || a->k_rows) && (!a->q_ptr || !a->k_ptr)) return fail(OEQ_ERR_INVALID, "%s: NULL buffer", who);
    if (!aligned(a->q) || !aligned(a->k) || !aligned(a->v)) return fail(OEQ_ERR_INVALID, "%s: unaligned buffer", who);
    return OEQ_OK;
}

// Tiles of rows by falling length of their walks: the longest first, so that a launch does not end with a few compute
// units at work on them. Lengths are those between the first and the last row's bounds; tiles of about the same length come in
// any order, on which no result depends. One block for query tiles, one for key tiles; order[tiles ..] is scratch.
__global__ __launch_bounds__(1024) void order_tiles(packed_attention::Args a, int* q_order, int q_tiles, int* k_order, int k_tiles) {
    __shared__ int count[256], longest;
    const bool keys = blockIdx.x == 1;
    int* order = keys ? k_order : q_order;
    const int tiles = keys ? k_tiles : q_tiles, rows = keys ? a.nk : a.nq, each = keys ? packed_attention::kKeyTile : packed_attention::kQueryTile;
    const int lane = threadIdx.x & 63;
    if (threadIdx.x < 256) count[threadIdx.x] = 0;
    if (threadIdx.x == 0) longest = 1;
    __syncthreads();
    for (int base = 0; base < tiles; base += 1024) {
        const int t = base + threadIdx.x, first = min(t * each, rows - 1), last = min(first + each - 1, rows - 1);
        const packed_attention::Bounds x = keys ? packed_attention::queries_of(a, first, lane) : packed_attention::keys_of(a, first, lane);
        const packed_attention::Bounds y = keys ? packed_attention::queries_of(a, last, lane) : packed_attention::keys_of(a, last, lane);
        const int n = x.lo < x.hi && y.lo < y.hi ? y.hi - x.lo : max(x.hi - x.lo, y.hi - y.lo);
        if (t < tiles) {
            order[tiles + t] = max(n, 0);
            atomicMax(&longest, n);
        }
    }
    __syncthreads();
    const float by = 255.0f / longest;
    for (int t = threadIdx.x; t < tiles; t += 1024) atomicAdd(&count[255 - min(255, (int)(order[tiles + t] * by))], 1);
    __syncthreads();
    if (threadIdx.x < 64) {  // where each class begins
        int c[4], sum = 0;
#pragma unroll
        for (int n = 0; n < 4; ++n) c[n] = count[4 * lane + n], sum += c[n];
        int before = sum;
#pragma unroll
        for (int n = 1; n < 64; n <<= 1) {
            const int x = __shfl_up(before, n);
            if (lane >= n) before += x;
        }
        before -= sum;
#pragma unroll
        for (int n = 0; n < 4; ++n) count[4 * lane + n] = before, before += c[n];
    }
    __syncthreads();
    for (int t = threadIdx.x; t < tiles; t += 1024)
        order[atomicAdd(&count[255 - min(255, (int)(order[tiles + t] * by))], 1)] = t;
}

int64_t query_tiles(const oeq_attention& a) { return (a.q_rows + packed_attention::kQueryTile - 1) / packed_attention::kQueryTile; }
int64_t key_tiles(const oeq_attention& a) { return (a.k_rows + packed_attention::kKeyTile - 1) / packed_attention::kKeyTile; }

packed_attention::Args attention_args(const oeq_attention& a) {
    packed_attention::Args g = {};
    g.q = a.q, g.k = a.k, g.v = a.v;
    g.q_ptr = a.q_ptr, g.k_ptr = a.k_ptr, g.k_len = a.k_len;
    g.q_row = a.q_row_stride, g.q_head = a.q_head_stride;
    g.k_row = a.k_row_stride, g.k_head = a.k_head_stride;
    g.v_row = a.v_row_stride, g.v_head = a.v_head_stride;
    g.stat_stride = oeq_attention_stat_stride(a.q_rows);
    g.segments = a.segments, g.nq = (int)a.q_rows, g.nk = (int)a.k_rows;
    g.hq = a.q_heads, g.hk = a.k_heads, g.d = a.head_dim, g.causal = a.causal != 0;
    // Below two blocks a compute unit a block has half as many rows, each shared by two waves that take every other group of
    // 32 keys. Forward, us, shared / not: 64 blocks of 128 rows, bf16 heads of 128 18 / 24, 150, fp16 of 72 25 / 33, 376, bf16 of 64
    // 29 / 35, 504, float32 of 128 240 / 296, 512, bf16 of 128 41 / 40, 1 008 80 / 60.
    g.split = query_tiles(a) * a.q_heads < 512 ? 2 : 1;
    const int rows = packed_attention::kQueryTile / g.split;
    g.tiles = (int)((a.q_rows + rows - 1) / rows);
    g.scale_log2 = a.scale * 1.4426950408889634f;
    return g;
}

// How many shares the form for few queries cuts a row's keys into; 0: the form for tiles of rows.
//
// Lengths are on the device, so the rule goes by their means over the segments and takes the smaller of two estimates, in
// steps of about a microsecond. Tiles: blocks of 128 rows walk the keys of all segments that their rows belong to, 64 a
// step. Few: blocks of a row and a key head walk that row's keys alone, 80 a step after some 5 steps of latency (a block's
// bounds, first reads and end). Either way two blocks a compute unit run at a time. Measured with 8 heads of 64, bf16,
// tiles / few in us: 128 segments of 1 row, 512 keys 336 / 26, of 2 rows, 16 keys 11 / 20, of 4 rows, 64 keys 17 / 39, of 8 rows,
// 64 keys 11 / 74, 512 keys 47 / 124; 1 024 segments of 1 row, 32 keys 29 / 74; a segment of 16 rows, 4 096 keys 39 / 23.
// (Means tell nothing of a prompt beside single tokens, or of one long cache among short ones: results are right there, but
// tiles then walk the single tokens' caches, and the long one has as few shares as the others.)
int parts_of(const oeq_attention& a) {
    constexpr int64_t kBlocks = 1024;   // (one token against 65 537 keys, again and again: 512 blocks 52 us, 1 024 51, 2 048 57)
    constexpr int64_t kLeastKeys = 256;  // a share is worth its block and its row of the join
    const int64_t segments = std::max(a.segments, 1), group = a.q_heads / a.k_heads;
    const int64_t blocks = a.q_rows * a.k_heads * ((group + 31) / 32);
    if (blocks > INT_MAX / packed_attention::kMostParts) return 0;
    const double keys = std::ceil((double)a.k_rows / segments), rows = std::max(1.0, (double)a.q_rows / segments);
    const int64_t parts = std::max<int64_t>(
        1, std::min({kBlocks / blocks, (int64_t)keys / kLeastKeys, (int64_t)packed_attention::kMostParts}));
    const double walk = std::min((double)a.k_rows, (127 / rows + 1) * keys);
    const double tiles = std::max(1.0, (a.q_rows + 127) / 128 * a.q_heads / 512.0) * std::ceil(walk / 64);
    const double few = std::max(1.0, blocks * parts / 512.0) * (5 + keys / parts / 80);
    return few < tiles ? (int)parts : 0;
}

// Whether tiles are put in the order of their walks' lengths first (a launch of 8 us): where there are segments, whose
// lengths can differ, long enough for a walk to last a while, and a few rounds of blocks on the compute units, so that
// the last of them counts. Out of order / in order, bf16, causal: 2.8 rounds, forward 173 / 157, gradients 705 / 608 us; 16 rounds,
// forward 1 823 / 1 870 (neighbours, which share keys, are no longer next to each other).
bool ordered(const oeq_attention& a) {
    const int64_t blocks = query_tiles(a) * a.q_heads;
    return a.segments > 1 && blocks > 512 && blocks <= 8 * 512 && a.k_rows / a.segments >= 512;
}

int head_tile(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }

int check_rotary(const char* who, const oeq_qk_rotary* a) {
    if (!a) return fail(OEQ_ERR_INVALID, "%s: NULL description", who);
    if (!element_bytes(a->type)) return fail(OEQ_ERR_INVALID, "%s: element type %d", who, a->type);
    if (a->rows < 0 || a->table_rows < 0 || a->q_heads < 0 || a->k_heads < 0)
        return fail(OEQ_ERR_INVALID, "%s: %lld rows, %lld rows of the table, %d and %d heads", who, (long long)a->rows,
                    (long long)a->table_rows, a->q_heads, a->k_heads);
    if (a->head_dim <= 0 || a->head_dim > 128 || a->head_dim % 8)
        return fail(OEQ_ERR_INVALID, "%s: heads of %d elements (multiples of 8 up to 128)", who, a->head_dim);
    if (a->rotary_dim < 0 || a->rotary_dim > a->head_dim || a->rotary_dim % 8)
        return fail(OEQ_ERR_INVALID, "%s: %d turned elements of %d (multiples of 8)", who, a->rotary_dim, a->head_dim);
    if (a->rows > INT_MAX) return fail(OEQ_ERR_INVALID, "%s: %lld rows", who, (long long)a->rows);
    for (int64_t s : {a->q_row_stride, a->q_head_stride, a->k_row_stride, a->k_head_stride})
        if (!aligned(s, a->type)) return fail(OEQ_ERR_INVALID, "%s: a stride of %lld elements", who, (long long)s);
    if (a->rows && ((a->q_heads && !a->q) || (a->k_heads && !a->k) || (a->rotary_dim && (!a->positions || !a->table))))
        return fail(OEQ_ERR_INVALID, "%s: NULL buffer", who);
    if (!aligned(a->q) || !aligned(a->k) || !aligned(a->q_weight) || !aligned(a->k_weight) || !aligned(a->table))
        return fail(OEQ_ERR_INVALID, "%s: unaligned buffer", who);
    return OEQ_OK;
}

// Lanes to a head, with eight elements each: a power of two.
int lanes_of(const qk_rotary::Args& g) { return g.d <= 8 ? 1 : g.d <= 16 ? 2 : g.d <= 32 ? 4 : g.d <= 64 ? 8 : 16; }

qk_rotary::Args rotary_args(const oeq_qk_rotary& a) {
    qk_rotary::Args g = {};
    g.q = a.q, g.k = a.k, g.q_weight = a.q_weight, g.k_weight = a.k_weight;
    g.positions = a.positions, g.table = a.table, g.table_rows = a.table_rows;
    g.q_row = a.q_row_stride, g.q_head = a.q_head_stride;
    g.k_row = a.k_row_stride, g.k_head = a.k_head_stride;
    g.q_heads = a.q_heads, g.k_heads = a.k_heads, g.d = a.head_dim, g.rotary = a.rotary_dim;
    g.interleaved = a.interleaved != 0;
    g.eps = a.eps, g.per_d = 1.0f / a.head_dim;
    g.rows = a.rows;
    g.groups = 1;
    while (g.groups < std::max(a.q_heads, a.k_heads) && g.groups * lanes_of(g) < 256) g.groups *= 2;
    return g;
}

int64_t rotary_blocks(const qk_rotary::Args& g) {
    const int each = 256 / (lanes_of(g) * g.groups);
    return (g.rows + each - 1) / each;
}

template <typename F>
void by_lanes(const qk_rotary::Args& g, F launch) {
    switch (lanes_of(g)) {
        case 1: return launch(std::integral_constant<int, 1>());
        case 2: return launch(std::integral_constant<int, 2>());
        case 4: return launch(std::integral_constant<int, 4>());
        case 8: return launch(std::integral_constant<int, 8>());
        default: return launch(std::integral_constant<int, 16>());
    }
}

template <bool APPEND>
int launch_rotary(int type, const qk_rotary::Args& g, hipStream_t stream) {
    const unsigned blocks = (unsigned)std::min<int64_t>(rotary_blocks(g), kMostBlocks);  // (the blocks walk the rest)
    by_lanes(g, [&](auto lanes) {
        constexpr int kLanes = decltype(lanes)::value;
        if (type == OEQ_FLOAT32)
            qk_rotary::forward<float, kLanes, APPEND><<<blocks, 256, 0, stream>>>(g);
        else if (type == OEQ_FLOAT16)
            qk_rotary::forward<_Float16, kLanes, APPEND><<<blocks, 256, 0, stream>>>(g);
        else
            qk_rotary::forward<__bf16, kLanes, APPEND><<<blocks, 256, 0, stream>>>(g);
    });
    HIP_TRY(hipGetLastError());
    return OEQ_OK;
}

// Blocks of the gradient: a few for each compute unit, so that the rows of partial sums stay few.
constexpr int kGradientBlocks = 1024;

unsigned gradient_blocks(const qk_rotary::Args& g) {
    return (unsigned)std::min<int64_t>(kGradientBlocks, rotary_blocks(g));
}

template <typename T>
int launch_rotary_gradient(const qk_rotary::Args& g, void* q_weight_grad, void* k_weight_grad, hipStream_t stream) {
    const unsigned blocks = gradient_blocks(g);
    if (blocks) {
        by_lanes(g, [&](auto lanes) { qk_rotary::backward<T, decltype(lanes)::value><<<blocks, 256, 0, stream>>>(g); });
        HIP_TRY(hipGetLastError());
    }
    if (g.partial) {
        qk_rotary::weight_gradient<T><<<lanes_of(g), 1024, 0, stream>>>(g, lanes_of(g), (int)blocks, (T*)q_weight_grad,
                                                                        (T*)k_weight_grad);
        HIP_TRY(hipGetLastError());
    }
    return OEQ_OK;
}

template <typename T, typename F>
int launch_dropout(int64_t rows, int64_t dim, const void* x, const void* residual, void* out, const int32_t* channels,
                   const int64_t* seed, unsigned drop, hipStream_t stream) {
    constexpr int V = 16 / (int)sizeof(T);
    const F scale = drop < 65536 ? (F)(65536.0 / (65536 - drop)) : (F)0;
    // elements are numbered in 32 bits: longer tensors go in parts of whole rows, a multiple of V of them so that every
    // part begins at 16 bytes
    const int64_t part = std::max<int64_t>(V, ((int64_t)1 << 31) / dim / V * V);
    for (int64_t first = 0; first < rows; first += part) {
        const int64_t at = first * dim;
        const unsigned count = (unsigned)(std::min(part, rows - first) * dim);
        const unsigned threads = (count + V - 1) / V;
        irrep_dropout::dropout<T, F, V><<<(threads + 255) / 256, 256, 0, stream>>>(
            (const T*)x + at, residual ? (const T*)residual + at : nullptr, (T*)out + at, channels, seed, count, (unsigned)dim,
            first, drop, scale);
        HIP_TRY(hipGetLastError());
    }
    return OEQ_OK;
}

}  // namespace

extern "C" {

int64_t oeq_attention_stat_stride(int64_t q_rows) { return (q_rows + 63) / 64 * 64 + 64; }

size_t oeq_attention_forward_workspace_bytes(const oeq_attention* a) {
    if (!a || a->k_heads <= 0 || a->q_heads <= 0 || a->segments < 0 || a->q_rows <= 0) return 0;
    const int parts = parts_of(*a);
    if (parts > 1) return (size_t)a->q_rows * a->q_heads * parts * (head_tile(a->head_dim) + 4) * sizeof(float);
    return parts == 0 && ordered(*a) ? 2 * (size_t)query_tiles(*a) * sizeof(int) : 0;
}

int oeq_attention_forward(const oeq_attention* a, void* out, void* out_rest, float* log2_sum, void* workspace,
                          size_t workspace_bytes, void* stream) {
    const char* who = "oeq_attention_forward";
    if (int rc = check_attention(who, a)) return rc;
    if (a->q_rows == 0) return OEQ_OK;
    if (!out || !log2_sum) return fail(OEQ_ERR_INVALID, "%s: NULL buffer", who);
    if (!aligned(out) || !aligned(out_rest)) return fail(OEQ_ERR_INVALID, "%s: unaligned buffer", who);
    if (workspace_bytes < oeq_attention_forward_workspace_bytes(a) || (workspace_bytes && !workspace))
        return fail(OEQ_ERR_INVALID, "%s: workspace too small", who);
    packed_attention::Args g = attention_args(*a);
    g.o = out, g.rest = out_rest, g.lse = log2_sum;
    g.parts = parts_of(*a), g.partial = (float*)workspace;
    const auto s = (hipStream_t)stream;
    if (g.parts == 0 && ordered(*a)) {
        g.q_order = (int*)workspace;
        order_tiles<<<1, 1024, 0, s>>>(g, (int*)workspace, g.tiles, nullptr, 0);
        HIP_TRY(hipGetLastError());
    }
    HIP_TRY(a->type == OEQ_FLOAT32 ? packed_attention::Launch<float>::forward(g, s)
            : a->type == OEQ_FLOAT16 ? packed_attention::Launch<_Float16>::forward(g, s)
                                     : packed_attention::Launch<__bf16>::forward(g, s));
    return OEQ_OK;
}

size_t oeq_attention_backward_workspace_bytes(const oeq_attention* a) {
    if (!a || a->q_heads <= 0 || a->q_rows < 0 || a->k_rows < 0) return 0;
    const size_t delta = (size_t)a->q_heads * oeq_attention_stat_stride(a->q_rows) * sizeof(float);
    // (of float16 a number for each tile of each head, where a tile has 64 rows or more)
    const size_t lifts = a->type == OEQ_FLOAT16 ? (size_t)a->q_heads * ((a->q_rows + 63) / 64) * sizeof(float) : 0;
    return delta + lifts + (ordered(*a) ? 2 * (size_t)(query_tiles(*a) + key_tiles(*a)) * sizeof(int) : 0);
}

int oeq_attention_backward(const oeq_attention* a, const void* out, const void* out_rest, const float* log2_sum,
                           const void* out_grad, int64_t grad_row_stride, int64_t grad_head_stride, void* q_grad,
                           void* k_grad, void* v_grad, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "oeq_attention_backward";
    if (int rc = check_attention(who, a)) return rc;
    if (!aligned(grad_row_stride, a->type) || !aligned(grad_head_stride, a->type) || grad_row_stride < 0 ||
        grad_row_stride * element_bytes(a->type) > kMostRowBytes)
        return fail(OEQ_ERR_INVALID, "%s: strides of %lld and %lld elements", who, (long long)grad_row_stride,
                    (long long)grad_head_stride);
    if ((a->q_rows && (!out || !log2_sum || !out_grad || !q_grad)) || (a->k_rows && (!k_grad || !v_grad)))
        return fail(OEQ_ERR_INVALID, "%s: NULL buffer", who);
    if (!aligned(out) || !aligned(out_rest) || !aligned(out_grad) || !aligned(q_grad) || !aligned(k_grad) || !aligned(v_grad))
        return fail(OEQ_ERR_INVALID, "%s: unaligned buffer", who);
    if (workspace_bytes < oeq_attention_backward_workspace_bytes(a) || !workspace)
        return fail(OEQ_ERR_INVALID, "%s: workspace too small", who);
    packed_attention::Args g = attention_args(*a);
    g.out = out, g.out_rest = out_rest, g.grad = out_grad, g.g_row = grad_row_stride, g.g_head = grad_head_stride;
    g.dq = q_grad, g.dk = k_grad, g.dv = v_grad, g.lse = (float*)log2_sum, g.delta = (float*)workspace;
    const auto s = (hipStream_t)stream;
    const int ktiles = (int)key_tiles(*a);
    g.lifts = g.delta + a->q_heads * g.stat_stride;
    g.q_tiles = g.tiles;
    if (ordered(*a)) {
        int* q_order = (int*)(g.lifts + (a->type == OEQ_FLOAT16 ? (int64_t)a->q_heads * g.tiles : 0));
        int* k_order = q_order + 2 * (int64_t)g.tiles;
        g.q_order = q_order, g.k_order = k_order;
        order_tiles<<<2, 1024, 0, s>>>(g, q_order, g.tiles, k_order, ktiles);
        HIP_TRY(hipGetLastError());
    }
    HIP_TRY(a->type == OEQ_FLOAT32 ? packed_attention::Launch<float>::backward(g, ktiles, s)
            : a->type == OEQ_FLOAT16 ? packed_attention::Launch<_Float16>::backward(g, ktiles, s)
                                     : packed_attention::Launch<__bf16>::backward(g, ktiles, s));
    return OEQ_OK;
}

int oeq_qk_norm_rotary(const oeq_qk_rotary* a, void* q_out, void* k_out, void* stream) {
    const char* who = "oeq_qk_norm_rotary";
    if (int rc = check_rotary(who, a)) return rc;
    qk_rotary::Args g = rotary_args(*a);
    if (g.rows == 0 || a->q_heads + a->k_heads == 0) return OEQ_OK;
    if ((a->q_heads && !q_out) || (a->k_heads && !k_out)) return fail(OEQ_ERR_INVALID, "%s: NULL buffer", who);
    if (!aligned(q_out) || !aligned(k_out)) return fail(OEQ_ERR_INVALID, "%s: unaligned buffer", who);
    g.q_out = q_out, g.k_out = k_out;
    g.ko_head = a->head_dim, g.ko_row = (int64_t)a->k_heads * a->head_dim;
    return launch_rotary<false>(a->type, g, (hipStream_t)stream);
}

int oeq_qk_norm_rotary_append(const oeq_qk_rotary* a, const void* v, int64_t v_row_stride, int64_t v_head_stride,
                              void* q_out, void* k_cache, int64_t k_cache_row_stride, int64_t k_cache_head_stride,
                              void* v_cache, int64_t v_cache_row_stride, int64_t v_cache_head_stride,
                              const int64_t* slots, int64_t cache_rows, void* stream) {
    const char* who = "oeq_qk_norm_rotary_append";
    if (int rc = check_rotary(who, a)) return rc;
    for (int64_t s : {v_row_stride, v_head_stride, k_cache_row_stride, k_cache_head_stride, v_cache_row_stride,
                      v_cache_head_stride})
        if (!aligned(s, a->type)) return fail(OEQ_ERR_INVALID, "%s: a stride of %lld elements", who, (long long)s);
    if (cache_rows < 0) return fail(OEQ_ERR_INVALID, "%s: %lld rows of the caches", who, (long long)cache_rows);
    qk_rotary::Args g = rotary_args(*a);
    if (g.rows == 0 || a->q_heads + a->k_heads == 0) return OEQ_OK;
    if ((a->q_heads && !q_out) || (a->k_heads && (!v || !slots || (cache_rows && (!k_cache || !v_cache)))))
        return fail(OEQ_ERR_INVALID, "%s: NULL buffer", who);
    if (!aligned(v) || !aligned(q_out) || !aligned(k_cache) || !aligned(v_cache))
        return fail(OEQ_ERR_INVALID, "%s: unaligned buffer", who);
    g.v = v, g.v_row = v_row_stride, g.v_head = v_head_stride;
    g.q_out = q_out, g.k_out = k_cache, g.v_out = v_cache;
    g.ko_row = k_cache_row_stride, g.ko_head = k_cache_head_stride;
    g.vo_row = v_cache_row_stride, g.vo_head = v_cache_head_stride;
    g.slots = slots, g.slots_end = cache_rows;
    return launch_rotary<true>(a->type, g, (hipStream_t)stream);
}

size_t oeq_qk_norm_rotary_backward_workspace_bytes(const oeq_qk_rotary* a) {
    if (!a || (!a->q_weight && !a->k_weight) || a->head_dim <= 0 || a->head_dim > 128) return 0;
    return (size_t)kGradientBlocks * 2 * 128 * sizeof(float);
}

int oeq_qk_norm_rotary_backward(const oeq_qk_rotary* a, const void* q_grad, int64_t q_grad_row_stride,
                                int64_t q_grad_head_stride, const void* k_grad, int64_t k_grad_row_stride,
                                int64_t k_grad_head_stride, void* q_in_grad, void* k_in_grad, void* q_weight_grad,
                                void* k_weight_grad, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "oeq_qk_norm_rotary_backward";
    if (int rc = check_rotary(who, a)) return rc;
    for (int64_t s : {q_grad_row_stride, q_grad_head_stride, k_grad_row_stride, k_grad_head_stride})
        if (!aligned(s, a->type)) return fail(OEQ_ERR_INVALID, "%s: a stride of %lld elements", who, (long long)s);
    qk_rotary::Args g = rotary_args(*a);
    if (g.rows && ((a->q_heads && (!q_grad || !q_in_grad)) || (a->k_heads && (!k_grad || !k_in_grad))))
        return fail(OEQ_ERR_INVALID, "%s: NULL buffer", who);
    if ((a->q_weight && !q_weight_grad) || (a->k_weight && !k_weight_grad))
        return fail(OEQ_ERR_INVALID, "%s: NULL buffer", who);
    const size_t need = oeq_qk_norm_rotary_backward_workspace_bytes(a);
    if (need && (workspace_bytes < need || !workspace)) return fail(OEQ_ERR_INVALID, "%s: workspace too small", who);
    if (!aligned(q_grad) || !aligned(k_grad) || !aligned(q_in_grad) || !aligned(k_in_grad))
        return fail(OEQ_ERR_INVALID, "%s: unaligned buffer", who);
    g.q_grad = q_grad, g.gq_row = q_grad_row_stride, g.gq_head = q_grad_head_stride;
    g.k_grad = k_grad, g.gk_row = k_grad_row_stride, g.gk_head = k_grad_head_stride;
    g.q_out = q_in_grad, g.k_out = k_in_grad;
    g.partial = need ? (float*)workspace : nullptr;
    if (!a->q_weight) q_weight_grad = nullptr;
    if (!a->k_weight) k_weight_grad = nullptr;
    const auto s = (hipStream_t)stream;
    if (a->type == OEQ_FLOAT32) return launch_rotary_gradient<float>(g, q_weight_grad, k_weight_grad, s);
    if (a->type == OEQ_FLOAT16) return launch_rotary_gradient<_Float16>(g, q_weight_grad, k_weight_grad, s);
    return launch_rotary_gradient<__bf16>(g, q_weight_grad, k_weight_grad, s);
}

int oeq_irrep_dropout(int type, int64_t rows, int64_t dim, const void* x, const void* residual, void* out,
                      const int32_t* channels, const int64_t* seed, double p, void* stream) {
    const char* who = "oeq_irrep_dropout";
    if (rows < 0 || dim < 0 || rows > INT_MAX || dim > (1 << 27))
        return fail(OEQ_ERR_INVALID, "%s: %lld rows of %lld", who, (long long)rows, (long long)dim);
    if (!(p >= 0.0 && p <= 1.0)) return fail(OEQ_ERR_INVALID, "%s: p = %g", who, p);
    if (type != OEQ_FLOAT64 && !element_bytes(type)) return fail(OEQ_ERR_INVALID, "%s: element type %d", who, type);
    if (rows == 0 || dim == 0) return OEQ_OK;
    if (!x || !out || !channels || !seed) return fail(OEQ_ERR_INVALID, "%s: NULL buffer", who);
    if (!aligned(x) || !aligned(residual) || !aligned(out)) return fail(OEQ_ERR_INVALID, "%s: unaligned buffer", who);
    const unsigned drop = (unsigned)std::nearbyint(p * 65536);
    const auto s = (hipStream_t)stream;
    switch (type) {
        case OEQ_FLOAT32: return launch_dropout<float, float>(rows, dim, x, residual, out, channels, seed, drop, s);
        case OEQ_FLOAT16: return launch_dropout<_Float16, float>(rows, dim, x, residual, out, channels, seed, drop, s);
        case OEQ_BFLOAT16: return launch_dropout<__bf16, float>(rows, dim, x, residual, out, channels, seed, drop, s);
        default: return launch_dropout<double, double>(rows, dim, x, residual, out, channels, seed, drop, s);
    }
}

}  // extern "C"
