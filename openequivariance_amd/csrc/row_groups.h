// Device code of rows grouped by type: the index itself, rows of a table by type and the sums of rows by type.
//
// The index of n rows with T types is `order`, the row numbers by type and ascending within a type, rows without a type
// (a type outside 0 .. T - 1) last, and `ptr`, where each type's rows begin in it: T + 1 numbers, ptr[T] the end of the last.
//
// It is a counting sort by eight bits of the type at a time, the lowest first; each pass keeps the order of rows whose bits are
// equal, so the last leaves rows of a type ascending and every sum over a type's rows has one order. A pass has two launches:
// blocks count the digits of their span of rows; then each block adds up the counts before its own (all digits below, and
// the same digit in the blocks before) and places its rows. Up to kOneBlock rows one block does all passes in LDS in one launch.
// Launches and chains of waits are all that it takes: 333 rows 3.7 us, 4 001 9, 20 000 3.5 and 6; of 32 003 types two passes and the
// search for their beginnings 24. (Every block counting all rows instead of the first launch: 18 us, not 9.)
#ifndef OEQ_ROW_GROUPS_H
#define OEQ_ROW_GROUPS_H

#include <hip/hip_runtime.h>

#include <cstdint>

namespace row_groups {

constexpr int kBits = 8, kDigits = 1 << kBits;
constexpr int kWaves = 16, kThreads = 64 * kWaves;
constexpr int kOneBlock = 8 * kThreads;  // rows that one block sorts in LDS
constexpr int kMostBlocks = 256;         // of a pass: every block adds up what all of them counted

__device__ __forceinline__ int key_of(int64_t type, int types) { return type >= 0 && type < types ? (int)type : types; }

// The lanes of a wave with the same digit as this one.
__device__ __forceinline__ uint64_t same_digit(int digit, bool valid) {
    uint64_t mask = __ballot(valid);
#pragma unroll
    for (int b = 0; b < kBits; ++b) {
        const uint64_t set = __ballot(digit >> b & 1);
        mask &= digit >> b & 1 ? set : ~set;
    }
    return mask;
}
__device__ __forceinline__ int lanes_before(uint64_t mask) {
    return __builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0));
}

// Sum over the digits before each thread's own (thread d < 256 brings digit d's); all threads call it.
__device__ __forceinline__ int before_digit(int count, int* wave_sums) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int sum = count;
#pragma unroll
    for (int n = 1; n < 64; n <<= 1) {
        const int x = __shfl_up(sum, n);
        if (lane >= n) sum += x;
    }
    if (wave < 4 && lane == 63) wave_sums[wave] = sum;
    __syncthreads();
    int before = sum - count;
    for (int w = 0; w < wave && w < 4; ++w) before += wave_sums[w];
    return before;
}

// All passes of up to kOneBlock rows: `each` rows to a thread, rows of a wave next to each other. Between passes keys and
// row numbers lie in LDS, in the order reached so far.
__global__ __launch_bounds__(kThreads) void sort_in_block(const int64_t* types, int rows, int count, int passes, int* order, int* ptr) {
    __shared__ int keys[kOneBlock], numbers[kOneBlock];
    __shared__ int counts[kWaves][kDigits], wave_sums[4];
    constexpr int kEach = kOneBlock / kThreads;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int rounds = (rows + kThreads - 1) / kThreads, span = rounds * 64;  // a wave's rows
    int key[kEach], number[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int at = wave * span + i * 64 + lane;
        number[i] = at;
        key[i] = i < rounds && at < rows ? key_of(types[at], count) : 0;
    }
    for (int pass = 0; pass < passes; ++pass) {
        for (int i = tid; i < kWaves * kDigits; i += kThreads) ((int*)counts)[i] = 0;
        __syncthreads();
        const int shift = pass * kBits;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int at = wave * span + i * 64 + lane;
            if (i >= rounds) break;
            const int digit = key[i] >> shift & (kDigits - 1);
            const uint64_t same = same_digit(digit, at < rows);
            if (at < rows && lanes_before(same) == 0) counts[wave][digit] += __popcll(same);
        }
        __syncthreads();
        int total = 0;
        if (tid < kDigits)
            for (int w = 0; w < kWaves; ++w) total += counts[w][tid];
        int before = before_digit(total, wave_sums);
        const bool last = pass + 1 == passes;
        if (passes == 1 && tid <= count) ptr[tid] = before;  // (the digit is the type)
        if (tid < kDigits)
            for (int w = 0; w < kWaves; ++w) {
                const int c = counts[w][tid];
                counts[w][tid] = before;
                before += c;
            }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int at = wave * span + i * 64 + lane;
            if (i >= rounds) break;
            const int digit = key[i] >> shift & (kDigits - 1);
            const uint64_t same = same_digit(digit, at < rows);
            if (at < rows) {
                const int to = counts[wave][digit] + lanes_before(same);
                if (last) order[to] = number[i];
                if (passes > 1) keys[to] = key[i], numbers[to] = number[i];
                if (lanes_before(same) == __popcll(same) - 1) counts[wave][digit] = to + 1;
            }
        }
        __syncthreads();
        if (!last) {
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const int at = wave * span + i * 64 + lane;
                if (i < rounds && at < rows) key[i] = keys[at], number[i] = numbers[at];
            }
        }
    }
    if (passes == 1) return;
    for (int t = tid; t <= count; t += kThreads) {  // the first place whose key is t or more
        int lo = 0, hi = rows;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (keys[mid] < t)
                lo = mid + 1;
            else
                hi = mid;
        }
        ptr[t] = lo;
    }
}

// Keys of a pass: from the types, or as the pass before left them.
struct Source {
    const int64_t* types;
    const int *keys, *numbers;
    int count;
    __device__ __forceinline__ int key(int at) const { return types ? key_of(types[at], count) : keys[at]; }
    __device__ __forceinline__ int number(int at) const { return types ? at : numbers[at]; }
};

// counts: [blocks, kDigits]. Each block has the next `span` rows.
__global__ __launch_bounds__(kThreads) void count_digits(Source from, int rows, int span, int shift, int* counts) {
    __shared__ int count[kDigits];
    const int tid = threadIdx.x;
    if (tid < kDigits) count[tid] = 0;
    __syncthreads();
    const int first = blockIdx.x * span, end = first + min(rows - first, span);
    for (int base = first; base < end; base += kThreads) {
        const int at = base + tid;
        const int digit = at < end ? from.key(at) >> shift & (kDigits - 1) : 0;
        const uint64_t same = same_digit(digit, at < end);
        if (at < end && lanes_before(same) == 0) atomicAdd(&count[digit], __popcll(same));
    }
    __syncthreads();
    if (tid < kDigits) counts[blockIdx.x * kDigits + tid] = count[tid];
}

// Places a block's rows by digit. Keys go on to the next pass, if there is one; a pass over all bits leaves ptr too.
__global__ __launch_bounds__(kThreads) void place_rows(Source from, int rows, int span, int shift, const int* counts, int blocks,
                                                       int* keys, int* numbers, int* ptr, int count) {
    __shared__ int next[kDigits], round[kWaves][kDigits], wave_sums[4], part[4][2][kDigits];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    {
        // four shares of the blocks are added up side by side
        const int d = tid & (kDigits - 1), share = tid / kDigits;
        int total = 0, mine = 0;
#pragma unroll 8
        for (int b = share; b < blocks; b += 4) {
            const int c = counts[b * kDigits + d];
            total += c;
            mine += b < (int)blockIdx.x ? c : 0;
        }
        part[share][0][d] = total, part[share][1][d] = mine;
    }
    __syncthreads();
    int total = 0, mine = 0;
    if (tid < kDigits)
        for (int s = 0; s < 4; ++s) total += part[s][0][tid], mine += part[s][1][tid];
    const int before = before_digit(total, wave_sums);
    if (tid < kDigits) {
        next[tid] = before + mine;
        if (ptr && blockIdx.x == 0 && tid <= count) ptr[tid] = before;
    }
    const int first = blockIdx.x * span, end = first + min(rows - first, span);
    for (int base = first; base < end; base += kThreads) {
        __syncthreads();
        for (int i = tid; i < kWaves * kDigits; i += kThreads) ((int*)round)[i] = 0;
        __syncthreads();
        const int at = base + tid;
        const bool valid = at < end;
        const int key = valid ? from.key(at) : 0, number = valid ? from.number(at) : 0;
        const int digit = key >> shift & (kDigits - 1);
        const uint64_t same = same_digit(digit, valid);
        const int rank = lanes_before(same);
        if (valid && rank == 0) round[wave][digit] = __popcll(same);
        __syncthreads();
        if (tid < kDigits) {
            int sum = next[tid];
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const int c = round[w][tid];
                round[w][tid] = sum;
                sum += c;
            }
            next[tid] = sum;
        }
        __syncthreads();
        if (valid) {
            const int to = round[wave][digit] + rank;
            numbers[to] = number;
            if (keys) keys[to] = key;
        }
    }
}

// ptr of many types: the first place whose key is t or more.
__global__ __launch_bounds__(256) void find_types(const int* keys, int rows, int count, int* ptr) {
    const int t = blockIdx.x * 256 + threadIdx.x;
    if (t > count) return;
    int lo = 0, hi = rows;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (keys[mid] < t)
            lo = mid + 1;
        else
            hi = mid;
    }
    ptr[t] = lo;
}

// ---------------------------------------------------------------------------
// rows of a table by type
// ---------------------------------------------------------------------------

// out[i] = scale table[types[i]], 0 where there is no type. V elements (16 bytes where everything is aligned, else one) at a
// time; `across` lanes, a power of two, share a row and have kLookups rows each, requested together. Bound by memory, or a launch.
constexpr int kLookups = 4;

template <typename T, int V>
__global__ __launch_bounds__(256) void lookup(const T* table, int64_t table_row, const int64_t* types, int64_t rows, int count,
                                              int channels, int across, float scale, T* out) {
    typedef T vec __attribute__((ext_vector_type(V)));
    const int lane = threadIdx.x & (across - 1), groups = 256 / across;
    const int64_t row0 = (int64_t)blockIdx.x * groups * kLookups + threadIdx.x / across;
    const T* from[kLookups];
    bool known[kLookups];
#pragma unroll
    for (int i = 0; i < kLookups; ++i) {
        const int64_t row = row0 + i * groups, type = row < rows ? types[row] : -1;
        known[i] = type >= 0 && type < count;
        from[i] = table + (known[i] ? type : 0) * table_row;
    }
    for (int c = lane * V; c < channels; c += across * V) {
        vec x[kLookups];
#pragma unroll
        for (int i = 0; i < kLookups; ++i) {
            x[i] = (T)0;
            if (known[i]) x[i] = *(const vec*)(from[i] + c);
        }
#pragma unroll
        for (int i = 0; i < kLookups; ++i) {
            const int64_t row = row0 + i * groups;
            if (row >= rows) break;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float y = known[i] ? (float)x[i][e] * scale : 0.0f;
                asm("" : "+v"(y));  // (a product of 32 bits, as elsewhere, not one that is rounded to 16 at once)
                x[i][e] = (T)y;
            }
            *(vec*)(out + row * channels + c) = x[i];
        }
    }
}

// ---------------------------------------------------------------------------
// sums of rows by type
// ---------------------------------------------------------------------------

// out[t] = scale sum_{i of type t} rows[i], in 32 bits and in an order that the index alone decides. A type of up to kChunk rows is
// summed by a group of lanes of its own, longer ones in two steps: chunks of kChunk places of the index sum what they hold of
// a longer type (a chunk holds parts of two at most: the one that it begins in and the one that it ends in), and the chunk in
// which a longer type begins adds up the chunks' sums.
// Bound by memory and a chain of waits (place, type, bounds, row): 20 000 rows of 512 floats, 89 types of which one has 12 400,
// 14 us and 9 for the long ones' join; 16 411 rows of 1 024, 32 003 types, bf16, 20 (98 MB, 4.8 TB/s) and 8. (Chunks of 64 rows:
// 16 and 7, 20 and 5. The join with a few groups of lanes, each with many chunks: 28.)
constexpr int kChunk = 32;

struct Sums {
    const void* rows;
    int64_t row, part;  // strides of a row and of its parts, which are summed too
    void* out;
    const int64_t* types;
    const int *order, *ptr;
    float* partial;  // [chunks, 2, channels]
    int count, n, parts, channels;
    float scale;
};

// The row at a place of the index. (An index that was not made here is kept inside the rows.)
__device__ __forceinline__ int row_at(const int* order, int at, int n) {
    const int row = order[at];
    return (unsigned)row < (unsigned)n ? row : 0;
}

template <typename T, int V>
struct Row {
    typedef T vec __attribute__((ext_vector_type(V)));
    float x[V];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = 0;
    }
    __device__ __forceinline__ void add(const vec& y) {
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] += (float)y[e];
    }
};

// Sum of the rows at places lo .. hi of the index for the V channels from c on; groups of lanes with the same channels take
// every `groups`-th row.
template <typename T, int V>
__device__ __forceinline__ Row<T, V> sum_places(const Sums& s, int lo, int hi, int c, int group, int groups) {
    typedef typename Row<T, V>::vec vec;
    Row<T, V> sum;
    sum.clear();
    const T* base = (const T*)s.rows + c;
    if (s.parts == 1) {
        int at = lo + group;
        for (; at + 7 * groups < hi; at += 8 * groups) {
            vec y[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) y[u] = *(const vec*)(base + row_at(s.order, at + u * groups, s.n) * s.row);
#pragma unroll
            for (int u = 0; u < 8; ++u) sum.add(y[u]);
        }
        for (; at < hi; at += groups) sum.add(*(const vec*)(base + row_at(s.order, at, s.n) * s.row));
    } else {
        for (int at = lo + group; at < hi; at += groups) {
            const T* from = base + row_at(s.order, at, s.n) * s.row;
            for (int p = 0; p < s.parts; ++p) sum.add(*(const vec*)(from + p * s.part));
        }
    }
    return sum;
}

template <typename T, int V>
__device__ __forceinline__ void store_sum(const Sums& s, const Row<T, V>& sum, int t, int c) {
    typename Row<T, V>::vec y;
#pragma unroll
    for (int e = 0; e < V; ++e) y[e] = (T)(sum.x[e] * s.scale);
    *(typename Row<T, V>::vec*)((T*)s.out + (int64_t)t * s.channels + c) = y;
}

// Threads of a block: `across` lanes next to each other for the channels (V each), 256 / across groups.
template <typename T, int V>
__device__ __forceinline__ void join_groups(Row<T, V>& sum, float* lds, int across, int lane, int group, int groups) {
    for (int half = groups >> 1; half; half >>= 1) {
        __syncthreads();
        if (group >= half && group < 2 * half)
#pragma unroll
            for (int e = 0; e < V; ++e) lds[((group - half) * across + lane) * V + e] = sum.x[e];
        __syncthreads();
        if (group < half)
#pragma unroll
            for (int e = 0; e < V; ++e) sum.x[e] += lds[(group * across + lane) * V + e];
    }
}

// The first blocks have a type for each of their groups of lanes, kTypes of them one after the other; the rest a chunk each.
// blockIdx.y: channels.
constexpr int kTypes = 4;

template <typename T, int V>
__global__ __launch_bounds__(256) void sum_types(Sums s, int across, int type_blocks) {
    __shared__ float lds[128 * V];
    const int lane = threadIdx.x % across, group = threadIdx.x / across, groups = 256 / across;
    const int c = (blockIdx.y * across + lane) * V;
    const bool valid = c < s.channels;
    if ((int)blockIdx.x < type_blocks) {
        if (!valid) return;
        const int t0 = (blockIdx.x * groups + group) * kTypes;
        int begin[kTypes + 1];
#pragma unroll
        for (int i = 0; i <= kTypes; ++i) begin[i] = t0 < s.count ? s.ptr[min(t0 + i, s.count)] : 0;
#pragma unroll
        for (int i = 0; i < kTypes; ++i) {
            const int lo = max(begin[i], 0), hi = min(begin[i + 1], s.n);
            if (t0 + i >= s.count || hi - lo > kChunk) continue;
            const Row<T, V> sum = sum_places<T, V>(s, lo, hi, c, 0, 1);
            store_sum(s, sum, t0 + i, c);
        }
        return;
    }
    const int chunk = blockIdx.x - type_blocks, first = chunk * kChunk, last = min(s.n, s.ptr[s.count]);
    if (first >= last) return;
    const int end = min(first + kChunk, last);
    const int ta = key_of(s.types[row_at(s.order, first, s.n)], s.count), tb = key_of(s.types[row_at(s.order, end - 1, s.n)], s.count);
    for (int side = 0; side < 2; ++side) {
        const int t = side ? tb : ta;
        if (t >= s.count || (side && tb == ta)) continue;
        const int lo = max(s.ptr[t], 0), hi = min(s.ptr[t + 1], s.n);
        if (hi - lo <= kChunk) continue;
        Row<T, V> sum;
        sum.clear();
        if (valid) sum = sum_places<T, V>(s, max(lo, first), min(hi, end), c, group, groups);
        join_groups(sum, lds, across, lane, group, groups);
        if (valid && group == 0)
#pragma unroll
            for (int e = 0; e < V; ++e) s.partial[((int64_t)chunk * 2 + side) * s.channels + c + e] = sum.x[e];
    }
}

// A block for each chunk: the longer types that begin in it. Few channels a block and many groups, each with a few of the
// chunks: what a long type waits for is one read after the other.
template <typename T, int V>
__global__ __launch_bounds__(256) void join_chunks(Sums s, int across) {
    __shared__ float lds[128 * V];
    const int lane = threadIdx.x % across, group = threadIdx.x / across, groups = 256 / across;
    const int c = (blockIdx.y * across + lane) * V;
    const bool valid = c < s.channels;
    const int chunk = blockIdx.x, first = chunk * kChunk, last = min(s.n, s.ptr[s.count]);
    if (first >= last) return;
    const int end = min(first + kChunk, last);
    const int ta = key_of(s.types[row_at(s.order, first, s.n)], s.count), tb = key_of(s.types[row_at(s.order, end - 1, s.n)], s.count);
    for (int side = 0; side < 2; ++side) {
        const int t = side ? tb : ta;
        if (t >= s.count || (side && tb == ta)) continue;
        const int lo = max(s.ptr[t], 0), hi = min(s.ptr[t + 1], s.n);
        if (hi - lo <= kChunk || lo < first) continue;
        const int chunks = (hi - 1) / kChunk - chunk + 1;
        Row<T, V> sum;
        sum.clear();
        // the first chunk's part is its end's, unless the type begins with the chunk; all others begin with the type
        if (valid)
#pragma unroll 4
            for (int k = group; k < chunks; k += groups) {
                const float* from = s.partial + ((int64_t)(chunk + k) * 2 + (k == 0 ? side : 0)) * s.channels + c;
#pragma unroll
                for (int e = 0; e < V; ++e) sum.x[e] += from[e];
            }
        join_groups(sum, lds, across, lane, group, groups);
        if (valid && group == 0) store_sum(s, sum, t, c);
    }
}

}  // namespace row_groups
#endif
