// The embedding of codebook tokens and its gradient (splat_labels.h).
//
// Lookup: out[i] = s T[t_i], a gather of whole rows, bound by the bytes of `out` (the table's
// rows are re-read from L2): 500,000 rows of 256 bf16 in 58 us, 4.4 TB/s written.
//
// Gradient: dT[v] = s sum_{i: t_i = v} dOut[i], without atomics on the sums, so that they have one
// order whatever the scheduling, in one of two ways:
//  - up to kFewTokens tokens: one kernel whose blocks each own a range of entries, pick their tokens
//    out of the whole list, order them by entry and position in shared memory and sum the rows
//    (latency: a sort of the list alone is four launches; 20,000 rows of 64 f32 in 13 us);
//  - more: the (token, position) pairs go through the renderer's stable radix sort (sort.cu), each
//    block sums the runs of a fixed stretch of the sorted list while dOut's rows stream past once
//    (bound by those bytes), and a token whose run crosses stretches is joined from their partial
//    sums, in order, by a second kernel. The kernel that makes the pairs zeroes the gradient first,
//    for the tokens nobody has. 500,000 rows of 256 bf16 in 88 us, 48 of them for the rows (5.4 TB/s).
#include <algorithm>
#include <new>

#include "elements.cuh"
#include "kernels.h"
#include "objects.h"

using namespace splat;

struct sp_embedding {
    sp_context* ctx = nullptr;
    uint64_t entries = 0;
    uint32_t dim = 0;
    sp_element element = SP_F32;
    uint64_t max_tokens = 0;
    SortPlan plan{};
    uint32_t sequence = 0;
    std::vector<void*> allocations;
    DeviceMeta* meta = nullptr;
    uint32_t* keys[2] = {nullptr, nullptr};
    uint32_t* values[2] = {nullptr, nullptr};
    uint32_t* histograms = nullptr;  // kSortMaxPasses * kSortRadix digit counts, then the tickets
    unsigned long long* lookback = nullptr;
    float* partials = nullptr;
};

namespace {

constexpr int kThreads = 256;
constexpr int kEmitItems = 8;
constexpr int kLookupRows = 4;   // rows in flight per thread
constexpr int kPieceRows = 4;    // rows in flight per thread while summing: 8 and 16 cost more in occupancy
constexpr int kFewRows = 4;      // ... in blocks of 1024 threads, 64 registers each
constexpr int kMinLanesLog2 = 2; // at least 4 threads a row while summing
constexpr uint32_t kShortPiece = 16, kLongPiece = 128, kMostStretch = 2048;
constexpr uint32_t kGroups = 148 * 16;         // of pieces, where there are enough tokens
constexpr uint32_t kFewTokens = 32768;         // 32 warps x 32 x 32 lanes
constexpr uint64_t kFewReads = 1ull << 24;     // token reads of all blocks together
constexpr uint32_t kFewThreads = 1024, kMostOwned = 512, kLongRun = 64;

// Sorted positions per group of threads, a power of two: long pieces make fewer partial sums (the
// gradient of 500,000 bf16 rows of 256: 102 us in pieces of 64, 94 us of 128), short ones give a small
// list groups enough to fill the SMs.
uint32_t piece_length(uint64_t count, int lanes_log2) {
    uint32_t piece = kShortPiece;
    while (piece < kLongPiece && count >= (uint64_t)piece * 2 * kGroups) piece *= 2;
    return std::min(piece, kMostStretch / ((uint32_t)kThreads >> lanes_log2));
}

// `lanes` threads (a power of two, at most 32) move one row, N elements at a time; kLookupRows rows
// a thread, the next ones' tokens read meanwhile. The rows are written past the caches' usual
// residents (the table stays in L2).
template <typename T, int N>
__global__ void __launch_bounds__(kThreads) k_lookup(const T* __restrict__ table, int64_t table_stride,
                                                     const void* __restrict__ tokens, int wide, uint64_t count,
                                                     uint64_t entries, uint32_t dim, float scale,
                                                     T* __restrict__ out, int64_t out_stride, int lanes_log2) {
    chain_enter();
    const uint32_t lanes = 1u << lanes_log2, lane = threadIdx.x & (lanes - 1);
    const uint64_t rows_per_pass = kThreads >> lanes_log2;
    const uint32_t packs = dim / N;
    const uint64_t step = (uint64_t)gridDim.x * rows_per_pass * kLookupRows;
    uint64_t row = (uint64_t)blockIdx.x * rows_per_pass * kLookupRows + (threadIdx.x >> lanes_log2);
    int64_t next[kLookupRows];
    auto read_tokens = [&](uint64_t from) {
#pragma unroll
        for (int k = 0; k < kLookupRows; ++k) {
            const uint64_t i = from + k * rows_per_pass;
            next[k] = i < count ? index_at(tokens, wide, i, entries) : -1;
        }
    };
    read_tokens(row);
    for (; row < count; row += step) {
        int64_t token[kLookupRows];
#pragma unroll
        for (int k = 0; k < kLookupRows; ++k) token[k] = next[k];
        read_tokens(row + step);
        for (uint32_t p = lane; p < packs; p += lanes) {
            Pack<T, N> v[kLookupRows];
#pragma unroll
            for (int k = 0; k < kLookupRows; ++k)
                if (token[k] >= 0) v[k] = load_pack<T, N>(table + token[k] * table_stride + (uint64_t)p * N);
#pragma unroll
            for (int k = 0; k < kLookupRows; ++k) {
                const uint64_t i = row + k * rows_per_pass;
                if (i >= count) continue;
                float scaled[N];
#pragma unroll
                for (int j = 0; j < N; ++j) scaled[j] = token[k] >= 0 ? v[k].get(j) * scale : 0.0f;
                Pack<T, N> o;
                o.set(scaled);
                store_streaming(out + (int64_t)i * out_stride + (uint64_t)p * N, o);
            }
        }
    }
}

// The sort's input: key = token (entries for none, which sorts last), value = position, with every
// pass's digit histogram; block 0 sets the sort's bookkeeping. The device status is left alone:
// it stays raised until it is read. The blocks also zero the gradient's `zero_rows` rows of `zero_units`
// U each (dense rows are one), so that entries without tokens need no look at the sorted list.
template <typename U>
__global__ void __launch_bounds__(kThreads) k_emit_tokens(const void* __restrict__ tokens, int wide, uint32_t count,
                                                          uint64_t entries, int passes, DeviceMeta* meta,
                                                          uint32_t* __restrict__ keys, uint32_t* __restrict__ values,
                                                          uint32_t* __restrict__ histograms,
                                                          U* __restrict__ zero, uint64_t zero_rows,
                                                          uint64_t zero_units, int64_t zero_stride) {
    chain_enter();
    __shared__ uint32_t hist[4][kSortRadix];
    for (int p = 0; p < passes; ++p) hist[p][threadIdx.x] = 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        meta->count = count;
        meta->partitions = (count + kSortShortPartition - 1) / kSortShortPartition;
        meta->key_shift = 0;
        meta->key_base = 0;
        meta->passes = (uint32_t)passes;
        meta->first_buffer = 0;
    }
    const uint64_t thread = (uint64_t)blockIdx.x * kThreads + threadIdx.x, threads = (uint64_t)gridDim.x * kThreads;
    if (zero_rows == 1) {
        for (uint64_t i = thread; i < zero_units; i += threads) zero[i] = U{};
    } else {
        for (uint64_t row = thread / 32; row < zero_rows; row += threads / 32)
            for (uint64_t i = lane_id(); i < zero_units; i += 32) zero[(int64_t)row * zero_stride + i] = U{};
    }
    __syncthreads();
    const uint32_t base = blockIdx.x * kThreads * kEmitItems;
#pragma unroll
    for (int k = 0; k < kEmitItems; ++k) {
        const uint32_t i = base + k * kThreads + threadIdx.x;
        if (i >= count) break;
        const int64_t token = index_at(tokens, wide, i, entries);
        const uint32_t key = token < 0 ? (uint32_t)entries : (uint32_t)token;
        keys[i] = key;
        values[i] = i;
        for (int p = 0; p < passes; ++p) atomicAdd(&hist[p][(key >> (8 * p)) & 255u], 1u);
    }
    __syncthreads();
    for (int p = 0; p < passes; ++p) {
        const uint32_t c = hist[p][threadIdx.x];
        if (c) atomicAdd(histograms + p * kSortRadix + threadIdx.x, c);
    }
}

// N columns of a row of sums, scaled and rounded.
template <typename T, int N>
__device__ __forceinline__ void store_row(T* to, const float (&sum)[N], float scale, bool packed) {
    if (packed) {
        float scaled[N];
#pragma unroll
        for (int j = 0; j < N; ++j) scaled[j] = sum[j] * scale;
        Pack<T, N> o;
        o.set(scaled);
        store_pack(to, o);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) to[j] = from_float<T>(sum[j] * scale);
    }
}

// A stretch of the sorted list per block, a piece of it per group of `lanes` threads, N columns a
// thread (blockIdx.y: the next lanes * N columns). A run inside its piece is a token's whole sum and
// is written out. A run over several pieces is added up from their partial sums in shared memory by
// the piece it begins in; one that crosses stretches leaves partial sums in memory: slot 0 of the
// stretch for a run that began before it, slot 1 for one that begins inside and goes on.
template <typename T, int N>
__global__ void __launch_bounds__(kThreads)
    k_sum_pieces(const uint32_t* __restrict__ keys, const uint32_t* __restrict__ positions, uint32_t count,
                 uint32_t entries, const T* __restrict__ upstream, int64_t upstream_stride, uint32_t dim, float scale,
                 T* __restrict__ out, int64_t out_stride, int out_packed, float* __restrict__ partials,
                 uint32_t partial_stride, uint32_t piece, int lanes_log2, const DeviceMeta* __restrict__ meta) {
    chain_enter();
    if (meta->status != 0) return;  // the list may be out of order: k_join_pieces writes NaN
    __shared__ uint32_t s_key[kMostStretch + 2];  // with the neighbours on both sides
    __shared__ alignas(16) uint32_t s_position[kMostStretch];
    __shared__ float s_part[2][kThreads][N];
    constexpr uint32_t kNobody = 0xffffffffu;
    const uint32_t lanes = 1u << lanes_log2, groups = kThreads >> lanes_log2;
    const uint32_t group = threadIdx.x >> lanes_log2, stretch = groups * piece;
    const uint64_t first = (uint64_t)blockIdx.x * stretch;
    for (uint32_t i = threadIdx.x; i < stretch + 2; i += kThreads) {
        const uint64_t at = first + i;  // of the list, plus 1
        s_key[i] = at >= 1 && at <= count ? keys[at - 1] : kNobody;
        if (i < stretch && at < count) s_position[i] = positions[at];
    }
    __syncthreads();
    const uint32_t* key = s_key + 1;
    const uint32_t here = (uint32_t)min((uint64_t)stretch, count - first);
    const uint32_t column = (blockIdx.y * lanes + (threadIdx.x & (lanes - 1))) * N;
    const bool inside = column < dim;
    const uint32_t begin = group * piece, end = min(begin + piece, here);
    T* const out_column = out + column;
    bool tail = false;  // the last run begins here and goes on
    if (inside && begin < here) {
        float acc[N];
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] = 0.0f;
        uint32_t current = key[begin];
        bool from_before = key[(int)begin - 1] == current;
        // Rows of a batch that is whole and has tokens throughout (the list is sorted) need no tests.
        auto load = [&](uint32_t i, Pack<T, N> (&v)[kPieceRows]) {
            if (i + kPieceRows <= end && key[i + kPieceRows - 1] < entries) {
                uint32_t at[kPieceRows];
#pragma unroll
                for (int k = 0; k < kPieceRows; k += 4) {
                    const uint4 four = *reinterpret_cast<const uint4*>(s_position + i + k);
                    at[k] = four.x, at[k + 1] = four.y, at[k + 2] = four.z, at[k + 3] = four.w;
                }
#pragma unroll
                for (int k = 0; k < kPieceRows; ++k)
                    v[k] = load_pack<T, N>(upstream + (int64_t)at[k] * upstream_stride + column);
            } else {
#pragma unroll
                for (int k = 0; k < kPieceRows; ++k)
                    if (i + k < end && key[i + k] < entries)
                        v[k] = load_pack<T, N>(upstream + (int64_t)s_position[i + k] * upstream_stride + column);
            }
        };
        auto add = [&](uint32_t i, const Pack<T, N> (&v)[kPieceRows]) {
            if (i + kPieceRows <= end && key[i + kPieceRows - 1] == current) {
                if (current >= entries) return;
#pragma unroll
                for (int k = 0; k < kPieceRows; ++k)
#pragma unroll
                    for (int j = 0; j < N; ++j) acc[j] += v[k].get(j);
                return;
            }
#pragma unroll
            for (int k = 0; k < kPieceRows; ++k) {
                if (i + k >= end) break;
                const uint32_t now = key[i + k];
                if (now != current) {
                    if (from_before) {
#pragma unroll
                        for (int j = 0; j < N; ++j) s_part[0][threadIdx.x][j] = acc[j];
                    } else if (current < entries) {
                        store_row<T, N>(out_column + (int64_t)current * out_stride, acc, scale, out_packed);
                    }
                    current = now;
                    from_before = false;
#pragma unroll
                    for (int j = 0; j < N; ++j) acc[j] = 0.0f;
                }
                if (now < entries) {
#pragma unroll
                    for (int j = 0; j < N; ++j) acc[j] += v[k].get(j);
                }
            }
        };
        for (uint32_t i = begin; i < end; i += kPieceRows) {
            Pack<T, N> v[kPieceRows];
            load(i, v);
            add(i, v);
        }
        const bool goes_on = key[end] == current;
        if (from_before || goes_on) {
            tail = !from_before;
#pragma unroll
            for (int j = 0; j < N; ++j) s_part[tail ? 1 : 0][threadIdx.x][j] = acc[j];
        } else if (current < entries) {
            store_row<T, N>(out_column + (int64_t)current * out_stride, acc, scale, out_packed);
        }
    }
    __syncthreads();
    if (!inside || begin >= here) return;
    // The run that ends piece `from` (its sum so far in `slot`), through the pieces it goes on over.
    auto follow = [&](uint32_t from, int slot, bool began_before) {
        const uint32_t token = key[min((from + 1) * piece, here) - 1];
        if (token >= entries) return;
        float sum[N];
#pragma unroll
        for (int j = 0; j < N; ++j) sum[j] = s_part[slot][threadIdx.x][j];
        uint32_t at = min((from + 1) * piece, here);  // where the run's next row would be
        for (uint32_t next = from + 1; at < here && key[at] == token; ++next) {
#pragma unroll
            for (int j = 0; j < N; ++j) sum[j] += s_part[0][threadIdx.x + (next - group) * lanes][j];
            at = min((next + 1) * piece, here);
            if (key[at - 1] != token) break;  // it ended inside piece `next`
        }
        const bool beyond = at == here && key[here - 1] == token && key[here] == token;
        if (!began_before && !beyond) {
            store_row<T, N>(out_column + (int64_t)token * out_stride, sum, scale, out_packed);
        } else {
            float* to = partials + ((uint64_t)blockIdx.x * 2 + (began_before ? 0 : 1)) * partial_stride + column;
#pragma unroll
            for (int j = 0; j < N; ++j) to[j] = sum[j];
        }
    };
    if (group == 0 && key[-1] == key[0]) {
        if (key[end - 1] == key[0]) {
            follow(0, 0, true);  // all of the first piece, and perhaps more
        } else if (key[0] < entries) {
            float* to = partials + (uint64_t)blockIdx.x * 2 * partial_stride + column;
#pragma unroll
            for (int j = 0; j < N; ++j) to[j] = s_part[0][threadIdx.x][j];
        }
    }
    if (tail) follow(group, 1, false);
}

// The runs that cross stretches: a warp looks whether one begins in its stretch and goes on, finds in
// how many stretches (the sorted list's keys at their starts), and adds up their partial sums in order,
// 4 columns a lane; a run with more than kWarpParts of them is joined by the block's eight warps
// together. blockIdx.y takes every gridDim.y-th 128 columns. If the sort failed, NaN throughout.
constexpr uint32_t kJoinWarps = kThreads / 32, kWarpParts = 16;
template <typename T>
__global__ void __launch_bounds__(kThreads)
    k_join_pieces(const uint32_t* __restrict__ keys, uint32_t count, uint32_t entries, uint32_t dim, float scale,
                  T* __restrict__ out, int64_t out_stride, const float* __restrict__ partials, uint32_t partial_stride,
                  uint32_t stretch, const DeviceMeta* __restrict__ meta) {
    chain_enter();
    __shared__ float4 shared[kJoinWarps][32];
    __shared__ uint2 long_runs[kJoinWarps];  // the stretch it begins in, its partial sums
    const uint32_t warp = threadIdx.x / 32, lane = lane_id();
    if (meta->status != 0) {
        const uint64_t block = (uint64_t)blockIdx.y * gridDim.x + blockIdx.x, blocks = (uint64_t)gridDim.x * gridDim.y;
        for (uint64_t row = block * kJoinWarps + warp; row < entries; row += blocks * kJoinWarps)
            for (uint32_t c = lane; c < dim; c += 32) out[(int64_t)row * out_stride + c] = from_float<T>(__int_as_float(0x7fffffff));
        return;
    }
    auto store = [&](uint32_t v, uint32_t column, float4 sum) {
        const float s[4] = {sum.x, sum.y, sum.z, sum.w};
        T* to = out + (int64_t)v * out_stride + column;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (column + j < dim) to[j] = from_float<T>(s[j] * scale);
    };
    // Partial sums p0..p1 of the run that begins in stretch `first`: its slot 1, then the next ones' slot 0.
    auto sum_of = [&](uint32_t first, uint32_t p0, uint32_t p1, uint32_t column) {
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
        for (uint32_t p = p0; p < p1; ++p) {
            const uint64_t slot = (uint64_t)(first + p) * 2 + (p == 0 ? 1 : 0);
            const float4 v = *reinterpret_cast<const float4*>(partials + slot * partial_stride + column);
            sum.x += v.x;
            sum.y += v.y;
            sum.z += v.z;
            sum.w += v.w;
        }
        return sum;
    };
    const uint32_t stretches = (count + stretch - 1) / stretch, mine = blockIdx.x * kJoinWarps + warp;
    uint32_t token = 0, parts = 0;
    if (mine + 1 < stretches) {
        const uint64_t next = (uint64_t)(mine + 1) * stretch;
        token = keys[next];
        const bool begins = mine == 0 || keys[next - stretch - 1] != token;
        if (token < entries && keys[next - 1] == token && begins) parts = 2;
    }
    // How far it goes: the last of `found` stretches is one of the run's; those from `end` on are not.
    // (The same in all of a warp's lanes.)
    if (parts != 0) {
        uint32_t found = mine + 1, end = stretches, step = 1;
        while (end - found > 1) {
            const uint64_t at = (uint64_t)found + (uint64_t)(lane + 1) * step;
            const bool in = at < end && keys[at * stretch] == token;
            const uint32_t many = __popc(__ballot_sync(0xffffffffu, in));  // the list is sorted: the first lanes
            const uint64_t beyond = (uint64_t)found + (uint64_t)(many + 1) * step;
            found += many * step;
            if (many < 32) end = (uint32_t)min((uint64_t)end, beyond);
            step = max((end - found) / 32, 1u);
        }
        parts = found - mine + 1;
    }
    if (lane == 0) long_runs[warp] = make_uint2(mine, parts > kWarpParts ? parts : 0u);
    const uint32_t first_column = blockIdx.y * 128 + lane * 4, step = gridDim.y * 128;
    if (parts != 0 && parts <= kWarpParts)
        for (uint32_t c = first_column; c < dim; c += step) store(token, c, sum_of(mine, 0, parts, c));
    __syncthreads();
    for (uint32_t k = 0; k < kJoinWarps; ++k) {
        const uint32_t first = long_runs[k].x, n = long_runs[k].y;
        if (n == 0) continue;
        const uint32_t p0 = (uint32_t)((uint64_t)n * warp / kJoinWarps);
        const uint32_t p1 = (uint32_t)((uint64_t)n * (warp + 1) / kJoinWarps);
        const uint32_t long_token = keys[(uint64_t)(first + 1) * stretch];
        for (uint32_t c0 = blockIdx.y * 128; c0 < dim; c0 += step) {
            const uint32_t c = c0 + lane * 4;
            if (c < dim) shared[warp][lane] = sum_of(first, p0, p1, c);
            __syncthreads();
            if (warp == 0 && c < dim) {
                float4 sum = shared[0][lane];
                for (uint32_t w = 1; w < kJoinWarps; ++w) {
                    const float4 v = shared[w][lane];
                    sum.x += v.x;
                    sum.y += v.y;
                    sum.z += v.z;
                    sum.w += v.w;
                }
                store(long_token, c, sum);
            }
            __syncthreads();
        }
    }
}

// Up to kFewTokens tokens: block b owns entries [b owned, (b + 1) owned). Each warp reads 1/32 of the
// tokens into registers and counts its entries' ones; the counts give every (entry, warp) its place in
// a list of positions in shared memory, ordered by entry and then position; the rows are summed from
// it, a run of at most kLongRun by one group of `lanes` threads in order, a longer one by all groups in
// equal parts, joined in order. Where the entries make too few blocks for the SMs, blockIdx.y takes
// every gridDim.y-th tile of columns.
template <typename T, int N>
__global__ void __launch_bounds__(kFewThreads)
    k_sum_few(const void* __restrict__ tokens, int wide, uint32_t count, uint64_t entries, uint32_t owned,
              const T* __restrict__ upstream, int64_t upstream_stride, uint32_t dim, float scale, T* __restrict__ out,
              int64_t out_stride, int out_packed, int lanes_log2) {
    chain_enter();
    constexpr uint32_t kWarps = kFewThreads / 32;
    extern __shared__ float4 few_smem[];
    __shared__ uint32_t start[kMostOwned + 1], warp_sums[kWarps], longs[kMostOwned], long_count;
    float* s_part = reinterpret_cast<float*>(few_smem);  // [kFewThreads][N]
    uint16_t* placed = reinterpret_cast<uint16_t*>(s_part + kFewThreads * N);  // [kWarps][owned]
    uint16_t* order = placed + kWarps * owned;                                 // [count], then the entries
    const uint32_t t = threadIdx.x, warp = t / 32, lane = lane_id();
    const uint32_t section = (count + kFewThreads - 1) / kFewThreads * 32;  // of the tokens, per warp
    const int64_t first_entry = (int64_t)blockIdx.x * owned;

    // The warp's tokens as entries of this block (kMostOwned: another block's).
    uint16_t* entry_of = order + count + warp * section;
#pragma unroll 8
    for (uint32_t k = lane; k < section; k += 32) {
        const uint32_t i = warp * section + k;
        uint32_t entry = kMostOwned;
        if (i < count) {
            const int64_t v = index_at(tokens, wide, i, entries) - first_entry;
            if (v >= 0 && v < (int64_t)owned) entry = (uint32_t)v;
        }
        entry_of[k] = (uint16_t)entry;
    }
    for (uint32_t i = t; i < kWarps * owned; i += kFewThreads) placed[i] = 0;
    if (t == 0) long_count = 0;
    __syncthreads();
    const uint32_t below = (1u << lane) - 1u;
    // place(entry, at, position): the warp's tokens, each `at` its next place in its entry, equal ones in
    // lane order.
    uint16_t* mine = placed + warp * owned;
    auto for_each_place = [&](auto&& place) {
#pragma unroll 2
        for (uint32_t k = lane; k < section; k += 32) {
            const uint32_t entry = entry_of[k];
            const bool here = entry < kMostOwned;
            if (!__any_sync(0xffffffffu, here)) continue;
            const uint32_t peers = __match_any_sync(0xffffffffu, entry);
            const uint32_t before = here ? mine[entry] : 0;
            __syncwarp();
            if (here) {
                if ((peers & below) == 0) mine[entry] = (uint16_t)(before + __popc(peers));
                place(entry, before + __popc(peers & below), warp * section + k);
            }
            __syncwarp();
        }
    };
    for_each_place([](uint32_t, uint32_t, uint32_t) {});
    __syncthreads();
    // Entry e's total, and in its column the running counts over the warps (a warp per entry); then the
    // entries' scan.
    auto scan = [&](uint32_t v) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t up = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= (uint32_t)o) v += up;
        }
        return v;
    };
    for (uint32_t e = warp; e < owned; e += kWarps) {
        const uint32_t c = placed[lane * owned + e], inclusive = scan(c);
        placed[lane * owned + e] = (uint16_t)(inclusive - c);
        if (lane == 31) start[e] = inclusive;
    }
    __syncthreads();
    const uint32_t total = t < owned ? start[t] : 0, inclusive = scan(total);
    if (lane == 31) warp_sums[warp] = inclusive;
    __syncthreads();
    const uint32_t before_warp = scan(warp_sums[lane]) - warp_sums[lane];
    const uint32_t offset = __shfl_sync(0xffffffffu, before_warp, warp);
    if (t < owned) {
        start[t] = offset + inclusive - total;
        if (t == owned - 1) start[owned] = offset + inclusive;
    }
    __syncthreads();
    for_each_place([&](uint32_t entry, uint32_t at, uint32_t position) { order[start[entry] + at] = (uint16_t)position; });
    __syncthreads();

    const uint32_t lanes = 1u << lanes_log2, groups = kFewThreads >> lanes_log2, group = t >> lanes_log2;
    const uint32_t entries_here = (uint32_t)min((int64_t)owned, (int64_t)entries - first_entry);
    auto sum_rows = [&](uint32_t from, uint32_t to, uint32_t column, float (&acc)[N]) {
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] = 0.0f;
        for (uint32_t i = from; i < to; i += kFewRows) {
            Pack<T, N> v[kFewRows];
#pragma unroll
            for (int k = 0; k < kFewRows; ++k)
                if (i + k < to) v[k] = load_pack<T, N>(upstream + (int64_t)order[i + k] * upstream_stride + column);
#pragma unroll
            for (int k = 0; k < kFewRows; ++k)
                if (i + k < to) {
#pragma unroll
                    for (int j = 0; j < N; ++j) acc[j] += v[k].get(j);
                }
        }
    };
    const uint32_t first_column = (t & (lanes - 1)) * N, tile = lanes * N;
    // An entry's run goes to a team of groups in equal parts, joined in order: as many groups as there
    // are to each entry, all of them for runs longer than kLongRun a group.
    const uint32_t groups_log2 = 31 - __clz(groups);
    uint32_t usual_log2 = 0;
    while (((uint32_t)2 << usual_log2) * entries_here <= groups) ++usual_log2;
    auto sum_entry = [&](uint32_t e, uint32_t team_log2, bool takes) {
        const uint32_t team = 1u << team_log2, member = group & (team - 1);
        const uint32_t from = takes ? start[e] : 0, n = takes ? start[e + 1] - from : 0;
        for (uint32_t base = blockIdx.y * tile; base < dim; base += gridDim.y * tile) {
            const uint32_t column = base + first_column;
            float acc[N];
            if (takes && column < dim) {
                sum_rows(from + (n * member >> team_log2), from + (n * (member + 1) >> team_log2), column, acc);
                if (member != 0)
#pragma unroll
                    for (int j = 0; j < N; ++j) s_part[t * N + j] = acc[j];
            }
            if (team > 1) __syncthreads();
            if (takes && member == 0 && column < dim) {
                for (uint32_t m = 1; m < team; ++m)
#pragma unroll
                    for (int j = 0; j < N; ++j) acc[j] += s_part[(t + m * lanes) * N + j];
                // A row of nobody's is 0 whatever the scale, as where the sorted list's rows are zeroed.
                store_row<T, N>(out + (first_entry + e) * out_stride + column, acc, n ? scale : 0.0f, out_packed);
            }
            if (team > 1) __syncthreads();
        }
    };
    // The teams' entries, then the long runs that were noted, each by itself: whatever their order.
    const uint32_t teams_log2 = groups_log2 - usual_log2, turns = (entries_here + (1u << teams_log2) - 1) >> teams_log2;
    for (uint32_t k = 0, long_runs = 0; k < turns + long_runs; ++k) {
        const bool all = k >= turns;
        const uint32_t e = all ? longs[k - turns] : (k << teams_log2) + (group >> usual_log2);
        const bool is_long = !all && usual_log2 < groups_log2 && e < entries_here &&
                             start[e + 1] - start[e] > kLongRun << usual_log2;
        if (is_long && (group & ((1u << usual_log2) - 1)) == 0 && (t & (lanes - 1)) == 0)
            longs[atomicAdd(&long_count, 1u)] = e;
        sum_entry(e, all ? groups_log2 : usual_log2, e < entries_here && !is_long);
        if (k + 1 == turns) {
            __syncthreads();
            long_runs = long_count;
        }
    }
}

template <typename T>
sp_status allocate(sp_embedding* e, T** out, uint64_t count) {
    void* p = nullptr;
    SP_CUDA(e->ctx, cudaMalloc(&p, std::max<uint64_t>(count * sizeof(T), 16)));
    e->allocations.push_back(p);
    *out = static_cast<T*>(p);
    return SP_OK;
}

int lanes_log2_for(uint32_t packs, int least = 0) {
    int log2 = least;
    while (log2 < 5 && (1u << log2) < packs) ++log2;
    return log2;
}

sp_status check_rows(sp_context* ctx, const void* p, int64_t stride, uint32_t dim, size_t size, const char* what) {
    SP_REQUIRE(ctx, p != nullptr, SP_ERR_INVALID, std::string("null ") + what);
    SP_REQUIRE(ctx, reinterpret_cast<uintptr_t>(p) % size == 0, SP_ERR_INVALID, std::string("misaligned ") + what);
    SP_REQUIRE(ctx, stride >= (int64_t)dim, SP_ERR_INVALID, std::string("row stride below dim: ") + what);
    return SP_OK;
}

template <typename T, int N>
cudaError_t lookup(const sp_embedding* e, const void* table, int64_t table_stride, const void* tokens, int wide,
                   uint64_t count, float scale, void* out, int64_t out_stride) {
    const int log2 = lanes_log2_for(e->dim / N);
    const uint64_t rows_per_block = (uint64_t)(kThreads >> log2) * kLookupRows;
    const unsigned grid = (unsigned)std::min<uint64_t>((count + rows_per_block - 1) / rows_per_block, 148 * 8);
    return launch_chained(k_lookup<T, N>, grid, kThreads, 0, e->ctx->stream, static_cast<const T*>(table),
                          table_stride, tokens, wide, count, e->entries, e->dim, scale, static_cast<T*>(out),
                          out_stride, log2);
}

// How the gradient's rows are laid over threads: N elements a thread, 2^lanes_log2 threads a row.
struct Rows {
    const void* upstream;
    int64_t upstream_stride;
    float scale;
    void* out;
    int64_t out_stride;
};

template <typename T, int N>
cudaError_t sum_pieces(const sp_embedding* e, const uint32_t* keys, const uint32_t* positions, uint32_t count,
                       const Rows& r, uint32_t partial_stride, uint32_t piece, int lanes_log2) {
    const uint32_t stretch = (kThreads >> lanes_log2) * piece, columns = N << lanes_log2;
    const dim3 grid((count + stretch - 1) / stretch, (e->dim + columns - 1) / columns);
    const int out_packed = pack_width(r.out, r.out_stride, e->dim, sizeof(T)) >= N;
    return launch_chained(k_sum_pieces<T, N>, grid, kThreads, 0, e->ctx->stream, keys, positions, count,
                          (uint32_t)e->entries, static_cast<const T*>(r.upstream), r.upstream_stride, e->dim, r.scale,
                          static_cast<T*>(r.out), r.out_stride, out_packed, e->partials, partial_stride, piece,
                          lanes_log2, static_cast<const DeviceMeta*>(e->meta));
}

// Entries per block of k_sum_few, 0 where the sorted list is the better way: a block an SM, or two where
// they have many rows to write (60,000 rows of 64 f32: 41 us in one, 17 us in two; 1000 rows 12 and 14).
uint32_t few_owned(uint64_t entries, uint64_t count) {
    if (count > kFewTokens) return 0;
    const uint64_t blocks = entries >= 148 * 128 ? 296 : 148;
    const uint64_t owned = std::min<uint64_t>((entries + blocks - 1) / blocks, kMostOwned);
    return (entries + owned - 1) / owned * count <= kFewReads ? (uint32_t)owned : 0;
}

template <typename T, int N>
cudaError_t sum_few(const sp_embedding* e, const void* tokens, int wide, uint32_t count, uint32_t owned, const Rows& r,
                    int lanes_log2) {
    const size_t smem = kFewThreads * N * sizeof(float) +
                        (kFewThreads / 32 * (size_t)owned + count + (count + kFewThreads - 1) / kFewThreads * kFewThreads) * sizeof(uint16_t);
    static std::atomic<unsigned long long> configured{0};
    constexpr size_t most = kFewThreads * N * sizeof(float) + (kFewThreads / 32 * kMostOwned + 2 * kFewTokens) * sizeof(uint16_t);
    const cudaError_t err = allow_smem_once(k_sum_few<T, N>, most, configured);
    if (err != cudaSuccess) return err;
    const int out_packed = pack_width(r.out, r.out_stride, e->dim, sizeof(T)) >= N;
    // Fewer threads a row where that makes column tiles for idle SMs.
    const unsigned blocks = grid_for(e->entries, owned);
    auto tiles = [&]() { return (e->dim + (N << lanes_log2) - 1) / (N << lanes_log2); };
    while (lanes_log2 > kMinLanesLog2 && blocks * tiles() < 148) --lanes_log2;
    const dim3 grid(blocks, std::max(1u, std::min(tiles(), 148 / blocks)));
    return launch_chained(k_sum_few<T, N>, grid, kFewThreads, smem, e->ctx->stream, tokens, wide,
                          count, e->entries, owned, static_cast<const T*>(r.upstream), r.upstream_stride, e->dim,
                          r.scale, static_cast<T*>(r.out), r.out_stride, out_packed, lanes_log2);
}

uint32_t partial_stride_of(uint32_t dim) { return (dim + 3) / 4 * 4; }

}  // namespace

// The entries catch whatever the host code may throw (a string or list that finds no memory).
extern "C" {

sp_status sp_embedding_create(sp_context* ctx, uint64_t entries, uint32_t dim, sp_element element,
                              uint64_t max_tokens, sp_embedding** out) try {
    if (!ctx || !out) return SP_ERR_INVALID;
    *out = nullptr;
    SP_REQUIRE(ctx, entries > 0 && entries < (1ull << 31), SP_ERR_INVALID, "entries outside [1, 2^31)");
    SP_REQUIRE(ctx, dim > 0 && dim < (1u << 20), SP_ERR_INVALID, "dim outside [1, 2^20)");
    SP_REQUIRE(ctx, element == SP_F32 || element == SP_BF16, SP_ERR_INVALID, "element type");
    SP_REQUIRE(ctx, max_tokens > 0 && max_tokens < (1ull << 30), SP_ERR_INVALID, "max_tokens outside [1, 2^30)");
    SP_CHECK(select_device(ctx));
    sp_embedding* e = new (std::nothrow) sp_embedding();
    SP_REQUIRE(ctx, e != nullptr, SP_ERR_OUT_OF_MEMORY, "host memory");
    e->ctx = ctx;
    e->entries = entries;
    e->dim = dim;
    e->element = element;
    e->max_tokens = max_tokens;
    uint32_t bits = 1;
    while ((1ull << bits) <= entries) ++bits;  // keys 0..entries
    e->plan.key_bits = (int)bits;
    e->plan.passes = (int)(bits + 7) / 8;
    e->plan.short_partitions = 1;
    // The most stretches any count up to max_tokens is cut into, at 8 pieces each (32 threads a row): a
    // count's pieces number below 2 kGroups until they are kLongPiece long.
    const uint64_t stretches = std::max<uint64_t>(2 * kGroups / 8 + 1, (max_tokens + 8 * kLongPiece - 1) / (8 * kLongPiece));
    sp_status s = SP_OK;
    auto all = [&]() -> sp_status {
        SP_CHECK(allocate(e, &e->meta, 1));
        for (int b = 0; b < 2; ++b) {
            SP_CHECK(allocate(e, &e->keys[b], max_tokens));
            SP_CHECK(allocate(e, &e->values[b], max_tokens));
        }
        SP_CHECK(allocate(e, &e->histograms, kSortMaxPasses * kSortRadix + kSortMaxPasses));
        const uint64_t partitions = (max_tokens + kSortShortPartition - 1) / kSortShortPartition;
        SP_CHECK(allocate(e, &e->lookback, partitions * kSortRadix));
        SP_CHECK(allocate(e, &e->partials, stretches * 2 * partial_stride_of(dim)));
        // The look-back words carry the pass's sequence number: zero is no pass's.
        SP_CUDA(ctx, cudaMemsetAsync(e->lookback, 0, partitions * kSortRadix * sizeof(unsigned long long), ctx->stream));
        SP_CUDA(ctx, cudaMemsetAsync(e->meta, 0, sizeof(DeviceMeta), ctx->stream));
        return SP_OK;
    };
    if ((s = all()) != SP_OK) {
        sp_embedding_destroy(e);
        return s;
    }
    *out = e;
    return SP_OK;
} catch (...) {
    return SP_ERR_OUT_OF_MEMORY;
}

void sp_embedding_destroy(sp_embedding* e) {
    if (!e) return;
    cudaSetDevice(e->ctx->device);
    cudaStreamSynchronize(e->ctx->stream);
    for (void* p : e->allocations) cudaFree(p);
    delete e;
}

sp_status sp_embedding_lookup(sp_embedding* e, const void* d_table, int64_t table_stride, const void* d_tokens,
                              sp_index index, uint64_t count, float scale, void* d_out, int64_t out_stride) try {
    if (!e) return SP_ERR_INVALID;
    sp_context* ctx = e->ctx;
    NvtxRange range("sp_embedding_lookup");
    const size_t size = element_size(e->element);
    SP_REQUIRE(ctx, index == SP_INDEX32 || index == SP_INDEX64, SP_ERR_INVALID, "index type");
    SP_REQUIRE(ctx, count <= e->max_tokens, SP_ERR_INVALID, "more tokens than the embedding was made for");
    SP_CHECK(check_rows(ctx, d_table, table_stride, e->dim, size, "table"));
    if (count == 0) return SP_OK;
    SP_REQUIRE(ctx, d_tokens != nullptr, SP_ERR_INVALID, "null tokens");
    SP_REQUIRE(ctx, reinterpret_cast<uintptr_t>(d_tokens) % (index == SP_INDEX64 ? 8 : 4) == 0, SP_ERR_INVALID,
               "misaligned tokens");
    SP_CHECK(check_rows(ctx, d_out, out_stride, e->dim, size, "output"));
    SP_CHECK(select_device(ctx));
    const int width = std::min(pack_width(d_table, table_stride, e->dim, size), pack_width(d_out, out_stride, e->dim, size));
    const int wide = index == SP_INDEX64;
    cudaError_t err = cudaErrorInvalidValue;
#define SPLAT_LOOKUP(T, N) \
    err = lookup<T, N>(e, d_table, table_stride, d_tokens, wide, count, scale, d_out, out_stride)
    if (e->element == SP_F32) {
        if (width == 4) SPLAT_LOOKUP(float, 4);
        else if (width == 2) SPLAT_LOOKUP(float, 2);
        else SPLAT_LOOKUP(float, 1);
    } else {
        if (width == 8) SPLAT_LOOKUP(bf16, 8);
        else if (width == 4) SPLAT_LOOKUP(bf16, 4);
        else if (width == 2) SPLAT_LOOKUP(bf16, 2);
        else SPLAT_LOOKUP(bf16, 1);
    }
#undef SPLAT_LOOKUP
    SP_CUDA(ctx, err);
    return SP_OK;
} catch (...) {
    return SP_ERR_OUT_OF_MEMORY;
}

sp_status sp_embedding_gradient(sp_embedding* e, const void* d_out_gradient, int64_t out_gradient_stride,
                                const void* d_tokens, sp_index index, uint64_t count, float scale,
                                void* d_table_gradient, int64_t table_gradient_stride) try {
    if (!e) return SP_ERR_INVALID;
    sp_context* ctx = e->ctx;
    NvtxRange range("sp_embedding_gradient");
    const size_t size = element_size(e->element);
    SP_REQUIRE(ctx, index == SP_INDEX32 || index == SP_INDEX64, SP_ERR_INVALID, "index type");
    SP_REQUIRE(ctx, count <= e->max_tokens, SP_ERR_INVALID, "more tokens than the embedding was made for");
    SP_CHECK(check_rows(ctx, d_table_gradient, table_gradient_stride, e->dim, size, "table gradient"));
    if (count > 0) {
        SP_REQUIRE(ctx, d_tokens != nullptr, SP_ERR_INVALID, "null tokens");
        SP_REQUIRE(ctx, reinterpret_cast<uintptr_t>(d_tokens) % (index == SP_INDEX64 ? 8 : 4) == 0, SP_ERR_INVALID,
                   "misaligned tokens");
        SP_CHECK(check_rows(ctx, d_out_gradient, out_gradient_stride, e->dim, size, "output gradient"));
    }
    SP_CHECK(select_device(ctx));
    cudaStream_t st = ctx->stream;
    const uint32_t n = (uint32_t)count;
    const int wide = index == SP_INDEX64;
    const Rows r{d_out_gradient, out_gradient_stride, scale, d_table_gradient, table_gradient_stride};
    // No rows to lay out where there are no tokens (and perhaps no pointer).
    const int width = n > 0 ? pack_width(d_out_gradient, out_gradient_stride, e->dim, size) : 1;
    const int lanes_log2 = lanes_log2_for(e->dim / width, kMinLanesLog2);
    cudaError_t err = cudaErrorInvalidValue;
#define SPLAT_ROWS(call)                                 \
    do {                                                 \
        if (e->element == SP_F32) {                      \
            if (width == 4) err = call(float, 4);        \
            else if (width == 2) err = call(float, 2);   \
            else err = call(float, 1);                   \
        } else {                                         \
            if (width == 8) err = call(bf16, 8);         \
            else if (width == 4) err = call(bf16, 4);    \
            else if (width == 2) err = call(bf16, 2);    \
            else err = call(bf16, 1);                    \
        }                                                \
    } while (0)
    if (const uint32_t owned = few_owned(e->entries, count)) {
#define SPLAT_FEW(T, N) sum_few<T, N>(e, d_tokens, wide, n, owned, r, lanes_log2)
        SPLAT_ROWS(SPLAT_FEW);
#undef SPLAT_FEW
        SP_CUDA(ctx, err);
        return SP_OK;
    }
    const uint32_t piece = piece_length(count, lanes_log2), partial_stride = partial_stride_of(e->dim);
    uint32_t* tickets = e->histograms + kSortMaxPasses * kSortRadix;
    SP_CUDA(ctx, cudaMemsetAsync(e->histograms, 0, (kSortMaxPasses * kSortRadix + kSortMaxPasses) * sizeof(uint32_t), st));
    // The gradient's rows as 16-byte units where they are whole ones, 4-byte or 2-byte ones otherwise.
    const bool dense = table_gradient_stride == (int64_t)e->dim;
    const uint64_t zero_rows = dense ? 1 : e->entries, zero_bytes = (dense ? e->entries : 1) * e->dim * size;
    const uint64_t alignment = reinterpret_cast<uintptr_t>(d_table_gradient) | zero_bytes |
                               (dense ? 0 : (uint64_t)table_gradient_stride * size);
    const unsigned emit_grid = std::max(grid_for(count, kThreads * kEmitItems),
                                        (unsigned)std::min<uint64_t>(148 * 8, zero_rows * zero_bytes / (kThreads * 256)));
#define SPLAT_EMIT(U)                                                                                                  \
    SP_CUDA(ctx, launch_chained(k_emit_tokens<U>, emit_grid, kThreads, 0, st, d_tokens, wide, n, e->entries,          \
                                e->plan.passes, e->meta, e->keys[0], e->values[0], e->histograms,                     \
                                static_cast<U*>(d_table_gradient), zero_rows, zero_bytes / sizeof(U),                  \
                                (int64_t)(table_gradient_stride * size / sizeof(U))))
    if (alignment % 16 == 0) SPLAT_EMIT(uint4);
    else if (alignment % 4 == 0) SPLAT_EMIT(uint32_t);
    else SPLAT_EMIT(uint16_t);
#undef SPLAT_EMIT
    const uint32_t partitions = (n + kSortShortPartition - 1) / kSortShortPartition;
    for (int pass = 0; pass < e->plan.passes; ++pass)
        SP_CUDA(ctx, launch_sort_pass(e->plan, pass, ++e->sequence, e->keys[0], e->values[0], e->keys[1], e->values[1],
                                      e->histograms, tickets, e->lookback, partitions, e->meta, st));
    const uint32_t* keys = e->keys[e->plan.passes & 1];
    const uint32_t* positions = e->values[e->plan.passes & 1];
#define SPLAT_PIECES(T, N) sum_pieces<T, N>(e, keys, positions, n, r, partial_stride, piece, lanes_log2)
    SPLAT_ROWS(SPLAT_PIECES);
#undef SPLAT_PIECES
#undef SPLAT_ROWS
    SP_CUDA(ctx, err);
    const uint32_t stretch = (kThreads >> lanes_log2) * piece;
    const unsigned join_blocks = grid_for((n + stretch - 1) / stretch, kJoinWarps);
    const dim3 join_grid(join_blocks, std::max(1u, std::min((e->dim + 127) / 128, 148 * 4 / join_blocks)));
#define SPLAT_JOIN(T)                                                                                                 \
    SP_CUDA(ctx, launch_chained(k_join_pieces<T>, join_grid, kThreads, 0, st, keys, n, (uint32_t)e->entries, e->dim,  \
                                scale, static_cast<T*>(d_table_gradient), table_gradient_stride,                      \
                                static_cast<const float*>(e->partials), partial_stride, stretch,                      \
                                static_cast<const DeviceMeta*>(e->meta)))
    if (e->element == SP_F32) SPLAT_JOIN(float);
    else SPLAT_JOIN(bf16);
#undef SPLAT_JOIN
    return SP_OK;
} catch (...) {
    return SP_ERR_OUT_OF_MEMORY;
}

sp_status sp_embedding_check(sp_embedding* e) try {
    if (!e) return SP_ERR_INVALID;
    sp_context* ctx = e->ctx;
    SP_CHECK(select_device(ctx));
    uint32_t status = 0;
    SP_CUDA(ctx, cudaMemcpyAsync(&status, &e->meta->status, sizeof(status), cudaMemcpyDeviceToHost, ctx->stream));
    SP_CHECK(sync_stream(ctx));
    if (status == 0) return SP_OK;
    SP_CUDA(ctx, cudaMemsetAsync(&e->meta->status, 0, sizeof(status), ctx->stream));
    return fail(ctx, (sp_status)status, "a device-side wait gave up (sort look-back timeout)");
} catch (...) {
    return SP_ERR_OUT_OF_MEMORY;
}

}  // extern "C"
