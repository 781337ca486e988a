// The embedding of codebook tokens and its gradient (splat_labels.h).
//
// Lookup: out[i] = s T[t_i], a gather of whole rows, bound by the bytes of `out` (the table's
// rows are re-read from L2).
//
// Gradient: dT[v] = s sum_{i: t_i = v} dOut[i], without atomics so that the sums have one order:
// the (token, position) pairs go through the renderer's stable radix sort (sort.cu), the sorted
// list is cut into pieces of a fixed length, each piece's runs are summed in f32 registers while
// dOut's rows stream past once (bound by those bytes), and a token whose run crosses pieces is
// joined from the pieces' partial sums, in order, by a second kernel, which also writes the zero
// rows of the tokens nobody has.
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
    uint2* ranges = nullptr;
    float* partials = nullptr;
};

namespace {

constexpr int kThreads = 256;
constexpr int kEmitItems = 8;
constexpr int kLookupRows = 4;   // rows in flight per thread
constexpr int kPieceRows = 8;    // rows in flight per thread while summing
constexpr uint32_t kShortPiece = 16, kLongPiece = 64;

// The sorted positions per piece: long pieces keep the partial sums few, short ones give a small
// list enough pieces to fill the SMs (148 SMs x 8 warps of pieces either way).
uint32_t piece_length(uint64_t count) { return count >= (uint64_t)kLongPiece * 148 * 8 ? kLongPiece : kShortPiece; }

// `lanes` threads (a power of two, at most 32) move one row, N elements at a time.
template <typename T, int N>
__global__ void __launch_bounds__(kThreads) k_lookup(const T* __restrict__ table, int64_t table_stride,
                                                     const void* __restrict__ tokens, int wide, uint64_t count,
                                                     uint64_t entries, uint32_t dim, float scale,
                                                     T* __restrict__ out, int64_t out_stride, int lanes_log2) {
    chain_enter();
    const uint32_t lanes = 1u << lanes_log2, lane = threadIdx.x & (lanes - 1);
    const uint64_t rows_per_pass = kThreads >> lanes_log2;
    const uint32_t packs = dim / N;
    for (uint64_t base = (uint64_t)blockIdx.x * rows_per_pass * kLookupRows; base < count;
         base += (uint64_t)gridDim.x * rows_per_pass * kLookupRows) {
        int64_t token[kLookupRows];
        uint64_t row[kLookupRows];
#pragma unroll
        for (int k = 0; k < kLookupRows; ++k) {
            row[k] = base + k * rows_per_pass + (threadIdx.x >> lanes_log2);
            token[k] = row[k] < count ? index_at(tokens, wide, row[k], entries) : -1;
        }
        for (uint32_t p = lane; p < packs; p += lanes) {
            Pack<T, N> v[kLookupRows];
#pragma unroll
            for (int k = 0; k < kLookupRows; ++k)
                if (token[k] >= 0)
                    v[k] = *reinterpret_cast<const Pack<T, N>*>(table + token[k] * table_stride + (uint64_t)p * N);
#pragma unroll
            for (int k = 0; k < kLookupRows; ++k) {
                if (row[k] >= count) continue;
                Pack<T, N> o;
#pragma unroll
                for (int j = 0; j < N; ++j)
                    o.v[j] = token[k] >= 0 ? from_float<T>(to_float(v[k].v[j]) * scale) : from_float<T>(0.0f);
                *reinterpret_cast<Pack<T, N>*>(out + (int64_t)row[k] * out_stride + (uint64_t)p * N) = o;
            }
        }
    }
}

// The sort's input: key = token (entries for none, which sorts last), value = position, with every
// pass's digit histogram; block 0 sets the sort's bookkeeping. The device status is left alone:
// it stays raised until it is read.
__global__ void __launch_bounds__(kThreads) k_emit_tokens(const void* __restrict__ tokens, int wide, uint32_t count,
                                                          uint64_t entries, int passes, DeviceMeta* meta,
                                                          uint32_t* __restrict__ keys, uint32_t* __restrict__ values,
                                                          uint32_t* __restrict__ histograms) {
    chain_enter();
    __shared__ uint32_t hist[4][kSortRadix];
    for (int p = 0; p < passes; ++p) hist[p][threadIdx.x] = 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        meta->count = count;
        meta->partitions = (count + kSortPartition - 1) / kSortPartition;
        meta->key_shift = 0;
        meta->key_base = 0;
        meta->passes = (uint32_t)passes;
        meta->first_buffer = 0;
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

// A piece of the sorted list per group of `lanes` threads, N columns a thread (blockIdx.y: the
// next lanes * N columns). A run that begins and ends inside its piece is a token's whole sum and
// is written out; the others leave partial sums: slot 0 of the piece for a run that began before
// it, slot 1 for one that begins inside and goes on.
template <typename T, int N>
__global__ void __launch_bounds__(kThreads)
    k_sum_pieces(const uint32_t* __restrict__ keys, const uint32_t* __restrict__ positions, uint32_t count,
                 uint32_t entries, const T* __restrict__ upstream, int64_t upstream_stride, uint32_t dim, float scale,
                 T* __restrict__ out, int64_t out_stride, int out_packed, float* __restrict__ partials,
                 uint32_t partial_stride, uint32_t piece, int lanes_log2, const DeviceMeta* __restrict__ meta) {
    chain_enter();
    if (meta->status != 0) return;  // the list may be out of order: k_join_pieces writes NaN
    const uint32_t lanes = 1u << lanes_log2;
    const uint32_t group = blockIdx.x * (kThreads >> lanes_log2) + (threadIdx.x >> lanes_log2);
    const uint32_t column = (blockIdx.y * lanes + (threadIdx.x & (lanes - 1))) * N;
    const uint64_t first = (uint64_t)group * piece;
    if (first >= count || column >= dim) return;
    const uint32_t begin = (uint32_t)first, end = (uint32_t)min((uint64_t)count, first + piece);
    float acc[N];
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = 0.0f;
    uint32_t current = keys[begin];
    bool from_before = begin > 0 && keys[begin - 1] == current;
    auto flush = [&](bool goes_on) {
        if (current >= entries) return;
        if (!from_before && !goes_on) {
            T* to = out + (int64_t)current * out_stride + column;
            Pack<T, N> o;
#pragma unroll
            for (int j = 0; j < N; ++j) o.v[j] = from_float<T>(acc[j] * scale);
            if (out_packed) {
                *reinterpret_cast<Pack<T, N>*>(to) = o;
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j) to[j] = o.v[j];
            }
        } else {
            float* to = partials + ((uint64_t)group * 2 + (from_before ? 0 : 1)) * partial_stride + column;
#pragma unroll
            for (int j = 0; j < N; ++j) to[j] = acc[j];
        }
    };
    for (uint32_t i = begin; i < end; i += kPieceRows) {
        uint32_t key[kPieceRows];
        Pack<T, N> v[kPieceRows];
#pragma unroll
        for (int k = 0; k < kPieceRows; ++k) {
            key[k] = entries;
            if (i + k < end) {
                key[k] = keys[i + k];
                if (key[k] < entries)
                    v[k] = *reinterpret_cast<const Pack<T, N>*>(upstream + (int64_t)positions[i + k] * upstream_stride +
                                                                column);
            }
        }
#pragma unroll
        for (int k = 0; k < kPieceRows; ++k) {
            if (i + k >= end) break;
            if (key[k] != current) {
                flush(false);
                current = key[k];
                from_before = false;
#pragma unroll
                for (int j = 0; j < N; ++j) acc[j] = 0.0f;
            }
            if (key[k] < entries) {
#pragma unroll
                for (int j = 0; j < N; ++j) acc[j] += to_float(v[k].v[j]);
            }
        }
    }
    flush(end < count && keys[end] == current);
}

// Per token: zeros where it has no rows, the ordered sum of its partials where its run crosses
// pieces, nothing where k_sum_pieces wrote it. A warp per token, 4 columns a lane; a token with
// more than kWarpPieces partials is joined by the block's eight warps together.
constexpr uint32_t kJoinWarps = kThreads / 32, kWarpPieces = 32;
template <typename T>
__global__ void __launch_bounds__(kThreads)
    k_join_pieces(const uint2* __restrict__ ranges, uint32_t entries, uint32_t dim, float scale, T* __restrict__ out,
                  int64_t out_stride, const float* __restrict__ partials, uint32_t partial_stride, uint32_t piece,
                  const DeviceMeta* __restrict__ meta) {
    chain_enter();
    __shared__ float4 shared[kJoinWarps][32];
    __shared__ uint2 span[kJoinWarps];
    const uint32_t warp = threadIdx.x / 32, lane = lane_id();
    const uint32_t token = blockIdx.x * kJoinWarps + warp;
    const bool failed = meta->status != 0;
    auto store = [&](uint32_t v, uint32_t column, float4 sum) {
        const float s[4] = {sum.x, sum.y, sum.z, sum.w};
        T* to = out + (int64_t)v * out_stride + column;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (column + j < dim) to[j] = from_float<T>(s[j] * scale);
    };
    // Partial p of a run over the sorted positions [s, e): slot 1 of its first piece, then slot 0.
    auto sum_of = [&](uint2 run, uint32_t p0, uint32_t p1, uint32_t column) {
        const uint32_t first = run.x / piece;
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
    uint2 run = make_uint2(0u, 0u);
    uint32_t pieces = 0;
    if (token < entries) {
        run = ranges[token];
        if (run.y > run.x) pieces = (run.y - 1) / piece - run.x / piece + 1;
        if (failed || pieces == 0) {
            const float fill = failed ? __int_as_float(0x7fffffff) : 0.0f;
            for (uint32_t c = lane; c < dim; c += 32) out[(int64_t)token * out_stride + c] = from_float<T>(fill);
        } else if (pieces > 1 && pieces <= kWarpPieces) {
            for (uint32_t c = lane * 4; c < dim; c += 128) store(token, c, sum_of(run, 0, pieces, c));
        }
    }
    if (lane == 0) span[warp] = !failed && pieces > kWarpPieces ? run : make_uint2(0u, 0u);
    __syncthreads();
    for (uint32_t w = 0; w < kJoinWarps; ++w) {
        const uint2 long_run = span[w];
        if (long_run.y == long_run.x) continue;
        const uint32_t n = (long_run.y - 1) / piece - long_run.x / piece + 1;
        const uint32_t p0 = (uint32_t)((uint64_t)n * warp / kJoinWarps);
        const uint32_t p1 = (uint32_t)((uint64_t)n * (warp + 1) / kJoinWarps);
        for (uint32_t c0 = 0; c0 < dim; c0 += 128) {
            const uint32_t c = c0 + lane * 4;
            if (c < dim) shared[warp][lane] = sum_of(long_run, p0, p1, c);
            __syncthreads();
            if (warp == 0 && c < dim) {
                float4 sum = shared[0][lane];
                for (uint32_t k = 1; k < kJoinWarps; ++k) {
                    const float4 v = shared[k][lane];
                    sum.x += v.x;
                    sum.y += v.y;
                    sum.z += v.z;
                    sum.w += v.w;
                }
                store(blockIdx.x * kJoinWarps + w, c, sum);
            }
            __syncthreads();
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

int lanes_log2_for(uint32_t packs) {
    int log2 = 0;
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
    const unsigned grid = (unsigned)std::min<uint64_t>((count + rows_per_block - 1) / rows_per_block, 1u << 20);
    return launch_chained(k_lookup<T, N>, grid, kThreads, 0, e->ctx->stream, static_cast<const T*>(table),
                          table_stride, tokens, wide, count, e->entries, e->dim, scale, static_cast<T*>(out),
                          out_stride, log2);
}

template <typename T, int N>
cudaError_t sum_pieces(const sp_embedding* e, const uint32_t* keys, const uint32_t* positions, uint32_t count,
                       const void* upstream, int64_t upstream_stride, float scale, void* out, int64_t out_stride,
                       uint32_t partial_stride, uint32_t piece) {
    const int log2 = lanes_log2_for(e->dim / N);
    const uint32_t per_block = kThreads >> log2;
    const uint32_t pieces = (count + piece - 1) / piece;
    const uint32_t columns = N << log2;
    const dim3 grid((pieces + per_block - 1) / per_block, (e->dim + columns - 1) / columns);
    const int out_packed = pack_width(out, out_stride, e->dim, sizeof(T)) >= N;
    return launch_chained(k_sum_pieces<T, N>, grid, kThreads, 0, e->ctx->stream, keys, positions, count,
                          (uint32_t)e->entries, static_cast<const T*>(upstream), upstream_stride, e->dim, scale,
                          static_cast<T*>(out), out_stride, out_packed, e->partials, partial_stride, piece, log2,
                          static_cast<const DeviceMeta*>(e->meta));
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
    // The most pieces any count up to max_tokens is cut into.
    const uint64_t most_short = std::min<uint64_t>(max_tokens, (uint64_t)kLongPiece * 148 * 8);
    const uint64_t pieces = std::max((most_short + kShortPiece - 1) / kShortPiece, (max_tokens + kLongPiece - 1) / kLongPiece);
    sp_status s = SP_OK;
    auto all = [&]() -> sp_status {
        SP_CHECK(allocate(e, &e->meta, 1));
        for (int b = 0; b < 2; ++b) {
            SP_CHECK(allocate(e, &e->keys[b], max_tokens));
            SP_CHECK(allocate(e, &e->values[b], max_tokens));
        }
        SP_CHECK(allocate(e, &e->histograms, kSortMaxPasses * kSortRadix + kSortMaxPasses));
        const uint64_t partitions = (max_tokens + kSortPartition - 1) / kSortPartition;
        SP_CHECK(allocate(e, &e->lookback, partitions * kSortRadix));
        SP_CHECK(allocate(e, &e->ranges, entries));
        SP_CHECK(allocate(e, &e->partials, pieces * 2 * partial_stride_of(dim)));
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
    const uint32_t piece = piece_length(count), partial_stride = partial_stride_of(e->dim);
    uint32_t* tickets = e->histograms + kSortMaxPasses * kSortRadix;
    SP_CUDA(ctx, cudaMemsetAsync(e->histograms, 0, (kSortMaxPasses * kSortRadix + kSortMaxPasses) * sizeof(uint32_t), st));
    SP_CUDA(ctx, launch_chained(k_emit_tokens, std::max(1u, grid_for(count, kThreads * kEmitItems)), kThreads, 0, st,
                                d_tokens, wide, n, e->entries, e->plan.passes, e->meta, e->keys[0], e->values[0],
                                e->histograms));
    const uint32_t partitions = (n + kSortPartition - 1) / kSortPartition;
    for (int pass = 0; pass < e->plan.passes && n > 0; ++pass)
        SP_CUDA(ctx, launch_sort_pass(e->plan, pass, ++e->sequence, e->keys[0], e->values[0], e->keys[1], e->values[1],
                                      e->histograms, tickets, e->lookback, partitions, e->meta, st));
    const uint32_t* keys = e->keys[e->plan.passes & 1];
    const uint32_t* positions = e->values[e->plan.passes & 1];
    SP_CUDA(ctx, launch_ranges(e->plan, keys, e->meta, std::max<uint64_t>(count, e->entries / 4), e->ranges,
                               (uint32_t)e->entries, st));
    if (n > 0) {
        const int width = pack_width(d_out_gradient, out_gradient_stride, e->dim, size);
        cudaError_t err = cudaErrorInvalidValue;
#define SPLAT_SUM(T, N)                                                                                       \
    err = sum_pieces<T, N>(e, keys, positions, n, d_out_gradient, out_gradient_stride, scale, d_table_gradient, \
                           table_gradient_stride, partial_stride, piece)
        if (e->element == SP_F32) {
            if (width == 4) SPLAT_SUM(float, 4);
            else if (width == 2) SPLAT_SUM(float, 2);
            else SPLAT_SUM(float, 1);
        } else {
            if (width == 8) SPLAT_SUM(bf16, 8);
            else if (width == 4) SPLAT_SUM(bf16, 4);
            else if (width == 2) SPLAT_SUM(bf16, 2);
            else SPLAT_SUM(bf16, 1);
        }
#undef SPLAT_SUM
        SP_CUDA(ctx, err);
    }
    const unsigned join_grid = grid_for(e->entries, kJoinWarps);
    if (e->element == SP_F32)
        SP_CUDA(ctx, launch_chained(k_join_pieces<float>, join_grid, kThreads, 0, st,
                                    static_cast<const uint2*>(e->ranges), (uint32_t)e->entries, e->dim, scale,
                                    static_cast<float*>(d_table_gradient), table_gradient_stride,
                                    static_cast<const float*>(e->partials), partial_stride, piece,
                                    static_cast<const DeviceMeta*>(e->meta)));
    else
        SP_CUDA(ctx, launch_chained(k_join_pieces<bf16>, join_grid, kThreads, 0, st,
                                    static_cast<const uint2*>(e->ranges), (uint32_t)e->entries, e->dim, scale,
                                    static_cast<bf16*>(d_table_gradient), table_gradient_stride,
                                    static_cast<const float*>(e->partials), partial_stride, piece,
                                    static_cast<const DeviceMeta*>(e->meta)));
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
