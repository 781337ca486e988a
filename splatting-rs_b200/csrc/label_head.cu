// The label head (splat_labels.h): cross entropy of features against a vocabulary of label rows,
// its gradient, and prediction, without ever storing the logits.
//
//   loss      z = c H W^T in tiles; per row the sum s of e^(z - base) over all labels but the target, base
//             following the largest; the tiles' (base, s) are joined, and with the target's
//             z: loss = log1p(s e^base / e^z[target]), log sum exp z = z[target] + loss
//   gradient  the logits again in tiles, turned into slopes G = exp(z - logsumexp) - [target]
//             where they are made and written as bf16 parts for a chunk of rows; then
//             dH = c g G W and dW = c g G^T H, the same tile pipeline (label_gemm.cuh)
//   predict   the loss's pass with the maximum's label kept
//
// Rows without a target are left out of every product: their indices are compacted first, and
// where there are such rows the features are copied in that order (whatever the rows left out
// hold, NaN included, is never read by a product).
#include <algorithm>
#include <cstring>
#include <new>

#include "label_thin.cuh"
#include "objects.h"

using namespace splat;
using namespace splat::label;

namespace {
constexpr uint64_t kFewSlopes = 1ull << 21;
}

struct sp_label_head {
    sp_context* ctx = nullptr;
    uint64_t labels = 0;
    uint32_t dim = 0;
    sp_element element = SP_F32;
    uint64_t max_rows = 0;
    bool training = false;
    uint32_t sms = 148;
    std::vector<void*> allocations;
    RowSet* rows = nullptr;
    uint32_t* row_of = nullptr;
    uint32_t* counts = nullptr;
    bf16* packed_features = nullptr;
    bf16* packed_weight = nullptr;
    float2* partials = nullptr;
    uint32_t* partial_labels = nullptr;
    float* target_logits = nullptr;
    double* loss_sums = nullptr;
    bf16* slopes = nullptr;
    float* sums = nullptr;  // partial sums of the output gradients

    uint32_t parts() const { return element == SP_F32 ? kParts : 1; }
    uint32_t products() const { return element == SP_F32 ? kPartProducts : 1; }
    // Parts of the slopes: f32's three, and two for bf16 operands where that costs little, or matters most. One
    // rounding to bf16 is nearly as much of the weight's gradient as its own last one (256 x 1000 x 64, features
    // that lean towards their label: 2.1e-3 of its norm in all, 1.65e-3 with two parts). Two parts cost the
    // gradient of 128 x 65,536 x 512 13 of 88 us, that of 2^21 slopes 1.4 to 3.5 us. With more rows a label's sums
    // average the rounding out, and a second part would double the bytes and half of the products. Not where the
    // rows have factors of their own, which are in their slopes: the targets' slopes of rows of one factor, near
    // minus that, are all rounded the same way (1.1e-3 of the weight's gradient at 20,000 x 32,768 x 512, which
    // takes 2.3 ms with two parts and 1.5 with one).
    uint32_t slope_parts(uint64_t rows, bool own_factors) const {
        return element == SP_F32 ? kParts : rows <= kTile || rows * labels <= kFewSlopes || own_factors ? 2 : 1;
    }
    uint64_t packed_stride() const { return ((uint64_t)dim + kBlockK - 1) / kBlockK * kBlockK; }
    uint64_t count_blocks() const { return (max_rows + 63) / 64; }
    uint64_t slope_stride() const { return (labels + kPairTile - 1) / kPairTile * kPairTile; }
};

namespace {

constexpr int kThreads = 256;
constexpr uint32_t kGatherRows = 64;        // rows a block compacts and copies
constexpr uint32_t kCountGroups = 16;       // such blocks' counts are summed this many at a time
constexpr uint32_t kRecountBlocks = 16;     // up to this many blocks each count all targets themselves
constexpr uint32_t kLogitWaves = 16, kOutWaves = 4;
constexpr uint32_t kLongestSum = 32;         // steps of 64 of K
constexpr double kLaunchUs = 3.0;           // of a small kernel in the chain
constexpr double kStepUs = 0.19;            // 64 of K of a 128 x 128 tile in a single block
constexpr double kPairCost = 1.4;           // of a 256 x 256 tile, in 128 x 128 tiles of one block
constexpr int kSlotsAhead = 8;                // partials a thread has under way
constexpr uint32_t kThreadSlots = 8;
// Slope elements kept at once (1.25 GiB). More rows go in chunks; their weight's gradient is summed over
// those, and a short last chunk fills few waves: 20,000 x 32,768 x 512 took 2036 us in chunks of a half
// of this, 1970 in one piece; 65,536 x 32,768 x 512 9350 and 9070.
constexpr uint64_t kSlopeBudget = 5ull << 27;

uint64_t round_up(uint64_t v, uint64_t to) { return (v + to - 1) / to * to; }

// ------------------------------------------------------------------ rows and operands

__device__ __forceinline__ bool has_target(const void* targets, int wide, uint64_t i, uint64_t labels) {
    return !targets || index_at(targets, wide, i, labels) >= 0;
}

// counts[b]: the targets among rows [b, b + 1) kGatherRows; group_counts: of kCountGroups such.
__global__ void __launch_bounds__(kCountGroups * 32)
    k_count_targets(const void* __restrict__ targets, int wide, uint64_t n, uint64_t labels,
                    uint32_t* __restrict__ counts, uint32_t* __restrict__ group_counts) {
    chain_enter();
    __shared__ uint32_t found[kCountGroups];
    const uint32_t warp = threadIdx.x / 32, block = blockIdx.x * kCountGroups + warp;
    uint32_t here = 0;
#pragma unroll
    for (uint32_t r = 0; r < kGatherRows; r += 32) {
        const uint64_t i = (uint64_t)block * kGatherRows + r + lane_id();
        here += __popc(__ballot_sync(0xffffffffu, i < n && has_target(targets, wide, i, labels)));
    }
    if (lane_id() == 0) {
        found[warp] = here;
        if ((uint64_t)block * kGatherRows < n) counts[block] = here;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        uint32_t sum = 0;
#pragma unroll
        for (uint32_t w = 0; w < kCountGroups; ++w) sum += found[w];
        group_counts[blockIdx.x] = sum;
    }
}

__device__ __forceinline__ uint32_t block_sum(uint32_t v) {
    __shared__ uint32_t warps[kThreads / 32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (lane_id() == 0) warps[threadIdx.x / 32] = v;
    __syncthreads();
    uint32_t sum = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) sum += warps[w];
    return sum;
}

// Eight columns of a row as bf16 parts: f32 in three (take_part), bf16 is copied.
template <typename T>
__device__ __forceinline__ void copy_parts(const T* from, uint32_t columns, bool vector, bf16* to, uint64_t part) {
    float v[8];
    if (vector && columns >= 8) {
        constexpr int N = 16 / sizeof(T);
#pragma unroll
        for (int q = 0; q < 8 / N; ++q) {
            const Pack<T, N> p = load_pack<T, N>(from + q * N);
#pragma unroll
            for (int j = 0; j < N; ++j) v[q * N + j] = p.get(j);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (uint32_t)j < columns ? to_float(from[j]) : 0.0f;
    }
    constexpr int parts = sizeof(T) == 4 ? (int)kParts : 1;
#pragma unroll
    for (int p = 0; p < parts; ++p) store_pack(to + p * part, take_part(v, p == parts - 1));
}

// The weight's copy as bf16 parts, where it cannot be read in place (`from` NULL: it can).
template <typename T>
struct PackWeight {
    const T* from;
    int64_t stride;
    int vector;
    bf16* to;
};

// Compacts the rows with targets (row_of), clears the outputs of the others, and copies the
// features where they cannot be read in place: `in_place` 0, or some rows left out. The first
// `gather_blocks` * `sharers` blocks do that (`sharers` of them find the same rows and share their
// copies, the first one writes the lists), the others copy the weight.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    k_gather_rows(const void* __restrict__ targets, int wide, uint64_t n, uint64_t labels, uint32_t gather_blocks,
                  uint32_t sharers,
                  const uint32_t* __restrict__ counts, const uint32_t* __restrict__ group_counts,
                  const T* __restrict__ features, int64_t stride, uint32_t dim, int vector, int in_place, RowSet* rows,
                  uint32_t* __restrict__ row_of, bf16* __restrict__ packed, uint64_t packed_stride, uint64_t part,
                  float* __restrict__ losses, double* __restrict__ normalizers, T* __restrict__ gradient,
                  int64_t gradient_stride, PackWeight<T> weight) {
    chain_enter();
    const uint32_t gathering = gather_blocks * sharers;
    if (blockIdx.x >= gathering) {
        // A warp per row, eight columns a lane.
        const uint64_t warps = (uint64_t)(gridDim.x - gathering) * (kThreads / 32);
        for (uint64_t r = (uint64_t)(blockIdx.x - gathering) * (kThreads / 32) + threadIdx.x / 32; r < labels;
             r += warps)
            for (uint32_t c = lane_id() * 8; c < packed_stride; c += 256)
                copy_parts(weight.from + (int64_t)r * weight.stride + c, c < dim ? dim - c : 0, weight.vector,
                           weight.to + r * packed_stride + c, labels * packed_stride);
        return;
    }
    __shared__ uint32_t chosen[kGatherRows];
    __shared__ uint32_t skipped[kGatherRows];
    __shared__ uint32_t half_count[2];
    const uint32_t t = threadIdx.x, lane = lane_id();
    const uint32_t block = blockIdx.x / sharers, share = blockIdx.x % sharers;
    const uint64_t first = (uint64_t)block * kGatherRows;
    uint32_t before = 0, all = 0;
    if (!targets) {
        before = (uint32_t)first;
        all = (uint32_t)n;
    } else if (counts) {
        const uint32_t group = block / kCountGroups, groups = (gather_blocks + kCountGroups - 1) / kCountGroups;
        for (uint32_t g = t; g < groups; g += kThreads) {
            const uint32_t c = group_counts[g];
            all += c;
            if (g < group) before += c;
        }
        if (t < block % kCountGroups) before += counts[group * kCountGroups + t];
        before = block_sum(before);
        all = block_sum(all);
    } else {
#pragma unroll 4
        for (uint64_t i = t; i < n; i += kThreads)
            if (has_target(targets, wide, i, labels)) {
                ++all;
                if (i < first) ++before;
            }
        before = block_sum(before);
        all = block_sum(all);
    }
    if (blockIdx.x == 0 && t == 0) {
        rows->count = all;
        rows->packed = !in_place || all != n;
    }
    bool live = false;
    uint32_t mask = 0;
    if (t < kGatherRows) {
        live = first + t < n && has_target(targets, wide, first + t, labels);
        mask = __ballot_sync(0xffffffffu, live);
        if (lane == 0) half_count[t / 32] = __popc(mask);
    }
    __syncthreads();
    const uint32_t here = half_count[0] + half_count[1];
    if (t < kGatherRows) {
        const uint32_t below = (t >= 32 ? half_count[0] : 0) + __popc(mask & ((1u << lane) - 1u));
        if (live) {
            chosen[below] = t;
            if (share == 0) row_of[before + below] = (uint32_t)(first + t);
        } else {
            skipped[t - below] = t;
            if (share == 0 && first + t < n) {
                if (losses) losses[first + t] = 0.0f;
                if (normalizers) normalizers[first + t] = 0.0;
            }
        }
    }
    __syncthreads();
    if (gradient) {
        const uint32_t last = (uint32_t)min((uint64_t)kGatherRows, n - first);
        for (uint32_t k = share; k < last - here; k += sharers)
            for (uint32_t c = t; c < dim; c += kThreads)
                gradient[(int64_t)(first + skipped[k]) * gradient_stride + c] = from_float<T>(0.0f);
    }
    if (in_place && all == n) return;
    // A warp per 256 columns of a row, eight a lane; then zero rows up to a whole tile, which the
    // weight's gradient sums over.
    const uint32_t column_parts = (uint32_t)((packed_stride + 255) / 256), warps = kThreads / 32 * sharers;
    for (uint32_t i = share * (kThreads / 32) + t / 32; i < here * column_parts; i += warps) {
        const uint32_t r = i / column_parts, c = (i - r * column_parts) * 256 + lane * 8;
        if (c < packed_stride)
            copy_parts(features + (int64_t)(first + chosen[r]) * stride + c, c < dim ? dim - c : 0, vector,
                       packed + (uint64_t)(before + r) * packed_stride + c, part);
    }
    const uint64_t padding = ((uint64_t)all + kTile - 1) / kTile * kTile - all;
    for (uint64_t i = blockIdx.x * (kThreads / 32) + t / 32; i < padding * column_parts; i += (uint64_t)gathering * (kThreads / 32)) {
        const uint64_t r = i / column_parts;
        const uint32_t c = (uint32_t)(i - r * column_parts) * 256 + lane * 8;
        if (c < packed_stride) copy_parts(features, 0, false, packed + (all + r) * packed_stride + c, part);
    }
}

// ------------------------------------------------------------------ joining

// LANES threads (1, 8 or 32) join a row's partial sums, each in units of its base's exponential: the highest base
// (and the largest logit with the lowest label) first, then the sum, in double, since a part may come
// close to f32's largest. With the rest, the sum without the target's logit (the largest's), in units of
// the latter's exponential, the loss (the negative log-probability) is log1p(rest): nothing cancels. The
// loss's mean is summed in double: per block, then by the last block.
template <int LANES>
__global__ void __launch_bounds__(kThreads)
    k_join_rows(RowSet* rows, const uint32_t* __restrict__ row_of, uint32_t all_rows,
                const float2* __restrict__ partials, const uint32_t* __restrict__ partial_labels,
                uint64_t partial_rows, uint32_t slots, float scale2, const float* __restrict__ target_logits,
                float* __restrict__ losses, double* __restrict__ normalizers, int32_t* __restrict__ labels_out,
                float* __restrict__ log_probability, double* __restrict__ block_sums, float* __restrict__ mean) {
    chain_enter();
    const uint32_t count = all_rows ? all_rows : rows->count;
    const bool failed = rows->status != 0;
    const float nan = __int_as_float(0x7fffffff);
    const uint64_t i = ((uint64_t)blockIdx.x * kThreads + threadIdx.x) / LANES;
    const uint32_t lane = threadIdx.x % LANES;
    double loss = 0.0;
    // Rows past the last go through with no partials: every lane takes part in the shuffles.
    const uint32_t mine = i < count ? slots : 0;
    float top = -INFINITY, largest = -INFINITY;
    uint32_t label = 0xffffffffu;
    double sum = 0.0;
    // Prediction: each part's largest goes into the sum here, and the row's out of it again (a 1, to double's
    // precision).
    const double one = partial_labels ? 1.0 : 0.0;
    for (uint32_t s0 = lane; s0 < mine; s0 += LANES * kSlotsAhead) {
        float2 p[kSlotsAhead];
        uint32_t l[kSlotsAhead];
#pragma unroll
        for (int k = 0; k < kSlotsAhead; ++k) {
            const uint32_t s = s0 + k * LANES;
            p[k] = s < mine ? partials[s * partial_rows + i] : make_float2(-INFINITY, 0.0f);
            l[k] = partial_labels && s < mine ? partial_labels[s * partial_rows + i] : 0xffffffffu;
        }
        const float before = top;
#pragma unroll
        for (int k = 0; k < kSlotsAhead; ++k) {
            if (partial_labels) {
                if (p[k].x > largest || (p[k].x == largest && l[k] < label)) largest = p[k].x, label = l[k];
            }
            top = fmaxf(top, p[k].x);
        }
        const float finite = finite_base(top);
        sum *= (double)exp2f((before - finite) * scale2);
#pragma unroll
        for (int k = 0; k < kSlotsAhead; ++k)
            if (s0 + k * LANES < mine) sum += ((double)p[k].y + one) * (double)exp2f((p[k].x - finite) * scale2);
    }
    float highest = top;
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
        highest = fmaxf(highest, __shfl_xor_sync(0xffffffffu, highest, o));
        const float x = __shfl_xor_sync(0xffffffffu, largest, o);
        const uint32_t l = __shfl_xor_sync(0xffffffffu, label, o);
        if (x > largest || (x == largest && l < label)) largest = x, label = l;
    }
    highest = finite_base(highest);
    sum *= (double)exp2f((top - highest) * scale2);
    top = highest;
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (i < count && lane == 0) {
        const uint32_t row = all_rows ? (uint32_t)i : row_of[i];
        const double ln2 = 0.6931471805599453;
        if (labels_out) {
            labels_out[row] = failed ? -1 : (int32_t)label;
            // An infinite largest logit has no softmax.
            log_probability[row] = failed || !(fabsf(largest) < INFINITY) ? nan : (float)-log1p(sum - 1.0);
        } else {
            const double target = target_logits[i], unit = (double)scale2 * ln2;
            const double rest = sum == 0.0 ? 0.0 : sum * exp2(((double)top - target) * scale2);
            double value, normalizer;
            if (rest <= 1.0) {
                value = log1p(rest);
                normalizer = target * unit + value;
            } else {
                const double others = log(sum) + log1p(1.0 / rest);
                normalizer = (double)top * unit + others;
                value = ((double)top - target) * unit + others;
            }
            // No softmax: the target's logit is infinite, or all are -inf.
            if (failed || target == INFINITY || (target == -INFINITY && sum == 0.0)) value = normalizer = nan;
            losses[row] = (float)value;
            normalizers[row] = normalizer;
            loss = (double)losses[row];
        }
    }
    if (labels_out) return;
    __shared__ double shared[kThreads / 32];
    __shared__ bool last;
    // The block's sum, in thread 0, added in a fixed order.
    auto block_total = [&](double v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane_id() == 0) shared[threadIdx.x / 32] = v;
        __syncthreads();
        double sum = 0.0;
        if (threadIdx.x == 0)
            for (int w = 0; w < kThreads / 32; ++w) sum += shared[w];
        return sum;
    };
    double total = block_total(loss);
    if (gridDim.x > 1) {
        if (threadIdx.x == 0) {
            block_sums[blockIdx.x] = total;
            __threadfence();
            last = atomicAdd(&rows->ticket, 1u) == gridDim.x - 1;
        }
        __syncthreads();
        if (!last) return;
        __threadfence();
        total = 0.0;
        for (uint32_t b = threadIdx.x; b < gridDim.x; b += kThreads) total += __ldcg(block_sums + b);
        total = block_total(total);
    }
    if (threadIdx.x == 0) {
        *mean = failed ? nan : (float)(total / (double)max(count, 1u));
        rows->ticket = 0;
    }
}

// A gradient from its f32 partial sums, added in order.
struct JoinArgs {
    const float* sums;  // NULL: the gradient is written already
    uint32_t splits;
    uint64_t rows, stride;
    int scatter;  // rows are compact rows from first_row on
    uint32_t first_row;
    void* out;
    int64_t out_stride;
    uint64_t all_rows;  // rows of the whole gradient
};

// Both gradients of a chunk; after the last chunk, NaN throughout if a device wait gave up (a gradient
// without sums got its own from k_label_gemm).
template <typename T>
__global__ void __launch_bounds__(kThreads) k_join_gradients(const RowSet* __restrict__ rows,
                                                             const uint32_t* __restrict__ row_of, uint32_t dim,
                                                             JoinArgs features, JoinArgs weight) {
    chain_enter();
    const bool failed = rows->status != 0;
    const uint64_t thread = (uint64_t)blockIdx.x * kThreads + threadIdx.x, threads = (uint64_t)gridDim.x * kThreads;
    const uint32_t quads = (dim + 3) / 4;
    for (int g = 0; g < 2; ++g) {
        const JoinArgs& a = g == 0 ? features : weight;
        T* out = static_cast<T*>(a.out);
        if (failed) {
            for (uint64_t i = thread; i < a.all_rows * dim; i += threads)
                out[(int64_t)(i / dim) * a.out_stride + i % dim] = from_float<T>(__int_as_float(0x7fffffff));
            continue;
        }
        if (!a.sums) continue;
        uint64_t live = a.rows;
        if (a.scatter) live = rows->count > a.first_row ? min(a.rows, (uint64_t)(rows->count - a.first_row)) : 0;
        for (uint64_t i = thread; i < live * quads; i += threads) {
            const uint64_t r = i / quads;
            const uint32_t c = (uint32_t)(i - r * quads) * 4;
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (uint32_t s = 0; s < a.splits; ++s) {
                const float4 v = *reinterpret_cast<const float4*>(a.sums + (s * a.rows + r) * a.stride + c);
                sum.x += v.x;
                sum.y += v.y;
                sum.z += v.z;
                sum.w += v.w;
            }
            const uint64_t row = a.scatter ? row_of[a.first_row + r] : r;
            T* to = out + (int64_t)row * a.out_stride + c;
            const float v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c + j < dim) to[j] = from_float<T>(v[j]);
        }
    }
}

// ------------------------------------------------------------------ host side

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// cuTensorMapEncodeTiled of the loaded driver (the library does not link libcuda).
EncodeTiled encode_tiled() {
    static const EncodeTiled function = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) !=
                cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<EncodeTiled>(f);
    }();
    return function;
}

// A bf16 matrix of `parts` planes as 64 x box_rows boxes in the 128-byte swizzle; elements outside read
// as zero.
sp_status make_map(sp_context* ctx, CUtensorMap* map, const void* base, uint64_t columns, uint64_t rows,
                   uint64_t stride, uint32_t parts, uint64_t part, uint32_t box_rows = 64) {
    const EncodeTiled encode = encode_tiled();
    SP_REQUIRE(ctx, encode != nullptr, SP_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
    const cuuint64_t dims[3] = {columns, rows, parts};
    const cuuint64_t strides[2] = {stride * 2, parts > 1 ? part * 2 : stride * 2};
    const cuuint32_t box[3] = {64, box_rows, 1}, steps[3] = {1, 1, 1};
    const CUresult r =
        encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, steps,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    SP_REQUIRE(ctx, r == CUDA_SUCCESS, SP_ERR_CUDA, "cuTensorMapEncodeTiled: error " + std::to_string((int)r));
    return SP_OK;
}

// Tiled copies need a 16-byte base and row pitch (below 2^40 bytes).
bool in_place(const sp_label_head* h, const void* p, int64_t stride) {
    return h->element == SP_BF16 && reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 8 == 0 &&
           (uint64_t)stride < (1ull << 39);
}

bool vector_rows(const sp_label_head* h, const void* p, int64_t stride) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % (16 / (int64_t)element_size(h->element)) == 0;
}

// How a product is cut up: pairs of blocks or single ones, and the pieces of the label tiles (of
// the inner dimension, for an output gradient).
struct Plan {
    bool pair;
    uint32_t m_tiles, n_tiles, splits;
    uint64_t items() const { return (uint64_t)m_tiles * splits; }
};

uint32_t tiles_of(uint64_t n, bool pair) { return (uint32_t)((n + (pair ? kPairTile : kTile) - 1) / (pair ? kPairTile : kTile)); }

// The cut that finishes soonest: whole waves of blocks times the longest piece, a pair's tile
// counted as kPairCost single ones (four times the products on two SMs that share their operands).
// At most kLogitWaves waves of pieces where there is more than one; starting a piece costs about a tenth
// of a tile.
Plan plan_logits(uint32_t sms, uint64_t rows, uint64_t labels) {
    Plan best{};
    double best_cost = 1e300;
    for (int pair = 0; pair < (rows <= kTile ? 1 : 2); ++pair) {  // no pair for half a pair's tile
        const uint32_t workers = pair ? std::max(sms / 2, 1u) : sms;
        const uint32_t m = tiles_of(rows, pair), n = tiles_of(labels, pair);
        for (uint32_t s = 1; s <= n && (s == 1 || (uint64_t)m * s <= (uint64_t)kLogitWaves * workers); ++s) {
            const double cost = (double)(((uint64_t)m * s + workers - 1) / workers) * ((n + s - 1) / s + 0.1) *
                                (pair ? kPairCost : 1.0);
            if (cost < best_cost) best_cost = cost, best = Plan{pair != 0, m, n, s};
        }
    }
    return best;
}

// The same for the two output gradients of a chunk of rows, whose tiles share the SMs, the longer
// ones first. Their pieces go through f32 sums, written and read at some 6.5 TB/s (and joined by a
// launch of their own) against kStepUs for a single block's step; at most kOutWaves waves of pieces,
// none below 4 steps. With `weight_splits` not 0 the weight's gradient is cut as before.
struct OutPlan {
    bool pair;
    uint32_t m_features, m_weight, n, features, weight;  // tiles, and the pieces of either
    bool weight_first;
    double us;
    uint64_t items() const { return ((uint64_t)m_features * features + (uint64_t)m_weight * weight) * n; }
};

OutPlan plan_out(uint32_t sms, uint64_t rows, uint64_t labels, uint32_t dim, uint32_t parts, bool sums_anyway,
                 uint32_t weight_splits = 0) {
    OutPlan best{};
    best.us = 1e300;
    const uint32_t label_k = (uint32_t)((labels + kBlockK - 1) / kBlockK), row_k = (uint32_t)((rows + kBlockK - 1) / kBlockK);
    const double products = parts > 1 ? kPartProducts : 1;
    for (int pair = 0; pair < 2; ++pair) {
        const uint32_t workers = pair ? std::max(sms / 2, 1u) : sms;
        const uint32_t mf = tiles_of(rows, pair), mw = tiles_of(labels, pair), n = tiles_of(dim, pair);
        const double step_us = products * kStepUs * (pair ? kPairCost : 1.0);
        // f32 operands' sums are cut at kLongestSum steps: the tensor cores' additions truncate.
        const uint32_t least_f = parts > 1 ? (label_k + kLongestSum - 1) / kLongestSum : 1;
        const uint32_t least_w = parts > 1 ? (row_k + kLongestSum - 1) / kLongestSum : 1;
        auto allowed = [&](uint64_t tiles, uint32_t s, uint32_t least, uint32_t k) {
            return s == least || (tiles * s <= (uint64_t)kOutWaves * workers && k >= 4 * s);
        };
        for (uint32_t sf = least_f; allowed((uint64_t)mf * n, sf, least_f, label_k); ++sf)
            for (uint32_t sw = weight_splits ? weight_splits : least_w;
                 (weight_splits && sw == weight_splits) || (!weight_splits && allowed((uint64_t)mw * n, sw, least_w, row_k)); ++sw) {
                const uint32_t kf = (label_k + sf - 1) / sf, kw = (row_k + sw - 1) / sw;
                const uint64_t fi = (uint64_t)mf * n * sf, wi = (uint64_t)mw * n * sw;
                // The first worker has the most pieces, and the most of the long ones.
                const bool weight_first = kw > kf;
                const uint64_t longs = ((weight_first ? wi : fi) + workers - 1) / workers;
                const uint64_t all = (fi + wi + workers - 1) / workers;
                const double steps = (double)longs * std::max(kf, kw) + (double)(all - longs) * std::min(kf, kw);
                double us = steps * step_us;
                if (sf > 1) us += (double)sf * rows * dim * 8.0 / 6.5e6;
                if (sw > 1 || sums_anyway) us += (double)sw * labels * dim * 8.0 / 6.5e6;
                if ((sf > 1 || sw > 1) && !sums_anyway) us += kLaunchUs;
                if (us < best.us) best = OutPlan{pair != 0, mf, mw, n, sf, sw, weight_first, us};
            }
    }
    return best;
}

// Rows whose slopes in one part (f32: in three) the workspace holds: all, twice where they may have two parts,
// or what the budget has room for, but a pair's tile of the most parts.
uint64_t slope_rows(const sp_label_head* h) {
    const uint64_t rows = kSlopeBudget / (h->slope_stride() * h->parts()) / kPairTile * kPairTile;
    const uint64_t twice = h->element == SP_BF16 && h->max_rows > kTile ? 2 : 1;
    return std::max(std::min(rows, twice * round_up(h->max_rows, kPairTile)), twice * kPairTile);
}

// The rows of slopes of `parts` taken at once: all of them, or else of the even cuts and of those that fill the
// SMs with whole tiles of the features' gradient, the one whose products finish soonest.
uint64_t chunk_for(const sp_label_head* h, uint64_t rows, uint32_t parts) {
    if (rows <= kTile) return parts == 2 ? kTile : kPairTile;  // two parts: what fits where one of a pair's tile does
    const uint64_t room = slope_rows(h) * h->parts() / parts / kPairTile * kPairTile;
    const uint64_t limit = std::min(room, round_up(rows, kPairTile));
    if (rows <= limit) return limit;
    const uint64_t wave = std::max<uint64_t>(h->sms / 2 / tiles_of(h->dim, true), 1) * kPairTile;
    const uint64_t fewest = (rows + limit - 1) / limit;
    uint64_t best = 0;
    double best_cost = 1e300;
    auto consider = [&](uint64_t chunk) {
        if (chunk == 0 || chunk > limit) return;
        double cost = 0.0;
        const uint64_t whole = rows / chunk, rest = rows % chunk;
        for (uint64_t part : {chunk, rest})
            if (part != 0)
                cost += plan_out(h->sms, part, h->labels, h->dim, h->parts(), true).us * (part == chunk ? (double)whole : 1.0);
        if (cost < best_cost) best_cost = cost, best = chunk;
    };
    for (uint64_t chunks = fewest; chunks < fewest + 3; ++chunks) consider(round_up((rows + chunks - 1) / chunks, kPairTile));
    consider(limit / wave * wave);
    return best;
}

// Rows of f32 sums that a gradient of `rows` rows over an inner dimension of up to `inner` may need. plan_out:
// pieces times tiles stay within kOutWaves waves, and a piece is 4 steps or longer; or f32's least pieces.
uint64_t sums_rows(const sp_label_head* h, uint64_t rows, uint64_t inner) {
    const uint64_t k = (inner + kBlockK - 1) / kBlockK, longest = h->parts() > 1 ? (k + kLongestSum - 1) / kLongestSum : 1;
    const uint64_t chosen = k >= 8 ? std::min((uint64_t)kOutWaves * h->sms * kTile, rows * (k / 4)) : 0;
    return std::max(chosen, longest > 1 ? rows * longest : 0);
}
// ... the features' gradient, and the weight's, which one piece of several chunks needs too.
uint64_t feature_sums_rows(const sp_label_head* h) {
    return sums_rows(h, std::min(h->max_rows, slope_rows(h)), h->labels);
}
uint64_t weight_sums_rows(const sp_label_head* h) {
    return std::max(h->labels, sums_rows(h, h->labels, std::min(h->max_rows, slope_rows(h))));
}

uint64_t sums_stride(const sp_label_head* h) { return ((uint64_t)h->dim + 3) / 4 * 4; }

template <typename T>
sp_status allocate(sp_label_head* h, T** out, uint64_t count) {
    void* p = nullptr;
    SP_CUDA(h->ctx, cudaMalloc(&p, std::max<uint64_t>(count * sizeof(T), 16)));
    h->allocations.push_back(p);
    *out = static_cast<T*>(p);
    return SP_OK;
}

// One call's inputs: the compacted rows and the operand maps.
struct Operands {
    CUtensorMap features, features_packed, weight;
    uint32_t all_rows;  // as in GemmArgs
};

template <int ENDING, bool PAIR, typename T>
cudaError_t launch_gemm(const sp_label_head* h, uint64_t items, const Operands& op, const CUtensorMap& slopes,
                        const GemmArgs& args) {
    auto kernel = k_label_gemm<ENDING, PAIR, T>;
    static std::atomic<unsigned long long> configured{0};
    using S = Shape<ENDING, PAIR, T>;
    const cudaError_t err = allow_smem_once(kernel, S::smem, configured);
    if (err != cudaSuccess) return err;
    constexpr unsigned blocks = PAIR ? 2 : 1;
    const unsigned workers = (unsigned)std::max<uint64_t>(1, std::min<uint64_t>(items, h->sms / blocks));
    cudaLaunchConfig_t config{};
    config.gridDim = workers * blocks;
    config.blockDim = S::threads;
    config.dynamicSmemBytes = S::smem;
    config.stream = h->ctx->stream;
    cudaLaunchAttribute attributes[2];
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = blocks;
    attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
    config.attrs = attributes;
    config.numAttrs = 2;
    return cudaLaunchKernelEx(&config, kernel, op.features, op.features_packed, op.weight, slopes, args);
}

template <int ENDING, typename T>
cudaError_t run_gemm(const sp_label_head* h, bool pair, uint64_t items, const Operands& op, const CUtensorMap& slopes,
                     const GemmArgs& args) {
    return pair ? launch_gemm<ENDING, true, T>(h, items, op, slopes, args)
                : launch_gemm<ENDING, false, T>(h, items, op, slopes, args);
}

template <typename T, bool DIRECT>
cudaError_t launch_thin(const sp_label_head* h, uint32_t blocks, const Operands& op, const ThinArgs& args) {
    constexpr size_t smem = thin_smem(sizeof(T) == 4);
    static std::atomic<unsigned long long> configured{0};
    const cudaError_t err = allow_smem_once(k_label_thin<T, DIRECT>, smem, configured);
    if (err != cudaSuccess) return err;
    return launch_chained(k_label_thin<T, DIRECT>, blocks, thin_threads(DIRECT), smem, h->ctx->stream, op.features,
                          op.features_packed, op.weight, args);
}

sp_status check_matrix(sp_context* ctx, const void* p, int64_t stride, uint32_t dim, size_t size, const char* what) {
    SP_REQUIRE(ctx, p != nullptr, SP_ERR_INVALID, std::string("null ") + what);
    SP_REQUIRE(ctx, reinterpret_cast<uintptr_t>(p) % size == 0, SP_ERR_INVALID, std::string("misaligned ") + what);
    SP_REQUIRE(ctx, stride >= (int64_t)dim, SP_ERR_INVALID, std::string("row stride below dim: ") + what);
    return SP_OK;
}

sp_status prepare(sp_label_head* h, const void* features, int64_t feature_stride, const void* weight,
                  int64_t weight_stride, const void* targets, int wide, uint64_t n, float* losses, double* normalizers,
                  void* gradient, int64_t gradient_stride, bool weight_needed, Operands* out) {
    sp_context* ctx = h->ctx;
    cudaStream_t st = ctx->stream;
    const uint64_t stride = h->packed_stride(), capacity = round_up(h->max_rows, kPairTile);
    const uint32_t parts = h->parts();
    const bool features_here = in_place(h, features, feature_stride), weight_here = in_place(h, weight, weight_stride);
    // Without targets every row counts: nothing to gather where the operands can be read in place.
    out->all_rows = !targets && features_here && (weight_here || !weight_needed) ? (uint32_t)n : 0;
    SP_CHECK(make_map(ctx, &out->features_packed, h->packed_features, h->dim, capacity, stride, parts, capacity * stride));
    if (features_here) SP_CHECK(make_map(ctx, &out->features, features, h->dim, n, feature_stride, 1, 0));
    else out->features = out->features_packed;
    if (weight_here) SP_CHECK(make_map(ctx, &out->weight, weight, h->dim, h->labels, weight_stride, 1, 0));
    else SP_CHECK(make_map(ctx, &out->weight, h->packed_weight, h->dim, h->labels, stride, parts, h->labels * stride));

    if (out->all_rows) return SP_OK;
    const unsigned blocks = grid_for(n, kGatherRows);
    const uint32_t* counts = nullptr;
    if (targets && blocks > kRecountBlocks) {
        SP_CUDA(ctx, launch_chained(k_count_targets, grid_for(blocks, kCountGroups), kCountGroups * 32, 0, st, targets,
                                    wide, n, h->labels, h->counts, h->counts + h->count_blocks()));
        counts = h->counts;
    }
    auto gather = [&](auto* typed) {
        using T = std::remove_pointer_t<decltype(typed)>;
        PackWeight<T> pack{nullptr, weight_stride, (int)vector_rows(h, weight, weight_stride), h->packed_weight};
        unsigned weight_blocks = 0;
        if (!weight_here && weight_needed) {
            pack.from = static_cast<const T*>(weight);
            weight_blocks = (unsigned)std::min<uint64_t>((h->labels + kThreads / 32 - 1) / (kThreads / 32), 148 * 16);
        }
        // Few blocks of rows share their copies among more, up to a wave of blocks.
        const uint32_t sharers = std::max(1u, std::min(16u, h->sms / blocks));
        return launch_chained(k_gather_rows<T>, blocks * sharers + weight_blocks, kThreads, 0, st, targets, wide, n,
                              h->labels, blocks, sharers, counts, static_cast<const uint32_t*>(h->counts + h->count_blocks()),
                              static_cast<const T*>(features), feature_stride, h->dim,
                              (int)vector_rows(h, features, feature_stride), (int)features_here, h->rows, h->row_of,
                              h->packed_features, stride, capacity * stride, losses, normalizers,
                              static_cast<T*>(gradient), gradient_stride, pack);
    };
    const cudaError_t err = h->element == SP_F32 ? gather((float*)nullptr) : gather((bf16*)nullptr);
    SP_CUDA(ctx, err);
    return SP_OK;
}

// The scale of logits that took `additions`, in powers of 2.
float scale2_for(float scale, uint32_t additions) { return (float)(scale * 1.4426950408889634 * given_back(additions)); }

GemmArgs common_args(const sp_label_head* h, const void* targets, int wide, float scale) {
    GemmArgs a;
    std::memset(&a, 0, sizeof(a));
    a.rows = h->rows;
    a.row_of = h->row_of;
    a.labels = (uint32_t)h->labels;
    a.dim = h->dim;
    a.products = h->products();
    a.parts_a = h->element == SP_F32 ? kPartsOfA : 0;
    a.parts_b = h->element == SP_F32 ? kPartsOfB : 0;
    a.chunk_rows = 0x80000000u;
    a.splits = 1;
    a.scale = scale;
    a.scale2 = scale2_for(scale, (h->dim + 15) / 16);
    a.per_scale = 1.4426950408889634 / a.scale2;
    a.targets = targets;
    a.wide = wide;
    return a;
}

sp_status check_call(sp_label_head* h, const void* features, int64_t feature_stride, const void* weight,
                     int64_t weight_stride, uint64_t rows, float scale) {
    sp_context* ctx = h->ctx;
    const size_t size = element_size(h->element);
    SP_REQUIRE(ctx, rows <= h->max_rows, SP_ERR_INVALID, "more rows than the label head was made for");
    SP_REQUIRE(ctx, scale > 0.0f && scale < INFINITY, SP_ERR_INVALID, "logit_scale must be positive and finite");
    SP_CHECK(check_matrix(ctx, weight, weight_stride, h->dim, size, "weight"));
    if (rows > 0) SP_CHECK(check_matrix(ctx, features, feature_stride, h->dim, size, "features"));
    return SP_OK;
}

sp_status check_targets(sp_context* ctx, const void* targets, sp_index index) {
    SP_REQUIRE(ctx, index == SP_INDEX32 || index == SP_INDEX64, SP_ERR_INVALID, "index type");
    SP_REQUIRE(ctx, targets != nullptr, SP_ERR_INVALID, "null targets");
    SP_REQUIRE(ctx, reinterpret_cast<uintptr_t>(targets) % (index == SP_INDEX64 ? 8 : 4) == 0, SP_ERR_INVALID,
               "misaligned targets");
    return SP_OK;
}

// Whether the few-row pass takes a call. Not a training head's loss: its gradient makes the logits again
// in the other pass, and a confident row's slope is the small difference of the two passes' numbers, which
// have to be rounded alike.
bool few_rows(const sp_label_head* h, uint64_t n, const void* targets) {
    return n <= kThinRows && !(targets && h->training);
}

// The pass over the logits shared by the loss and the prediction.
sp_status run_stats(sp_label_head* h, const Operands& op, const void* weight, int64_t weight_stride,
                    const void* targets, int wide, uint64_t n, float scale,
                    float* mean, float* losses, double* normalizers, int32_t* labels_out, float* log_probability) {
    sp_context* ctx = h->ctx;
    GemmArgs a = common_args(h, targets, wide, scale);
    a.all_rows = op.all_rows;
    a.k_blocks = (h->dim + kBlockK - 1) / kBlockK;
    a.partials = h->partials;
    a.partial_labels = labels_out ? h->partial_labels : nullptr;
    a.target_logits = h->target_logits;
    uint32_t slots = 0;
    if (few_rows(h, n, targets)) {
        ThinArgs thin;
        thin.weight = weight;
        thin.weight_stride = weight_stride;
        thin.dim = h->dim;
        thin.vector = vector_rows(h, weight, weight_stride);
        thin.known_rows = targets || op.all_rows ? 0 : (uint32_t)n;
        thin.columns = (uint32_t)round_up(n, 16);
        // Whole rounds of tiles over the SMs; converted weights come in tiles of the height that fills
        // the last round too.
        const bool direct = in_place(h, weight, weight_stride);
        const uint64_t round = (uint64_t)(direct ? kTile : kConvertTile) * h->sms, rounds = (h->labels + round - 1) / round;
        thin.tile = direct ? kTile : (uint32_t)round_up((h->labels + rounds * h->sms - 1) / (rounds * h->sms), 8);
        thin.tiles = (uint32_t)((h->labels + thin.tile - 1) / thin.tile);
        const uint32_t blocks = std::min(thin.tiles, h->sms);
        a.partial_rows = kThinRows;
        slots = blocks;
        a.scale2 = scale2_for(scale, ((h->dim + 15) / 16 + 1) / 2);  // two accumulators
        thin.g = a;
        const cudaError_t err = h->element == SP_F32                 ? launch_thin<float, false>(h, blocks, op, thin)
                                : direct                             ? launch_thin<bf16, true>(h, blocks, op, thin)
                                                                     : launch_thin<bf16, false>(h, blocks, op, thin);
        SP_CUDA(ctx, err);
    } else {
        const Plan plan = plan_logits(h->sms, n, h->labels);
        a.n_tiles = plan.n_tiles;
        a.splits = plan.splits;
        a.partial_rows = (uint64_t)plan.m_tiles * (plan.pair ? kPairTile : kTile);
        if (h->element == SP_F32) {
            slots = (plan.pair ? Shape<kStats, true, float>::column_parts : Shape<kStats, false, float>::column_parts) * a.splits;
            SP_CUDA(ctx, (run_gemm<kStats, float>(h, plan.pair, plan.items(), op, op.weight, a)));
        } else {
            slots = (plan.pair ? Shape<kStats, true, bf16>::column_parts : Shape<kStats, false, bf16>::column_parts) * a.splits;
            SP_CUDA(ctx, (run_gemm<kStats, bf16>(h, plan.pair, plan.items(), op, op.weight, a)));
        }
    }
    auto join = [&](auto kernel, uint32_t lanes) {
        return launch_chained(kernel, grid_for(n * lanes, kThreads), kThreads, 0, ctx->stream, h->rows,
                              static_cast<const uint32_t*>(h->row_of), a.all_rows,
                              static_cast<const float2*>(h->partials),
                              static_cast<const uint32_t*>(a.partial_labels), a.partial_rows, slots, a.scale2,
                              static_cast<const float*>(h->target_logits), losses, normalizers, labels_out,
                              log_probability, h->loss_sums, mean);
    };
        // About kThreadSlots partials a thread, as far as a warp goes.
    SP_CUDA(ctx, slots <= kThreadSlots       ? join(k_join_rows<1>, 1)
                 : slots <= 8 * kThreadSlots ? join(k_join_rows<8>, 8)
                                             : join(k_join_rows<32>, 32));
    return SP_OK;
}

}  // namespace

// The entries catch whatever the host code may throw (a string or list that finds no memory).
extern "C" {

sp_status sp_label_head_create(sp_context* ctx, uint64_t labels, uint32_t dim, sp_element element, uint64_t max_rows,
                               int training, sp_label_head** out) try {
    if (!ctx || !out) return SP_ERR_INVALID;
    *out = nullptr;
    SP_REQUIRE(ctx, labels > 0 && labels < (1ull << 31) - 512, SP_ERR_INVALID, "labels outside [1, 2^31 - 512)");
    SP_REQUIRE(ctx, dim > 0 && dim < (1u << 20), SP_ERR_INVALID, "dim outside [1, 2^20)");
    SP_REQUIRE(ctx, element == SP_F32 || element == SP_BF16, SP_ERR_INVALID, "element type");
    SP_REQUIRE(ctx, max_rows > 0 && max_rows < (1ull << 31) - 512, SP_ERR_INVALID, "max_rows outside [1, 2^31 - 512)");
    SP_CHECK(select_device(ctx));
    sp_label_head* h = new (std::nothrow) sp_label_head();
    SP_REQUIRE(ctx, h != nullptr, SP_ERR_OUT_OF_MEMORY, "host memory");
    h->ctx = ctx;
    h->labels = labels;
    h->dim = dim;
    h->element = element;
    h->max_rows = max_rows;
    h->training = training != 0;
    sp_status s = SP_OK;
    auto all = [&]() -> sp_status {
        int sms = 0;
        SP_CUDA(ctx, cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, ctx->device));
        h->sms = (uint32_t)std::max(sms, 1);
        const uint64_t capacity = round_up(max_rows, kPairTile), stride = h->packed_stride();
        SP_CHECK(allocate(h, &h->rows, 1));
        SP_CUDA(ctx, cudaMemsetAsync(h->rows, 0, sizeof(RowSet), ctx->stream));
        SP_CHECK(allocate(h, &h->row_of, max_rows));
        SP_CHECK(allocate(h, &h->counts, h->count_blocks() + (h->count_blocks() + kCountGroups - 1) / kCountGroups));
        SP_CHECK(allocate(h, &h->packed_features, capacity * stride * h->parts()));
        SP_CHECK(allocate(h, &h->packed_weight, labels * stride * h->parts()));
        // plan_logits: pieces times row tiles stay within kLogitWaves waves, or one piece.
        const uint64_t slots = 4 * kTile * std::max<uint64_t>(capacity / kTile, (uint64_t)kLogitWaves * h->sms);
        SP_CHECK(allocate(h, &h->partials, slots));
        SP_CHECK(allocate(h, &h->partial_labels, slots));
        SP_CHECK(allocate(h, &h->target_logits, capacity));
        SP_CHECK(allocate(h, &h->loss_sums, (max_rows * 32 + kThreads - 1) / kThreads));
        if (h->training) {
            SP_CHECK(allocate(h, &h->slopes, slope_rows(h) * h->slope_stride() * h->parts()));
            SP_CHECK(allocate(h, &h->sums, (feature_sums_rows(h) + weight_sums_rows(h)) * sums_stride(h)));
        }
        return SP_OK;
    };
    if ((s = all()) != SP_OK) {
        sp_label_head_destroy(h);
        return s;
    }
    *out = h;
    return SP_OK;
} catch (...) {
    return SP_ERR_OUT_OF_MEMORY;
}

void sp_label_head_destroy(sp_label_head* h) {
    if (!h) return;
    cudaSetDevice(h->ctx->device);
    cudaStreamSynchronize(h->ctx->stream);
    for (void* p : h->allocations) cudaFree(p);
    delete h;
}

sp_status sp_label_head_loss(sp_label_head* h, const void* d_features, int64_t feature_stride, const void* d_weight,
                             int64_t weight_stride, const void* d_targets, sp_index index, uint64_t rows,
                             float logit_scale, float* d_mean, float* d_losses, double* d_log_normalizers) try {
    if (!h) return SP_ERR_INVALID;
    sp_context* ctx = h->ctx;
    NvtxRange range("sp_label_head_loss");
    SP_CHECK(check_call(h, d_features, feature_stride, d_weight, weight_stride, rows, logit_scale));
    SP_REQUIRE(ctx, d_mean != nullptr, SP_ERR_INVALID, "null mean");
    SP_CHECK(select_device(ctx));
    if (rows == 0) {
        SP_CUDA(ctx, cudaMemsetAsync(d_mean, 0, sizeof(float), ctx->stream));
        return SP_OK;
    }
    SP_CHECK(check_targets(ctx, d_targets, index));
    SP_REQUIRE(ctx, d_losses != nullptr && d_log_normalizers != nullptr, SP_ERR_INVALID, "null output");
    Operands op;
    const int wide = index == SP_INDEX64;
    SP_CHECK(prepare(h, d_features, feature_stride, d_weight, weight_stride, d_targets, wide, rows, d_losses,
                     d_log_normalizers, nullptr, 0, !few_rows(h, rows, d_targets), &op));
    return run_stats(h, op, d_weight, weight_stride, d_targets, wide, rows, logit_scale, d_mean, d_losses, d_log_normalizers, nullptr, nullptr);
} catch (...) {
    return SP_ERR_OUT_OF_MEMORY;
}

sp_status sp_label_head_predict(sp_label_head* h, const void* d_features, int64_t feature_stride,
                                const void* d_weight, int64_t weight_stride, uint64_t rows, float logit_scale,
                                int32_t* d_labels, float* d_log_probabilities) try {
    if (!h) return SP_ERR_INVALID;
    sp_context* ctx = h->ctx;
    NvtxRange range("sp_label_head_predict");
    SP_CHECK(check_call(h, d_features, feature_stride, d_weight, weight_stride, rows, logit_scale));
    if (rows == 0) return SP_OK;
    SP_REQUIRE(ctx, d_labels != nullptr && d_log_probabilities != nullptr, SP_ERR_INVALID, "null output");
    SP_CHECK(select_device(ctx));
    Operands op;
    SP_CHECK(prepare(h, d_features, feature_stride, d_weight, weight_stride, nullptr, 0, rows, nullptr, nullptr,
                     nullptr, 0, !few_rows(h, rows, nullptr), &op));
    return run_stats(h, op, d_weight, weight_stride, nullptr, 0, rows, logit_scale, nullptr, nullptr, nullptr, d_labels, d_log_probabilities);
} catch (...) {
    return SP_ERR_OUT_OF_MEMORY;
}

sp_status sp_label_head_gradient(sp_label_head* h, const void* d_features, int64_t feature_stride,
                                 const void* d_weight, int64_t weight_stride, const void* d_targets, sp_index index,
                                 uint64_t rows, float logit_scale, const double* d_log_normalizers,
                                 const float* d_row_gradient, void* d_feature_gradient,
                                 int64_t feature_gradient_stride, void* d_weight_gradient,
                                 int64_t weight_gradient_stride) try {
    if (!h) return SP_ERR_INVALID;
    sp_context* ctx = h->ctx;
    NvtxRange range("sp_label_head_gradient");
    const size_t size = element_size(h->element);
    SP_REQUIRE(ctx, h->training, SP_ERR_INVALID, "the label head was not made for training");
    SP_CHECK(check_call(h, d_features, feature_stride, d_weight, weight_stride, rows, logit_scale));
    SP_CHECK(check_matrix(ctx, d_weight_gradient, weight_gradient_stride, h->dim, size, "weight gradient"));
    SP_CHECK(select_device(ctx));
    if (rows == 0) {
        SP_CUDA(ctx, cudaMemset2DAsync(d_weight_gradient, weight_gradient_stride * size, 0, h->dim * size, h->labels,
                                       ctx->stream));
        return SP_OK;
    }
    SP_CHECK(check_targets(ctx, d_targets, index));
    SP_REQUIRE(ctx, d_log_normalizers != nullptr, SP_ERR_INVALID, "null log normalizers");
    SP_CHECK(check_matrix(ctx, d_feature_gradient, feature_gradient_stride, h->dim, size, "feature gradient"));
    const int wide = index == SP_INDEX64;
    Operands op;
    SP_CHECK(prepare(h, d_features, feature_stride, d_weight, weight_stride, d_targets, wide, rows, nullptr, nullptr,
                     d_feature_gradient, feature_gradient_stride, true, &op));

    const uint32_t slope_parts = h->slope_parts(rows, d_row_gradient != nullptr);
    const uint64_t chunk = chunk_for(h, rows, slope_parts), chunks = (rows + chunk - 1) / chunk;
    const uint64_t sum_stride = sums_stride(h);
    CUtensorMap slopes, slopes_out;
    const uint32_t panels = (uint32_t)(h->slope_stride() / 64);
    SP_CHECK(make_map(ctx, &slopes, h->slopes, 64, chunk, 64, panels * slope_parts, chunk * 64));
    SP_CHECK(make_map(ctx, &slopes_out, h->slopes, 64, chunk, 64, panels * slope_parts, chunk * 64, 32));
    // One cut of the weight's gradient for every chunk: its pieces' sums go on from one to the next.
    const OutPlan first = plan_out(h->sms, std::min(chunk, rows), h->labels, h->dim, h->parts(), chunks > 1);
    const bool weight_sums = first.weight > 1 || chunks > 1;
    float* weight_sum = h->sums;
    float* feature_sum = h->sums + weight_sums_rows(h) * sum_stride;

    for (uint64_t c = 0; c < chunks; ++c) {
        const uint64_t here = std::min(chunk, rows - c * chunk);
        const Plan logits = plan_logits(h->sms, here, h->labels);
        const OutPlan plan = c == 0 ? first
                                    : plan_out(h->sms, here, h->labels, h->dim, h->parts(), true, first.weight);
        const bool feature_sums = plan.features > 1;
        SP_REQUIRE(ctx, (!feature_sums || plan.features * here <= feature_sums_rows(h)) &&
                            (!weight_sums || plan.weight * h->labels <= weight_sums_rows(h)),
                   SP_ERR_OVERFLOW, "the gradients' sums exceed their workspace");
        GemmArgs a = common_args(h, d_targets, wide, logit_scale);
        a.first_row = (uint32_t)(c * chunk);
        a.chunk_rows = (uint32_t)chunk;
        a.k_blocks = (h->dim + kBlockK - 1) / kBlockK;
        a.n_tiles = logits.n_tiles;
        a.splits = logits.splits;
        a.log_normalizers = d_log_normalizers;
        a.row_gradient = d_row_gradient;
        a.panels = panels;
        a.residuals = h->target_logits;  // free in a gradient
        const bool weight_here = in_place(h, d_weight, weight_stride);
        a.weight = weight_here ? static_cast<const bf16*>(d_weight) : h->packed_weight;
        a.weight_stride = weight_here ? weight_stride : (int64_t)h->packed_stride();
        SP_CUDA(ctx, h->element == SP_F32 ? (run_gemm<kSlopes, float>(h, logits.pair, logits.items(), op, slopes_out, a))
                     : slope_parts == 1   ? (run_gemm<kSlopes, bf16>(h, logits.pair, logits.items(), op, slopes_out, a))
                                          : (run_gemm<kFineSlopes, bf16>(h, logits.pair, logits.items(), op, slopes_out, a)));

        if (slope_parts == 2) a.products = 2, a.only_weight = 1, a.parts_a = 0x01;  // the small part first
        OutArgs& f = a.out[0];
        f.n_tiles = plan.n;
        f.splits = plan.features;
        f.k_blocks = (uint32_t)((h->labels + kBlockK - 1) / kBlockK);
        f.partial = feature_sums;
        f.out = feature_sums ? (void*)feature_sum : d_feature_gradient;
        f.stride = feature_sums ? (int64_t)sum_stride : feature_gradient_stride;
        f.rows = here;
        f.packed = vector_rows(h, d_feature_gradient, feature_gradient_stride);
        OutArgs& w = a.out[1];
        w.m_tiles = plan.m_weight;
        w.n_tiles = plan.n;
        w.splits = plan.weight;
        w.partial = weight_sums;
        w.add = c > 0;
        w.out = weight_sums ? (void*)weight_sum : d_weight_gradient;
        w.stride = weight_sums ? (int64_t)sum_stride : weight_gradient_stride;
        w.rows = h->labels;
        w.packed = vector_rows(h, d_weight_gradient, weight_gradient_stride);
        a.weight_first = plan.weight_first;
        SP_CUDA(ctx, h->element == SP_F32 ? (run_gemm<kOut, float>(h, plan.pair, plan.items(), op, slopes, a))
                                          : (run_gemm<kOut, bf16>(h, plan.pair, plan.items(), op, slopes, a)));

        const bool last = c + 1 == chunks;
        JoinArgs jf{feature_sums ? feature_sum : nullptr, plan.features, here, sum_stride, 1, a.first_row,
                    d_feature_gradient, feature_gradient_stride, last ? rows : 0};
        JoinArgs jw{weight_sums && last ? weight_sum : nullptr, plan.weight, h->labels, sum_stride, 0, 0,
                    d_weight_gradient, weight_gradient_stride, last ? h->labels : 0};
        if (!jf.sums && !jw.sums) continue;  // written already, NaN included
        const uint64_t quads = std::max(feature_sums ? here * (sum_stride / 4) : (uint64_t)0,
                                        jw.sums ? h->labels * (sum_stride / 4) : (uint64_t)0);
        const unsigned grid = (unsigned)std::min<uint64_t>((quads + kThreads - 1) / kThreads, 148 * 16);
        SP_CUDA(ctx, h->element == SP_F32
                         ? launch_chained(k_join_gradients<float>, grid, kThreads, 0, ctx->stream,
                                          static_cast<const RowSet*>(h->rows), static_cast<const uint32_t*>(h->row_of),
                                          h->dim, jf, jw)
                         : launch_chained(k_join_gradients<bf16>, grid, kThreads, 0, ctx->stream,
                                          static_cast<const RowSet*>(h->rows), static_cast<const uint32_t*>(h->row_of),
                                          h->dim, jf, jw));
    }
    return SP_OK;
} catch (...) {
    return SP_ERR_OUT_OF_MEMORY;
}

sp_status sp_label_head_check(sp_label_head* h) try {
    if (!h) return SP_ERR_INVALID;
    sp_context* ctx = h->ctx;
    SP_CHECK(select_device(ctx));
    uint32_t status = 0;
    SP_CUDA(ctx, cudaMemcpyAsync(&status, &h->rows->status, sizeof(status), cudaMemcpyDeviceToHost, ctx->stream));
    SP_CHECK(sync_stream(ctx));
    if (status == 0) return SP_OK;
    SP_CUDA(ctx, cudaMemsetAsync(&h->rows->status, 0, sizeof(status), ctx->stream));
    return fail(ctx, (sp_status)status, "a device-side wait gave up (label head pipeline)");
} catch (...) {
    return SP_ERR_OUT_OF_MEMORY;
}

}  // extern "C"
