// The tensor-core pipeline of the label head: D = A B^T over bf16 operands in tiles of 256 x 256
// per pair of thread blocks (or 128 x 128 per block), f32 accumulators in tensor memory, and three
// endings for a tile:
//   kStats   the logits' running sum of exponentials per row, and the target's logit or the
//            largest one and its label
//   kSlopes  the softmax slopes p - [target] (times c g of the row, if rows have their own), written as
//            bf16 parts: f32's three, or one; kFineSlopes in two
//   kOut     the tile itself, or a partial sum of it, of the two output gradients dH = G W and
//            dW = G^T H, in one launch: the tiles of one fill the SMs the other's leave
//
// A block is one producer warp (tiled bulk copies into a ring of shared-memory stages), one warp
// that issues the products, and eight or sixteen warps that empty one accumulator while the other fills. In a
// pair each block keeps 128 rows of A and of B and the accumulator of its A rows; the products are
// issued by the first block and read B from both.
//
// Bound by the tensor cores: 20,000 rows x 32,768 labels x 512 bf16 take 397 us for the logits' sums (94 % of
// the tensor pipe's cycles, at 1.50 GHz), 516 us for the slopes (71 %, at 1.52: 1.26 GB written, exponentials and
// roundings beside the products) and 895 us for both gradients (92 %, at 1.35). Tiles of 256 x 256 per pair
// because a block's 128 x 128 reads twice the bytes per product from shared memory; the latter is for few rows or
// labels.
#pragma once

#include "elements.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

namespace splat {
namespace label {

constexpr int kTile = 128;     // rows of A, and of B, per block
constexpr int kPairTile = 2 * kTile;
constexpr int kBlockK = 64;    // 128 bytes of bf16
constexpr uint32_t kOperandBytes = kTile * kBlockK * 2;
constexpr uint32_t kBoxBytes = kOperandBytes / 2;  // a box is 64 x 64 elements
constexpr uint32_t kStageBytes = 2 * kOperandBytes;
constexpr uint32_t kStoreBytes = 32 * 128;  // a warp's 32 x 64 slopes on their way out

// f32 operands: three bf16 parts each, the six products of parts whose weights sum to 2^-16 or
// more of the whole, smallest first so that they are added while the sum is small. One hex digit
// per product, the first in the low one.
constexpr uint32_t kParts = 3, kPartProducts = 6;
constexpr uint32_t kPartsOfA = 0x001012, kPartsOfB = 0x010210;

// The next part of eight f32 operands, what it leaves stays in v: the upper 16 bits, then those of the rest,
// then (`last`) the other 8 bits, exact to 24 bits in all for magnitudes from 2^-110 on. Truncated, not rounded:
// no part of a finite value is infinite, and all have its sign, so that no two products of one pair of values
// overflow in opposite directions. The products left out are then 6e-8 of a logit (rounded parts: 6e-9), a
// third of what the sums lose. An infinite value is infinite in its last part alone, which meets only the other
// operand's first: against a part of 0 it would make NaN.
__device__ __forceinline__ Pack<bf16, 8> take_part(float (&v)[8], bool last) {
    Pack<bf16, 8> o;
    uint32_t* two = reinterpret_cast<uint32_t*>(&o.word);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (last) asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(two[j]) : "f"(v[2 * j + 1]), "f"(v[2 * j]));
        else asm("cvt.rz.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(two[j]) : "f"(v[2 * j + 1]), "f"(v[2 * j]));
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] -= o.get(j);
    return o;
}

// The rows that have a target, in order: row_of[i] is the i-th one's row. Where `packed`, the
// features were copied to the workspace in that order; else every row counts and they are read
// in place.
struct RowSet {
    uint32_t count;
    uint32_t packed;
    uint32_t status;  // SP_ERR_* raised on the device, kept until it is read
    uint32_t ticket;  // of the loss sum's blocks
};

constexpr uint32_t kNoTarget = 0xffffffffu;  // index_at's -1

enum Ending { kStats = 0, kSlopes = 1, kOut = 2, kFineSlopes = 3 };
constexpr bool makes_slopes(int ending) { return ending == kSlopes || ending == kFineSlopes; }

// Warps that empty the accumulators: 8, or 16 for a pair's logits of bf16 operands, where the
// exponentials take as long as the products up to some 256 columns and need more warps to overlap
// (f32 operands' products are six times as many). 227 KB of shared memory hold the outgoing slopes and
// as many stages as fit.
template <int ENDING, bool PAIR, typename T>
struct Shape {
    static constexpr int epilogue_warps = ENDING != kOut && PAIR && sizeof(T) == 2 ? 16 : 8;
    static constexpr int threads = 128 + 32 * epilogue_warps;
    static constexpr int stages = makes_slopes(ENDING) && epilogue_warps == 16 ? 5 : 6;
    static constexpr uint32_t store_bytes = makes_slopes(ENDING) ? epilogue_warps * kStoreBytes : 0;
    static constexpr size_t smem = 1024 + (size_t)stages * kStageBytes + store_bytes + 256;
    static constexpr int column_parts = epilogue_warps / 4;  // of a tile, one per four warps
    static_assert(smem <= 227 * 1024, "shared memory of a block");
};

// One of the output gradients of a chunk of rows.
struct OutArgs {
    uint32_t m_tiles, n_tiles, splits;  // m_tiles: dW's; dH's follow the row count
    uint32_t k_blocks;                  // dH's; dW's follow the row count
    void* out;            // the gradient itself, or f32 partial sums [splits][rows][stride]
    int64_t stride;
    uint64_t rows;        // of the partial sums, or of dW
    int partial;          // out holds partial sums
    int add;              // ... and this call adds to them
    int packed;           // 16-byte stores are aligned
};

struct GemmArgs {
    RowSet* rows;
    const uint32_t* row_of;
    uint32_t all_rows;     // not 0: that many rows, all of them count and are read in place
    uint32_t labels, dim;
    uint32_t products;     // 1, or more for operands in parts: those of the p-th product are the p-th hex
    uint32_t parts_a, parts_b;  // digits of these
    uint32_t only_weight;  // kOut: so many first products are dW's alone
    uint32_t k_blocks;     // kStats, kSlopes: of the features' columns
    uint32_t n_tiles;      // kStats, kSlopes: of the labels
    uint32_t splits;       // ... and the pieces they are cut into
    uint32_t first_row, chunk_rows;  // kSlopes, kOut: the rows of this call's slopes
    float scale, scale2;   // the logits' scale, and times log2(e)
    const void* targets;
    int wide;
    // kStats
    float2* partials;      // [Shape::column_parts * splits][partial_rows]: base and sum
    uint32_t* partial_labels;  // the maximum's label, or NULL
    uint64_t partial_rows;
    float* target_logits;
    // kSlopes
    const double* log_normalizers;
    double per_scale;      // log2(e) / scale2: a division per tile and row took 5 of 73 us (4096 x 8191 x 256 f32)
    const float* row_gradient;
    uint32_t panels;       // of 64 labels in a part of the slopes
    // bf16 operands: what rounding left of each row's target slope, by far the row's largest. dH takes it
    // in in f32 from the weight's rows, which undoes most of the slopes' rounding there.
    float* residuals;
    const bf16* weight;
    int64_t weight_stride;
    // kOut
    OutArgs out[2];        // dH, dW
    int weight_first;      // dW's tiles, the longer ones, come first
};

// The tensor cores truncate their f32 additions (16 products each), so that a sum ends low: by a slope,
// measured, of 0.09 to 0.16 2^-23 of itself an addition for terms of both signs at 4 to 256 additions, and 0.15
// to 0.47 for terms of one. An eighth is given back: 4096 logits over 512 random bf16 columns were off by
// 4.7e-7 of their root mean square, 4.2e-7 of that slope. A sum that loses nothing (a feature of one 1) is off by
// as much instead, so that no more is given back than for the most additions measured: 3.8e-6.
constexpr uint32_t kMostGivenBack = 256;
__host__ __device__ inline double given_back(uint32_t additions) {
    return 1.0 + ((additions < kMostGivenBack ? additions : kMostGivenBack) + 1) / 8.0 / 8388608.0;
}

struct Work {
    uint32_t m, n0, n1, k0, k1, split, which;
};

template <int ENDING, int TILE>
struct Schedule {
    uint32_t items, m_tiles, k_blocks, row_blocks, before;
    __device__ Schedule(const GemmArgs& a, uint32_t count) {
        const uint32_t here = count > a.first_row ? min(count - a.first_row, a.chunk_rows) : 0;
        m_tiles = (here + TILE - 1) / TILE;
        k_blocks = a.k_blocks;
        row_blocks = (here + kBlockK - 1) / kBlockK;
        items = m_tiles * a.splits;
        before = 0;
        if (ENDING == kOut) {
            const uint32_t features = m_tiles * a.out[0].n_tiles * a.out[0].splits;
            const uint32_t weight = a.out[1].m_tiles * a.out[1].n_tiles * a.out[1].splits;
            items = features + weight;
            before = a.weight_first ? weight : features;
        }
    }
    __device__ Work at(const GemmArgs& a, uint32_t item) const {
        Work w;
        w.which = 0;
        if (ENDING == kOut) {
            const bool second = item >= before;
            if (second) item -= before;
            w.which = (a.weight_first != 0) != second ? 1 : 0;
            const OutArgs& o = a.out[w.which];
            const uint32_t tiles = w.which ? o.m_tiles : m_tiles, blocks = w.which ? row_blocks : o.k_blocks;
            // Neighbours share the slopes' tiles, the larger operand.
            w.n0 = item % o.n_tiles;
            w.n1 = w.n0 + 1;
            w.m = item / o.n_tiles % tiles;
            w.split = item / o.n_tiles / tiles;
            w.k0 = (uint32_t)((uint64_t)blocks * w.split / o.splits);
            w.k1 = (uint32_t)((uint64_t)blocks * (w.split + 1) / o.splits);
        } else {
            // Neighbours share the label tiles.
            w.m = item % m_tiles;
            w.split = item / m_tiles;
            w.n0 = (uint32_t)((uint64_t)a.n_tiles * w.split / a.splits);
            w.n1 = (uint32_t)((uint64_t)a.n_tiles * (w.split + 1) / a.splits);
            w.k0 = 0;
            w.k1 = k_blocks;
        }
        return w;
    }
};

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two f32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)),
          "l"(reinterpret_cast<unsigned long long&>(c)));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
    return d;
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
    return d;
}

// A row's running softmax: sum of 2^((z - base) scale2) over its logits z so far, without the one that
// matters: the target's for the loss, the largest for prediction. What is left of 1 after its probability
// is then known to full precision however near 1 that is. The loss takes any logit as base that keeps the sum
// in range; prediction's is the largest. The difference comes before the scale: 2^(z scale2 - base scale2) in
// one operation is off by a whole rounding of base scale2 in the exponent, which passes f32's range at logits
// of 2^31 (the type's lowest values, as masks), and so does base scale2 itself near the largest.
constexpr float kLargestSum = 18446744073709551616.0f;  // 2^64
struct RowStats {
    float base, sum, target_logit, largest;
    uint32_t label;
};

// base, or for one of -inf (no logits so far, or none above it) any that counts those as 0.
__device__ __forceinline__ float finite_base(float base) { return base == -INFINITY ? 0.0f : base; }

template <int W>
__device__ __forceinline__ float largest_of(const float (&v)[W]) {
    float m[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
    for (int j = 4; j < W; ++j) m[j & 3] = fmaxf(m[j & 3], v[j]);
    return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}

// sum of 2^((v - base) scale2): packed operations around the exponentials, four sums.
template <int W>
__device__ __forceinline__ float sum_exp2(const float (&v)[W], float scale2, float base) {
    const float2 s2 = make_float2(scale2, scale2), below = make_float2(-base, -base);
    float2 t[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
    for (int j = 0; j < W; j += 2) {
        const float2 x = mul2(add2(make_float2(v[j], v[j + 1]), below), s2);
        t[(j / 2) & 1] = add2(t[(j / 2) & 1], make_float2(exp2_fast(x.x), exp2_fast(x.y)));
    }
    t[0] = add2(t[0], t[1]);
    return t[0].x + t[0].y;
}

// W more logits of a row, labels first..first + W - 1 (those from `labels` on are absent). The loss
// takes its base from the row's first chunk and looks for the largest logit again only when a sum
// passes 2^64 (which leaves room to join sums in f32), so that a chunk's exponentials wait for
// nothing: the running maximum in every chunk cost a quarter of the pass at width 512. The caller
// says whether the target is in the chunk of any of the lanes that are here (`near`).
template <bool LABEL, int W>
__device__ __forceinline__ void add_logits(RowStats& s, float (&v)[W], uint32_t first, uint32_t labels, float scale2,
                                           uint32_t target, bool near) {
    if (first + W > labels) {
#pragma unroll
        for (int j = 0; j < W; ++j)
            if (first + j >= labels) v[j] = -INFINITY;
    }
    if (LABEL) {
        const float m = largest_of(v);
        if (m > s.largest) {
            // The one that was the largest joins the others (exp2(-inf) = 0 where there was none).
            s.sum = (s.sum + 1.0f) * exp2_fast((s.base - m) * scale2);
            s.base = s.largest = m;
            uint32_t place = 0;
#pragma unroll
            for (int j = W - 1; j >= 0; --j)
                if (v[j] == m) place = j;
#pragma unroll
            for (int j = 0; j < W; ++j)
                if (place == (uint32_t)j) v[j] = -INFINITY;
            s.label = first + place;
        }
        s.sum += sum_exp2(v, scale2, finite_base(s.base));
        return;
    }
    if (near) {
        const uint32_t at = target - first;
#pragma unroll
        for (int j = 0; j < W; ++j)
            if (at == (uint32_t)j) {
                s.target_logit = v[j];
                v[j] = -INFINITY;
            }
    }
    if (s.base == -INFINITY) {
        const float m = largest_of(v);
        if (m != -INFINITY) s.base = m;  // NaN stays NaN
    }
    float base = finite_base(s.base), sum;
    for (;;) {
        sum = s.sum + sum_exp2(v, scale2, base);
        if (sum <= kLargestSum) break;
        const float higher = fmaxf(base, largest_of(v));
        if (!(higher > base)) break;  // the sum of many, an infinite logit, or NaN
        s.sum *= exp2_fast((base - higher) * scale2);
        base = s.base = higher;
    }
    s.sum = sum;
}

// The slopes of 32 logits of a row, in place (the target's only if PLACE); zeros past the labels and in rows that
// do not count. The target's, if it is among them, also in `target_slope`: p - 1 from the difference of its logit
// and the normalizer, since p itself may round to 1. The normalizer over the scale is `normalizer`, to f32's
// precision, less shift_low / scale2.
template <bool PLACE>
__device__ __forceinline__ void to_slopes(float (&v)[32], uint32_t first, uint32_t labels, float scale2,
                                          float normalizer, float weight, uint32_t target, bool live,
                                          float shift_low, float& target_slope) {
    const uint32_t at = target - first;
    const bool near = __any_sync(0xffffffffu, at < 32);
    float logit = 0.0f;
    if (near) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
            if (at == (uint32_t)j) logit = v[j];
    }
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
        const float2 x = fma2(add2(make_float2(v[j], v[j + 1]), make_float2(-normalizer, -normalizer)),
                              make_float2(scale2, scale2), make_float2(shift_low, shift_low));
        v[j] = exp2_fast(x.x);
        v[j + 1] = exp2_fast(x.y);
    }
    if (near) {
        const float slope = expm1f(fmaf(logit - normalizer, scale2, shift_low) * 0.693147181f);
        if (at < 32) target_slope = slope * weight;
        if (PLACE) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (at == (uint32_t)j) v[j] = slope;
        }
    }
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = live ? v[j] * weight : 0.0f;
    if (first + 32 > labels) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
            if (first + j >= labels) v[j] = 0.0f;
    }
}

// 32 values as bf16 into half a 128-byte row of the swizzled shared tile (16-byte unit u of row r
// lies at u ^ (r & 7)); what the rounding left stays in v for the next part.
__device__ __forceinline__ void stage_part(uint32_t tile, uint32_t row, int half, float (&v)[32]) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const __nv_bfloat162 pair = __floats2bfloat162_rn(v[q * 8 + 2 * j], v[q * 8 + 2 * j + 1]);
            w[j] = reinterpret_cast<const uint32_t&>(pair);
            v[q * 8 + 2 * j] -= __low2float(pair);
            v[q * 8 + 2 * j + 1] -= __high2float(pair);
        }
        const uint32_t unit = (uint32_t)(half * 4 + q) ^ (row & 7u);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(tile + row * 128 + unit * 16), "r"(w[0]),
                     "r"(w[1]), "r"(w[2]), "r"(w[3])
                     : "memory");
    }
}

// What the first part leaves of 32 values.
__device__ __forceinline__ void round_off(float (&v)[32]) {
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
        const __nv_bfloat162 pair = __floats2bfloat162_rn(v[j], v[j + 1]);
        v[j] -= __low2float(pair);
        v[j + 1] -= __high2float(pair);
    }
}

// Column `column` of that row.
__device__ __forceinline__ void stage_one(uint32_t tile, uint32_t row, uint32_t column, bf16 v) {
    const uint32_t at = tile + row * 128 + ((column / 8) ^ (row & 7u)) * 16 + column % 8 * 2;
    asm volatile("st.shared.b16 [%0], %1;" ::"r"(at), "h"(__bfloat16_as_ushort(v)) : "memory");
}

template <typename T>
__device__ __forceinline__ void store_out(T* to, const float (&v)[32], uint32_t columns, bool packed) {
    constexpr int N = 16 / sizeof(T);
    if (packed && columns >= 32) {
#pragma unroll
        for (int q = 0; q < 32 / N; ++q) {
            float part[N];
#pragma unroll
            for (int j = 0; j < N; ++j) part[j] = v[q * N + j];
            Pack<T, N> o;
            o.set(part);
            store_pack(to + q * N, o);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 32; ++j)
            if ((uint32_t)j < columns) to[j] = from_float<T>(v[j]);
    }
}

// v += factor * (a row's 32 columns, of which `columns` exist), rows being 16-byte aligned.
__device__ __forceinline__ void add_scaled(float (&v)[32], float factor, const bf16* row, uint32_t columns) {
    if (columns >= 32) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const Pack<bf16, 8> p = load_pack<bf16, 8>(row + q * 8);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[q * 8 + j] = fmaf(factor, p.get(j), v[q * 8 + j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 32; ++j)
            if ((uint32_t)j < columns) v[j] = fmaf(factor, to_float(row[j]), v[j]);
    }
}

// Adds to 32 f32 sums in memory where they lie: each has one adder in a launch, so the order of the
// additions is that of the launches.
__device__ __forceinline__ void add_out(float* to, const float (&v)[32], uint32_t columns) {
    if (columns >= 32) {
#pragma unroll
        for (int j = 0; j < 32; j += 4)
            asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(to + j), "f"(v[j]),
                         "f"(v[j + 1]), "f"(v[j + 2]), "f"(v[j + 3])
                         : "memory");
    } else {
#pragma unroll
        for (int j = 0; j < 32; ++j)
            if ((uint32_t)j < columns) to[j] += v[j];
    }
}

// map_slopes: the slopes as [part][64 labels][row][64], so that every box of a tile is one contiguous
// stretch (row by row over all labels the writes alone kept the slopes' pass at 250 us, 9472 x 32,768 x
// 512, against 190 us without them); boxes of 64 rows to read (kOut), 32 to write (kSlopes).
template <int ENDING, bool PAIR, typename T>
__global__ void __launch_bounds__(Shape<ENDING, PAIR, T>::threads, 1)
    k_label_gemm(const __grid_constant__ CUtensorMap map_features,
                 const __grid_constant__ CUtensorMap map_features_packed,
                 const __grid_constant__ CUtensorMap map_weight, const __grid_constant__ CUtensorMap map_slopes,
                 const __grid_constant__ GemmArgs a) {
    constexpr int kBlocks = PAIR ? 2 : 1;
    constexpr int kSide = kTile * kBlocks;  // the pair's tile
    using S = Shape<ENDING, PAIR, T>;
    constexpr int kStages = S::stages, kSpan = kSide / S::column_parts;  // columns per warp
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem = (tc::smem_address(smem_raw) + 1023u) & ~1023u;
    const uint32_t store_at = smem + kStages * kStageBytes;
    const uint32_t barriers = store_at + S::store_bytes;
    const uint32_t full = barriers, empty = full + 8 * kStages, done = empty + 8 * kStages, drained = done + 16;
    const uint32_t tmem_slot = drained + 16;
    uint8_t* generic_base = smem_raw + (smem - tc::smem_address(smem_raw));
    const uint32_t warp = threadIdx.x / 32, lane = lane_id();
    const uint32_t rank = PAIR ? tc::cluster_rank() : 0;
    // Workers take the items round by round. The output gradients', the long ones first, go in turns from
    // either end, so that the workers with one long item more have a short one less.
    auto item_of = [](uint32_t round) {
        const uint32_t worker = blockIdx.x / kBlocks, workers = gridDim.x / kBlocks;
        return round * workers + (ENDING == kOut && round % 2 ? workers - 1 - worker : worker);
    };

    if (warp == 0 && lane == 0) {
        for (int s = 0; s < kStages; ++s) {
            tc::barrier_init(full + 8 * s, 1);
            tc::barrier_init(empty + 8 * s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            tc::barrier_init(done + 8 * b, 1);
            tc::barrier_init(drained + 8 * b, S::epilogue_warps * kBlocks);
        }
        tc::barrier_init_fence();
        tc::prefetch_map(&map_features);
        tc::prefetch_map(&map_weight);
    }
    if (warp == 2) tc::tmem_alloc<PAIR>(tmem_slot, 2 * kSide);
    tc::fence_before_sync();
    __syncthreads();
    if constexpr (PAIR) tc::cluster_sync();  // the other block's barriers are set up too
    tc::fence_after_sync();
    const uint32_t tmem = *reinterpret_cast<uint32_t*>(generic_base + (tmem_slot - smem));
    chain_enter();

    const uint32_t count = a.all_rows ? a.all_rows : a.rows->count;
    const bool packed = !a.all_rows && a.rows->packed != 0;
    const Schedule<ENDING, kSide> schedule(a, count);
    bool ok = true;

    if (warp == 0) {
        if (tc::elect_one()) {
            const CUtensorMap* features = packed ? &map_features_packed : &map_features;
            uint32_t stage = 0, phase = 0;
            for (uint32_t round = 0; ok && item_of(round) < schedule.items; ++round) {
                const Work w = schedule.at(a, item_of(round));
                const int am = (int)(w.m * kSide + rank * kTile), first_row = (int)a.first_row;
                for (uint32_t n = w.n0; ok && n < w.n1; ++n) {
                    const int bn = (int)(n * kSide + rank * kTile);
                    for (uint32_t p = ENDING == kOut && w.which == 0 ? a.only_weight : 0; ok && p < a.products; ++p) {
                        const int za = (int)((a.parts_a >> (4 * p)) & 15u), zb = (int)((a.parts_b >> (4 * p)) & 15u);
                        for (uint32_t k = w.k0; k < w.k1; ++k) {
                            if (!(ok = tc::barrier_wait(empty + 8 * stage, phase ^ 1))) break;
                            // Both blocks' copies count on the first one's barrier.
                            const uint32_t to = smem + stage * kStageBytes;
                            const uint32_t bar = PAIR ? tc::map_to_rank(full + 8 * stage, 0) : full + 8 * stage;
                            if (rank == 0) tc::barrier_expect(full + 8 * stage, kStageBytes * kBlocks);
                            const int kk = (int)k * kBlockK;
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const uint32_t ta = to + h * kBoxBytes, tb = ta + kOperandBytes;
                                const int m = am + h * 64, bm = bn + h * 64;
                                if (ENDING != kOut) {  // H W^T
                                    tc::load_box<PAIR>(ta, features, bar, kk, first_row + m, za);
                                    tc::load_box<PAIR>(tb, &map_weight, bar, kk, bm, zb);
                                } else if (w.which == 0) {  // G W
                                    tc::load_box<PAIR>(ta, &map_slopes, bar, 0, m, za * (int)a.panels + (int)k);
                                    tc::load_box<PAIR>(tb, &map_weight, bar, bm, kk, zb);
                                } else {  // G^T H
                                    tc::load_box<PAIR>(ta, &map_slopes, bar, 0, kk, za * (int)a.panels + m / 64);
                                    tc::load_box<PAIR>(tb, features, bar, bm, first_row + kk, zb);
                                }
                            }
                            if (++stage == kStages) stage = 0, phase ^= 1;
                        }
                    }
                }
            }
            // The products' last arrivals reach this block before it may leave.
            for (int i = 0; ok && i < kStages; ++i) {
                ok = tc::barrier_wait(empty + 8 * stage, phase ^ 1);
                if (++stage == kStages) stage = 0, phase ^= 1;
            }
        }
    } else if (warp == 1) {
        if (rank == 0 && tc::elect_one()) {
            uint32_t stage = 0, phase = 0, buffer = 0, buffer_phase = 0;
            for (uint32_t round = 0; ok && item_of(round) < schedule.items; ++round) {
                const Work w = schedule.at(a, item_of(round));
                const uint32_t steps = (w.k1 - w.k0) * (a.products - (ENDING == kOut && w.which == 0 ? a.only_weight : 0));
                if (steps == 0) continue;
                // Which operands run along K in memory: W in dH; G and H in dW. 16 of K are 32 bytes along
                // a row, or 16 rows of 128 bytes.
                const bool a_transposed = w.which != 0;
                constexpr bool b_transposed = ENDING == kOut;
                const uint32_t desc = tc::instruction(kSide, kSide, a_transposed, b_transposed);
                const uint32_t a_step = a_transposed ? 2048 : 32, b_step = b_transposed ? 2048 : 32;
                for (uint32_t n = w.n0; ok && n < w.n1; ++n) {
                    if (!(ok = tc::barrier_wait(drained + 8 * buffer, buffer_phase ^ 1))) break;
                    tc::fence_after_sync();
                    for (uint32_t k = 0; k < steps; ++k) {
                        if (!(ok = tc::barrier_wait(full + 8 * stage, phase))) break;
                        tc::fence_after_sync();
                        const uint32_t at = smem + stage * kStageBytes;
#pragma unroll
                        for (int q = 0; q < kBlockK / 16; ++q) {
                            const uint64_t da = tc::operand(at + q * a_step, kBoxBytes);
                            const uint64_t db = tc::operand(at + kOperandBytes + q * b_step, kBoxBytes);
                            tc::multiply<PAIR>(tmem + buffer * kSide, da, db, desc, k != 0 || q != 0);
                        }
                        tc::commit<PAIR>(empty + 8 * stage);
                        if (++stage == kStages) stage = 0, phase ^= 1;
                    }
                    if (!ok) break;
                    tc::commit<PAIR>(done + 8 * buffer);
                    if (++buffer == 2) buffer = 0, buffer_phase ^= 1;
                }
            }
        }
    } else if (warp >= 4) {
        // An equal part of the tile's columns per four warps; thread = row.
        const uint32_t part = (warp - 4) / 4, quarter = warp % 4;
        const uint32_t lane_row = rank * kTile + quarter * 32 + lane;
        const uint32_t tmem_at = tmem + ((quarter * 32) << 16) + part * kSpan;
        const uint32_t stage_tile = store_at + (warp - 4) * kStoreBytes;
        uint32_t buffer = 0, buffer_phase = 0;
        // Output gradients of a call that gave up, here or in a kernel before, are NaN.
        const bool poisoned = ENDING == kOut && a.rows->status != 0;
        for (uint32_t round = 0; (ok || ENDING == kOut) && item_of(round) < schedule.items; ++round) {
            const Work w = schedule.at(a, item_of(round));
            const bool empty_sum = w.k0 == w.k1;
            const OutArgs& o = a.out[w.which];
            if (ENDING == kOut && empty_sum && o.add) continue;
            const uint32_t row = w.m * kSide + lane_row;  // in this call's rows (or labels)
            const uint32_t compact = a.first_row + row;
            const bool live = compact < count;
            RowStats stats{-INFINITY, 0.0f, 0.0f, -INFINITY, 0u};
            uint32_t target = kNoTarget;
            float normalizer = 0.0f, shift_low = 0.0f, weight = 0.0f;
            float residual = 0.0f;
            if (ENDING == kOut && sizeof(T) == 2 && live && w.which == 0) {
                target = (uint32_t)index_at(a.targets, a.wide, a.row_of[compact], a.labels);
                residual = a.residuals[row];
            }
            if (ENDING != kOut && live) {
                const uint32_t original = a.all_rows ? compact : a.row_of[compact];
                if (a.targets) target = (uint32_t)index_at(a.targets, a.wide, original, a.labels);
                if (makes_slopes(ENDING)) {
                    const double exact = a.log_normalizers[original] * a.per_scale;
                    normalizer = (float)exact;
                    shift_low = (float)(((double)normalizer - exact) * a.scale2);
                    weight = a.row_gradient ? a.scale * a.row_gradient[original] : 1.0f;
                }
            }
            // The mean's factor comes after the sums: the target's slope p - 1, by far the largest, is then near
            // -1 and loses little where it is rounded to bf16 (the factor in it, all rows' lost the same up to
            // 2^-9, which adds up in dW). bf16 gradients lose more than the truncation in their last rounding.
            float factor = 1.0f;
            if (ENDING == kOut) {
                if (!a.row_gradient) factor = a.scale / (float)max(count, 1u);
                if (sizeof(T) == 4) factor *= (float)given_back((w.k1 - w.k0) * (kBlockK / 16));
            }
            for (uint32_t n = w.n0; (ok || ENDING == kOut) && n < w.n1; ++n) {
                if (!empty_sum && ok) {
                    ok = __all_sync(0xffffffffu, tc::barrier_wait(done + 8 * buffer, buffer_phase));
                    if (ENDING != kOut && !ok) break;
                    tc::fence_after_sync();
                }
                // After the last load the accumulator may fill again.
                auto drain = [&]() {
                    tc::fence_before_sync();
                    __syncwarp();
                    if (lane == 0)
                        tc::barrier_arrive_cluster(PAIR ? tc::map_to_rank(drained + 8 * buffer, 0) : drained + 8 * buffer);
                };
                const uint32_t accumulator = tmem_at + buffer * kSide, columns_at = n * kSide + part * kSpan;
                if constexpr (makes_slopes(ENDING)) {
                    // 64 columns at a time: each part fills the warp's 32 x 64 tile, which a bulk copy
                    // writes out while the next is computed.
#pragma unroll
                    for (int c = 0; c < kSpan; c += 64) {
                        auto reclaim = [&]() {
                            if (lane == 0) tc::store_wait_read();
                            __syncwarp();
                        };
                        auto store = [&](int p) {
                            tc::fence_async_shared();
                            __syncwarp();
                            if (lane == 0) tc::store_box(&map_slopes, stage_tile, 0, (int)row, (int)(p * a.panels + (columns_at + c) / 64));
                        };
                        if constexpr (sizeof(T) == 2) {
                            // A second part takes the slopes from the accumulator again: 64 of them and what
                            // the first one left do not fit a thread's registers. A kernel of its own: as a
                            // loop over an argument it made the pass with one part an eighth slower (9803 x
                            // 12,379 x 28: 76 us, 67 without).
                            constexpr int kSlopeParts = ENDING == kFineSlopes ? 2 : 1;
#pragma unroll 1
                            for (int p = 0; p < kSlopeParts; ++p) {
#pragma unroll
                                for (int q = 0; q < 2; ++q) {
                                    float v[32];
                                    __syncwarp();
                                    tc::tmem_load32(accumulator + c + 32 * q, v);
                                    tc::tmem_load_wait();
                                    if (q == 1 && c + 64 == kSpan && p + 1 == kSlopeParts) drain();
                                    const uint32_t column = columns_at + c + 32 * q;
                                    float slope = 0.0f;
                                    to_slopes<false>(v, column, a.labels, a.scale2, normalizer, weight, target, live, shift_low, slope);
                                    if (p != 0) round_off(v);
                                    if (q == 0) reclaim();
                                    stage_part(stage_tile, lane, q, v);
                                    if (target - column < 32) {
                                        const bf16 rounded = __float2bfloat16_rn(slope);
                                        const float left = slope - __bfloat162float(rounded);
                                        stage_one(stage_tile, lane, 32 * q + target - column, p == 0 ? rounded : __float2bfloat16_rn(left));
                                        a.residuals[row] = left;
                                    }
                                }
                                store(p);
                            }
                        } else {
                            float v[2][32], unused;
                            __syncwarp();
                            tc::tmem_load32(accumulator + c, v[0]);
                            tc::tmem_load32(accumulator + c + 32, v[1]);
                            tc::tmem_load_wait();
                            if (c + 64 == kSpan) drain();
#pragma unroll
                            for (int q = 0; q < 2; ++q)
                                to_slopes<true>(v[q], columns_at + c + 32 * q, a.labels, a.scale2, normalizer, weight, target,
                                                live, shift_low, unused);
                            for (int p = 0; p < (int)kParts; ++p) {
                                reclaim();
                                stage_part(stage_tile, lane, 0, v[0]);
                                stage_part(stage_tile, lane, 1, v[1]);
                                store(p);
                            }
                        }
                    }
                } else if constexpr (ENDING == kStats) {
                    // One chunk's code for the whole tile: unrolled it overflows the instruction cache.
#pragma unroll 1
                    for (int c = 0; c < kSpan; c += 32) {
                        float v[32];
                        __syncwarp();
                        tc::tmem_load32(accumulator + c, v);
                        tc::tmem_load_wait();
                        if (c + 32 == kSpan) drain();
                        const uint32_t column = columns_at + c;
                        const bool near = __any_sync(0xffffffffu, target - column < 32);
                        if (a.partial_labels) add_logits<true>(stats, v, column, a.labels, a.scale2, target, near);
                        else add_logits<false>(stats, v, column, a.labels, a.scale2, target, near);
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < kSpan; c += 32) {
                        float v[32];
                        if (empty_sum || !ok) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] = 0.0f;
                        } else {
                            __syncwarp();
                            tc::tmem_load32(accumulator + c, v);
                            tc::tmem_load_wait();
                            if (c + 32 == kSpan) drain();
                        }
                        if (poisoned || !ok) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] = __int_as_float(0x7fffffff);
                        }
                        const uint32_t column = columns_at + c;
                        if ((w.which ? row < o.rows : live) && column < a.dim) {
                            const uint32_t columns = a.dim - column;
                            if (sizeof(T) == 2 && w.which == 0 && w.k0 == 0)
                                add_scaled(v, residual, a.weight + (int64_t)target * a.weight_stride + column, columns);
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] *= factor;
                            if (o.partial) {
                                float* to = static_cast<float*>(o.out) + ((uint64_t)w.split * o.rows + row) * (uint64_t)o.stride +
                                            column;
                                if (o.add) add_out(to, v, columns);
                                else store_out<float>(to, v, columns, true);
                            } else {
                                const uint64_t r = w.which ? row : a.row_of[compact];
                                store_out<T>(static_cast<T*>(o.out) + (int64_t)r * o.stride + column, v, columns, o.packed);
                            }
                        }
                    }
                }
                if (!empty_sum && ++buffer == 2) buffer = 0, buffer_phase ^= 1;
            }
            if (ENDING == kStats && ok && live) {
                const uint64_t slot = (uint64_t)(w.split * S::column_parts + part) * a.partial_rows + row;
                a.partials[slot] = make_float2(stats.base, stats.sum);
                if (a.partial_labels) a.partial_labels[slot] = stats.label;
                // The target is in exactly one thread's columns.
                if (target != kNoTarget && target / kSide >= w.n0 && target / kSide < w.n1 &&
                    target % kSide / kSpan == part)
                    a.target_logits[row] = stats.target_logit;
            }
        }
        if (makes_slopes(ENDING) && lane == 0) tc::store_wait();
    }
    __syncwarp();
    if (!ok) {
        atomicCAS(&a.rows->status, 0u, (uint32_t)SP_ERR_TIMEOUT);
        // Copies and products issued before the wait that ran out finish meanwhile.
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    }
    tc::fence_before_sync();
    __syncthreads();
    if constexpr (PAIR) tc::cluster_sync();  // no block leaves while the other may reach into it
    if (warp == 2) {
        tc::fence_after_sync();
        tc::tmem_free<PAIR>(tmem, 2 * kSide);
    }
}

}  // namespace label
}  // namespace splat
