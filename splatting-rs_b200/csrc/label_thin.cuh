// The logits' pass for at most kThinRows rows, where the weight's bytes are what it costs: the roles
// of label_gemm.cuh swapped (128 labels on the accumulator's lanes, the rows its columns), so that
// the products are no wider than the rows, and the weight read once and in place: bf16 by tiled bulk
// copies where it is aligned for them, else (f32, odd strides) by 24 warps that split it into
// its bf16 parts on the way into shared memory.
//
// One bf16 row against 65,536 labels of 512 takes 20 us, 67 MB at 3.3 TB/s: four tiles a block at most, so the
// first copies' latency and the last tile's sums are a good part. 60 f32 rows against 20,011 labels of 768 take 34
// us for 62 MB: bound by the instructions of the conversion and its hand-over from stage to stage (without the
// loads it takes 25).
//
// f32 parts of the rows lie one below the other, so that one product of a weight part covers all the
// rows' parts it meets: accumulator groups hi hi | hi mid + mid hi | hi lo + mid mid + lo hi. Grouped
// by size, and hi hi by even and odd steps of K, they also lose less to the tensor cores' truncating
// additions before they are added in f32.
#pragma once

#include "label_gemm.cuh"

namespace splat {
namespace label {

constexpr int kThinRows = 64;
constexpr int kConvertWarps = 24;
constexpr uint32_t kConvertTile = kConvertWarps * 4;  // labels of a converted tile, at most: eight threads a row
constexpr int kConvertAhead = 5;                      // steps whose loads a thread has under way
constexpr int thin_threads(bool direct) { return direct ? 256 : 256 + kConvertWarps * 32; }
constexpr int kThinStagesF32 = 2, kThinStagesBf16 = 6;
constexpr uint32_t kRowsBytes = kThinRows * kBlockK * 2;
constexpr int kLogitStride = kTile + 1;  // of a row's logits in shared memory: no bank twice
constexpr uint32_t kThinColumns = 512;

constexpr uint32_t thin_stage_bytes(bool f32) { return (f32 ? kParts : 1) * (kOperandBytes + kRowsBytes); }
constexpr size_t thin_smem(bool f32) {
    return 1024 + (size_t)(f32 ? kThinStagesF32 : kThinStagesBf16) * thin_stage_bytes(f32) +
           kThinRows * kLogitStride * sizeof(float) + 256;
}

struct ThinArgs {
    GemmArgs g;
    const void* weight;
    int64_t weight_stride;
    uint32_t dim;
    int vector;          // 16-byte loads are aligned
    uint32_t tile;       // labels per tile: kTile, or for converted weights a multiple of 8 up to kConvertTile
    uint32_t known_rows; // not 0: the rows' count, known before the launch that gathers them is done
    uint32_t columns;    // of the accumulators: the rows, rounded up to 16
    uint32_t tiles;
};

__device__ __forceinline__ void tmem_load16(uint32_t address, float (&v)[16]) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(address));
}

// One thread's eight columns of a weight row on their way to shared memory.
template <typename T>
struct RawEight {
    static constexpr int N = 16 / sizeof(T);
    Pack<T, N> p[8 / N];
    __device__ __forceinline__ void load(const T* from, uint32_t columns, bool vector) {
        if (vector && columns >= 8) {
#pragma unroll
            for (int q = 0; q < 8 / N; ++q) p[q] = load_pack<T, N>(from + q * N);
        } else {
#pragma unroll
            for (int q = 0; q < 8 / N; ++q) {
                float v[N];
#pragma unroll
                for (int j = 0; j < N; ++j) v[j] = (uint32_t)(q * N + j) < columns ? to_float(from[q * N + j]) : 0.0f;
                p[q].set(v);
            }
        }
    }
};

// DIRECT: the weight arrives by bulk copies; else through the converting warps.
template <typename T, bool DIRECT>
__global__ void __launch_bounds__(thin_threads(DIRECT), 1)
    k_label_thin(const __grid_constant__ CUtensorMap map_rows, const __grid_constant__ CUtensorMap map_rows_packed,
                 const __grid_constant__ CUtensorMap map_weight, const __grid_constant__ ThinArgs a) {
    constexpr bool kF32 = sizeof(T) == 4;
    constexpr int kParted = kF32 ? (int)kParts : 1;
    constexpr int kRing = kF32 ? kThinStagesF32 : kThinStagesBf16;
    constexpr uint32_t kBytes = thin_stage_bytes(kF32);
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem = (tc::smem_address(smem_raw) + 1023u) & ~1023u;
    uint8_t* generic_base = smem_raw + (smem - tc::smem_address(smem_raw));
    float* logits = reinterpret_cast<float*>(generic_base + kRing * kBytes);
    const uint32_t barriers = smem + kRing * kBytes + (kThinRows * kLogitStride * sizeof(float) + 15) / 16 * 16;
    const uint32_t full = barriers, empty = full + 8 * kRing, done = empty + 8 * kRing, drained = done + 16;
    const uint32_t tmem_slot = drained + 16;
    const uint32_t warp = threadIdx.x / 32, lane = lane_id();

    if (warp == 0 && lane == 0) {
        for (int s = 0; s < kRing; ++s) {
            tc::barrier_init(full + 8 * s, 1 + (DIRECT ? 0 : kConvertWarps));
            tc::barrier_init(empty + 8 * s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            tc::barrier_init(done + 8 * b, 1);
            tc::barrier_init(drained + 8 * b, 4);
        }
        tc::barrier_init_fence();
    }
    if (warp == 2) tc::tmem_alloc<false>(tmem_slot, kThinColumns);
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = *reinterpret_cast<uint32_t*>(generic_base + (tmem_slot - smem));
    // The gathering launch before this one has itself waited for all that came earlier, the weight among
    // it: the converting warps need not wait for the rows.
    if (DIRECT || warp < 8 || a.known_rows == 0) chain_enter();

    const uint32_t count = a.known_rows ? a.known_rows : a.g.all_rows ? a.g.all_rows : a.g.rows->count;
    const uint32_t tiles = count ? a.tiles : 0;
    // A buffer's accumulator groups: f32's three, then hi hi (all, for bf16) of the odd steps.
    const uint32_t buffer_columns = 4 * kThinRows;
    bool ok = true;

    if (warp == 0) {
        if (tc::elect_one()) {
            const CUtensorMap* rows = !a.g.all_rows && a.g.rows->packed ? &map_rows_packed : &map_rows;
            uint32_t stage = 0, phase = 0;
            for (uint32_t tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x)
                for (uint32_t k = 0; k < a.g.k_blocks; ++k) {
                    if (!(ok = tc::barrier_wait(empty + 8 * stage, phase ^ 1))) break;
                    const uint32_t bar = full + 8 * stage, to = smem + stage * kBytes;
                    tc::barrier_expect(bar, kParted * kRowsBytes + (DIRECT ? kOperandBytes : 0));
                    if (DIRECT)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            tc::load_box<false>(to + h * kBoxBytes, &map_weight, bar, (int)k * kBlockK,
                                                (int)(tile * a.tile) + h * 64, 0);
#pragma unroll
                    for (int p = 0; p < kParted; ++p)
                        tc::load_box<false>(to + kParted * kOperandBytes + p * kRowsBytes, rows, bar, (int)k * kBlockK, 0, p);
                    if (++stage == kRing) stage = 0, phase ^= 1;
                }
            for (int i = 0; ok && i < kRing; ++i) {
                ok = tc::barrier_wait(empty + 8 * stage, phase ^ 1);
                if (++stage == kRing) stage = 0, phase ^= 1;
            }
        }
    } else if (warp == 1) {
        if (tc::elect_one()) {
            uint32_t stage = 0, phase = 0, buffer = 0, buffer_phase = 0;
            for (uint32_t tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x) {
                if (!(ok = tc::barrier_wait(drained + 8 * buffer, buffer_phase ^ 1))) break;
                tc::fence_after_sync();
                const uint32_t into = tmem + buffer * buffer_columns;
                for (uint32_t k = 0; k < a.g.k_blocks; ++k) {
                    if (!(ok = tc::barrier_wait(full + 8 * stage, phase))) break;
                    tc::fence_after_sync();
                    const uint32_t w_at = smem + stage * kBytes, r_at = w_at + kParted * kOperandBytes;
#pragma unroll
                    for (int q = 0; q < kBlockK / 16; ++q) {
                        auto product = [&](int weight_part, int rows_part, uint32_t group, uint32_t n, bool add) {
                            tc::multiply<false>(into + group * kThinRows,
                                                tc::operand(w_at + weight_part * kOperandBytes + q * 32, kBoxBytes),
                                                tc::operand(r_at + rows_part * kRowsBytes + q * 32, kBoxBytes),
                                                tc::instruction(kTile, n, false, false), add);
                        };
                        const bool again = k > 1 || q != 0;
                        if (!kF32) {
                            product(0, 0, k & 1 ? 3 : 0, a.columns, again);
                        } else {
                            if (k & 1) {
                                product(0, 0, 3, kThinRows, again);
                                product(0, 1, 1, 2 * kThinRows, true);
                            } else {
                                product(0, 0, 0, 3 * kThinRows, again);
                            }
                            product(1, 0, 1, 2 * kThinRows, true);
                            product(2, 0, 2, kThinRows, true);
                        }
                    }
                    tc::commit<false>(empty + 8 * stage);
                    if (++stage == kRing) stage = 0, phase ^= 1;
                }
                if (!ok) break;
                tc::commit<false>(done + 8 * buffer);
                if (++buffer == 2) buffer = 0, buffer_phase ^= 1;
            }
        }
    } else if (warp >= 4 && warp < 8) {
        // The tile's logits turn over in shared memory: a thread reads a label's, then 128 / columns
        // threads (to a power of two) take a row's, 16 at a time.
        const uint32_t t = threadIdx.x - 128;
        const uint32_t split = a.columns <= 16 ? 3 : a.columns <= 32 ? 2 : 1;
        const uint32_t row = t >> split, part = t & ((1u << split) - 1), span = kTile >> split;
        const bool live = row < count;
        RowStats stats{-INFINITY, 0.0f, 0.0f, -INFINITY, 0u};
        uint32_t target = kNoTarget;
        if (live && a.g.targets)
            target = (uint32_t)index_at(a.g.targets, a.g.wide, a.g.all_rows ? row : a.g.row_of[row], a.g.labels);
        uint32_t buffer = 0, buffer_phase = 0;
        for (uint32_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
            // All four warps agree whether to go on: they meet at barriers below.
            const bool here = tc::barrier_wait(done + 8 * buffer, buffer_phase);
            uint32_t all;
            asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.and.pred q, 1, 128, p;\n\t"
                         "selp.u32 %0, 1, 0, q;\n\t}" : "=r"(all) : "r"((uint32_t)here) : "memory");
            if (!(ok = all != 0)) break;
            tc::fence_after_sync();
            const uint32_t from = tmem + buffer * buffer_columns + (((warp - 4) * 32) << 16);
            for (uint32_t c = 0; c < a.columns; c += 16) {
                float v[16], w[16];
                auto add_group = [&](uint32_t group) {
                    tmem_load16(from + group * kThinRows + c, w);
                    tc::tmem_load_wait();
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] += w[j];
                };
                tmem_load16(from + c, v);
                tc::tmem_load_wait();
                if (a.g.k_blocks > 1) add_group(3);
                if (kF32) {
                    add_group(1);
                    add_group(2);
                }
#pragma unroll
                for (int j = 0; j < 16; ++j) logits[(c + j) * kLogitStride + t] = v[j];
            }
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) tc::barrier_arrive_cluster(drained + 8 * buffer);
            asm volatile("barrier.cta.sync 1, 128;" ::: "memory");
            if (row < a.columns) {
#pragma unroll 1
                for (uint32_t c = 0; c < span; c += 16) {
                    const uint32_t at = part * span + c, first = tile * a.tile + at;
                    if (at >= a.tile) break;
                    float v[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] = logits[row * kLogitStride + at + j];
                    const bool near = target - first < min(16u, a.tile - at);
                    const uint32_t end = min(a.g.labels, (tile + 1) * a.tile);
                    if (a.g.partial_labels) add_logits<true>(stats, v, first, end, a.g.scale2, target, near);
                    else add_logits<false>(stats, v, first, end, a.g.scale2, target, near);
                    if (near) a.g.target_logits[row] = stats.target_logit;
                }
            }
            asm volatile("barrier.cta.sync 1, 128;" ::: "memory");
            if (++buffer == 2) buffer = 0, buffer_phase ^= 1;
        }
        // The row's parts, in neighbouring lanes, as one; of prediction's two largest logits the one that
        // is not joins the sum.
        __syncwarp();
        for (uint32_t o = 1; o < (1u << split); o <<= 1) {
            const float base = __shfl_xor_sync(0xffffffffu, stats.base, o), sum = __shfl_xor_sync(0xffffffffu, stats.sum, o);
            const float largest = __shfl_xor_sync(0xffffffffu, stats.largest, o);
            const uint32_t label = __shfl_xor_sync(0xffffffffu, stats.label, o);
            const bool other = largest > stats.largest || (largest == stats.largest && label < stats.label);
            const float one = a.g.partial_labels ? 1.0f : 0.0f;
            const float top = fmaxf(stats.base, base), finite = finite_base(top);
            const float mine = (stats.sum + (other ? one : 0.0f)) * exp2_fast((stats.base - finite) * a.g.scale2);
            const float theirs = (sum + (other ? 0.0f : one)) * exp2_fast((base - finite) * a.g.scale2);
            stats.sum = part & o ? theirs + mine : mine + theirs;
            stats.base = top;
            if (other) stats.largest = largest, stats.label = label;
        }
        if (ok && live && part == 0) {
            const uint64_t slot = (uint64_t)blockIdx.x * a.g.partial_rows + row;
            a.g.partials[slot] = make_float2(stats.base, stats.sum);
            if (a.g.partial_labels) a.g.partial_labels[slot] = stats.label;
        }
    } else if (warp >= 8 && !DIRECT) {
        // Eight lanes a row of 64 columns, a tile a turn; the next steps' loads are under way: 60 rows, 20,011
        // labels, 768 columns take 38 us with gather and join, 39 with three steps', 45 with seven (more code
        // than the instruction caches like); 41 with sixteen warps, two turns and two steps'.
        const uint32_t t = threadIdx.x - 256, unit = t % 8, in_tile = t / 8;
        const T* weight = static_cast<const T*>(a.weight);
        RawEight<T> raw[kConvertAhead];
        const uint32_t mine = blockIdx.x < tiles ? (tiles - 1 - blockIdx.x) / gridDim.x + 1 : 0;  // tiles
        const uint32_t steps = mine * a.g.k_blocks;
        uint32_t load_tile = blockIdx.x, load_k = 0;
        auto load_next = [&](RawEight<T>& to) {
            const uint32_t column = load_k * kBlockK + unit * 8, label = load_tile * a.tile + in_tile;
            const uint32_t columns = column < a.dim ? a.dim - column : 0;
            const bool there = in_tile < a.tile && label < a.g.labels && load_tile < tiles;
            to.load(weight + (there ? (int64_t)label * a.weight_stride + column : 0), there ? columns : 0, a.vector);
            if (++load_k == a.g.k_blocks) load_k = 0, load_tile += gridDim.x;
        };
        auto convert = [&](const RawEight<T>& from, uint32_t to) {
            if (in_tile >= a.tile) return;  // those accumulator lanes are not read
            float v[8];
            constexpr int N = RawEight<T>::N;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = from.p[j / N].get(j % N);
            const uint32_t at = to + in_tile * 128 + ((unit ^ (in_tile & 7u)) * 16);
#pragma unroll
            for (int p = 0; p < kParted; ++p) {
                const Pack<bf16, 8> o = take_part(v, p == kParted - 1);
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + p * kOperandBytes), "r"(o.word.x),
                             "r"(o.word.y), "r"(o.word.z), "r"(o.word.w)
                             : "memory");
            }
        };
#pragma unroll
        for (int b = 0; b < kConvertAhead; ++b)
            if ((uint32_t)b < steps) load_next(raw[b]);
        uint32_t stage = 0, phase = 0;
        for (uint32_t s = 0; s < steps; s += kConvertAhead) {
#pragma unroll
            for (int b = 0; b < kConvertAhead; ++b) {
                if (s + b >= steps || !ok) break;
                if (!(ok = tc::barrier_wait(empty + 8 * stage, phase ^ 1))) break;
                convert(raw[b], smem + stage * kBytes);
                tc::fence_async_shared();
                __syncwarp();
                if (lane == 0) tc::barrier_arrive_cluster(full + 8 * stage);
                if (s + b + kConvertAhead < steps) load_next(raw[b]);
                if (++stage == kRing) stage = 0, phase ^= 1;
            }
            if (!ok) break;
        }
    }
    __syncwarp();
    if (!ok) {
        atomicCAS(&a.g.rows->status, 0u, (uint32_t)SP_ERR_TIMEOUT);
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    }
    tc::fence_before_sync();
    __syncthreads();
    if (warp == 2) {
        tc::fence_after_sync();
        tc::tmem_free<false>(tmem, kThinColumns);
    }
}

}  // namespace label
}  // namespace splat
