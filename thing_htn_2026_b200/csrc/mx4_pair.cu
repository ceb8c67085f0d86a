// out[M, N] = x[M, K] @ W[N, K]^T (+ bias) for many rows, W in microscaled 4-bit floating point (mx4.cuh), on pairs of
// multiprocessors (tcgen05 with cta_group::2, the scales applied by the tensor core).
//
//  * A pair's tile is 256 rows of W (the accumulator's lanes, 128 a block) by up to kCols rows of x (its columns, of which each block
//    brings half), so that a multiprocessor brings half of what a block alone would for the same products.
//  * Rows in 4 bits (kQuantized): both operands as they lie, 256 columns of the sum in 128 bytes a row, kind::mxf4, four times
//    the rate of bfloat16.
//  * Rows in bfloat16 or float32 (kRows2, kRows2Apart, kRows6): two or six terms of 8-bit floats (mx4_tcgen05.cuh) that mx4_terms_kernel has
//    prepared, 128 columns of the sum at a time, kind::mxf8f6f4; W's codes are spread over 8-bit containers by TMA as they are
//    copied.  Two terms at twice the rate of bfloat16 cost what a bfloat16 product costs; W is a quarter of the bytes.
//  * Scales: 512 bytes for 128 rows and 128 columns, by TMA like the operands, to tensor memory by tcgen05.cp just ahead of the
//    products that use them.  A tile's rows of x begin at a multiple of 64 rows of its operand, two columns of scales.
//
// A row's result depends on its own entries and its place in a tile alone.  Every wait on an mbarrier is bounded: after
// kWaitLimitNs, and more for the stages of a sum, the waiter sets THN_ERR_WAIT_TIMEOUT in the caller's error word, what is left to store becomes NaN, and tensor
// memory is given back.  A pair's two blocks are one cluster and always resident together; no wait depends on another pair.
#include "mx4_tcgen05.cuh"

namespace {

// Rows in 4 bits; bfloat16 rows for a result in bfloat16 (kRows2) and in float32 (kRows2Apart); float32 rows.
enum Mode { kQuantized, kRows2, kRows2Apart, kRows6 };

constexpr int kFeatures = 256;                             // of a pair
constexpr int kEpilogueWarps = 8, kThreads = 64 + 32 * kEpilogueWarps;      // warp 0: TMA, warp 1: products and tensor memory

template <int MODE>
struct Shape {
    static constexpr int kT = MODE == kQuantized ? 1 : MODE == kRows6 ? 6 : 2;
    static constexpr int kCols = 192;                                        // of an accumulator
    // Accumulators of a tile, and tiles that are held at once.  The tensor core cuts a sum's last bits off at every step of 32 columns, and six terms in one
    // accumulator would be six times as many cuts: 300 float32 rows, K = 4,096: 6.8e-6 off in relation to the result, 1.1e-6 for products
    // added one after the other in float32.  So float32's first terms have an accumulator of their own, and a bfloat16's where the result keeps what it
    // saves: 300 bfloat16 rows, K = 12,288, 4.1e-6 off in one accumulator, 0.8e-6 in two, 2.7e-6 for float32 additions; 2,048 by 24,576 x 4,096 269
    // and 331 us.  A bfloat16 result is rounded by 2^-9 and takes one.
    static constexpr int kSums = MODE == kRows6 || MODE == kRows2Apart ? 2 : 1, kBuffers = 2 / kSums;
    static constexpr int kSteps = MODE == kQuantized ? 2 : 1;                // pieces of 128 columns of the sum that a stage holds
    static constexpr int kAtoms = (kCols + 64 + 127) / 128;                  // of scales that a tile's rows of x can touch
    static constexpr uint32_t kASmem = 128 * 128, kBSmem = kCols / 2 * 128;  // of one block, a term
    static constexpr uint32_t kScaleBytes = kSteps * (1 + kT * kAtoms) * kMx4AtomBytes;      // W's, then x's: [term][128 rows][piece]
    static constexpr uint32_t kStageStride = kASmem + kT * kBSmem + (kScaleBytes + 1023) / 1024 * 1024;
    static constexpr int kFit = (int)((226 * 1024 - 2048) / kStageStride);
    static constexpr int kStages = kFit < 8 ? kFit : 8;
    static constexpr size_t kSmemBytes = kStages * kStageStride + 1024 /* alignment */ + 512 /* barriers */;
    static constexpr uint32_t kScaleCol = kCols * kSums * kBuffers;          // W's scales, then x's
    static constexpr uint32_t kScaleCols = kSteps * 4 * (1 + kT * kAtoms);   // of a stage; two stages' in turn
    static_assert(kScaleCol + 2 * kScaleCols <= 512, "tensor memory");
    static_assert(kStages >= 2, "shared memory");
};

struct Args {
    void* out;
    const void* bias;
    int bias_dtype, M, N, atoms;                // atoms: pieces of 128 columns of the sum
    int cuts, size, n_tiles;        // the rows of x in equal tiles
    int band;                       // how many of them are multiplied by all of W before the next
    int pitch;                      // rows of x's operand from one tile to the next
    int* err;
    int skip_loads;                 // the test of the bounded waits: nothing is loaded
};

__device__ __forceinline__ uint32_t block_in_pair() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// the address, as a cluster sees it, of the leading block's copy of something in shared memory
__device__ __forceinline__ uint32_t leader_addr(const void* p) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_addr(p)));
    return a;
}
// All threads of both blocks.  (Not the .aligned form, which counts warps: a warp whose lanes come one after the other would count twice.)
__device__ __forceinline__ void pair_barrier() {
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
// A box to this block's shared memory, its bytes counted by the leading block's barrier.
__device__ __forceinline__ void load_box(void* dst, const CUtensorMap* map, uint32_t leader_bar, int x, int y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(smem_addr(dst)), "l"(map), "r"(leader_bar), "r"(x), "r"(y)
        : "memory");
}
__device__ __forceinline__ void load_box(void* dst, const CUtensorMap* map, uint32_t leader_bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(smem_addr(dst)), "l"(map), "r"(leader_bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}
__device__ __forceinline__ void load_box(void* dst, const CUtensorMap* map, uint32_t leader_bar, int x, int y, int z, int w) {
    asm volatile(
        "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(smem_addr(dst)), "l"(map), "r"(leader_bar), "r"(x), "r"(y), "r"(z), "r"(w)
        : "memory");
}
// 512 bytes of scales in each block's shared memory to four columns of its tensor memory.
__device__ __forceinline__ void pair_scales(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
template <int MODE>
__device__ __forceinline__ void pair_mma(uint32_t tmem_d, uint64_t a_desc, uint64_t b_desc, uint32_t instr, uint32_t a_scales, uint32_t b_scales,
                                         uint32_t accumulate) {
    if constexpr (MODE == kQuantized)
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "setp.ne.b32 p, %6, 0;\n"
            "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n"
            "}\n"
            ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(instr), "r"(a_scales), "r"(b_scales), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "setp.ne.b32 p, %6, 0;\n"
            "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%4], [%5], p;\n"
            "}\n"
            ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(instr), "r"(a_scales), "r"(b_scales), "r"(accumulate)
            : "memory");
}
// The barrier at this place in both blocks hears of the products issued so far.
__device__ __forceinline__ void pair_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(smem_addr(bar)), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void tmem_load_32(uint32_t taddr, float (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
          "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]),
          "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]),
          "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
        : "r"(taddr)
        : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// Rows [row0, row0 + here) of x, which begin at row x_row of its operand, by features from `feature` on; columns: the rows rounded up to 32.
struct Tile {
    int row0, here, columns, x_row, feature;
};

template <int MODE, typename OutT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) mx4_pair_kernel(
    const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_w_scales, const __grid_constant__ CUtensorMap map_x,
    const __grid_constant__ CUtensorMap map_x_scales, const Args a) {
    using S = Shape<MODE>;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* tiles = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(tiles + (size_t)S::kStages * S::kStageStride);
    uint64_t* empty = full + S::kStages;
    uint64_t* acc_full = empty + S::kStages;               // accumulator ready to be stored
    uint64_t* acc_empty = acc_full + S::kBuffers;          // accumulator read by both blocks (the leader's counts)
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + S::kBuffers);
    volatile int* give_up = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    const int rank = (int)block_in_pair(), pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
    const int n_k = (a.atoms + S::kSteps - 1) / S::kSteps;
    const uint32_t b_smem = a.size / 2 * 128;              // of x, one block, a term

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) {
            mbar_init(full + s, 1);
            mbar_init(empty + s, 1);
        }
        for (int i = 0; i < S::kBuffers; ++i) {
            mbar_init(acc_full + i, 1);
            mbar_init(acc_empty + i, 2 * kEpilogueWarps);
        }
        *give_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    if (warp == 1) {   // the same warp of both blocks allocates
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    pair_barrier();                            // both blocks' barriers stand
    __syncwarp();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    constexpr uint32_t tmem_base = 0;          // all columns are this pair's

    // Neighbouring tiles share their rows of W: the tiles of rows run fastest, within a band of them that stays in L2.
    const int n_features = (a.N + kFeatures - 1) / kFeatures;
    auto tile_of = [&](int i) {
        Tile t;
        const int first = i / (a.band * n_features) * a.band, here = min(a.band, a.cuts - first), j = i - first * n_features;
        const int f = j / here, cut = first + j - f * here;
        t.row0 = cut * a.size;
        t.here = min(a.size, a.M - t.row0);
        t.columns = (t.here + 31) / 32 * 32;
        t.x_row = cut * a.pitch;
        t.feature = f * kFeatures;
        return t;
    };

    if (warp == 0) {
        // ---- the copies: a whole warp walks, one thread of it issues
        const bool issues = elect_one();
        const uint32_t leader_full = leader_addr(full);
        int it = 0;
        for (int i = pair; i < a.n_tiles && !__any_sync(0xffffffffu, *give_up); i += n_pairs) {
            const Tile t = tile_of(i);
            const int b_row = t.x_row + rank * (t.columns / 2), a_row = t.feature + rank * 128;
            // (a last tile of fewer columns brings what a whole one does)
            const uint32_t bytes = (MODE == kQuantized ? S::kASmem : S::kASmem / 2) + S::kT * b_smem + S::kScaleBytes;
            for (int kb = 0; kb < n_k && !a.skip_loads; ++kb, ++it) {
                const int s = it % S::kStages;
                if (!__all_sync(0xffffffffu, mbar_wait(empty + s, ((it / S::kStages) & 1) ^ 1))) {
                    if (lane == 0 && a.err) atomicOr(a.err, THN_ERR_WAIT_TIMEOUT);
                    *give_up = 1;
                    break;
                }
                unsigned char* dst = tiles + (size_t)s * S::kStageStride;
                unsigned char* scales = dst + S::kASmem + S::kT * S::kBSmem;
                const uint32_t bar = leader_full + s * (uint32_t)sizeof(uint64_t);
                if (issues) {
                    if (rank == 0) mbar_expect_tx(full + s, 2 * bytes);
                    load_box(dst, &map_w, bar, kb * 128, a_row);           // (bytes of codes, or entries)
                    load_box(dst + S::kASmem, &map_x, bar, kb * 128, b_row, 0);
                    load_box(scales, &map_w_scales, bar, 0, kb * S::kSteps, a_row >> 7, 0);
                    load_box(scales + S::kSteps * kMx4AtomBytes, &map_x_scales, bar, 0, kb * S::kSteps, t.x_row >> 7, 0);
                }
                __syncwarp();
            }
        }
    } else if (warp == 1 && rank == 0) {
        // ---- the leading block issues the pair's products: a whole warp walks, one thread of it issues.  A stage's scales go to tensor memory ahead of
        // the products of the stage before it, so that they are copied under those; two sets of columns take them in turn.
        const bool issues = elect_one();
        auto bring_scales = [&](int s, uint32_t set) {           // W's, then x's, [term][piece of K][128 rows]
            const uint32_t from = smem_addr(tiles + (size_t)s * S::kStageStride) + S::kASmem + S::kT * S::kBSmem;
            const uint32_t to = tmem_base + S::kScaleCol + set * S::kScaleCols;
#pragma unroll
            for (int p = 0; p < S::kSteps; ++p) pair_scales(to + 4 * p, scale_desc(from + p * kMx4AtomBytes));
#pragma unroll
            for (int term = 0; term < S::kT; ++term)
#pragma unroll
                for (int j = 0; j < S::kAtoms; ++j)
#pragma unroll
                    for (int p = 0; p < S::kSteps; ++p)
                        pair_scales(to + 4 * (S::kSteps + (term * S::kSteps + p) * S::kAtoms + j),
                                    scale_desc(from + (S::kSteps + (term * S::kAtoms + j) * S::kSteps + p) * kMx4AtomBytes));
        };
        const int total = n_k * ((a.n_tiles - pair + n_pairs - 1) / n_pairs);
        bool ok = true, brought = false;                         // whether this stage has come, and its scales are on their way
        int it = 0, s = 0, local = 0;
        uint32_t phase = 0;                                      // of the stage s
        for (int i = pair; i < a.n_tiles && ok; i += n_pairs, ++local) {
            const Tile t = tile_of(i);
            const uint32_t instr = MODE == kQuantized ? scaled_instr(1, 1, kFeatures, t.columns) : scaled_instr(kE2M1, kE4M3, kFeatures, t.columns);
            const uint32_t first = (t.x_row & 127) >> 5;          // the tile's first column of scales
            const int buf = local % S::kBuffers;
            ok = __all_sync(0xffffffffu, mbar_wait(acc_empty + buf, ((local / S::kBuffers) & 1) ^ 1) && !*give_up);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t tmem_d = tmem_base + buf * S::kSums * S::kCols;
            for (int kb = 0; kb < n_k && ok; ++kb, ++it) {
                const int next = s + 1 == S::kStages ? 0 : s + 1;
                const uint32_t next_phase = next == 0 ? phase ^ 1 : phase;
                if (!brought) {
                    ok = __all_sync(0xffffffffu, mbar_wait(full + s, phase));
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    if (issues) bring_scales(s, it & 1);
                }
                brought = it + 1 < total && __all_sync(0xffffffffu, mbar_here(full + next, next_phase));
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t at = smem_addr(tiles + (size_t)s * S::kStageStride);
                const uint32_t w_col = tmem_base + S::kScaleCol + (it & 1) * S::kScaleCols, x_col = w_col + 4 * S::kSteps + first;
                const uint64_t a_desc = smem_desc(at);
                if (issues) {
                    if (brought) bring_scales(next, (it + 1) & 1);
#pragma unroll
                    for (int term = 0; term < S::kT; ++term) {
                        const uint64_t b_desc = smem_desc(at + S::kASmem + term * b_smem);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {      // 32 bytes further along K: + 2 in the address field
                            if constexpr (MODE == kQuantized) {    // 64 entries, two of a piece's four scales
                                if (k >= 2 && kb * 2 + 1 >= a.atoms) break;
                                pair_mma<MODE>(tmem_d, a_desc + 2 * k, b_desc + 2 * k, with_scale_byte(instr, (k & 1) * 2), w_col + 4 * (k >> 1),
                                               x_col + (k >> 1) * S::kAtoms * 4, (kb | k) != 0);
                            } else {                               // 32 entries, one scale
                                const bool second = S::kSums == 2 && term > 0;
                                pair_mma<MODE>(tmem_d + (second ? S::kCols : 0), a_desc + 2 * k, b_desc + 2 * k, with_scale_byte(instr, k), w_col,
                                               x_col + term * S::kAtoms * 4, (kb | k | (second ? term - 1 : term)) != 0);
                            }
                        }
                    }
                    pair_commit(empty + s);                // the stage is free in both blocks when these products are done
                }
                __syncwarp();
                s = next;
                phase = next_phase;
            }
            if (ok && issues) pair_commit(acc_full + buf);
            __syncwarp();
        }
        if (!ok) {                                         // (the warps that wait for an accumulator, in both blocks, give up by themselves)
            if (lane == 0 && a.err) atomicOr(a.err, THN_ERR_WAIT_TIMEOUT);
            *give_up = 1;
        }
    } else if (warp >= 2) {
        // ---- epilogue: a warp reads tensor-memory lanes 32 * (warp % 4) .. + 31 (= features), its group every second chunk of 32 columns (= rows)
        const int quarter = warp & 3, group = (warp - 2) >> 2;
        int local = 0;
        bool dead = false;
        for (int i = pair; i < a.n_tiles; i += n_pairs, ++local) {
            const Tile t = tile_of(i);
            const int buf = local % S::kBuffers;
            const int feature = t.feature + rank * 128 + quarter * 32 + lane;
            const bool there = feature < a.N;
            const float bias = bias_of(a.bias, a.bias_dtype, feature, a.N);
            if (!dead) {
                const bool came = mbar_wait(acc_full + buf, (local / S::kBuffers) & 1, sum_limit_ns(n_k));
                dead = !__all_sync(0xffffffffu, came && !*give_up);      // all lanes together before tcgen05.ld
                if (dead) {
                    if (lane == 0 && a.err) atomicOr(a.err, THN_ERR_WAIT_TIMEOUT);
                    *give_up = 1;
                }
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t taddr = tmem_base + buf * S::kSums * S::kCols + ((uint32_t)(quarter * 32) << 16);
#pragma unroll 1
            for (int c = 32 * group; c < t.here; c += 32 * (kEpilogueWarps / 4)) {
                float v[32];
                if (dead) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(0x7fffffffu);
                } else {
                    tmem_load_32(taddr + c, v);
                    if constexpr (S::kSums == 2) {
                        float rest[32];
                        tmem_load_32(taddr + S::kCols + c, rest);
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] += rest[j];
                    }
                }
                if (there) {
                    OutT* out = static_cast<OutT*>(a.out) + (long long)(t.row0 + c) * a.N + feature;
                    if (c + 32 <= t.here) {
#pragma unroll
                        for (int j = 0; j < 32; ++j, out += a.N) *out = from_f32<OutT>(v[j] + bias);
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; ++j, out += a.N)
                            if (c + j < t.here) *out = from_f32<OutT>(v[j] + bias);
                    }
                }
                __syncwarp();
            }
            // this warp has read its share of the accumulator: the leader may fill it again
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0)
                asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(leader_addr(acc_empty + buf)) : "memory");
        }
    }
    if (*give_up) let_copies_land();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    pair_barrier();                            // neither block leaves while the other may reach into it
    __syncwarp();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(*tmem_slot), "r"(512) : "memory");
    }
    // neither block leaves before both have given their tensor memory back
    __syncthreads();
    pair_barrier();
}

// A tensor map of up to four dimensions, the strides in bytes from the second on.
bool make_map(CUtensorMap* map, CUtensorMapDataType type, int n, const void* base, const cuuint64_t (&dims)[4], const cuuint64_t (&strides)[3],
              const cuuint32_t (&box)[4], CUtensorMapSwizzle swizzle) {
    const EncodeTiled encode = encode_tiled();
    if (encode == nullptr) return false;
    const cuuint32_t elem[4] = {1, 1, 1, 1};
    return encode(map, type, n, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// Scales [planes][rows / 128][pieces of K][512 bytes] for boxes of `steps` pieces for 128 `box_atoms` rows of each plane.
bool map_scales(CUtensorMap* map, const void* scales, long long atoms, long long row_atoms, int planes, int steps, int box_atoms) {
    const cuuint64_t row = (cuuint64_t)atoms * kMx4AtomBytes;
    return make_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, scales, {kMx4AtomBytes / 4, (cuuint64_t)atoms, (cuuint64_t)row_atoms, (cuuint64_t)planes},
                    {kMx4AtomBytes, row, row * (cuuint64_t)row_atoms}, {kMx4AtomBytes / 4, (cuuint32_t)steps, (cuuint32_t)box_atoms, (cuuint32_t)planes},
                    CU_TENSOR_MAP_SWIZZLE_NONE);
}
// Bytes [planes][rows][width] for boxes of 128 bytes of box_rows rows of each plane, 128-byte swizzle.
bool map_planes(CUtensorMap* map, const void* base, long long width, long long rows, int planes, int box_rows) {
    return make_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, base, {(cuuint64_t)width, (cuuint64_t)rows, (cuuint64_t)planes, 1},
                    {(cuuint64_t)width, (cuuint64_t)(width * rows), 0}, {128, (cuuint32_t)box_rows, (cuuint32_t)planes, 1}, CU_TENSOR_MAP_SWIZZLE_128B);
}

int pair_count() {
    int device = 0, n_sms = 0;
    cudaGetDevice(&device);
    if (cudaDeviceGetAttribute(&n_sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) cudaGetLastError();
    return n_sms >= 2 ? n_sms / 2 : 1;
}

template <int MODE, typename OutT>
int launch(const CUtensorMap (&maps)[4], const Args& args, cudaStream_t stream) {
    constexpr auto kernel = mx4_pair_kernel<MODE, OutT>;
    const int status = reserve_smem<kernel>("mx4_pair", Shape<MODE>::kSmemBytes);
    if (status != 0) return status;
    const int most = pair_count(), pairs = args.n_tiles < most ? args.n_tiles : most;
    // In plain stream order, and no kernel is scheduled early behind it: a pair holds all tensor memory of two multiprocessors from its start to its end,
    // and a long chain of such kernels and small ones, each scheduled under the one before, was seen to stop for good.
    thn_launch_ordered(kernel, dim3((unsigned)(2 * pairs)), kThreads, Shape<MODE>::kSmemBytes, stream, maps[0], maps[1], maps[2], maps[3], args);
    return thn_launch_status("mx4_pair");
}

// The bytes of x's operand that are multiplied by all of W before the next ones: less than half of L2, beside W and the results on their way.  16,384
// bfloat16 rows by 24,576 x 4,096 are 134 MB of terms: 2.6 ms in three bands, 3.4 in one, which every 256 rows of W bring from memory again; by 4,096 x
// 12,288 1.28 and 1.64 ms; bands of 24 or 96 MB are level or slower.
constexpr long long kBandBytes = 48 << 20;

template <int MODE>
int run(Args args, const void* codes, const void* scales, const void* x, const void* x_scales, int out_dtype, cudaStream_t stream) {
    using S = Shape<MODE>;
    const long long padded = (long long)args.atoms * kMx4Atom;
    const long long n_tiles = (long long)args.cuts * ((args.N + kFeatures - 1) / kFeatures);
    THN_UNSUPPORTED_IF(n_tiles > 0x3fffffff, "mx4_pair: M=%d N=%d are too many tiles", args.M, args.N);
    args.n_tiles = (int)n_tiles;
    const long long x_bytes = (long long)args.M * padded * S::kT / (MODE == kQuantized ? 2 : 1);
    const long long bands = (x_bytes + kBandBytes - 1) / kBandBytes;
    args.band = bands < args.cuts ? (int)((args.cuts + bands - 1) / bands) : 1;
    const long long x_rows = MODE == kQuantized ? args.M : (long long)args.cuts * args.pitch;
    CUtensorMap maps[4];
    bool made = map_scales(&maps[1], scales, args.atoms, (args.N + 127) / 128, 1, S::kSteps, 1) &&
                map_scales(&maps[3], x_scales, args.atoms, (x_rows + 127) / 128, S::kT, S::kSteps, S::kAtoms);
    if (MODE == kQuantized)
        made = made && map_bytes(&maps[0], codes, args.N, padded / 2, 128) && map_planes(&maps[2], x, padded / 2, x_rows, 1, args.size / 2);
    else
        made = made && map_unpacked(&maps[0], codes, args.N, padded, 128) &&
               map_planes(&maps[2], x, padded, x_rows, S::kT, args.size / 2);
    if (!made) {
        thn_set_error("mx4_pair: cuTensorMapEncodeTiled failed for M=%d N=%d and %d pieces of K", args.M, args.N, args.atoms);
        return THN_BAD_ARGUMENT;
    }
    if constexpr (MODE == kRows2) return launch<MODE, __nv_bfloat16>(maps, args, stream);
    else if constexpr (MODE == kRows2Apart) return launch<MODE, float>(maps, args, stream);
    else return out_dtype == THN_F32 ? launch<MODE, float>(maps, args, stream) : launch<MODE, __nv_bfloat16>(maps, args, stream);
}

}  // namespace

// How M rows are cut into tiles by N outputs: the size (a multiple of 32) with which the pairs' rounds take the least time, a stage of a tile counted
// with its products' time, 2 clocks a column and term, or that of its bytes of shared memory at 64 a clock, whichever is longer; the rows of x's operand from one tile to
// the next.  Terms are written by a kernel of this library, which begins every tile at a whole piece of 128 rows of scales; rows in 4 bits lie as they
// do, and their tiles begin at multiples of 64.  (2,048 rows by 2,560 outputs are 130 tiles of 160 rows and not 110 of 192: two rounds of 74 pairs
// either way.)
struct RowCuts {
    int cuts, size, pitch;
};
static RowCuts cuts_for(int x_type, int M, int N, int pairs) {
    const bool quantized = x_type == 2;
    const int most = Shape<kQuantized>::kCols, grain = quantized ? 64 : 32, terms = quantized ? 1 : x_type == THN_F32 ? kTerms<float> : kTerms<__nv_bfloat16>;
    const long long features = (N + kFeatures - 1) / kFeatures;
    RowCuts best = {};
    long long least = 0;
    for (int size = most; size >= grain; size -= grain) {
        const int cuts = (M + size - 1) / size, columns = cuts == 1 ? (M + 31) / 32 * 32 : size;
        const long long rounds = (cuts * features + pairs - 1) / pairs, products = 2 * terms * columns;
        const long long loads = (16384 + terms * columns * 64) / 64;
        const long long time = rounds * (products < loads ? loads : products);
        if (best.cuts == 0 || time < least) {
            best = {cuts, columns, quantized ? columns : (columns + 127) / 128 * 128};
            least = time;
        }
    }
    return best;
}

// The bytes of `terms` that M rows of a type need by N outputs.
static long long terms_needed(int x_type, int M, int N, int K) {
    if (x_type == 2) return 0;
    const RowCuts c = cuts_for(x_type, M, N, pair_count());
    const long long rows = (long long)c.cuts * c.pitch * (x_type == THN_F32 ? kTerms<float> : kTerms<__nv_bfloat16>), padded = mx4_padded(K);
    return rows * padded + rows / 128 * (padded / kMx4Atom) * kMx4AtomBytes;
}

THN_API int thn_mx4_pair_scratch(int x_type, int M, int N, int K, long long* bytes) {
    *bytes = terms_needed(x_type, M, N, K);
    return THN_OK;
}

// out [M, N] of out_dtype = x [M, K] @ w [N, K]^T (+ bias [N] of bias_dtype, or null).
//   x          [M, K] of x_type; 2: codes [M, padded / 2] with x_scales (mx4.cuh)
//   codes, scales: W;  terms: scratch of thn_mx4_pair_scratch
// Scales and terms 16-byte, 4-bit codes 32-byte aligned.  err: device error word (THN_ERR_WAIT_TIMEOUT if a wait gave up).
// skip_loads: 0; otherwise no operand is loaded, so that the waits run out (for the test of the waits only).
THN_API int thn_mx4_pair(void* out, int out_dtype, const void* x, const void* x_scales, int x_type, const void* codes, const void* scales,
                         const void* bias, int bias_dtype, void* terms, long long terms_bytes, int M, int N, int K, int skip_loads, int* err,
                         cudaStream_t stream) {
    THN_CHECK_ARG(x_type >= 0 && x_type <= 2 && (out_dtype == THN_F32 || out_dtype == THN_BF16) && (bias_dtype == THN_F32 || bias_dtype == THN_BF16),
                  "mx4_pair: unknown type %d, %d or %d", x_type, out_dtype, bias_dtype);
    THN_UNSUPPORTED_IF(M < 1 || M > (1 << 24) || N < 1 || N > (1 << 24) || K < 1 || K > (1 << 24), "mx4_pair: M=%d N=%d K=%d not supported", M, N, K);
    THN_CHECK_ARG((((uintptr_t)codes | (uintptr_t)(x_type == 2 ? x : codes)) & 31) == 0 &&
                  (((uintptr_t)scales | (uintptr_t)x_scales | (uintptr_t)terms) & 15) == 0, "mx4_pair: codes must be 32-byte, scales and terms 16-byte aligned");
    THN_CHECK_ARG(terms_bytes >= terms_needed(x_type, M, N, K), "mx4_pair: %lld bytes of scratch, %lld needed", terms_bytes,
                  terms_needed(x_type, M, N, K));
    Args args = {};
    args.out = out;
    args.bias = bias;
    args.bias_dtype = bias_dtype;
    args.M = M;
    args.N = N;
    args.atoms = (int)(mx4_padded(K) / kMx4Atom);
    args.err = err;
    args.skip_loads = skip_loads;
    const RowCuts rows = cuts_for(x_type, M, N, pair_count());
    args.cuts = rows.cuts;
    args.size = rows.size;
    args.pitch = rows.pitch;
    const long long plane = (long long)rows.cuts * rows.pitch;
    THN_UNSUPPORTED_IF((long long)(N + 127) / 128 * args.atoms > 0x7fffffff || plane / 128 * 6 * args.atoms > 0x7fffffff || plane * 6 > 0x7fffffff,
                       "mx4_pair: M=%d N=%d K=%d is too large", M, N, K);
    if (x_type == 2) return run<kQuantized>(args, codes, scales, x, x_scales, out_dtype, stream);
    uint8_t* bytes = static_cast<uint8_t*>(terms);
    uint8_t* term_scales = bytes + plane * (x_type == THN_F32 ? kTerms<float> : kTerms<__nv_bfloat16>) * mx4_padded(K);
    const int status = mx4_terms(bytes, term_scales, x, x_type, M, K, (int)plane, rows.size, rows.pitch, stream);
    if (status != THN_OK) return status;
    if (x_type == THN_F32) return run<kRows6>(args, codes, scales, bytes, term_scales, out_dtype, stream);
    if (out_dtype == THN_F32) return run<kRows2Apart>(args, codes, scales, bytes, term_scales, out_dtype, stream);
    return run<kRows2>(args, codes, scales, bytes, term_scales, out_dtype, stream);
}
