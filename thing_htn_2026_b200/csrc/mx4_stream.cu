// out[M, N] = x[M, K] @ W[N, K]^T (+ bias) for few rows, W in microscaled 4-bit floating point (mx4.cuh): bound by reading W once.
//
//  * 128 rows of W are the wide operand of tcgen05.mma (kind::mxf8f6f4, scales applied by the tensor core), the rows of x its
//    narrow one.  W comes by TMA, which spreads its 4-bit codes over 8-bit containers as it copies, so no thread touches a weight;
//    its scales come as 512 bytes for 128 rows and 128 columns, in the order of tensor memory, and go there by tcgen05.cp.
//  * Rows in bfloat16 or float32 become two or six terms of 8-bit floats (mx4_tcgen05.cuh), a column of the narrow operand each;
//    their sums are added at the end.  Up to kConverted rows this happens in the kernel, a warp for 128 columns of
//    them, beside the copies of W; more rows are prepared by a kernel of their own (mx4_terms_kernel), since every block would
//    do it again, and come by TMA.  Rows in 4 bits are brought as W is.
//  * Few tiles of 128 outputs: each is cut along K among the blocks of a cluster, whose partial sums meet in distributed shared
//    memory and are added in ascending order: no scratch memory, no counters, the same result every time.  More tiles: a block
//    alone walks several, and brings the next one's while the last one's sums are stored.
//  * Two blocks a multiprocessor while the rows are few: the bytes in flight cover the memory's latency.
//  * W of the first stages is asked for while the kernels before still run; those that write a weight in this form (mx4.cu) let nothing run ahead of
//    their end.
//
// Every wait on an mbarrier is bounded: after kWaitLimitNs, and more for the stages of a sum, the waiter sets THN_ERR_WAIT_TIMEOUT in the caller's
// error word, the block's partial sums become NaN, and tensor memory is given back.  These waits are for the block's own copies and products.  The
// blocks of a cluster, which are resident together, wait for one another at its barrier, without a limit of its own: each comes there after bounded waits.
#include "mx4_tcgen05.cuh"

namespace {

constexpr int BW = 128, BK = 128, UMMA_K = 32;
constexpr uint32_t kWSmem = BW * BK, kWBytes = kWSmem / 2;     // in shared memory; as the barrier counts
constexpr int kMaxStages = 12;
constexpr int kMaxCluster = 8;
// Rows that the kernel itself brings to terms.  Five to eight float32 rows, with six terms to compute, only by a weight of few pieces (four pieces of
// K a block): by 19,456 x 2,560 eight of them took 26 us so and 13.7 us prepared, five by 1,333 x 1,000 4.6 us either way, a launch more.
constexpr int kConverted = 8;
constexpr long long kFewPieces = 4 * 296;      // (two blocks on each of 148 multiprocessors)
inline bool converts(int x_type, int M, int N, int K) {
    return M <= 4 || (M <= kConverted && (x_type != THN_F32 || (N + 127LL) / 128 * ((K + 127) / 128) <= kFewPieces));
}

// RT: the rows' type (float, __nv_bfloat16, or uint8_t: 4 bits); MR: rows the block has room for; PAIRS: how many pairs of rows the
// kernel itself brings to terms (0: they come prepared, or in 4 bits)
template <typename RT, int MR, int PAIRS>
struct Shape {
    static constexpr bool kQuantized = sizeof(RT) == 1, kConverts = PAIRS > 0;
    static constexpr int kT = kQuantized ? 1 : kTerms<RT>;
    static constexpr int NX = MR * kT < 16 ? 16 : MR * kT;           // columns of the product
    static constexpr int kThreads = 192 + (kConverts ? 128 : 0);     // warp 0: TMA, warp 1: products and tensor memory, 2-5: sums, 6-9: rows to terms
    static constexpr int kXAtoms = (NX + 127) / 128;
    static constexpr uint32_t kXSmem = NX * BK;
    static constexpr uint32_t kStageBytes = kWSmem + kXSmem + (1 + kXAtoms) * kMx4AtomBytes;
    static constexpr uint32_t kStageStride = (kStageBytes + 1023) / 1024 * 1024;
    static constexpr int kRecvFloats = (MR + kMaxCluster) * BW;      // [own row][sending block][output]
    static constexpr size_t kFixed = 1024 /* alignment */ + 512 /* barriers */;
    static constexpr int kScaleCols = 4 + 4 * kXAtoms;               // of a stage; two stages' in turn, behind the two accumulators
    static constexpr int kUsedCols = 2 * NX + 2 * kScaleCols;
    static constexpr int kTmemCols = kUsedCols <= 64 ? 64 : kUsedCols <= 128 ? 128 : kUsedCols <= 256 ? 256 : 512;
    static_assert(kUsedCols <= 512, "tensor memory");
    // (four warps bring rows to terms in turn: as many stages as warps keep each of them within a round of the ring)
    static constexpr int kMinStages = kConverts ? 4 : 3;
    // bytes of a block of a cluster or alone, and the stages that fit a multiprocessor's or half of its shared memory
    static constexpr size_t recv_bytes(bool cluster) { return cluster ? kRecvFloats * 4 : 0; }
    // (blocks that can share a multiprocessor have tensor memory for both: the blocks of two clusters that wait for each other's would wait for good.
    // A block alone fills it, too, so that a third never fits.)
    static constexpr int stages_for(int blocks, bool cluster) {
        if (blocks == 2 && kTmemCols > 256) return 0;
        const int n = (int)(((blocks == 2 ? 113 : 226) * 1024 - kFixed - recv_bytes(cluster)) / kStageStride);
        return n < kMaxStages ? n : kMaxStages;
    }
    static_assert(stages_for(1, true) >= 4, "shared memory");
    static constexpr uint32_t kInstr = scaled_instr(kE2M1, kQuantized ? kE2M1 : kE4M3, BW, NX);
};

struct Args {
    void* out;
    const void* x;                // [M, K] of RT
    const uint8_t* x_scales;      // 4 bits, and terms that were prepared
    const uint8_t* w_scales;
    const void* bias;
    int bias_dtype, M, N, K, chunks, n_tiles, stages, vector;      // vector: x's rows are whole aligned 16-byte pieces
    int* err;
    int skip_loads;               // the test of the bounded waits: nothing is loaded
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
// *mine as it lies in block `rank` of the cluster <- v
__device__ __forceinline__ void store_to_block(float* mine, uint32_t rank, float v) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_addr(mine)), "r"(rank));
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote), "f"(v) : "memory");
}

template <typename RT, int MR, int PAIRS, typename OutT>
__global__ void __launch_bounds__(Shape<RT, MR, PAIRS>::kThreads) mx4_stream_kernel(const __grid_constant__ CUtensorMap map_w,
                                                                             const __grid_constant__ CUtensorMap map_x, const Args a) {
    using S = Shape<RT, MR, PAIRS>;
    pdl_launch_dependents();
    extern __shared__ unsigned char smem_raw[];
    unsigned char* tiles = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const int stages = a.stages;
    uint64_t* full = reinterpret_cast<uint64_t*>(tiles + (size_t)stages * S::kStageStride);
    uint64_t* empty = full + kMaxStages;
    uint64_t* acc_full = empty + kMaxStages;   // [2] accumulator ready to be summed
    uint64_t* acc_empty = acc_full + 2;        // [2] accumulator read
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
    volatile int* give_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
    float* recv = reinterpret_cast<float*>(reinterpret_cast<unsigned char*>(full) + 512);      // (a cluster's blocks)
    static_assert((2 * kMaxStages + 4) * 8 + 8 <= 512, "barriers");

    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank(), n_ranks = (int)cluster_size();
    // A cluster of several blocks has one tile; a block alone walks tiles first, first + grid, ...
    const int first_tile = blockIdx.x / n_ranks, step = gridDim.x / n_ranks;
    const int c0 = (int)((long long)a.chunks * rank / n_ranks), n = (int)((long long)a.chunks * (rank + 1) / n_ranks) - c0;
    auto give_up_at = [&] {
        if (a.err) atomicOr(a.err, THN_ERR_WAIT_TIMEOUT);
        *give_up = 1;
    };

    auto load_w = [&](int s, int tile, int c) {
        constexpr uint32_t kBytes = kWBytes + kMx4AtomBytes + (S::kConverts ? 0 : S::kXSmem / (S::kQuantized ? 2 : 1) + kMx4AtomBytes * S::kXAtoms);
        unsigned char* dst = tiles + (size_t)s * S::kStageStride;
        mbar_expect_tx(full + s, kBytes);
        tma_load_2d(dst, &map_w, full + s, c * BK, tile * BW);
        bulk_load(dst + kWSmem + S::kXSmem, a.w_scales + ((long long)tile * a.chunks + c) * kMx4AtomBytes, kMx4AtomBytes, full + s);
    };
    const int early = a.skip_loads ? 0 : min(stages, n);
    if (warp == 0 && elect_one()) {
        // W of the first stages, before anything else: nobody but this thread need know of the barriers yet
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
        for (int s = 0; s < stages; ++s) {
            mbar_init(full + s, S::kConverts ? 2 : 1);     // the copies, and the warp that brings x
            mbar_init(empty + s, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(acc_full + i, 1);
            mbar_init(acc_empty + i, 4);
        }
        *give_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        for (int i = 0; i < early; ++i) load_w(i, first_tile, c0 + i);
    }
    __syncwarp();
    __syncthreads();
    __syncwarp();
    uint32_t tmem_base = 0;                    // of the warps of the products and the sums
    if (n_ranks > 1) cluster_arrive();         // this block has begun: the others may reach into it

    if (warp == 0) {
        // ---- the copies: the whole warp walks, one thread of it issues
        const bool issues = elect_one();
        auto load_x = [&](int s, int c) {
            if constexpr (!S::kConverts) {
                unsigned char* dst = tiles + (size_t)s * S::kStageStride;
                tma_load_2d(dst + kWSmem, &map_x, full + s, c * BK, 0);
#pragma unroll
                for (int j = 0; j < S::kXAtoms; ++j)
                    bulk_load(dst + kWSmem + S::kXSmem + (1 + j) * kMx4AtomBytes, a.x_scales + ((long long)j * a.chunks + c) * kMx4AtomBytes,
                              kMx4AtomBytes, full + s);
            }
        };
        pdl_wait();
        if (issues)
            for (int i = 0; i < early; ++i) load_x(i, c0 + i);
        __syncwarp();
        int s = early == stages ? 0 : early;
        uint32_t phase = early == stages ? 0 : 1;            // of the stage's last use; 1: never used
        bool ok = !a.skip_loads;
        for (int tile = first_tile, i0 = early; tile < a.n_tiles && ok; tile += step, i0 = 0) {
            for (int i = i0; i < n; ++i) {
                ok = __all_sync(0xffffffffu, mbar_wait(empty + s, phase) && !*give_up);
                if (!ok) break;
                if (issues) {
                    load_w(s, tile, c0 + i);
                    load_x(s, c0 + i);
                }
                __syncwarp();
                if (++s == stages) {
                    s = 0;
                    phase ^= 1;
                }
            }
        }
        if (!ok && !a.skip_loads && lane == 0) give_up_at();
        __syncwarp();
    } else if (warp == 1) {
        // ---- the products: the whole warp walks, one thread of it issues.  A stage's scales go to tensor memory ahead of the products of the stage
        // before it, so that they are copied under those; two sets of columns take them in turn.
        // (Tensor memory is taken once the kernels before are done: a block that held it while it waits for them could hold what one of theirs, or of another
        // stream's kernels beside them, still has to take, and that wait has no bound.
        // Blocks that walk alone, two a multiprocessor, pay for it: one row by 19,456 x 2,560 9.9 us, 8.1 with columns taken ahead of the wait, eight rows 10.9 and
        // 9.7, 32 by 34,816 x 5,120 23.1 and 22.3; clusters are level, 5.3 and 5.1 by 6,144 x 2,560.)
        pdl_wait();
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)),
                     "r"(S::kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        asm volatile("bar.sync 1, 160;" ::: "memory");         // the warps of the sums
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
        const bool issues = elect_one();
        auto bring_scales = [&](int s, uint32_t set) {
            const uint32_t from = smem_addr(tiles + (size_t)s * S::kStageStride) + kWSmem + S::kXSmem;
#pragma unroll
            for (int j = 0; j < 1 + S::kXAtoms; ++j)
                scales_to_tmem(tmem_base + 2 * S::NX + set * S::kScaleCols + 4 * j, scale_desc(from + j * kMx4AtomBytes));
        };
        const int total = n * ((a.n_tiles - first_tile + step - 1) / step);
        bool ok = true, brought = false;       // whether this stage has come, and its scales are on their way
        int it = 0, s = 0, local = 0;
        uint32_t phase = 0;                    // of the stage s
        for (int tile = first_tile; tile < a.n_tiles && ok; tile += step, ++local) {
            const int buf = local & 1;
            ok = __all_sync(0xffffffffu, mbar_wait(acc_empty + buf, ((local >> 1) & 1) ^ 1) && !*give_up);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t tmem_d = tmem_base + buf * S::NX;
            for (int i = 0; i < n && ok; ++i, ++it) {
                const int next = s + 1 == stages ? 0 : s + 1;
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
                const uint32_t w_col = tmem_base + 2 * S::NX + (it & 1) * S::kScaleCols;
                const uint64_t w_desc = smem_desc(at), x_desc = smem_desc(at + kWSmem);
                if (issues) {
                    if (brought) bring_scales(next, (it + 1) & 1);
#pragma unroll
                    for (int k = 0; k < BK / UMMA_K; ++k)  // 32 bytes further along K: + 2 in the address field
                        mma_scaled(tmem_d, w_desc + 2 * k, x_desc + 2 * k, with_scale_byte(S::kInstr, k), w_col, w_col + 4, (i | k) != 0);
                    umma_commit(empty + s);
                }
                __syncwarp();
                s = next;
                phase = next_phase;
            }
            if (ok && issues) umma_commit(acc_full + buf);
            __syncwarp();
        }
        if (!ok && lane == 0) give_up_at();    // (the warps that wait for an accumulator give up by themselves)
        __syncwarp();
    } else if (warp >= 6) {
        if constexpr (S::kConverts) {
            // ---- rows of x to terms: chunk by chunk in turn among four warps, a half warp a row, a thread eight columns, the rows of a warp's next
            // two chunks under way.  A warp is within a round of the ring, because the stage that it filled last was free (and there are as many
            // stages as warps).  Rows behind the last one are zeros in columns that nobody reads.
            const int half = lane >> 4, piece = lane & 15;
            Eight<RT> held[2][PAIRS];
            const int total = n * (first_tile < a.n_tiles ? (a.n_tiles - first_tile + step - 1) / step : 0);
            auto fetch = [&](int it, Eight<RT> (&e)[PAIRS]) {
                if (it >= total) return;
                const int c = (c0 + it % n) * BK + piece * 8;
#pragma unroll
                for (int p = 0; p < PAIRS; ++p) {
                    const int row = 2 * p + half;
                    e[p].load(static_cast<const RT*>(a.x) + (long long)min(row, a.M - 1) * a.K, c, row < a.M ? a.K : 0, a.vector);
                }
            };
            auto convert = [&](int it, const Eight<RT> (&e)[PAIRS]) {
                if (__any_sync(0xffffffffu, *give_up)) return false;           // all lanes together
                const int round = it / stages, s = it - round * stages;
                if (round > 0 && !__all_sync(0xffffffffu, mbar_wait(empty + s, (round & 1) ^ 1))) {
                    if (lane == 0) give_up_at();
                    return false;
                }
                unsigned char* dst = tiles + (size_t)s * S::kStageStride + kWSmem;
#pragma unroll
                for (int p = 0; p < PAIRS; ++p) {
                    uint32_t top = e[p].top();
                    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    const uint32_t b = row_scale_byte(top);
                    e[p].terms(b, [&](int term, uint2 bytes) {
                        const int column = term * MR + 2 * p + half;
                        *reinterpret_cast<uint2*>(dst + column * BK + (((piece >> 1) ^ (column & 7)) << 4) + (piece & 1) * 8) = bytes;
                        if ((piece & 3) == 0)
                            dst[S::kXSmem + kMx4AtomBytes + (column & 31) * 16 + (column >> 5) * 4 + (piece >> 2)] = (uint8_t)term_scale_byte(b, term);
                    });
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(full + s);
                return true;
            };
            pdl_wait();
            fetch(warp - 6, held[0]);
            fetch(warp - 2, held[1]);
            for (int it = warp - 6; it < total; it += 8) {
                if (!convert(it, held[0])) break;
                fetch(it + 8, held[0]);
                if (it + 4 >= total || !convert(it + 4, held[1])) break;
                fetch(it + 12, held[1]);
            }
            __syncwarp();
        }
    } else {
        // ---- the sums: a thread has an output of the tile
        pdl_wait();
        __syncwarp();
        asm volatile("bar.sync 1, 160;" ::: "memory");         // tensor memory is there
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
        const int r = (warp & 3) * 32 + lane;
        bool dead = false;
        int local = 0;
        for (int tile = first_tile; tile < a.n_tiles; tile += step, ++local) {
            const int buf = local & 1, out_n = tile * BW + r;
            const float bias = bias_of(a.bias, a.bias_dtype, out_n, a.N);
            if (!dead) {
                const bool came = mbar_wait(acc_full + buf, (local >> 1) & 1, sum_limit_ns(n));
                dead = !__all_sync(0xffffffffu, came && !*give_up);              // all lanes together before tcgen05.ld
                if (dead && lane == 0) give_up_at();
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t taddr = tmem_base + buf * S::NX + ((uint32_t)((warp & 3) * 32) << 16);
            // calls put(row, sum) for the rows
            auto rows = [&](auto put) {
#pragma unroll
                for (int j = 0; j < MR; j += 8) {
                    if (j >= a.M) break;                             // the same for all
                    float v[S::kT][8];
                    if (dead) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[0][e] = __uint_as_float(0x7fffffffu);
#pragma unroll
                        for (int term = 1; term < S::kT; ++term)
#pragma unroll
                            for (int e = 0; e < 8; ++e) v[term][e] = 0.f;
                    } else {
#pragma unroll
                        for (int term = 0; term < S::kT; ++term) tmem_load_8(taddr + term * MR + j, v[term]);
                        tmem_wait_load();
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float sum = v[S::kT - 1][e];                 // the smallest first
#pragma unroll
                        for (int term = S::kT - 2; term >= 0; --term) sum += v[term][e];
                        if (j + e < a.M) put(j + e, sum);
                    }
                }
            };
            if (n_ranks == 1) {
                rows([&](int row, float sum) {
                    if (out_n < a.N) static_cast<OutT*>(a.out)[(long long)row * a.N + out_n] = from_f32<OutT>(sum + bias);
                });
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(acc_empty + buf);
            } else {
                // this block's partial sums to the rows' owners: row j goes to block j % n_ranks, as its row j / n_ranks, sender `rank`
                __syncwarp();
                cluster_wait();                                      // every block has begun
                int owner = 0, slot = rank;                          // slot = (j / n_ranks) * n_ranks + rank, kept without divisions
                rows([&](int, float sum) {
                    store_to_block(recv + slot * BW + r, (uint32_t)owner, sum);
                    if (++owner == n_ranks) {
                        owner = 0;
                        slot += n_ranks;
                    }
                });
                __syncwarp();
                cluster_arrive();
                cluster_wait();                                      // the partial sums are where they are added
                for (int j = rank, own = 0; j < a.M; j += n_ranks, ++own) {
                    float v[kMaxCluster];
#pragma unroll
                    for (int q = 0; q < kMaxCluster; ++q) v[q] = q < n_ranks ? recv[(own * n_ranks + q) * BW + r] : 0.f;
                    float sum = 0.f;                                 // in ascending order of K
#pragma unroll
                    for (int q = 0; q < kMaxCluster; ++q) sum += v[q];
                    if (out_n < a.N) static_cast<OutT*>(a.out)[(long long)j * a.N + out_n] = from_f32<OutT>(sum + bias);
                }
            }
        }
    }
    if (n_ranks > 1 && (warp < 2 || warp >= 6)) {          // (the warps of the sums have been through both)
        __syncwarp();
        cluster_wait();
        cluster_arrive();
        cluster_wait();
    }
    if (*give_up) let_copies_land();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    __syncwarp();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(S::kTmemCols) : "memory");
    }
}

// Rows as terms of 8-bit floats (mx4_terms).  A thread takes sixteen columns; two of them have a block's, eight the columns of four scale bytes.  2,048 rows of
// 9,728 bfloat16 entries 15.3 us (eight columns a thread: 22.4; two units a thread: 15.7).
constexpr int kTermThreads = 256, kTermEntries = 16;

template <typename RT>
__global__ void __launch_bounds__(kTermThreads) mx4_terms_kernel(uint8_t* __restrict__ bytes, uint8_t* __restrict__ scales, const RT* __restrict__ x,
                                                                 uint32_t units, Mx4Divisor pieces, Mx4Divisor size, int pitch, int K, int padded, int plane,
                                                                 bool vector) {
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t unit = blockIdx.x * (uint32_t)kTermThreads + threadIdx.x;
    const uint32_t from = pieces.of(unit), piece = unit - from * pieces.d;
    Eight<RT> held[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) held[h].load(x + (long long)from * K, piece * kTermEntries + 8 * h, unit < units ? K : 0, vector);
    uint32_t top = max(held[0].top(), held[1].top());
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    const uint32_t b = row_scale_byte(top);
    // the eight threads' four scale bytes of the first term as one word
    uint32_t four = b << (8 * ((threadIdx.x >> 1) & 3));
    four |= __shfl_xor_sync(0xffffffffu, four, 2);
    four |= __shfl_xor_sync(0xffffffffu, four, 4);
    if (unit >= units) return;
    const uint32_t tile = size.of(from), row = tile * pitch + (from - tile * size.d);
    uint2 low[kTerms<RT>];
    held[0].terms(b, [&](int term, uint2 v) { low[term] = v; });
    held[1].terms(b, [&](int term, uint2 v) {
        const long long at = (long long)term * plane + row;
        *reinterpret_cast<uint4*>(bytes + at * padded + piece * kTermEntries) = make_uint4(low[term].x, low[term].y, v.x, v.y);
        if ((threadIdx.x & 7) == 0) {
            uint32_t w = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) w |= term_scale_byte(four >> (8 * i) & 255, term) << (8 * i);
            *reinterpret_cast<uint32_t*>(scales + mx4_scale_at(at, piece / 8, padded / kMx4Atom)) = w;
        }
    });
}

// Clusters of `c` blocks that are resident together on the current device, `blocks` a multiprocessor.
template <typename S, auto KERNEL>
int resident_clusters(int device, int c, int blocks) {
    static NumberPerDevice held[2][kMaxCluster + 1];
    return held[blocks - 1][c](device, [&] {
        cudaLaunchConfig_t config = {};
        config.gridDim = dim3((unsigned)(c * 512));
        config.blockDim = dim3(S::kThreads);
        config.dynamicSmemBytes = S::stages_for(blocks, true) * S::kStageStride + S::kFixed + S::recv_bytes(true);
        cudaLaunchAttribute attribute[1];
        attribute[0].id = cudaLaunchAttributeClusterDimension;
        attribute[0].val.clusterDim.x = (unsigned)c;
        attribute[0].val.clusterDim.y = 1;
        attribute[0].val.clusterDim.z = 1;
        config.attrs = attribute;
        config.numAttrs = 1;
        int found = 0;
        if (cudaOccupancyMaxActiveClusters(&found, KERNEL, &config) != cudaSuccess) {
            cudaGetLastError();
            return -1;
        }
        return found;
    });
}

// How a weight is cut: blocks of a cluster, and blocks a multiprocessor.
struct Cut {
    int cluster, blocks;
};

// Few tiles: the largest cluster of which all are resident together and that has a piece of K a block, two blocks a multiprocessor where a half of
// its shared memory holds four stages, else one.  More tiles: blocks alone, two a multiprocessor where there are more tiles than those and four
// stages fit (34,816 x 5,120 is 272 tiles: 1.84 rounds of single blocks, of which the second leaves the memory idle in part).
template <typename S, auto KERNEL>
Cut cut_for(int device, int n_tiles, int chunks, int n_sms) {
    if (n_tiles <= n_sms) {
        const int most = chunks < kMaxCluster ? chunks : kMaxCluster;
        if (S::stages_for(2, true) >= 4)
            for (int c = most; c >= 2; --c)
                if (n_tiles * c <= 2 * n_sms && resident_clusters<S, KERNEL>(device, c, 2) >= n_tiles) return {c, 2};
        for (int c = most; c >= 2; --c)
            if (n_tiles * c <= n_sms && resident_clusters<S, KERNEL>(device, c, 1) >= n_tiles) return {c, 1};
        if (S::stages_for(2, true) >= S::kMinStages)
            for (int c = most; c >= 2; --c)
                if (n_tiles * c <= 2 * n_sms && resident_clusters<S, KERNEL>(device, c, 2) >= n_tiles) return {c, 2};
    }
    return {1, n_tiles > n_sms && S::stages_for(2, false) >= 4 ? 2 : 1};
}

template <typename RT, int MR, int PAIRS, typename OutT>
int launch(const CUtensorMap& map_w, const CUtensorMap& map_x, Args args, cudaStream_t stream) {
    using S = Shape<RT, MR, PAIRS>;
    constexpr auto kernel = mx4_stream_kernel<RT, MR, PAIRS, OutT>;
    const int status = reserve_smem<kernel>("mx4_stream", 226 * 1024);
    if (status != 0) return status;
    int device = 0, n_sms = 0;
    cudaGetDevice(&device);
    cudaDeviceGetAttribute(&n_sms, cudaDevAttrMultiProcessorCount, device);
    const Cut cut = cut_for<S, kernel>(device, args.n_tiles, args.chunks, n_sms);
    args.stages = S::stages_for(cut.blocks, cut.cluster > 1);
    const size_t smem = args.stages * S::kStageStride + S::kFixed + S::recv_bytes(cut.cluster > 1);
    const int slots = n_sms * cut.blocks;
    const int grid = cut.cluster > 1 ? args.n_tiles * cut.cluster : args.n_tiles < slots ? args.n_tiles : slots;
    thn_launch_cluster(kernel, dim3((unsigned)grid), dim3(S::kThreads), smem, stream, dim3((unsigned)cut.cluster, 1, 1), map_w, map_x, args);
    return thn_launch_status("mx4_stream");
}

// terms: for the rows' terms, kT * MR rows of `padded` bytes, then their scales (null where the kernel brings them itself)
template <typename RT, int MR, int PAIRS = 0>
int launch_rows(Args args, const void* codes, long long padded, void* terms, int out_dtype, cudaStream_t stream) {
    using S = Shape<RT, MR, PAIRS>;
    CUtensorMap map_w, map_x;
    bool made = map_unpacked(&map_w, codes, args.N, padded, BW);
    if constexpr (S::kQuantized) made = made && map_unpacked(&map_x, args.x, args.M, padded, S::NX);
    else if constexpr (!S::kConverts) {
        uint8_t* bytes = static_cast<uint8_t*>(terms);
        uint8_t* scales = bytes + (long long)S::kT * MR * padded;
        const int status = mx4_terms(bytes, scales, args.x, sizeof(RT) == 4 ? THN_F32 : THN_BF16, args.M, args.K, MR, MR, MR, stream);
        if (status != THN_OK) return status;
        args.x_scales = scales;
        made = made && map_bytes(&map_x, bytes, S::kT * MR, padded, S::NX);
    } else map_x = map_w;
    if (!made) {
        thn_set_error("mx4_stream: cuTensorMapEncodeTiled failed for M=%d N=%d K=%d", args.M, args.N, args.K);
        return THN_BAD_ARGUMENT;
    }
    return out_dtype == THN_F32 ? launch<RT, MR, PAIRS, float>(map_w, map_x, args, stream) : launch<RT, MR, PAIRS, __nv_bfloat16>(map_w, map_x, args, stream);
}

// the rows that a block has room for
int room_for(int M) { return M <= 8 ? 8 : M <= 16 ? 16 : M <= 32 ? 32 : 64; }

}  // namespace

int mx4_terms(void* bytes, void* scales, const void* x, int x_type, int M, int K, int plane, int size, int pitch, cudaStream_t stream) {
    const long long padded = mx4_padded(K), units = (long long)M * (padded / kTermEntries);
    THN_UNSUPPORTED_IF(units > 0x7ffff000, "mx4_terms: %d rows of %d entries are too many", M, K);
    const unsigned blocks = (unsigned)((units + kTermThreads - 1) / kTermThreads);
    const bool vector = ((uintptr_t)x & 15) == 0 && K % 8 == 0;
    const Mx4Divisor pieces((uint32_t)(padded / kTermEntries)), rows((uint32_t)size);
    if (x_type == THN_F32)
        thn_launch(mx4_terms_kernel<float>, blocks, kTermThreads, 0, stream, (uint8_t*)bytes, (uint8_t*)scales, (const float*)x, (uint32_t)units, pieces, rows,
                   pitch, K, (int)padded, plane, vector);
    else
        thn_launch(mx4_terms_kernel<__nv_bfloat16>, blocks, kTermThreads, 0, stream, (uint8_t*)bytes, (uint8_t*)scales, (const __nv_bfloat16*)x,
                   (uint32_t)units, pieces, rows, pitch, K, (int)padded, plane, vector);
    return thn_launch_status("mx4_terms");
}

// How many rows of a type (THN_F32, THN_BF16, 2: 4 bits) thn_mx4_stream takes.
static int rows_taken(int x_type) { return x_type == THN_F32 ? 32 : 64; }
THN_API int thn_mx4_stream_rows(int x_type) { return rows_taken(x_type); }

// The bytes of `terms` that M rows of a type need.
static long long terms_needed(int x_type, int M, int N, int K) {
    if (x_type == 2 || converts(x_type, M, N, K)) return 0;
    const long long rows = (long long)(M <= 16 ? 16 : room_for(M)) * (x_type == THN_F32 ? kTerms<float> : kTerms<__nv_bfloat16>), padded = mx4_padded(K);
    return rows * padded + (rows + 127) / 128 * (padded / kMx4Atom) * kMx4AtomBytes;
}

THN_API int thn_mx4_stream_scratch(int x_type, int M, int N, int K, long long* bytes) {
    *bytes = terms_needed(x_type, M, N, K);
    return THN_OK;
}

// out [M, N] of out_dtype = x [M, K] @ w [N, K]^T (+ bias [N] of bias_dtype, or null).
//   x          [M, K] of x_type; 2: codes [M, padded / 2] with x_scales (mx4.cuh)
//   codes, scales: W;  terms: scratch of thn_mx4_stream_scratch
// Scales and terms 16-byte, 4-bit codes 32-byte aligned.  err: device error word (THN_ERR_WAIT_TIMEOUT if a wait gave up).
// skip_loads: 0; otherwise no operand is loaded, so that the waits run out (for the test of the waits only).
THN_API int thn_mx4_stream(void* out, int out_dtype, const void* x, const void* x_scales, int x_type, const void* codes, const void* scales,
                           const void* bias, int bias_dtype, void* terms, long long terms_bytes, int M, int N, int K, int skip_loads, int* err,
                           cudaStream_t stream) {
    THN_CHECK_ARG(x_type >= 0 && x_type <= 2 && (out_dtype == THN_F32 || out_dtype == THN_BF16) && (bias_dtype == THN_F32 || bias_dtype == THN_BF16),
                  "mx4_stream: unknown type %d, %d or %d", x_type, out_dtype, bias_dtype);
    THN_UNSUPPORTED_IF(M < 1 || M > rows_taken(x_type) || N < 1 || K < 1 || K > (1 << 24), "mx4_stream: M=%d N=%d K=%d not supported", M, N, K);
    THN_CHECK_ARG((((uintptr_t)codes | (uintptr_t)(x_type == 2 ? x : codes)) & 31) == 0 &&
                  (((uintptr_t)scales | (uintptr_t)x_scales | (uintptr_t)terms) & 15) == 0, "mx4_stream: codes must be 32-byte, scales and terms 16-byte aligned");
    THN_CHECK_ARG(terms_bytes >= terms_needed(x_type, M, N, K), "mx4_stream: %lld bytes of scratch, %lld needed", terms_bytes,
                  terms_needed(x_type, M, N, K));
    const long long padded = mx4_padded(K);
    Args args = {};
    args.out = out;
    args.x = x;
    args.x_scales = (const uint8_t*)x_scales;
    args.w_scales = (const uint8_t*)scales;
    args.bias = bias;
    args.bias_dtype = bias_dtype;
    args.M = M;
    args.N = N;
    args.K = K;
    args.chunks = (int)(padded / BK);
    args.n_tiles = (N + BW - 1) / BW;
    args.vector = ((uintptr_t)x & 15) == 0 && K % 8 == 0;
    args.err = err;
    args.skip_loads = skip_loads;
#define GO(...) return launch_rows<__VA_ARGS__>(args, codes, padded, terms, out_dtype, stream)
    const int room = room_for(M);
    if (x_type == THN_F32) {
        if (M <= 2) GO(float, 8, 1);
        if (M <= 4) GO(float, 8, 2);
        if (converts(x_type, M, N, K)) GO(float, 8, 4);
        if (room <= 16) GO(float, 16);
        GO(float, 32);
    }
    if (x_type == THN_BF16) {
        if (M <= 2) GO(__nv_bfloat16, 8, 1);
        if (M <= 4) GO(__nv_bfloat16, 8, 2);
        if (room == 8) GO(__nv_bfloat16, 8, 4);
        if (room == 16) GO(__nv_bfloat16, 16);
        if (room == 32) GO(__nv_bfloat16, 32);
        GO(__nv_bfloat16, 64);
    }
    if (room <= 16) GO(uint8_t, 16);
    if (room == 32) GO(uint8_t, 32);
    GO(uint8_t, 64);
#undef GO
}
