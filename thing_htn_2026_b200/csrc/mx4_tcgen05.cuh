// What the block-scaled products on tensor memory share: barriers, copies, descriptors.
#pragma once

#include <cuda.h>

#include "mx4.cuh"
#include "per_device.h"

// Rows x [M, K] of a type (THN_F32, THN_BF16) as terms of 8-bit floats, see below: term t of row r is row t * plane + r / size * pitch + r % size of a
// matrix of bytes [terms * plane, padded], whose scales lie as mx4.cuh says (mx4_stream.cu).
int mx4_terms(void* bytes, void* scales, const void* x, int x_type, int M, int K, int plane, int size, int pitch, cudaStream_t stream);

namespace {

// A wait gives up after 20 ms.  One for an accumulator waits for all stages of its sum, and a stage takes 2.3 us of a float32 tile's products at 1 GHz, or 4 us
// where all pairs bring theirs from memory at half its rate: 10 us more for each (1.3 s for 2^24 columns, the most that a product takes).
constexpr unsigned long long kWaitLimitNs = 20ull * 1000 * 1000, kStageLimitNs = 10ull * 1000;
__device__ __forceinline__ unsigned long long sum_limit_ns(int stages) { return kWaitLimitNs + (unsigned)stages * kStageLimitNs; }

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// The warp of this thread, as a number that the compiler knows to be the same for the whole warp.  What a warp computes from such
// numbers alone stands in uniform registers, where the tensor core's instructions want their operands: with a single thread's
// numbers an instruction took 55 to 75 clocks to issue, most of it on the way of its operands there.
__device__ __forceinline__ int uniform_warp() { return __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0); }
// One thread of a whole warp says yes.
__device__ __forceinline__ bool elect_one() {
    uint32_t yes;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(yes));
    return yes != 0;
}

__device__ __forceinline__ void mbar_init(uint64_t* bar, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
// Bounded wait for the phase with the given parity.  Returns false when it gave up.  (A try may sleep for as long as the hardware lets it; the clock, which
// counts a part of a long step alone, is looked at after each.)
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, unsigned long long limit_ns = kWaitLimitNs) {
    const uint32_t addr = smem_addr(bar);
    WaitClock clock;
    for (;;) {
        uint32_t done;
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
            "selp.u32 %0, 1, 0, p;\n"
            "}\n"
            : "=r"(done)
            : "r"(addr), "r"(parity)
            : "memory");
        if (done) return true;
        if (clock.ran_out(limit_ns)) return false;
    }
}
// Whether that phase is over, without waiting.
__device__ __forceinline__ bool mbar_here(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(done)
        : "r"(smem_addr(bar)), "r"(parity)
        : "memory");
    return done != 0;
}
__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(smem_addr(dst)), "l"(map), "r"(smem_addr(bar)), "r"(x), "r"(y)
        : "memory");
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_addr(dst)), "l"(src), "r"(bytes), "r"(smem_addr(bar)) : "memory");
}

// Shared-memory matrix descriptor of a K-major tile in rows of 128 bytes with the 128-byte swizzle (see gemm_tcgen05.cu).
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// The same of 512 bytes of scales: 32 rows of 16 bytes, no swizzle, eight rows (128 bytes) a step.
__device__ __forceinline__ uint64_t scale_desc(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
}
// 512 bytes of scales to four columns of tensor memory, the same in all four quarters of its lanes.
__device__ __forceinline__ void scales_to_tmem(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// Element types of kind::mxf8f6f4
constexpr uint32_t kE4M3 = 0, kE2M1 = 5;
// Instruction descriptor of the block-scaled kinds: which of a word's four scale bytes at bits 4-5 (B) and 29-30 (A), element
// types at 7 (A) and 10 (B), N / 8 at 17, scales that are powers of two (bit 23), M / 16 at 24; both operands K-major.
__host__ __device__ constexpr uint32_t scaled_instr(uint32_t a_type, uint32_t b_type, int m, int n) {
    return (a_type << 7) | (b_type << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ uint32_t with_scale_byte(uint32_t instr, uint32_t k) { return instr | (k << 4) | (k << 29); }

// 32 columns of the sum: D += A B with 8-bit containers, one scale byte a row
__device__ __forceinline__ void mma_scaled(uint32_t tmem_d, uint64_t a_desc, uint64_t b_desc, uint32_t instr, uint32_t a_scales,
                                           uint32_t b_scales, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %6, 0;\n"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%4], [%5], p;\n"
        "}\n"
        ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(instr), "r"(a_scales), "r"(b_scales), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
// Eight consecutive columns of this warp's 32 lanes; the caller waits with tmem_wait_load().
__device__ __forceinline__ void tmem_load_8(uint32_t taddr, float* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7])
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// The bias of output n of N (null: none), whose type is a number of ThnDtype.
__device__ __forceinline__ float bias_of(const void* bias, int dtype, int n, int N) {
    if (bias == nullptr || n >= N) return 0.f;
    return dtype == THN_F32 ? static_cast<const float*>(bias)[n] : __bfloat162float(static_cast<const __nv_bfloat16*>(bias)[n]);
}

// ---- rows as they are, as sums of 8-bit floats.
//
// A block of 32 entries with its largest magnitude in [2^e, 2^(e+1)) is brought to [2^7, 2^8) by the scale 2^(e-7); its entries
// are rounded to e4m3 (four significant bits, down to 2^-9), what that leaves is brought up by 2^4 and rounded again, and so on.
// Two terms hold a bfloat16 (eight bits) exactly down to 2^-13 of the block's largest entry, and below that to 2^-21 of it; six hold a
// float32 (24 bits), down to 2^-13, and below that to 2^-37.  A term's products cost the tensor core half of a bfloat16's.
template <typename T>
constexpr int kTerms = sizeof(T) == 2 ? 2 : 6;

// The scale byte of a block's first term, from its largest magnitude's bits; 255: not a number.
__device__ __forceinline__ uint32_t row_scale_byte(uint32_t top_bits) {
    const uint32_t field = top_bits >> 23;
    return field == 255 ? 255 : field > 7 ? field - 7 : 0;
}
// The scale byte of term t: 2^-4 for each, as far as there are bytes.
__device__ __forceinline__ uint32_t term_scale_byte(uint32_t first, int t) { return first == 255 ? 255 : first > 4u * t ? first - 4 * t : 0; }

// Eight neighbouring entries of a row, as they lie in memory.
template <typename T>
struct Eight;

template <>
struct Eight<__nv_bfloat16> {
    uint4 raw;
    // what lies behind the last column is zero; vector: the row is whole aligned 16-byte pieces
    __device__ __forceinline__ void load(const __nv_bfloat16* row, int c, int K, bool vector) {
        if (vector) {
            raw = c < K ? *reinterpret_cast<const uint4*>(row + c) : make_uint4(0, 0, 0, 0);
        } else {
            const uint16_t* bits = reinterpret_cast<const uint16_t*>(row);
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                w[i] = (c + 2 * i < K ? bits[c + 2 * i] : 0u) | (c + 2 * i + 1 < K ? (uint32_t)bits[c + 2 * i + 1] << 16 : 0u);
            raw = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    // the largest magnitude, as the bits of a float32
    __device__ __forceinline__ uint32_t top() const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) m = __vmaxu2(m, (&raw.x)[i] & 0x7fff7fffu);
        return max(m << 16, m & 0xffff0000u);
    }
    // The terms: put(term, bytes).  Two-wide: the scaled entries and what their first term leaves are float16 numbers (eight bits below 2^8).
    template <typename Put>
    __device__ __forceinline__ void terms(uint32_t b, Put put) const {
        const uint32_t up = (254 - min(b, 253u)) << 7, next = (15 + b - term_scale_byte(b, 1)) << 10;      // powers of two: bfloat16, float16
        uint32_t t0[4], t1[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t w = (&raw.x)[i], half, back, rest;
            uint16_t first, second;
            asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(w) : "r"(w), "r"(up | up << 16));
            asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(half) : "f"(__uint_as_float(w & 0xffff0000u)), "f"(__uint_as_float(w << 16)));
            asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(first) : "r"(half));
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(back) : "h"(first));
            asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(rest) : "r"(half), "r"(back));
            asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(rest) : "r"(rest), "r"(next | next << 16));
            asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(second) : "r"(rest));
            t0[i] = first;
            t1[i] = second;
        }
        const bool no = b == 255;
        put(0, no ? make_uint2(0, 0) : make_uint2(t0[0] | t0[1] << 16, t0[2] | t0[3] << 16));
        put(1, no ? make_uint2(0, 0) : make_uint2(t1[0] | t1[1] << 16, t1[2] | t1[3] << 16));
    }
};

template <>
struct Eight<float> {
    float v[8];
    __device__ __forceinline__ void load(const float* row, int c, int K, bool vector) {
#pragma unroll
        for (int h = 0; h < 8; h += 4) {
            if (vector) {
                const float4 q = c + h < K ? *reinterpret_cast<const float4*>(row + c + h) : make_float4(0.f, 0.f, 0.f, 0.f);
                v[h] = q.x; v[h + 1] = q.y; v[h + 2] = q.z; v[h + 3] = q.w;
            } else {
#pragma unroll
                for (int i = h; i < h + 4; ++i) v[i] = c + i < K ? row[c + i] : 0.f;
            }
        }
    }
    __device__ __forceinline__ uint32_t top() const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
        return m;
    }
    template <typename Put>
    __device__ __forceinline__ void terms(uint32_t b, Put put) const {
        const float up = __uint_as_float((254 - min(b, 253u)) << 23);
        float rest[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) rest[i] = b == 255 ? 0.f : v[i] * up;
#pragma unroll
        for (int term = 0; term < kTerms<float>; ++term) {
            const float next = __uint_as_float((127 + term_scale_byte(b, term) - term_scale_byte(b, term + 1)) << 23);
            uint32_t w[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint16_t pair;
                uint32_t back;
                float lo, hi;
                asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(pair) : "f"(rest[2 * i + 1]), "f"(rest[2 * i]));
                asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(back) : "h"(pair));
                asm("{\n.reg .f16 a, b;\nmov.b32 {a, b}, %2;\ncvt.f32.f16 %0, a;\ncvt.f32.f16 %1, b;\n}" : "=f"(lo), "=f"(hi) : "r"(back));
                rest[2 * i] = (rest[2 * i] - lo) * next;
                rest[2 * i + 1] = (rest[2 * i + 1] - hi) * next;
                w[i >> 1] |= (uint32_t)pair << (16 * (i & 1));
            }
            put(term, make_uint2(w[0], w[1]));
        }
    }
};

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult result;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &result) != cudaSuccess ||
            result != cudaDriverEntryPointSuccess)
            p = nullptr;
        return (EncodeTiled)p;
    }();
    return fn;
}

// Lets a kernel take so much dynamic shared memory on the current device.
template <auto KERNEL>
int reserve_smem(const char* what, size_t bytes) {
    static OncePerDevice reserved;
    int device = -1;
    cudaGetDevice(&device);
    const int status = reserved(device, [&] { return (int)cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes); });
    if (status != 0) {
        cudaGetLastError();
        thn_set_error("%s: cannot reserve %zu bytes of shared memory: %s", what, bytes, cudaGetErrorString((cudaError_t)status));
    }
    return status;
}

// Codes [rows][padded / 2] for boxes of 128 columns x box_rows, which arrive as 8-bit containers of 16 bytes for 16 entries, the
// first eight of them filled (and counted by the barrier).
inline bool map_unpacked(CUtensorMap* map, const void* codes, long long rows, long long padded, int box_rows) {
    const EncodeTiled encode = encode_tiled();
    if (encode == nullptr) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)padded, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)padded / 2};
    const cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
    const cuuint32_t elem[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, 2, const_cast<void*>(codes), dims, strides, box, elem,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// Rows of `width` bytes for boxes of 128 bytes x box_rows.
inline bool map_bytes(CUtensorMap* map, const void* base, long long rows, long long width, int box_rows) {
    const EncodeTiled encode = encode_tiled();
    if (encode == nullptr) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)width};
    const cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
    const cuuint32_t elem[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, elem,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace
