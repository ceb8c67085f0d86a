// To and from microscaled 4-bit floating point (layout: mx4.cuh).
//
// Quantising a block of 32 entries x: b = max(floor(log2 max|x|) - 2 + 127, 0), which makes 4 <= max|x| 2^(127 - b) < 8 (or
// less, where the scale is already the smallest), and an entry's code is that of the nearest magnitude to |x| 2^(127 - b), of two
// equally near ones the even code, and 6 above 6.  All of it is exact but that one rounding: the scale is a power of two.  A
// block that holds an infinity or a NaN gets the scale byte 255 and codes of zero.
//
// What these kernels write may be the next product's weight, which a product reads while the kernels before it still run.  So
// they let no later kernel be scheduled ahead of their end, and a kernel that begins after their end has all that they wrote; but
// for rows that are quantised to be multiplied (early), which a product reads after its wait.
#include "mx4.cuh"

namespace {

constexpr int kThreads = 256;

// How many pieces of 32 bytes of entries a thread takes: one where there are few, for the latency, two where there are enough for every
// multiprocessor's threads, half of 148 times 2,048 (2,048 x 9,728 bfloat16 entries to 4 bits: 9.6 us, 10.8 with four).
constexpr int kAhead = 2;
inline int ahead_of(long long units) { return units < 148 * 1024 ? 1 : kAhead; }

// Two float32 to their codes, the first in the low half of the byte (nearest, ties to the even code, at most 6).
__device__ __forceinline__ uint32_t codes_of(float lo, float hi) {
    uint32_t r;
    asm("{\n.reg .b8 b, z;\nmov.b16 {b, z}, 0;\ncvt.rn.satfinite.e2m1x2.f32 b, %2, %1;\nmov.b32 %0, {b, z, z, z};\n}" : "=r"(r) : "f"(lo), "f"(hi));
    return r;
}

// 32 bytes at a multiple of 32.
__device__ __forceinline__ void load_32(const void* p, uint32_t (&w)[8]) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(p));
}
__device__ __forceinline__ void store_32(void* p, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
                 "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

// The 32 bytes of neighbouring entries that a thread has, sixteen bfloat16 or eight float32, as they lie in memory; what lies behind the last column
// is zero.  wide: the bytes, 32, 16 or 0, to whose multiples the rows are aligned and of which they are a whole number.  top(): the largest
// magnitude as the bits of a float32; codes(b): the codes under the scale byte b, eight a word.
template <typename T>
struct Piece {
    static constexpr int kEntries = 32 / (int)sizeof(T), kWords = kEntries / 8, kShare = kMx4Block / kEntries;      // threads of a block
    uint32_t w[8];
    __device__ __forceinline__ void load(const T* row, int c, int columns, int wide) {
        if (wide == 32) {
            if (c < columns) {
                load_32(row + c, w);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = 0;
            }
        } else if (wide == 16) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint4 q = c + h * (kEntries / 2) < columns ? *reinterpret_cast<const uint4*>(row + c + h * (kEntries / 2)) : make_uint4(0, 0, 0, 0);
                w[4 * h] = q.x; w[4 * h + 1] = q.y; w[4 * h + 2] = q.z; w[4 * h + 3] = q.w;
            }
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = c + i < columns ? __float_as_uint(row[c + i]) : 0u;
        } else {
            const uint16_t* bits = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                w[i] = (c + 2 * i < columns ? bits[c + 2 * i] : 0u) | (c + 2 * i + 1 < columns ? (uint32_t)bits[c + 2 * i + 1] << 16 : 0u);
        }
    }
    __device__ __forceinline__ uint32_t top() const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (sizeof(T) == 4) m = max(m, w[i] & 0x7fffffffu);
            else m = __vmaxu2(m, w[i] & 0x7fff7fffu);
        }
        return sizeof(T) == 4 ? m : max(m << 16, m & 0xffff0000u);
    }
    __device__ __forceinline__ void codes(uint32_t b, uint32_t (&word)[kWords]) const {
#pragma unroll
        for (int j = 0; j < kWords; ++j) {
            word[j] = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (sizeof(T) == 4) {
                    const float factor = __uint_as_float((254 - min(b, 253u)) << 23);
                    word[j] |= codes_of(__uint_as_float(w[2 * i]) * factor, __uint_as_float(w[2 * i + 1]) * factor) << (8 * i);
                } else {
                    const uint32_t factor = (254 - min(b, 253u)) << 7;
                    uint32_t x;
                    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(x) : "r"(w[4 * j + i]), "r"(factor | factor << 16));      // exact, but for what is nothing beside 1/4
                    word[j] |= codes_of(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u)) << (8 * i);
                }
            }
        }
    }
};

// A thread takes AHEAD pieces, kThreads apart, and asks for all of them before it works on the first.  Bound by the memory where there are many:
// 19,456 x 2,560 bfloat16 entries 21.9 us, 5.8 TB/s (28.2 us in pieces of 16 bytes, four a thread), and back 20.7 us, 6.1 TB/s (26.4).
template <int AHEAD, typename T>
__global__ void __launch_bounds__(kThreads) mx4_quantize_kernel(uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                                const T* __restrict__ x, uint32_t units, Mx4Divisor pieces, long long columns,
                                                                long long padded, int wide, bool early) {
    using P = Piece<T>;
    if (early) pdl_launch_dependents();
    pdl_wait();
    const uint32_t first = blockIdx.x * (uint32_t)(kThreads * AHEAD) + threadIdx.x;
    P held[AHEAD];
    Mx4Place<kThreads> at(first, pieces);
#pragma unroll
    for (int a = 0; a < AHEAD; ++a, at.step(pieces))
        held[a].load(x + (long long)at.row * columns, (int)(at.piece * P::kEntries), first + a * kThreads < units ? (int)columns : 0, wide);
    at = Mx4Place<kThreads>(first, pieces);
#pragma unroll
    for (int a = 0; a < AHEAD; ++a, at.step(pieces)) {
        uint32_t top = held[a].top();
#pragma unroll
        for (int m = 1; m < P::kShare; m *= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, m));
        const uint32_t field = top >> 23;
        const uint32_t b = field == 255 ? 255 : field > 2 ? field - 2 : 0;
        uint32_t word[P::kWords];
        held[a].codes(b, word);
        // the four scale bytes of 128 columns as one word
        uint32_t four = b << (8 * ((threadIdx.x / P::kShare) & 3));
        four |= __shfl_xor_sync(0xffffffffu, four, P::kShare);
        four |= __shfl_xor_sync(0xffffffffu, four, 2 * P::kShare);
        if (first + a * kThreads >= units) continue;
        uint8_t* dst = codes + (long long)at.row * (padded / 2) + at.piece * (P::kEntries / 2);
        if constexpr (P::kWords == 2) *reinterpret_cast<uint2*>(dst) = b == 255 ? make_uint2(0, 0) : make_uint2(word[0], word[1]);
        else *reinterpret_cast<uint32_t*>(dst) = b == 255 ? 0 : word[0];
        if (threadIdx.x % (4 * P::kShare) == 0)
            *reinterpret_cast<uint32_t*>(scales + mx4_scale_at(at.row, at.piece / (4 * P::kShare), padded / kMx4Atom)) = four;
    }
}

template <int AHEAD, typename T>
__global__ void __launch_bounds__(kThreads) mx4_dequantize_kernel(T* __restrict__ out, const uint8_t* __restrict__ codes,
                                                                  const uint8_t* __restrict__ scales, uint32_t units, Mx4Divisor pieces,
                                                                  long long columns, long long padded, int wide) {
    using P = Piece<T>;
    pdl_wait();
    const uint32_t first = blockIdx.x * (uint32_t)(kThreads * AHEAD) + threadIdx.x;
    uint32_t words[AHEAD][P::kWords];
    uint8_t bytes[AHEAD];
    Mx4Place<kThreads> at(first, pieces);
#pragma unroll
    for (int a = 0; a < AHEAD; ++a, at.step(pieces)) {
        if (first + a * kThreads < units) {
            const uint8_t* src = codes + (long long)at.row * (padded / 2) + at.piece * (P::kEntries / 2);
            if constexpr (P::kWords == 2) {
                const uint2 q = *reinterpret_cast<const uint2*>(src);
                words[a][0] = q.x;
                words[a][1] = q.y;
            } else {
                words[a][0] = *reinterpret_cast<const uint32_t*>(src);
            }
            bytes[a] = scales[mx4_scale_at(at.row, at.piece / (4 * P::kShare), padded / kMx4Atom) + at.piece % (4 * P::kShare) / P::kShare];
        }
    }
    at = Mx4Place<kThreads>(first, pieces);
#pragma unroll
    for (int a = 0; a < AHEAD; ++a, at.step(pieces)) {
        const bool there = first + a * kThreads < units;
        const int c = at.piece * P::kEntries;
        const float s = mx4_scale(bytes[a]);
        const long long dst = (long long)at.row * columns + c;
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (sizeof(T) == 4) {
                w[i] = __float_as_uint(mx4_value(words[a][0] >> (4 * i)) * s);
            } else {
                const uint32_t two = words[a][i / 4] >> (8 * (i & 3));
                const __nv_bfloat162 v = __floats2bfloat162_rn(mx4_value(two) * s, mx4_value(two >> 4) * s);
                w[i] = *reinterpret_cast<const uint32_t*>(&v);
            }
        }
        if (wide == 32) {
            if (there) store_32(out + dst, w);
        } else if (wide == 16) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (there && c + h * (P::kEntries / 2) < columns)
                    *reinterpret_cast<uint4*>(out + dst + h * (P::kEntries / 2)) = make_uint4(w[4 * h], w[4 * h + 1], w[4 * h + 2], w[4 * h + 3]);
        } else {
            // rows that begin anywhere: a warp's entries through shared memory, so that neighbouring threads store neighbouring entries (2,048 x
            // 1,001 bfloat16 entries: 3.3 us, 15.3 with a thread's own)
            __shared__ __align__(16) T turned[kThreads * P::kEntries];
            T* mine = turned + threadIdx.x / 32 * 32 * P::kEntries;
            const int lane = threadIdx.x & 31, left = there ? (int)columns - c : 0;
            __syncwarp();
#pragma unroll
            for (int h = 0; h < 2; ++h)
                reinterpret_cast<uint4*>(mine)[2 * lane + h] = make_uint4(w[4 * h], w[4 * h + 1], w[4 * h + 2], w[4 * h + 3]);
            __syncwarp();
#pragma unroll
            for (int i = 0; i < P::kEntries; ++i) {
                const int from = i * (32 / P::kEntries) + lane / P::kEntries, e = lane % P::kEntries;
                T* to = out + __shfl_sync(0xffffffffu, dst, from) + e;
                if (e < __shfl_sync(0xffffffffu, left, from)) *to = mine[i * 32 + lane];
            }
        }
    }
}

// Codes and scales as they are stored, row by row, into this library's layout.  A thread has a block, four the columns of four scale bytes; wide: the
// stored rows are whole aligned 16-byte pieces.  24,576 x 4,096: 18.6 us, 5.7 TB/s (eight codes a thread: 58).
__global__ void __launch_bounds__(kThreads) mx4_arrange_kernel(uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                               const uint8_t* __restrict__ stored, const uint8_t* __restrict__ stored_scales,
                                                               uint32_t units, Mx4Divisor pieces, int columns, int padded, bool wide) {
    pdl_wait();
    const uint32_t unit = blockIdx.x * (uint32_t)kThreads + threadIdx.x, row = pieces.of(unit), piece = unit - row * pieces.d;
    const int row_bytes = (columns + 1) / 2, blocks = (columns + kMx4Block - 1) / kMx4Block, from = (int)piece * (kMx4Block / 2);
    const uint8_t* src = stored + (long long)row * row_bytes + from;
    const bool there = unit < units && (int)piece < blocks;
    uint32_t word[4] = {0, 0, 0, 0};
    if (there && wide) {
        const uint4 q = *reinterpret_cast<const uint4*>(src);
        word[0] = q.x; word[1] = q.y; word[2] = q.z; word[3] = q.w;
    } else if (there) {
#pragma unroll
        for (int i = 0; i < kMx4Block / 2; ++i) {
            uint32_t byte = from + i < row_bytes ? src[i] : 0;
            if (2 * (from + i) + 1 >= columns) byte &= 15;
            word[i / 4] |= byte << (8 * (i & 3));
        }
    }
    uint32_t four = there ? (uint32_t)stored_scales[(long long)row * blocks + piece] << (8 * (piece & 3)) : 0;
    four |= __shfl_xor_sync(0xffffffffu, four, 1);
    four |= __shfl_xor_sync(0xffffffffu, four, 2);
    if (unit >= units) return;
    *reinterpret_cast<uint4*>(codes + (long long)row * (padded / 2) + from) = make_uint4(word[0], word[1], word[2], word[3]);
    if ((piece & 3) == 0) *reinterpret_cast<uint32_t*>(scales + mx4_scale_at(row, piece >> 2, padded / kMx4Atom)) = four;
}

int refuse_sizes(const char* what, long long rows, long long columns) {
    THN_CHECK_ARG(rows >= 0 && columns >= 1 && columns <= (1 << 26), "%s: %lld rows of %lld entries", what, rows, columns);
    THN_UNSUPPORTED_IF(rows > 0x7fffffff, "%s: %lld rows of %lld entries are too many", what, rows, columns);
    return THN_OK;
}

// Rows in steps of whole pieces of scales, so that a launch has fewer than 2^31 units: go(first row, rows).
template <typename Go>
int in_steps(long long rows, long long units_a_row, Go go) {
    long long most = 0x7ffffff0 / units_a_row - kThreads * kAhead;
    most = most < 128 ? 128 : most / 128 * 128;
    for (long long row = 0; row < rows; row += most) {
        const int status = go(row, rows - row < most ? rows - row : most);
        if (status != THN_OK) return status;
    }
    return THN_OK;
}

// To how many bytes, 32, 16 or 0, rows of `columns` entries at `p` are aligned.
template <typename T>
int alignment(const T* p, long long columns) {
    const uintptr_t bits = (uintptr_t)p | (uintptr_t)(columns * sizeof(T));
    return bits % 32 == 0 ? 32 : bits % 16 == 0 ? 16 : 0;
}

template <typename T>
int quantize(uint8_t* codes, uint8_t* scales, const T* x, long long rows, long long columns, bool early, cudaStream_t stream) {
    const long long padded = mx4_padded(columns), pieces = padded / Piece<T>::kEntries;
    const int wide = alignment(x, columns);
    return in_steps(rows, pieces, [&](long long row, long long n) {
        const int ahead = ahead_of(n * pieces);
        thn_launch(ahead == 1 ? mx4_quantize_kernel<1, T> : mx4_quantize_kernel<kAhead, T>,
                   (unsigned)((n * pieces + kThreads * ahead - 1) / (kThreads * ahead)), kThreads, 0, stream, codes + row * (padded / 2),
                   scales + row / 128 * (padded / kMx4Atom) * kMx4AtomBytes, x + row * columns, (uint32_t)(n * pieces), Mx4Divisor((uint32_t)pieces), columns,
                   padded, wide, early);
        return thn_launch_status("mx4_quantize");
    });
}

template <typename T>
int dequantize(T* out, const uint8_t* codes, const uint8_t* scales, long long rows, long long columns, cudaStream_t stream) {
    const long long padded = mx4_padded(columns), pieces = (columns + Piece<T>::kEntries - 1) / Piece<T>::kEntries;
    const int wide = alignment(out, columns);
    return in_steps(rows, pieces, [&](long long row, long long n) {
        const int ahead = ahead_of(n * pieces);
        thn_launch(ahead == 1 ? mx4_dequantize_kernel<1, T> : mx4_dequantize_kernel<kAhead, T>,
                   (unsigned)((n * pieces + kThreads * ahead - 1) / (kThreads * ahead)), kThreads, 0, stream, out + row * columns,
                   codes + row * (padded / 2), scales + row / 128 * (padded / kMx4Atom) * kMx4AtomBytes, (uint32_t)(n * pieces),
                   Mx4Divisor((uint32_t)pieces), columns, padded, wide);
        return thn_launch_status("mx4_dequantize");
    });
}

}  // namespace

// x [rows, columns] of dtype -> codes and scales (mx4.cuh).  codes and scales 16-byte aligned.  early: what they become is never read as a weight.
THN_API int thn_mx4_quantize(void* codes, void* scales, const void* x, long long rows, long long columns, int dtype, int early,
                             cudaStream_t stream) {
    const int status = refuse_sizes("mx4_quantize", rows, columns);
    if (status != THN_OK) return status;
    THN_CHECK_ARG(dtype == THN_F32 || dtype == THN_BF16, "mx4_quantize: unknown dtype %d", dtype);
    if (rows == 0) return THN_OK;
    return dtype == THN_F32 ? quantize((uint8_t*)codes, (uint8_t*)scales, (const float*)x, rows, columns, early != 0, stream)
                            : quantize((uint8_t*)codes, (uint8_t*)scales, (const __nv_bfloat16*)x, rows, columns, early != 0, stream);
}

// out [rows, columns] of dtype: what codes and scales stand for.
THN_API int thn_mx4_dequantize(void* out, const void* codes, const void* scales, long long rows, long long columns, int dtype,
                               cudaStream_t stream) {
    const int status = refuse_sizes("mx4_dequantize", rows, columns);
    if (status != THN_OK) return status;
    THN_CHECK_ARG(dtype == THN_F32 || dtype == THN_BF16, "mx4_dequantize: unknown dtype %d", dtype);
    if (rows == 0) return THN_OK;
    return dtype == THN_F32 ? dequantize((float*)out, (const uint8_t*)codes, (const uint8_t*)scales, rows, columns, stream)
                            : dequantize((__nv_bfloat16*)out, (const uint8_t*)codes, (const uint8_t*)scales, rows, columns, stream);
}

// stored [rows, ceil(columns / 2)] and stored_scales [rows, ceil(columns / 32)], both row by row -> codes and scales.
THN_API int thn_mx4_arrange(void* codes, void* scales, const void* stored, const void* stored_scales, long long rows, long long columns,
                            cudaStream_t stream) {
    const int status = refuse_sizes("mx4_arrange", rows, columns);
    if (status != THN_OK) return status;
    if (rows == 0) return THN_OK;
    const long long padded = mx4_padded(columns), pieces = padded / kMx4Block, row_bytes = (columns + 1) / 2, blocks = (columns + kMx4Block - 1) / kMx4Block;
    const bool wide = columns % kMx4Block == 0 && ((uintptr_t)stored & 15) == 0;
    return in_steps(rows, pieces, [&](long long row, long long n) {
        thn_launch(mx4_arrange_kernel, (unsigned)((n * pieces + kThreads - 1) / kThreads), kThreads, 0, stream, (uint8_t*)codes + row * (padded / 2),
                   (uint8_t*)scales + row / 128 * (padded / kMx4Atom) * kMx4AtomBytes, (const uint8_t*)stored + row * row_bytes,
                   (const uint8_t*)stored_scales + row * blocks, (uint32_t)(n * pieces), Mx4Divisor((uint32_t)pieces), (int)columns, (int)padded, wide);
        return thn_launch_status("mx4_arrange");
    });
}
