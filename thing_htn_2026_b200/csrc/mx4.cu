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

// Two float32 to their codes, the first in the low half of the byte (nearest, ties to the even code, at most 6).
__device__ __forceinline__ uint32_t codes_of(float lo, float hi) {
    uint32_t r;
    asm("{\n.reg .b8 b, z;\nmov.b16 {b, z}, 0;\ncvt.rn.satfinite.e2m1x2.f32 b, %2, %1;\nmov.b32 %0, {b, z, z, z};\n}" : "=r"(r) : "f"(lo), "f"(hi));
    return r;
}

// Eight neighbouring entries of a row as they lie in memory; what lies behind the last column is zero.  vector: the row is whole aligned 16-byte
// pieces.  top(): the largest magnitude as the bits of a float32; codes(b): the codes under the scale byte b.
template <typename T>
struct Piece;

template <>
struct Piece<float> {
    float v[8];
    __device__ __forceinline__ void load(const float* row, int c, int columns, bool vector) {
#pragma unroll
        for (int h = 0; h < 8; h += 4) {
            if (vector) {
                const float4 q = c + h < columns ? *reinterpret_cast<const float4*>(row + c + h) : make_float4(0.f, 0.f, 0.f, 0.f);
                v[h] = q.x; v[h + 1] = q.y; v[h + 2] = q.z; v[h + 3] = q.w;
            } else {
#pragma unroll
                for (int i = h; i < h + 4; ++i) v[i] = c + i < columns ? row[c + i] : 0.f;
            }
        }
    }
    __device__ __forceinline__ uint32_t top() const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
        return m;
    }
    __device__ __forceinline__ uint32_t codes(uint32_t b) const {
        const float factor = __uint_as_float((254 - min(b, 253u)) << 23);
        uint32_t word = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) word |= codes_of(v[2 * i] * factor, v[2 * i + 1] * factor) << (8 * i);
        return word;
    }
};

template <>
struct Piece<__nv_bfloat16> {
    uint32_t w[4];
    __device__ __forceinline__ void load(const __nv_bfloat16* row, int c, int columns, bool vector) {
        if (vector) {
            const uint4 q = c < columns ? *reinterpret_cast<const uint4*>(row + c) : make_uint4(0, 0, 0, 0);
            w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
        } else {
            const uint16_t* bits = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                w[i] = (c + 2 * i < columns ? bits[c + 2 * i] : 0u) | (c + 2 * i + 1 < columns ? (uint32_t)bits[c + 2 * i + 1] << 16 : 0u);
        }
    }
    __device__ __forceinline__ uint32_t top() const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
        return max(m << 16, m & 0xffff0000u);
    }
    __device__ __forceinline__ uint32_t codes(uint32_t b) const {
        const uint32_t factor = (254 - min(b, 253u)) << 7;
        uint32_t word = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t x;
            asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(x) : "r"(w[i]), "r"(factor | factor << 16));      // exact, but for what is nothing beside 1/4
            word |= codes_of(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u)) << (8 * i);
        }
        return word;
    }
};

// Pieces of eight entries: a thread takes AHEAD of them, kThreads apart, and asks for all of them before it works on the first.  Four threads have a
// block's entries, sixteen the columns of four scale bytes.  Bound by the memory where there are many: 2,048 x 9,728 bfloat16 entries 12.5 us, 4.0
// TB/s (one piece a thread: 19 us).
template <int AHEAD, typename T>
__global__ void __launch_bounds__(kThreads) mx4_quantize_kernel(uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                                const T* __restrict__ x, uint32_t units, Mx4Divisor pieces, long long columns,
                                                                long long padded, bool vector, bool early) {
    if (early) pdl_launch_dependents();
    pdl_wait();
    const uint32_t first = blockIdx.x * (uint32_t)(kThreads * AHEAD) + threadIdx.x;
    Piece<T> held[AHEAD];
    Mx4Place<kThreads> at(first, pieces);
#pragma unroll
    for (int a = 0; a < AHEAD; ++a, at.step(pieces))
        held[a].load(x + (long long)at.row * columns, (int)(at.piece * 8), first + a * kThreads < units ? (int)columns : 0, vector);
    at = Mx4Place<kThreads>(first, pieces);
#pragma unroll
    for (int a = 0; a < AHEAD; ++a, at.step(pieces)) {
        uint32_t top = held[a].top();
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const uint32_t field = top >> 23;
        const uint32_t b = field == 255 ? 255 : field > 2 ? field - 2 : 0;
        const uint32_t word = b == 255 ? 0 : held[a].codes(b);
        // the sixteen threads' four scale bytes as one word
        uint32_t four = b << (8 * ((threadIdx.x >> 2) & 3));
        four |= __shfl_xor_sync(0xffffffffu, four, 4);
        four |= __shfl_xor_sync(0xffffffffu, four, 8);
        if (first + a * kThreads >= units) continue;
        *reinterpret_cast<uint32_t*>(codes + (long long)at.row * (padded / 2) + at.piece * 4) = word;
        if ((threadIdx.x & 15) == 0)
            *reinterpret_cast<uint32_t*>(scales + mx4_scale_at(at.row, at.piece / 16, padded / kMx4Atom)) = four;
    }
}

template <int AHEAD, typename T>
__global__ void __launch_bounds__(kThreads) mx4_dequantize_kernel(T* __restrict__ out, const uint8_t* __restrict__ codes,
                                                                  const uint8_t* __restrict__ scales, uint32_t units, Mx4Divisor pieces,
                                                                  long long columns, long long padded, bool vector) {
    pdl_wait();
    const uint32_t first = blockIdx.x * (uint32_t)(kThreads * AHEAD) + threadIdx.x;
    uint32_t words[AHEAD];
    uint8_t bytes[AHEAD];
    Mx4Place<kThreads> at(first, pieces);
#pragma unroll
    for (int a = 0; a < AHEAD; ++a, at.step(pieces)) {
        if (first + a * kThreads < units) {
            words[a] = *reinterpret_cast<const uint32_t*>(codes + (long long)at.row * (padded / 2) + at.piece * 4);
            bytes[a] = scales[mx4_scale_at(at.row, at.piece / 16, padded / kMx4Atom) + (at.piece % 16) / 4];
        }
    }
    at = Mx4Place<kThreads>(first, pieces);
#pragma unroll
    for (int a = 0; a < AHEAD; ++a, at.step(pieces)) {
        if (first + a * kThreads >= units) break;
        const long long c = (long long)at.piece * 8;
        const float s = mx4_scale(bytes[a]);
        T* dst = out + (long long)at.row * columns + c;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = mx4_value(words[a] >> (4 * i)) * s;
        if (vector && c + 8 <= columns) {
            if constexpr (sizeof(T) == 2) {
                uint4 packed;
                __nv_bfloat162* p = reinterpret_cast<__nv_bfloat162*>(&packed);
#pragma unroll
                for (int i = 0; i < 4; ++i) p[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                *reinterpret_cast<uint4*>(dst) = packed;
            } else {
                *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
                *reinterpret_cast<float4*>(dst + 4) = make_float4(v[4], v[5], v[6], v[7]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < columns) dst[i] = from_f32<T>(v[i]);
        }
    }
}

// Codes and scales as they are stored, row by row, into this library's layout.  A thread has eight codes, sixteen the columns of four scale bytes; words:
// the stored rows are whole aligned words.
__global__ void __launch_bounds__(kThreads) mx4_arrange_kernel(uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                               const uint8_t* __restrict__ stored, const uint8_t* __restrict__ stored_scales,
                                                               uint32_t units, Mx4Divisor pieces, int columns, int padded, bool words) {
    pdl_wait();
    const uint32_t unit = blockIdx.x * (uint32_t)kThreads + threadIdx.x, row = pieces.of(unit), piece = unit - row * pieces.d;
    if (unit >= units) return;
    const int row_bytes = (columns + 1) / 2, blocks = (columns + kMx4Block - 1) / kMx4Block;
    const uint8_t* src = stored + (long long)row * row_bytes;
    uint32_t word = 0;
    if (words) {
        if ((int)piece * 4 < row_bytes) word = *reinterpret_cast<const uint32_t*>(src + piece * 4);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = (int)piece * 4 + i;
            uint32_t byte = at < row_bytes ? src[at] : 0;
            if (2 * at + 1 >= columns) byte &= 15;
            word |= byte << (8 * i);
        }
    }
    *reinterpret_cast<uint32_t*>(codes + (long long)row * (padded / 2) + piece * 4) = word;
    if ((piece & 15) == 0) {
        uint32_t four = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = (int)(piece >> 4) * 4 + i;
            if (at < blocks) four |= (uint32_t)stored_scales[(long long)row * blocks + at] << (8 * i);
        }
        *reinterpret_cast<uint32_t*>(scales + mx4_scale_at(row, piece >> 4, padded / kMx4Atom)) = four;
    }
}

int refuse_sizes(const char* what, long long rows, long long columns) {
    THN_CHECK_ARG(rows >= 0 && columns >= 1 && columns <= (1 << 26), "%s: %lld rows of %lld entries", what, rows, columns);
    THN_UNSUPPORTED_IF(rows > 0x7fffffff, "%s: %lld rows of %lld entries are too many", what, rows, columns);
    return THN_OK;
}

// Rows in steps of whole pieces of scales, so that a launch has fewer than 2^31 units: go(first row, rows).
template <typename Go>
int in_steps(long long rows, long long units_a_row, Go go) {
    long long most = 0x7ffffff0 / units_a_row - kThreads * kMx4Ahead;
    most = most < 128 ? 128 : most / 128 * 128;
    for (long long row = 0; row < rows; row += most) {
        const int status = go(row, rows - row < most ? rows - row : most);
        if (status != THN_OK) return status;
    }
    return THN_OK;
}

template <typename T>
int quantize(uint8_t* codes, uint8_t* scales, const T* x, long long rows, long long columns, bool early, cudaStream_t stream) {
    const long long padded = mx4_padded(columns), pieces = padded / 8;
    const bool vector = ((uintptr_t)x & 15) == 0 && columns % (16 / sizeof(T)) == 0;
    return in_steps(rows, pieces, [&](long long row, long long n) {
        const int ahead = mx4_ahead(n * pieces);
        thn_launch(ahead == 1 ? mx4_quantize_kernel<1, T> : mx4_quantize_kernel<kMx4Ahead, T>,
                   (unsigned)((n * pieces + kThreads * ahead - 1) / (kThreads * ahead)), kThreads, 0, stream, codes + row * (padded / 2),
                   scales + row / 128 * (padded / kMx4Atom) * kMx4AtomBytes, x + row * columns, (uint32_t)(n * pieces), Mx4Divisor((uint32_t)pieces), columns,
                   padded, vector, early);
        return thn_launch_status("mx4_quantize");
    });
}

template <typename T>
int dequantize(T* out, const uint8_t* codes, const uint8_t* scales, long long rows, long long columns, cudaStream_t stream) {
    const long long padded = mx4_padded(columns), pieces = (columns + 7) / 8;
    const bool vector = ((uintptr_t)out & 15) == 0 && columns % (16 / sizeof(T)) == 0;
    return in_steps(rows, pieces, [&](long long row, long long n) {
        const int ahead = mx4_ahead(n * pieces);
        thn_launch(ahead == 1 ? mx4_dequantize_kernel<1, T> : mx4_dequantize_kernel<kMx4Ahead, T>,
                   (unsigned)((n * pieces + kThreads * ahead - 1) / (kThreads * ahead)), kThreads, 0, stream, out + row * columns,
                   codes + row * (padded / 2), scales + row / 128 * (padded / kMx4Atom) * kMx4AtomBytes, (uint32_t)(n * pieces),
                   Mx4Divisor((uint32_t)pieces), columns, padded, vector);
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
    const long long padded = mx4_padded(columns), pieces = padded / 8, row_bytes = (columns + 1) / 2, blocks = (columns + kMx4Block - 1) / kMx4Block;
    const bool words = columns % 8 == 0 && ((uintptr_t)stored & 3) == 0;
    return in_steps(rows, pieces, [&](long long row, long long n) {
        thn_launch(mx4_arrange_kernel, (unsigned)((n * pieces + kThreads - 1) / kThreads), kThreads, 0, stream, (uint8_t*)codes + row * (padded / 2),
                   (uint8_t*)scales + row / 128 * (padded / kMx4Atom) * kMx4AtomBytes, (const uint8_t*)stored + row * row_bytes,
                   (const uint8_t*)stored_scales + row * blocks, (uint32_t)(n * pieces), Mx4Divisor((uint32_t)pieces), (int)columns, (int)padded, words);
        return thn_launch_status("mx4_arrange");
    });
}
