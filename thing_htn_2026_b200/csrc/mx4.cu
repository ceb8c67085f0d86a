// To and from microscaled 4-bit floating point (layout: mx4.cuh).
//
// Quantising a block of 32 entries x: b = max(floor(log2 max|x|) - 2 + 127, 0), which makes 4 <= max|x| 2^(127 - b) < 8 (or
// less, where the scale is already the smallest), and an entry's code is that of the nearest magnitude to |x| 2^(127 - b), of two
// equally near ones the even code, and 6 above 6.  All of it is exact but that one rounding: the scale is a power of two.  A
// block that holds an infinity or a NaN gets the scale byte 255 and codes of zero.
#include "mx4.cuh"

namespace {

constexpr int kThreads = 256;

// Eight neighbouring entries of a row as float32; what lies behind the last column is zero.
template <typename T>
__device__ __forceinline__ void load8(const T* row, long long c, long long columns, bool vector, float (&v)[8]) {
    if (vector && c + 8 <= columns) {
        if constexpr (sizeof(T) == 2) {
            const uint4 raw = *reinterpret_cast<const uint4*>(row + c);
            const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        } else {
            const float4 a = *reinterpret_cast<const float4*>(row + c), b = *reinterpret_cast<const float4*>(row + c + 4);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < columns ? to_f32<T>(row[c + i]) : 0.f;
    }
}

// Two float32 to their codes, the first in the low half of the byte (nearest, ties to the even code, at most 6).
__device__ __forceinline__ uint32_t codes_of(float lo, float hi) {
    uint32_t r;
    asm("{\n.reg .b8 b, z;\nmov.b16 {b, z}, 0;\ncvt.rn.satfinite.e2m1x2.f32 b, %2, %1;\nmov.b32 %0, {b, z, z, z};\n}" : "=r"(r) : "f"(lo), "f"(hi));
    return r;
}

// A thread takes eight entries, four threads a block, sixteen the columns of four scale bytes.
template <typename T>
__global__ void __launch_bounds__(kThreads) mx4_quantize_kernel(uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                                const T* __restrict__ x, long long rows, long long columns,
                                                                long long padded, bool vector) {
    pdl_launch_dependents();
    pdl_wait();
    const long long pieces = padded / 8, unit = (long long)blockIdx.x * kThreads + threadIdx.x;
    const long long row = unit / pieces, piece = unit - row * pieces;
    const bool there = row < rows;
    float v[8];
    if (there) {
        load8(x + row * columns, piece * 8, columns, vector, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.f;
    }
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const uint32_t field = top >> 23;
    const uint32_t b = field == 255 ? 255 : field > 2 ? field - 2 : 0;
    const float factor = __uint_as_float((254 - min(b, 253u)) << 23);
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) word |= codes_of(v[2 * i] * factor, v[2 * i + 1] * factor) << (8 * i);
    if (b == 255) word = 0;
    // the sixteen threads' four scale bytes as one word
    uint32_t four = b << (8 * ((threadIdx.x >> 2) & 3));
    four |= __shfl_xor_sync(0xffffffffu, four, 4);
    four |= __shfl_xor_sync(0xffffffffu, four, 8);
    if (!there) return;
    *reinterpret_cast<uint32_t*>(codes + row * (padded / 2) + piece * 4) = word;
    if ((threadIdx.x & 15) == 0)
        *reinterpret_cast<uint32_t*>(scales + mx4_scale_at(row, piece / 16, padded / kMx4Atom)) = four;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) mx4_dequantize_kernel(T* __restrict__ out, const uint8_t* __restrict__ codes,
                                                                  const uint8_t* __restrict__ scales, long long rows,
                                                                  long long columns, long long padded, bool vector) {
    pdl_launch_dependents();
    pdl_wait();
    const long long pieces = (columns + 7) / 8, unit = (long long)blockIdx.x * kThreads + threadIdx.x;
    const long long row = unit / pieces, c = (unit - row * pieces) * 8;
    if (row >= rows) return;
    const uint32_t word = *reinterpret_cast<const uint32_t*>(codes + row * (padded / 2) + c / 2);
    const float s = mx4_scale(scales[mx4_scale_at(row, c / kMx4Atom, padded / kMx4Atom) + (c % kMx4Atom) / kMx4Block]);
    T* dst = out + row * columns + c;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = mx4_value(word >> (4 * i)) * s;
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

// Codes and scales as they are stored, row by row, into this library's layout: a thread per 128 columns of a row.
__global__ void __launch_bounds__(kThreads) mx4_arrange_kernel(uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                               const uint8_t* __restrict__ stored, const uint8_t* __restrict__ stored_scales,
                                                               long long rows, long long columns, long long padded) {
    pdl_launch_dependents();
    pdl_wait();
    const long long atoms = padded / kMx4Atom, unit = (long long)blockIdx.x * kThreads + threadIdx.x;
    const long long row = unit / atoms, atom = unit - row * atoms;
    if (row >= rows) return;
    const long long row_bytes = (columns + 1) / 2, blocks = (columns + kMx4Block - 1) / kMx4Block;
    const uint8_t* src = stored + row * row_bytes;
    uint32_t* dst = reinterpret_cast<uint32_t*>(codes + row * (padded / 2) + atom * (kMx4Atom / 2));
    for (int w = 0; w < kMx4Atom / 8; ++w) {
        uint32_t word = 0;
        for (int i = 0; i < 4; ++i) {
            const long long at = atom * (kMx4Atom / 2) + w * 4 + i;
            uint32_t byte = at < row_bytes ? src[at] : 0;
            if (2 * at + 1 >= columns) byte &= 15;
            word |= byte << (8 * i);
        }
        dst[w] = word;
    }
    uint32_t four = 0;
    for (int i = 0; i < 4; ++i) {
        const long long at = atom * 4 + i;
        if (at < blocks) four |= (uint32_t)stored_scales[row * blocks + at] << (8 * i);
    }
    *reinterpret_cast<uint32_t*>(scales + mx4_scale_at(row, atom, atoms)) = four;
}

int refuse_sizes(const char* what, long long rows, long long columns) {
    THN_CHECK_ARG(rows >= 0 && columns >= 1 && columns <= (1 << 30), "%s: %lld rows of %lld entries", what, rows, columns);
    THN_UNSUPPORTED_IF(rows * (mx4_padded(columns) / 8) > (long long)0x7fffffff * kThreads, "%s: %lld rows of %lld entries are too many",
                       what, rows, columns);
    return THN_OK;
}

unsigned blocks_for(long long units) { return (unsigned)((units + kThreads - 1) / kThreads); }

}  // namespace

// x [rows, columns] of dtype -> codes and scales (mx4.cuh).  codes and scales 16-byte aligned.
THN_API int thn_mx4_quantize(void* codes, void* scales, const void* x, long long rows, long long columns, int dtype, cudaStream_t stream) {
    const int status = refuse_sizes("mx4_quantize", rows, columns);
    if (status != THN_OK) return status;
    THN_CHECK_ARG(dtype == THN_F32 || dtype == THN_BF16, "mx4_quantize: unknown dtype %d", dtype);
    if (rows == 0) return THN_OK;
    const long long padded = mx4_padded(columns);
    const unsigned blocks = blocks_for(rows * (padded / 8));
    const bool vector = ((uintptr_t)x & 15) == 0 && columns % (dtype == THN_F32 ? 4 : 8) == 0;
    if (dtype == THN_F32)
        thn_launch(mx4_quantize_kernel<float>, blocks, kThreads, 0, stream, (uint8_t*)codes, (uint8_t*)scales, (const float*)x, rows, columns,
                   padded, vector);
    else
        thn_launch(mx4_quantize_kernel<__nv_bfloat16>, blocks, kThreads, 0, stream, (uint8_t*)codes, (uint8_t*)scales,
                   (const __nv_bfloat16*)x, rows, columns, padded, vector);
    return thn_launch_status("mx4_quantize");
}

// out [rows, columns] of dtype: what codes and scales stand for.
THN_API int thn_mx4_dequantize(void* out, const void* codes, const void* scales, long long rows, long long columns, int dtype,
                               cudaStream_t stream) {
    const int status = refuse_sizes("mx4_dequantize", rows, columns);
    if (status != THN_OK) return status;
    THN_CHECK_ARG(dtype == THN_F32 || dtype == THN_BF16, "mx4_dequantize: unknown dtype %d", dtype);
    if (rows == 0) return THN_OK;
    const long long padded = mx4_padded(columns);
    const unsigned blocks = blocks_for(rows * ((columns + 7) / 8));
    const bool vector = ((uintptr_t)out & 15) == 0 && columns % (dtype == THN_F32 ? 4 : 8) == 0;
    if (dtype == THN_F32)
        thn_launch(mx4_dequantize_kernel<float>, blocks, kThreads, 0, stream, (float*)out, (const uint8_t*)codes, (const uint8_t*)scales,
                   rows, columns, padded, vector);
    else
        thn_launch(mx4_dequantize_kernel<__nv_bfloat16>, blocks, kThreads, 0, stream, (__nv_bfloat16*)out, (const uint8_t*)codes,
                   (const uint8_t*)scales, rows, columns, padded, vector);
    return thn_launch_status("mx4_dequantize");
}

// stored [rows, ceil(columns / 2)] and stored_scales [rows, ceil(columns / 32)], both row by row -> codes and scales.
THN_API int thn_mx4_arrange(void* codes, void* scales, const void* stored, const void* stored_scales, long long rows, long long columns,
                            cudaStream_t stream) {
    const int status = refuse_sizes("mx4_arrange", rows, columns);
    if (status != THN_OK) return status;
    if (rows == 0) return THN_OK;
    const long long padded = mx4_padded(columns);
    thn_launch(mx4_arrange_kernel, blocks_for(rows * (padded / kMx4Atom)), kThreads, 0, stream, (uint8_t*)codes, (uint8_t*)scales,
               (const uint8_t*)stored, (const uint8_t*)stored_scales, rows, columns, padded);
    return thn_launch_status("mx4_arrange");
}
