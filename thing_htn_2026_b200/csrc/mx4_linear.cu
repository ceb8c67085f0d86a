// out[M, N] = x[M, K] @ W[N, K]^T (+ bias) with W in microscaled 4-bit floating point (mx4.cuh) and x in float32, bfloat16 or that form.
// float32 sums, one rounding.
//
// A block computes 64 x 64 outputs: 32 columns of both operands at a time, as float32 in shared memory, four by four outputs a thread.
#include "mx4.cuh"

namespace {

constexpr int kTile = 64, kThreads = 256;

struct Mx4Rows {                    // x in 4 bits
    const uint8_t* codes;
    const uint8_t* scales;
};

__device__ __forceinline__ float entry(const uint8_t* codes, const uint8_t* scales, long long row, long long c, long long padded) {
    const uint32_t byte = codes[row * (padded / 2) + c / 2];
    return mx4_value(c & 1 ? byte >> 4 : byte & 15) * mx4_scale(scales[mx4_scale_at(row, c / 128, padded / 128) + c % 128 / 32]);
}

// XT: float, __nv_bfloat16 or Mx4Rows
template <typename XT, typename OutT, typename BiasT>
__global__ void __launch_bounds__(kThreads) mx4_linear_kernel(OutT* __restrict__ out, const void* __restrict__ x, const uint8_t* __restrict__ x_scales,
                                                              const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                              const BiasT* __restrict__ bias, int M, int N, int K, int padded) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ float xs[32][kTile + 1], ws[32][kTile + 1];
    const int n0 = blockIdx.x * kTile, m0 = blockIdx.y * kTile;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float acc[4][4] = {};
    for (int k0 = 0; k0 < K; k0 += 32) {
        for (int i = threadIdx.x; i < 32 * kTile; i += kThreads) {
            const int c = i & 31, r = i >> 5;
            float v = 0.f, w = 0.f;
            if (m0 + r < M && k0 + c < K) {
                if constexpr (sizeof(XT) == sizeof(Mx4Rows)) v = entry((const uint8_t*)x, x_scales, m0 + r, k0 + c, padded);
                else v = to_f32<XT>(((const XT*)x)[(long long)(m0 + r) * K + k0 + c]);
            }
            if (n0 + r < N && k0 + c < K) w = entry(codes, scales, n0 + r, k0 + c, padded);
            xs[c][r] = v;
            ws[c][r] = w;
        }
        __syncthreads();
#pragma unroll 8
        for (int c = 0; c < 32; ++c) {
            float a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] = xs[c][ty * 4 + i];
                b[i] = ws[c][tx + 16 * i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int m = m0 + ty * 4 + i, n = n0 + tx + 16 * j;
            if (m < M && n < N) out[(long long)m * N + n] = from_f32<OutT>(acc[i][j] + (bias ? to_f32<BiasT>(bias[n]) : 0.f));
        }
}

template <typename XT, typename OutT>
void launch(void* out, const void* x, const void* x_scales, const void* codes, const void* scales, const void* bias, int bias_dtype, int M, int N,
            int K, cudaStream_t stream) {
    const dim3 grid((N + kTile - 1) / kTile, (M + kTile - 1) / kTile);
    const int padded = (int)mx4_padded(K);
    if (bias_dtype == THN_F32)
        thn_launch(mx4_linear_kernel<XT, OutT, float>, grid, kThreads, 0, stream, (OutT*)out, x, (const uint8_t*)x_scales, (const uint8_t*)codes,
                   (const uint8_t*)scales, (const float*)bias, M, N, K, padded);
    else
        thn_launch(mx4_linear_kernel<XT, OutT, __nv_bfloat16>, grid, kThreads, 0, stream, (OutT*)out, x, (const uint8_t*)x_scales,
                   (const uint8_t*)codes, (const uint8_t*)scales, (const __nv_bfloat16*)bias, M, N, K, padded);
}

}  // namespace

enum Mx4RowsType { THN_X_F32 = 0, THN_X_BF16 = 1, THN_X_MX4 = 2 };

THN_API int thn_mx4_linear(void* out, int out_dtype, const void* x, const void* x_scales, int x_type, const void* codes, const void* scales,
                           const void* bias, int bias_dtype, int M, int N, int K, int* err, cudaStream_t stream) {
    (void)err;
    THN_CHECK_ARG(M >= 0 && N >= 0 && K >= 1 && K <= (1 << 30), "mx4_linear: M=%d N=%d K=%d", M, N, K);
    THN_UNSUPPORTED_IF(M > 65535 * kTile, "mx4_linear: %d rows", M);
    THN_CHECK_ARG((out_dtype == THN_F32 || out_dtype == THN_BF16) && (bias_dtype == THN_F32 || bias_dtype == THN_BF16),
                  "mx4_linear: unknown dtype %d or %d", out_dtype, bias_dtype);
    if (M == 0 || N == 0) return THN_OK;
#define GO(XT)                                                                                                            \
    do {                                                                                                                  \
        if (out_dtype == THN_F32) launch<XT, float>(out, x, x_scales, codes, scales, bias, bias_dtype, M, N, K, stream);  \
        else launch<XT, __nv_bfloat16>(out, x, x_scales, codes, scales, bias, bias_dtype, M, N, K, stream);               \
    } while (0)
    if (x_type == THN_X_F32) GO(float);
    else if (x_type == THN_X_BF16) GO(__nv_bfloat16);
    else GO(Mx4Rows);
#undef GO
    return thn_launch_status("mx4_linear");
}
