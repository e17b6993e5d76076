// Row kernels of the 8-bit operators: floats -> 8-bit integers with one scale a row, and the weighted sum of the
// experts' results of a token.
#include "dtype.cuh"
#include "internal.h"

namespace {

// q = x * 127 / a of the real numbers, to the nearest integer, ties to even.  r = x * fl(127 / a) is off by at most two
// roundings of 2^-24 relative, 127 * 2^-23 < 2^-16 in all, so its nearest integer is the quotient's unless r lies within 2^-15 of
// a half; there the quotient is formed in 64 bits, where x * 127 is exact (24 + 7 bits) and one rounding of the division
// cannot reach a half that the quotient does not: they differ by 2^-32 relative or more.
__device__ __forceinline__ int quantise_one(float x, float inv, float a) {
    const float r = x * inv;
    float q = rintf(r);
    if (!(fabsf(fabsf(r - q) - 0.5f) > 0x1p-15f)) q = (float)rint((double)x * 127.0 / (double)a);
    return (int)q;
}

// largest magnitude as the bits of a float: NaN above infinity above every number
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

constexpr int Q_THREADS = 256;

// One block a row: the largest magnitude, then the row again.
template <typename T>
__global__ void __launch_bounds__(Q_THREADS) quantise_i8_kernel(const T* __restrict__ x, long long x_stride, int8_t* __restrict__ q, long long q_stride,
                                                                float* __restrict__ scale, int M, int K) {
    __shared__ uint32_t s_max[Q_THREADS / 32];
    for (int m = blockIdx.x; m < M; m += gridDim.x) {
        const T* row = x + (long long)m * x_stride;
        uint32_t top = 0;
        for (int k = threadIdx.x; k < K; k += Q_THREADS) top = max(top, magnitude(to_f32(row[k])));
        top = __reduce_max_sync(0xFFFFFFFFu, top);
        if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = top;
        __syncthreads();
        top = 0;
        for (int i = 0; i < Q_THREADS / 32; i++) top = max(top, s_max[i]);
        __syncthreads();
        const float a = __uint_as_float(top);
        const bool zero = top == 0 || top >= 0x7F800000u;
        const float inv = __fdiv_rn(127.0f, a);
        if (threadIdx.x == 0) scale[m] = top >= 0x7F800000u ? __int_as_float(0x7FC00000) : __fdiv_rn(a, 127.0f);
        int8_t* out = q + (long long)m * q_stride;
        for (int k = threadIdx.x; k < K; k += Q_THREADS) out[k] = zero ? (int8_t)0 : (int8_t)quantise_one(to_f32(row[k]), inv, a);
    }
}

// One block a token, one thread a column.
template <typename T, typename TO>
__global__ void __launch_bounds__(256) combine_kernel(const T* __restrict__ y, long long y_stride, int places, const int32_t* __restrict__ slots,
                                                      const float* __restrict__ weights, int top_k, TO* __restrict__ out, long long out_stride, int tokens,
                                                      int N) {
    for (int t = blockIdx.x; t < tokens; t += gridDim.x)
        for (int n = threadIdx.x; n < N; n += blockDim.x) {
            float sum = 0.f;
            for (int j = 0; j < top_k; j++) {
                const int p = slots[(long long)t * top_k + j];
                if (p >= 0 && p < places) sum = fmaf(weights[(long long)t * top_k + j], to_f32(y[(long long)p * y_stride + n]), sum);
            }
            out[(long long)t * out_stride + n] = from_f32<TO>(sum);
        }
}

}  // namespace

extern "C" {

int tnns_cuda_quantise_i8(tnns_cuda_ctx* ctx, const void* d_x, int dtype, long long x_stride, int8_t* d_q, long long q_stride,
                          float* d_scale, int M, int K, void* stream) {
    if (!ctx) return tnns_fail(TNNS_ERR_INVALID, "ctx is NULL");
    if (!tnns_dtype_ok(dtype)) return tnns_fail(TNNS_ERR_INVALID, "unknown element type %d", dtype);
    if (M < 0 || K <= 0) return tnns_fail(TNNS_ERR_INVALID, "bad size: %d rows of %d", M, K);
    if (x_stride < K || q_stride < K || q_stride % 16) return tnns_fail(TNNS_ERR_INVALID, "rows of %d elements at strides %lld and %lld (8-bit rows: a multiple of 16)", K, x_stride, q_stride);
    if (M == 0) return TNNS_OK;
    if (!d_x || !d_q || !d_scale) return tnns_fail(TNNS_ERR_INVALID, "NULL argument");
    if ((uintptr_t)d_x % tnns_dtype_bytes(dtype) || (uintptr_t)d_q % 16 || (uintptr_t)d_scale % 4) return tnns_fail(TNNS_ERR_INVALID, "unaligned pointer");
    const int rc = tnns_enter(ctx);
    if (rc) return rc;
    const int grid = M < 16 * ctx->sm_count ? M : 16 * ctx->sm_count;
    TNNS_FOR_DTYPE(dtype, T, (quantise_i8_kernel<T><<<grid, Q_THREADS, 0, (cudaStream_t)stream>>>((const T*)d_x, x_stride, d_q, q_stride, d_scale, M, K)));
    tnns_count_launch();
    TNNS_CUDA_TRY(cudaGetLastError());
    return TNNS_OK;
}

int tnns_cuda_combine(tnns_cuda_ctx* ctx, const void* d_y, int dtype, long long y_stride, int places, const int32_t* d_slots,
                      const float* d_weights, int top_k, void* d_out, int out_dtype, long long out_stride, int T, int N, void* stream) {
    if (!ctx) return tnns_fail(TNNS_ERR_INVALID, "ctx is NULL");
    if (!tnns_dtype_ok(dtype) || !tnns_dtype_ok(out_dtype)) return tnns_fail(TNNS_ERR_INVALID, "unknown element type %d / %d", dtype, out_dtype);
    if (T < 0 || N <= 0 || places < 0 || top_k < 1) return tnns_fail(TNNS_ERR_INVALID, "bad size: %d tokens of %d, %d places, top_k %d", T, N, places, top_k);
    if (y_stride < N || out_stride < N) return tnns_fail(TNNS_ERR_INVALID, "rows of %d elements at strides %lld and %lld", N, y_stride, out_stride);
    if (T == 0) return TNNS_OK;
    if ((!d_y && places) || !d_slots || !d_weights || !d_out) return tnns_fail(TNNS_ERR_INVALID, "NULL argument");
    if ((uintptr_t)d_y % tnns_dtype_bytes(dtype) || (uintptr_t)d_out % tnns_dtype_bytes(out_dtype) || (uintptr_t)d_slots % 4 || (uintptr_t)d_weights % 4)
        return tnns_fail(TNNS_ERR_INVALID, "unaligned pointer");
    const int rc = tnns_enter(ctx);
    if (rc) return rc;
    const int grid = T < 16 * ctx->sm_count ? T : 16 * ctx->sm_count;
    TNNS_FOR_DTYPE(dtype, TI, TNNS_FOR_DTYPE(out_dtype, TO, (combine_kernel<TI, TO><<<grid, 256, 0, (cudaStream_t)stream>>>((const TI*)d_y, y_stride, places, d_slots, d_weights, top_k, (TO*)d_out, out_stride, T, N))));
    tnns_count_launch();
    TNNS_CUDA_TRY(cudaGetLastError());
    return TNNS_OK;
}

}  // extern "C"
