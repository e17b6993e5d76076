// Row kernels of the 8-bit operators: floats -> 8-bit integers with one scale a row, and the weighted sum of the
// experts' results of a token.
#include <algorithm>

#include "dtype.cuh"
#include "internal.h"

namespace {

// ---------------------------------------------------------------------------------------
// quantise
// ---------------------------------------------------------------------------------------

// A chunk = the 16 bytes of a row that hold elements VE*i .. VE*i + VE - 1.
template <typename T>
struct Chunk {
    static constexpr int VE = 16 / sizeof(T);
    uint32_t w[4];
};
__device__ __forceinline__ void unpack(const Chunk<float>& c, float (&f)[4]) {
#pragma unroll
    for (int j = 0; j < 4; j++) f[j] = __uint_as_float(c.w[j]);
}
__device__ __forceinline__ void unpack(const Chunk<__half>& c, float (&f)[8]) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&c.w[j]));
        f[2 * j] = v.x;
        f[2 * j + 1] = v.y;
    }
}
__device__ __forceinline__ void unpack(const Chunk<__nv_bfloat16>& c, float (&f)[8]) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        f[2 * j] = __uint_as_float(c.w[j] << 16);
        f[2 * j + 1] = __uint_as_float(c.w[j] & 0xFFFF0000u);
    }
}
// Chunk i of a row of K elements, zeros past the row's end.  MIS: rows need not start on 16 bytes; the two aligned vectors that
// overlap the chunk are fetched (the second only where it holds elements of the row, so that no other 16 bytes than those that
// the row touches are read) and shifted together.
template <typename T, bool MIS>
__device__ __forceinline__ Chunk<T> load_chunk(const T* row, int i, int K) {
    constexpr int VE = Chunk<T>::VE;
    Chunk<T> c;
    if (!MIS) {
        const uint4 v = *reinterpret_cast<const uint4*>(row + (long long)i * VE);
        c.w[0] = v.x; c.w[1] = v.y; c.w[2] = v.z; c.w[3] = v.w;
    } else {
        const int off = (int)((uintptr_t)row & 15);  // bytes; alike for the whole row
        const uint4* base = reinterpret_cast<const uint4*>((uintptr_t)row - off) + i;
        const uint4 a = base[0];
        uint4 b = make_uint4(0, 0, 0, 0);
        if (off && ((long long)(i + 1) * 16 - off) < (long long)K * (int)sizeof(T)) b = base[1];
        const uint32_t v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        uint32_t u[5];
        switch (off >> 2) {
            case 0: u[0] = v[0]; u[1] = v[1]; u[2] = v[2]; u[3] = v[3]; u[4] = v[4]; break;
            case 1: u[0] = v[1]; u[1] = v[2]; u[2] = v[3]; u[3] = v[4]; u[4] = v[5]; break;
            case 2: u[0] = v[2]; u[1] = v[3]; u[2] = v[4]; u[3] = v[5]; u[4] = v[6]; break;
            default: u[0] = v[3]; u[1] = v[4]; u[2] = v[5]; u[3] = v[6]; u[4] = v[7]; break;
        }
#pragma unroll
        for (int j = 0; j < 4; j++) c.w[j] = sizeof(T) == 4 ? u[j] : __funnelshift_r(u[j], u[j + 1], (off & 2) * 8);
    }
    const int have = K - i * VE;
    if (have < VE) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (sizeof(T) == 4) {
                if (j >= have) c.w[j] = 0;
            } else {
                if (2 * j >= have) c.w[j] = 0;
                else if (2 * j + 1 >= have) c.w[j] &= 0xFFFFu;
            }
        }
    }
    return c;
}
// Largest magnitude so far, as the bits of the type (16-bit types: two at a time): NaN above infinity above every number.
template <typename T>
__device__ __forceinline__ uint32_t widen_max(uint32_t top, const Chunk<T>& c) {
#pragma unroll
    for (int j = 0; j < 4; j++) top = sizeof(T) == 4 ? max(top, c.w[j] & 0x7FFFFFFFu) : __vmaxu2(top, c.w[j] & 0x7FFF7FFFu);
    return top;
}
// .. -> the bits of a float
template <typename T>
__device__ __forceinline__ uint32_t magnitude_bits(uint32_t top);
template <>
__device__ __forceinline__ uint32_t magnitude_bits<float>(uint32_t top) { return top; }
template <>
__device__ __forceinline__ uint32_t magnitude_bits<__nv_bfloat16>(uint32_t top) { return max(top & 0xFFFFu, top >> 16) << 16; }
template <>
__device__ __forceinline__ uint32_t magnitude_bits<__half>(uint32_t top) {
    return __float_as_uint(__half2float(__ushort_as_half((unsigned short)max(top & 0xFFFFu, top >> 16))));
}

struct RowScale {
    float a, inv;
    bool zero, exact;  // every q is 0; every q by the quotient in 64 bits
};
__device__ __forceinline__ RowScale row_scale(uint32_t bits, float* scale) {
    RowScale r;
    const bool bad = bits >= 0x7F800000u;
    r.a = __uint_as_float(bits);
    r.zero = bits == 0 || bad;
    r.exact = !r.zero && r.a < 1e-36f;  // 127 / a would leave the range of fp32
    r.inv = r.zero || r.exact ? 0.f : __fdiv_rn(127.0f, r.a);
    if (scale) *scale = bad ? __int_as_float(0x7FC00000) : __fdiv_rn(r.a, 127.0f);
    return r;
}
// q = x * 127 / a of the real numbers, to the nearest integer, ties to even, for a chunk, as bytes.  r = x * fl(127 / a) is off by two
// roundings, 2^-23 relative; adding 1.5 * 2^23 then rounds it to an integer, ties to even, and leaves that in the low byte.  What
// remains is the quotient next to a half, h = n + 1/2:
//   16-bit types  with x = X * 2^i, a = A * 2^j (X, A at most 11 bits) a quotient that is not h differs from it by
//                 1 / max((2n + 1) * A, 127 * X) > 2^-19 relative.  So r, rounded to 21 bits, is h exactly where the quotient is,
//                 and on the quotient's side of h where it is not: no case is left.
//   fp32          where r lies within 2^-15 of a half, x * 127 and h * a are compared in 64 bits, where both are exact.
// Rows whose largest magnitude is too small for 127 / a to be a float divide in 64 bits.
template <typename T, int VE>
__device__ __forceinline__ void quantise_chunk(const float (&x)[VE], const RowScale& s, uint32_t (&out)[VE / 4]) {
    constexpr float MAGIC = 12582912.0f;
    uint32_t q[VE];
    if (sizeof(T) == 2) {
#pragma unroll
        for (int j = 0; j < VE; j++) q[j] = __float_as_uint(__uint_as_float((__float_as_uint(x[j] * s.inv) + 4u) & ~7u) + MAGIC);
    } else {
        float far = 0.f;
#pragma unroll
        for (int j = 0; j < VE; j++) {
            const float r = x[j] * s.inv, m = r + MAGIC;
            far = fmaxf(far, fabsf(r - (m - MAGIC)));
            q[j] = __float_as_uint(m);
        }
        if (far > 0.5f - 0x1p-15f) {
#pragma unroll
            for (int j = 0; j < VE; j++) {
                const float r = fabsf(x[j] * s.inv), n = floorf(r);
                if (fabsf(r - n - 0.5f) < 0x1p-15f) {
                    const double d = (double)fabsf(x[j]) * 127.0 - ((double)n + 0.5) * (double)s.a;
                    const int even = (int)n + ((int)n & 1), up = d > 0 ? (int)n + 1 : d < 0 ? (int)n : even;
                    q[j] = (uint32_t)(x[j] < 0 ? -up : up);
                }
            }
        }
    }
    if (s.exact) {
#pragma unroll
        for (int j = 0; j < VE; j++) q[j] = (uint32_t)(int)rint((double)x[j] * 127.0 / (double)s.a);
    }
#pragma unroll
    for (int j = 0; j < VE / 4; j++) out[j] = s.zero ? 0u : __byte_perm(__byte_perm(q[4 * j], q[4 * j + 1], 0x0040), __byte_perm(q[4 * j + 2], q[4 * j + 3], 0x0040), 0x5410);
}
template <int VE>
__device__ __forceinline__ void store_chunk(int8_t* out, int i, int K, const uint32_t (&q)[VE / 4]) {
    int8_t* at = out + (long long)i * VE;
    const int have = K - i * VE;
    if (have >= VE) {
        if constexpr (VE == 8) *reinterpret_cast<uint2*>(at) = make_uint2(q[0], q[1]);
        else *reinterpret_cast<uint32_t*>(at) = q[0];
    } else {
#pragma unroll
        for (int j = 0; j < VE; j++)
            if (j < have) at[j] = (int8_t)(q[j >> 2] >> (8 * (j & 3)));
    }
}

// GROUP threads a row (a warp, or the whole block), which keeps the row in registers between its largest magnitude and its
// integers, NV chunks a thread: every element is read once.  LONG: rows that do not fit; the chunks past the kept ones are
// read a second time.  Bounded by memory: M = 8192, K = 4096 (figures beside the launch).
template <typename T, int GROUP, int NV, bool MIS, bool LONG>
__global__ void __launch_bounds__(GROUP < 256 ? 256 : GROUP) quantise_i8_kernel(const T* __restrict__ x, long long x_stride, int8_t* __restrict__ q, long long q_stride,
                                                                              float* __restrict__ scale, int M, int K) {
    constexpr int VE = Chunk<T>::VE, ROWS = GROUP < 256 ? 256 / GROUP : 1;
    __shared__ uint32_t s_top[32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int m = blockIdx.x * ROWS + (ROWS > 1 ? threadIdx.x / GROUP : 0), lane = threadIdx.x % GROUP;
    if (m >= M) return;  // (a whole group, and with ROWS > 1 a whole warp)
    const T* row = x + (long long)m * x_stride;
    const int chunks = (K + VE - 1) / VE;
    Chunk<T> c[NV];
    uint32_t top = 0;
#pragma unroll
    for (int v = 0; v < NV; v++)
        if (lane + v * GROUP < chunks) c[v] = load_chunk<T, MIS>(row, lane + v * GROUP, K);
#pragma unroll
    for (int v = 0; v < NV; v++)
        if (lane + v * GROUP < chunks) top = widen_max(top, c[v]);
    if (LONG)
        for (int i = lane + NV * GROUP; i < chunks; i += GROUP) top = widen_max(top, load_chunk<T, MIS>(row, i, K));
    uint32_t bits = __reduce_max_sync(0xFFFFFFFFu, magnitude_bits<T>(top));
    if (GROUP > 32) {
        if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = bits;
        __syncthreads();
        bits = __reduce_max_sync(0xFFFFFFFFu, (threadIdx.x & 31) < GROUP / 32 ? s_top[threadIdx.x & 31] : 0u);
    }
    const RowScale s = row_scale(bits, lane == 0 ? scale + m : nullptr);
    int8_t* out = q + (long long)m * q_stride;
    auto finish = [&](const Chunk<T>& ch, int i) {
        float f[VE];
        uint32_t w[VE / 4];
        unpack(ch, f);
        quantise_chunk<T, VE>(f, s, w);
        store_chunk<VE>(out, i, K, w);
    };
#pragma unroll
    for (int v = 0; v < NV; v++)
        if (lane + v * GROUP < chunks) finish(c[v], lane + v * GROUP);
    if (LONG)
        for (int i = lane + NV * GROUP; i < chunks; i += GROUP) finish(load_chunk<T, MIS>(row, i, K), i);
}

template <typename... Args>
int launch(void (*kern)(Args...), long long grid, int threads, cudaStream_t stream, Args... args) {
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(threads);
    cfg.stream = stream;
    cfg.attrs = attr;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
    TNNS_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, args...));
    tnns_count_launch();
    TNNS_CUDA_TRY(cudaGetLastError());
    return TNNS_OK;
}

// The fewest threads that hold a row in four chunks each, so that many rows are on their way at once; one row by itself takes
// more threads instead (the launch is all latency then).
template <typename T, bool MIS>
int launch_quantise(tnns_cuda_ctx* ctx, const T* x, long long x_stride, int8_t* q, long long q_stride, float* scale, int M, int K, cudaStream_t st) {
    const int chunks = (K + Chunk<T>::VE - 1) / Chunk<T>::VE;
    if (chunks <= 32) return launch<const T*, long long, int8_t*, long long, float*, int, int>(quantise_i8_kernel<T, 32, 1, MIS, false>, ((long long)M + 7) / 8, 256, st, x, x_stride, q, q_stride, scale, M, K);
    if (chunks <= 128 && M > ctx->sm_count) return launch<const T*, long long, int8_t*, long long, float*, int, int>(quantise_i8_kernel<T, 32, 4, MIS, false>, ((long long)M + 7) / 8, 256, st, x, x_stride, q, q_stride, scale, M, K);
    if (chunks <= 256) return launch<const T*, long long, int8_t*, long long, float*, int, int>(quantise_i8_kernel<T, 256, 1, MIS, false>, M, 256, st, x, x_stride, q, q_stride, scale, M, K);
    if (chunks <= 1024 && M > ctx->sm_count) return launch<const T*, long long, int8_t*, long long, float*, int, int>(quantise_i8_kernel<T, 256, 4, MIS, false>, M, 256, st, x, x_stride, q, q_stride, scale, M, K);
    if (chunks <= 1024) return launch<const T*, long long, int8_t*, long long, float*, int, int>(quantise_i8_kernel<T, 1024, 1, MIS, false>, M, 1024, st, x, x_stride, q, q_stride, scale, M, K);
    if (chunks <= 4096) return launch<const T*, long long, int8_t*, long long, float*, int, int>(quantise_i8_kernel<T, 1024, 4, MIS, false>, M, 1024, st, x, x_stride, q, q_stride, scale, M, K);
    return launch<const T*, long long, int8_t*, long long, float*, int, int>(quantise_i8_kernel<T, 1024, 4, MIS, true>, M, 1024, st, x, x_stride, q, q_stride, scale, M, K);
}

// ---------------------------------------------------------------------------------------
// combine
// ---------------------------------------------------------------------------------------

struct CombineArgs {
    const void* y;
    long long y_stride;
    const int32_t* slots;
    const float* weights;
    void* out;
    long long out_stride;
    int places, top_k, T, N, out_dtype, per_row;  // per_row: vectors of V columns
};
template <int V>
__device__ __forceinline__ void store_vec(const CombineArgs& p, long long at, const float (&f)[V]) {
    if (p.out_dtype == TNNS_F32) {
        float* o = (float*)p.out + at;
        if constexpr (V == 8) {
            reinterpret_cast<float4*>(o)[0] = make_float4(f[0], f[1], f[2], f[3]);
            reinterpret_cast<float4*>(o)[1] = make_float4(f[4], f[5], f[6], f[7]);
        } else if constexpr (V == 2) *reinterpret_cast<float2*>(o) = make_float2(f[0], f[1]);
        else *o = f[0];
        return;
    }
    uint16_t h[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
        if (p.out_dtype == TNNS_F16) h[j] = __half_as_ushort(__float2half_rn(f[j]));
        else h[j] = __bfloat16_as_ushort(__float2bfloat16_rn(f[j]));
    }
    uint16_t* o = (uint16_t*)p.out + at;
    if constexpr (V == 8) *reinterpret_cast<uint4*>(o) = make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16, h[4] | (uint32_t)h[5] << 16, h[6] | (uint32_t)h[7] << 16);
    else if constexpr (V == 2) *reinterpret_cast<uint32_t*>(o) = h[0] | (uint32_t)h[1] << 16;
    else *o = h[0];
}
template <typename T, int V>
struct RawVec {
    uint32_t w[V * sizeof(T) <= 4 ? 1 : V * sizeof(T) / 4];
};
template <typename T, int V>
__device__ __forceinline__ RawVec<T, V> load_vec(const T* at) {
    RawVec<T, V> r;
    constexpr int B = V * sizeof(T);
    if constexpr (B >= 16) {
#pragma unroll
        for (int i = 0; i < B / 16; i++) {
            const uint4 v = reinterpret_cast<const uint4*>(at)[i];
            r.w[4 * i] = v.x; r.w[4 * i + 1] = v.y; r.w[4 * i + 2] = v.z; r.w[4 * i + 3] = v.w;
        }
    } else if constexpr (B == 8) {
        const uint2 v = *reinterpret_cast<const uint2*>(at);
        r.w[0] = v.x; r.w[1] = v.y;
    } else if constexpr (B == 4) r.w[0] = *reinterpret_cast<const uint32_t*>(at);
    else r.w[0] = *reinterpret_cast<const uint16_t*>(at);
    return r;
}
template <typename T, int V>
__device__ __forceinline__ void add_vec(const RawVec<T, V>& r, float w, float (&sum)[V]) {
#pragma unroll
    for (int j = 0; j < V; j++) {
        float v;
        if constexpr (sizeof(T) == 4) v = __uint_as_float(r.w[j]);
        else {
            const unsigned short h = (unsigned short)(r.w[j >> 1] >> (16 * (j & 1)));
            if constexpr (sizeof(T) == 2) v = to_f32(*reinterpret_cast<const T*>(&h));
        }
        sum[j] = fmaf(w, v, sum[j]);
    }
}

// One thread V neighbouring columns of a token, the rows of eight slots on their way at once.  Bounded by memory: every row of y is
// read once, V * 32 neighbouring columns a warp.
template <typename T, int V>
__global__ void __launch_bounds__(256) combine_kernel(CombineArgs p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    constexpr int U = 8;
    const long long item = (long long)blockIdx.x * 256 + threadIdx.x;
    if (item >= (long long)p.T * p.per_row) return;
    const int t = item < 0xFFFFFFFFLL ? (int)((uint32_t)item / (uint32_t)p.per_row) : (int)(item / p.per_row);
    const int n = (int)(item - (long long)t * p.per_row) * V;
    const int32_t* slots = p.slots + (long long)t * p.top_k;
    const float* weights = p.weights + (long long)t * p.top_k;
    const T* y = (const T*)p.y + n;
    float sum[V] = {};
    for (int j0 = 0; j0 < p.top_k; j0 += U) {
        int at[U];
        float w[U];
        RawVec<T, V> r[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            at[u] = j0 + u < p.top_k ? __ldg(slots + j0 + u) : -1;
            w[u] = j0 + u < p.top_k ? __ldg(weights + j0 + u) : 0.f;
        }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (at[u] >= 0 && at[u] < p.places) r[u] = load_vec<T, V>(y + (long long)at[u] * p.y_stride);
#pragma unroll
        for (int u = 0; u < U; u++)
            if (at[u] >= 0 && at[u] < p.places) add_vec<T, V>(r[u], w[u], sum);
    }
    store_vec<V>(p, (long long)t * p.out_stride + n, sum);
}

template <typename T, int V>
int launch_combine(const CombineArgs& a, cudaStream_t st) {
    const long long blocks = ((long long)a.T * a.per_row + 255) / 256;
    if (blocks > 0x7FFFFFFFLL) return tnns_fail(TNNS_ERR_UNSUPPORTED, "%d tokens of %d columns", a.T, a.N);
    return launch<CombineArgs>(combine_kernel<T, V>, blocks, 256, st, a);
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
    const cudaStream_t st = (cudaStream_t)stream;
    const bool mis = ((uintptr_t)d_x | (uintptr_t)(x_stride * tnns_dtype_bytes(dtype))) % 16 != 0 || K % (16 / tnns_dtype_bytes(dtype)) != 0;
    TNNS_FOR_DTYPE(dtype, T, return mis ? (launch_quantise<T, true>(ctx, (const T*)d_x, x_stride, d_q, q_stride, d_scale, M, K, st)) : (launch_quantise<T, false>(ctx, (const T*)d_x, x_stride, d_q, q_stride, d_scale, M, K, st)));
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
    CombineArgs a;
    a.y = d_y; a.y_stride = y_stride; a.slots = d_slots; a.weights = d_weights; a.out = d_out; a.out_stride = out_stride;
    a.places = places; a.top_k = top_k; a.T = T; a.N = N; a.out_dtype = out_dtype;
    // columns of a thread: as many as rows and bases allow to move at once (8 elements: 16 or 32 bytes)
    const int bi = tnns_dtype_bytes(dtype), bo = tnns_dtype_bytes(out_dtype);
    auto fits = [&](int v) {
        const int ai = std::min(16, v * bi), ao = std::min(16, v * bo);
        return N % v == 0 && ((uintptr_t)d_y | (uintptr_t)(y_stride * bi)) % ai == 0 && ((uintptr_t)d_out | (uintptr_t)(out_stride * bo)) % ao == 0;
    };
    const int v = fits(8) ? 8 : fits(2) ? 2 : 1;
    a.per_row = N / v;
    const cudaStream_t st = (cudaStream_t)stream;
    TNNS_FOR_DTYPE(dtype, TI, return v == 8 ? (launch_combine<TI, 8>(a, st)) : v == 2 ? (launch_combine<TI, 2>(a, st)) : (launch_combine<TI, 1>(a, st)));
}

}  // extern "C"
