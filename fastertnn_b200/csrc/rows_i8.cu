// Row kernels of the 8-bit operators: floats -> 8-bit integers with one scale a row, and the weighted sum of the
// experts' results of a token.
#include <algorithm>

#include "dtype.cuh"
#include "internal.h"
#include "mbar.cuh"

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
// The 16 bytes from byte `off` on of the 32 that a and b hold.
template <typename T>
__device__ __forceinline__ void realign(const uint4& a, const uint4& b, int off, uint32_t (&w)[4]) {
    uint32_t v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int j = 0; j < 7; j++) v[j] = off & 4 ? v[j + 1] : v[j];
#pragma unroll
    for (int j = 0; j < 5; j++) v[j] = off & 8 ? v[j + 2] : v[j];
#pragma unroll
    for (int j = 0; j < 4; j++) w[j] = sizeof(T) == 4 ? v[j] : __funnelshift_r(v[j], v[j + 1], (off & 2) * 8);
}
// Chunk i of a row of K elements, zeros past the row's end.  MIS: rows need not start on 16 bytes; the two aligned vectors that
// overlap the chunk are fetched (the second only where it holds elements of the row, so that no other 16 bytes than those that
// the row touches are read) and shifted together.  WHOLE: the caller knows that the chunk is complete.
template <typename T, bool MIS, bool WHOLE = false>
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
        if (off && (WHOLE || ((long long)(i + 1) * 16 - off) < (long long)K * (int)sizeof(T))) b = base[1];
        realign<T>(a, b, off, c.w);
    }
    const int have = K - i * VE;
    if (!WHOLE && have < VE) {
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
// Rows whose largest magnitude is too small for 127 / a to be a float divide in 64 bits.  PLAIN: the row is neither of those nor all
// zeros.
template <typename T, int VE, bool PLAIN>
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
    if (!PLAIN && s.exact) {
#pragma unroll
        for (int j = 0; j < VE; j++) q[j] = (uint32_t)(int)rint((double)x[j] * 127.0 / (double)s.a);
    }
#pragma unroll
    for (int j = 0; j < VE / 4; j++) out[j] = !PLAIN && s.zero ? 0u : __byte_perm(__byte_perm(q[4 * j], q[4 * j + 1], 0x0040), __byte_perm(q[4 * j + 2], q[4 * j + 3], 0x0040), 0x5410);
}
template <int VE, bool WHOLE>
__device__ __forceinline__ void store_chunk(int8_t* out, int i, int K, const uint32_t (&q)[VE / 4]) {
    int8_t* at = out + (long long)i * VE;
    const int have = K - i * VE;
    if (WHOLE || have >= VE) {
        if constexpr (VE == 8) *reinterpret_cast<uint2*>(at) = make_uint2(q[0], q[1]);
        else *reinterpret_cast<uint32_t*>(at) = q[0];
    } else {
#pragma unroll
        for (int j = 0; j < VE; j++)
            if (j < have) at[j] = (int8_t)(q[j >> 2] >> (8 * (j & 3)));
    }
}

template <typename T, bool WHOLE = false>
__device__ __forceinline__ void finish_chunk(const Chunk<T>& c, int8_t* out, int i, int K, const RowScale& s) {
    constexpr int VE = Chunk<T>::VE;
    float f[VE];
    uint32_t w[VE / 4];
    unpack(c, f);
    quantise_chunk<T, VE, WHOLE>(f, s, w);
    store_chunk<VE, WHOLE>(out, i, K, w);
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// GROUP threads a row (a warp, or the whole block), which keeps the row in registers between its largest magnitude and its
// integers, NV chunks a thread: every element is read once.  LONG: rows that do not fit; the chunks past the kept ones are read a
// second time.  The form for few rows (all latency) and for rows too long for the ring below.  (Groups that went on to another row and
// requested it ahead were slower, 51 against 33 us for 8192 x 4096 bf16: their registers cost more rows in flight than that gave.)
// The input may be what the launch in front is still writing: no __restrict__ on it and no __ldg in this file, which would promise that
// it does not change while the kernel runs.
template <typename T, int GROUP, int NV, bool MIS, bool LONG>
__global__ void __launch_bounds__(GROUP < 256 ? 256 : GROUP) quantise_i8_kernel(const T* x, long long x_stride, int8_t* __restrict__ q, long long q_stride,
                                                                              float* __restrict__ scale, int M, int K) {
    constexpr int VE = Chunk<T>::VE, ROWS = GROUP < 256 ? 256 / GROUP : 1;
    __shared__ uint32_t s_top[32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const long long m = (long long)blockIdx.x * ROWS + (ROWS > 1 ? threadIdx.x / GROUP : 0);
    const int lane = threadIdx.x % GROUP, chunks = K / VE + (K % VE != 0);
    if (m >= M) return;  // (a whole group, and with several a whole warp)
    const T* row = x + m * x_stride;
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
    int8_t* out = q + m * q_stride;
#pragma unroll
    for (int v = 0; v < NV; v++)
        if (lane + v * GROUP < chunks) finish_chunk(c[v], out, lane + v * GROUP, K, s);
    if (LONG)
        for (int i = lane + NV * GROUP; i < chunks; i += GROUP) finish_chunk(load_chunk<T, MIS>(row, i, K), out, i, K, s);
}

// Many rows: persistent blocks, RING_WARPS warps, each with rows of its own that the copy engine brings into its slots of shared
// memory (the aligned 16 bytes that the row touches), `slots` a warp, ahead of the warp's work: the bytes on their way do not
// depend on registers.  A warp goes over its row twice, for the largest magnitude and for the integers.  Bounded by memory for fp32 (8192 x
// 4096: 31 us = 5.4 TB/s, 0.82 of the measured copy; rows in registers 45), by instructions for 16-bit types (19.6 us = 5.1 TB/s;
// rows in registers 33) and short rows (20000 x 512 bf16: 12.4 us).
constexpr int RING_WARPS = 12, RING_MAX_SLOTS = 8, RING_BYTES = 200 * 1024;
template <typename T, bool MIS>
__global__ void __launch_bounds__(RING_WARPS * 32, 1) quantise_ring_kernel(const T* x, long long x_stride, int8_t* __restrict__ q, long long q_stride,
                                                                         float* __restrict__ scale, int M, int K, int slots, int slot_bytes, unsigned int* status) {
    extern __shared__ __align__(16) unsigned char s_ring[];
    __shared__ uint64_t s_bar[RING_WARPS * RING_MAX_SLOTS];
    __shared__ int s_abort;
    constexpr int VE = Chunk<T>::VE;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, chunks = K / VE + (K % VE != 0), whole = K / VE;
    const uint32_t bars = smem_u32(s_bar + warp * RING_MAX_SLOTS);
    unsigned char* ring = s_ring + (size_t)warp * slots * slot_bytes;
    if (threadIdx.x == 0) s_abort = 0;
    if (lane == 0) {
        for (int s = 0; s < slots; s++) mbar_init(bars + 8 * s, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const long long step = (long long)gridDim.x * RING_WARPS;
    auto request = [&](long long m, int s) {  // lane 0
        const uintptr_t from = (uintptr_t)(x + m * x_stride), lo = from & ~(uintptr_t)15, hi = (from + (size_t)K * sizeof(T) + 15) & ~(uintptr_t)15;
        mbar_arrive_expect_tx(bars + 8 * s, (uint32_t)(hi - lo));
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(ring + s * slot_bytes)), "l"(lo),
                     "r"((uint32_t)(hi - lo)), "r"(bars + 8 * s)
                     : "memory");
    };
    const long long m0 = (long long)blockIdx.x * RING_WARPS + warp;
    if (lane == 0)
        for (int s = 0; s < slots; s++)
            if (m0 + s * step < M) request(m0 + s * step, s);
    __syncwarp();
    int s = 0;
    uint32_t ph = 0;
    for (long long m = m0; m < M; m += step) {
        if (!__all_sync(0xFFFFFFFFu, mbar_wait(bars + 8 * s, ph, &s_abort, status, 13))) {
            // a wait gave up: give the copies already requested time to land before shared memory is released
            for (int i = 0; i < 1000; i++) __nanosleep(1000);
            break;
        }
        const T* row = reinterpret_cast<const T*>(ring + s * slot_bytes + (MIS ? (uintptr_t)(x + m * x_stride) & 15 : 0));
        uint32_t top = 0;
        // (whole chunks without the tests that the last one needs)
#pragma unroll 4
        for (int i = lane; i < whole; i += 32) top = widen_max(top, load_chunk<T, MIS, true>(row, i, K));
        if (whole < chunks && lane == 0) top = widen_max(top, load_chunk<T, MIS>(row, whole, K));
        const RowScale sc = row_scale(__reduce_max_sync(0xFFFFFFFFu, magnitude_bits<T>(top)), lane == 0 ? scale + m : nullptr);
        int8_t* out = q + m * q_stride;
        if (sc.zero || sc.exact) {
            for (int i = lane; i < chunks; i += 32) finish_chunk(load_chunk<T, MIS>(row, i, K), out, i, K, sc);
        } else {
#pragma unroll 4
            for (int i = lane; i < whole; i += 32) finish_chunk<T, true>(load_chunk<T, MIS, true>(row, i, K), out, i, K, sc);
            if (whole < chunks && lane == 0) finish_chunk(load_chunk<T, MIS>(row, whole, K), out, whole, K, sc);
        }
        __syncwarp();
        if (lane == 0 && m + slots * step < M) {
            fence_async();  // the warp's reads before the copy's writes
            request(m + slots * step, s);
        }
        if (++s == slots) { s = 0; ph ^= 1; }
    }
}

template <typename... Args>
int launch(void (*kern)(Args...), long long grid, int threads, size_t smem, cudaStream_t stream, Args... args) {
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
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

template <typename T, int GROUP, int NV, bool MIS, bool LONG = false>
int launch_rows(const T* x, long long x_stride, int8_t* q, long long q_stride, float* scale, int M, int K, cudaStream_t st) {
    constexpr int THREADS = GROUP < 256 ? 256 : GROUP, ROWS = THREADS / GROUP;
    return launch<const T*, long long, int8_t*, long long, float*, int, int>(quantise_i8_kernel<T, GROUP, NV, MIS, LONG>, ((long long)M + ROWS - 1) / ROWS, THREADS, 0, st, x,
                                                                             x_stride, q, q_stride, scale, M, K);
}
// Rows enough for every warp of the ring form to have two: that one, where its slots hold the row.  Else the fewest threads that hold a
// row in four chunks each; a few rows by themselves take more threads (the launch is all latency then).
template <typename T, bool MIS>
int launch_quantise(tnns_cuda_ctx* ctx, const T* x, long long x_stride, int8_t* q, long long q_stride, float* scale, int M, int K, cudaStream_t st) {
    const int chunks = K / Chunk<T>::VE + (K % Chunk<T>::VE != 0);  // (K may be any int)
    const bool many = M > ctx->sm_count;
    const long long slot = (((long long)K * sizeof(T) + 15) / 16 + 1) * 16;  // a row may touch one 16-byte vector more than its size
    if (M >= 2LL * RING_WARPS * ctx->sm_count && slot * RING_WARPS <= RING_BYTES) {
        auto kern = quantise_ring_kernel<T, MIS>;
        static bool set[64] = {false};  // the attribute belongs to (function, device)
        if (!set[ctx->device & 63]) {
            TNNS_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, RING_BYTES));
            set[ctx->device & 63] = true;
        }
        const int slots = (int)std::min<long long>(RING_MAX_SLOTS, RING_BYTES / (slot * RING_WARPS));
        return launch<const T*, long long, int8_t*, long long, float*, int, int, int, int, unsigned int*>(kern, ctx->sm_count, RING_WARPS * 32, (size_t)slots * RING_WARPS * slot, st, x,
                                                                                                          x_stride, q, q_stride, scale, M, K, slots, (int)slot, ctx->d_status);
    }
    if (chunks <= 32) return launch_rows<T, 32, 1, MIS>(x, x_stride, q, q_stride, scale, M, K, st);
    if (chunks <= 128 && many) return launch_rows<T, 32, 4, MIS>(x, x_stride, q, q_stride, scale, M, K, st);
    if (chunks <= 256) return launch_rows<T, 256, 1, MIS>(x, x_stride, q, q_stride, scale, M, K, st);
    if (chunks <= 1024 && many) return launch_rows<T, 256, 4, MIS>(x, x_stride, q, q_stride, scale, M, K, st);
    if (chunks <= 1024) return launch_rows<T, 1024, 1, MIS>(x, x_stride, q, q_stride, scale, M, K, st);
    if (chunks <= 4096) return launch_rows<T, 1024, 4, MIS>(x, x_stride, q, q_stride, scale, M, K, st);
    return launch_rows<T, 1024, 4, MIS, true>(x, x_stride, q, q_stride, scale, M, K, st);
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
    int places, top_k, T, N, out_dtype, per_row;  // per_row: chunks of VE columns
};
template <int VE>
__device__ __forceinline__ void store_sums(const CombineArgs& p, long long row, int c0, const float (&f)[VE]) {
    const bool whole = c0 >= 0 && c0 + VE <= p.N;
    if (p.out_dtype == TNNS_F32) {
        float* o = (float*)p.out + row + c0;
        if (whole) {
#pragma unroll
            for (int j = 0; j < VE; j += 4) *reinterpret_cast<float4*>(o + j) = make_float4(f[j], f[j + 1], f[j + 2], f[j + 3]);
        } else {
#pragma unroll
            for (int j = 0; j < VE; j++)
                if (c0 + j >= 0 && c0 + j < p.N) o[j] = f[j];
        }
        return;
    }
    uint16_t h[VE];
#pragma unroll
    for (int j = 0; j < VE; j++) {
        if (p.out_dtype == TNNS_F16) h[j] = __half_as_ushort(__float2half_rn(f[j]));
        else h[j] = __bfloat16_as_ushort(__float2bfloat16_rn(f[j]));
    }
    uint16_t* o = (uint16_t*)p.out + row + c0;
    if (whole) {
        uint32_t w[VE / 2];
#pragma unroll
        for (int j = 0; j < VE / 2; j++) w[j] = h[2 * j] | (uint32_t)h[2 * j + 1] << 16;
        if constexpr (VE == 8) *reinterpret_cast<uint4*>(o) = make_uint4(w[0], w[1], w[2], w[3]);
        else *reinterpret_cast<uint2*>(o) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
        for (int j = 0; j < VE; j++)
            if (c0 + j >= 0 && c0 + j < p.N) o[j] = h[j];
    }
}

// One thread a chunk of VE neighbouring columns (16 bytes of y) of a token, the rows of eight slots on their way at once.  Bounded by
// memory: every row of y is read once (8192 tokens of 8 x 2048 bf16: 50 us = 6.1 TB/s, 0.93 of the measured copy; fp32 92 us = 6.6; rows of 2047: 95 us).  MIS: rows need not start on 16 bytes; the first chunk of a row begins where its results are
// aligned (at a column up to VE - 1 below 0), and y is fetched as the aligned vectors that hold the chunk.
template <typename T, bool MIS>
__global__ void __launch_bounds__(256) combine_kernel(CombineArgs p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    constexpr int U = 8, VE = Chunk<T>::VE;
    const long long item = (long long)blockIdx.x * 256 + threadIdx.x;
    if (item >= (long long)p.T * p.per_row) return;
    const int t = item < 0xFFFFFFFFLL ? (int)((uint32_t)item / (uint32_t)p.per_row) : (int)(item / p.per_row);
    const long long out_row = (long long)t * p.out_stride;
    int c0 = (int)(item - (long long)t * p.per_row) * VE;
    if (MIS) {
        const uintptr_t elements = ((uintptr_t)p.out >> (p.out_dtype == TNNS_F32 ? 2 : 1)) + (uintptr_t)out_row;
        c0 -= (int)(elements % VE);
        if (c0 >= p.N) return;
    }
    const int32_t* slots = p.slots + (long long)t * p.top_k;
    const float* weights = p.weights + (long long)t * p.top_k;
    float sum[VE] = {};
    for (int j0 = 0; j0 < p.top_k; j0 += U) {
        int at[U];
        float w[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            at[u] = j0 + u < p.top_k ? slots[j0 + u] : -1;
            w[u] = j0 + u < p.top_k ? weights[j0 + u] : 0.f;
        }
        uint4 a[U], b[MIS ? U : 1];
#pragma unroll
        for (int u = 0; u < U; u++) {
            a[u] = make_uint4(0, 0, 0, 0);
            if (MIS) b[u] = make_uint4(0, 0, 0, 0);
            if (at[u] >= 0 && at[u] < p.places) {
                const T* row = (const T*)p.y + (long long)at[u] * p.y_stride;
                if (!MIS) a[u] = *reinterpret_cast<const uint4*>(row + c0);
                else {
                    // of the two aligned vectors those that hold elements of the row
                    const uintptr_t from = (uintptr_t)(row + c0), lo = from & ~(uintptr_t)15;
                    if (lo + 16 > (uintptr_t)row) a[u] = *reinterpret_cast<const uint4*>(lo);
                    if (from != lo && lo + 16 < (uintptr_t)(row + min(c0 + VE, p.N))) b[u] = *reinterpret_cast<const uint4*>(lo + 16);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (at[u] >= 0 && at[u] < p.places) {
                Chunk<T> c;
                float f[VE];
                if (MIS) realign<T>(a[u], b[u], (int)((uintptr_t)((const T*)p.y + (long long)at[u] * p.y_stride + c0) & 15), c.w);
                else { c.w[0] = a[u].x; c.w[1] = a[u].y; c.w[2] = a[u].z; c.w[3] = a[u].w; }
                unpack(c, f);
#pragma unroll
                for (int j = 0; j < VE; j++) sum[j] = fmaf(w[u], f[j], sum[j]);
            }
    }
    store_sums<VE>(p, out_row, c0, sum);
}

template <typename T>
int launch_combine(CombineArgs a, cudaStream_t st) {
    constexpr int VE = Chunk<T>::VE;
    const int bo = tnns_dtype_bytes(a.out_dtype);
    const bool mis = a.N % VE || ((uintptr_t)a.y | (uintptr_t)(a.y_stride * (long long)sizeof(T))) % 16 || ((uintptr_t)a.out | (uintptr_t)(a.out_stride * bo)) % (VE * bo);
    a.per_row = mis ? (int)(((long long)a.N + 2 * VE - 2) / VE) : a.N / VE;
    const long long blocks = ((long long)a.T * a.per_row + 255) / 256;
    if (blocks > 0x7FFFFFFFLL || a.N > 0x7FFFFF00) return tnns_fail(TNNS_ERR_UNSUPPORTED, "%d tokens of %d columns", a.T, a.N);
    if (mis) return launch<CombineArgs>(combine_kernel<T, true>, blocks, 256, 0, st, a);
    return launch<CombineArgs>(combine_kernel<T, false>, blocks, 256, 0, st, a);
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
    a.per_row = 0;
    const cudaStream_t st = (cudaStream_t)stream;
    TNNS_FOR_DTYPE(dtype, TI, return launch_combine<TI>(a, st));
}

}  // extern "C"
