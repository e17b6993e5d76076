// Products of quantised rows with 8-bit weights: y = PReLU(row scale * channel scale * sum q w), dense and over the places of
// every expert.
#include <algorithm>
#include <new>

#include "dtype.cuh"
#include "internal.h"

// Weights as the kernels read them: tiles of 128 channels x 128 elements of K, 16 KB each, [expert][channel tile][K tile], zeros
// past N and K.  Within a tile a channel's 128 bytes lie in the 128-byte swizzle pattern (of its eight 16-byte pieces, piece c
// sits at c ^ (channel % 8)): what the tensor core reads from shared memory, so that a tile is one contiguous copy.
struct tnns_cuda_weights_i8 {
    int experts, N, K, device;
    int n_tiles, k_tiles;
    int8_t* d_img;
    float* d_scale;  // [expert][n_tiles * 128], zeros past N
};

namespace {

constexpr int WT = 128, WT_BYTES = WT * WT;

__global__ void __launch_bounds__(256) tile_weights_kernel(const int8_t* __restrict__ w, int8_t* __restrict__ img, int N, int K, int n_tiles, int k_tiles,
                                                           long long pieces) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < pieces; i += (long long)gridDim.x * 256) {
        const int c = (int)(i & 7), r = (int)((i >> 3) & 127);  // 16-byte piece of a channel of a tile
        const long long tile = i >> 10;
        const int kt = (int)(tile % k_tiles);
        const long long et = tile / k_tiles;
        const int n = (int)(et % n_tiles) * WT + r, k0 = kt * WT + c * 16;
        const long long e = et / n_tiles;
        union { int8_t b[16]; uint4 v; } u;
        for (int j = 0; j < 16; j++) u.b[j] = n < N && k0 + j < K ? w[(e * N + n) * K + k0 + j] : (int8_t)0;
        *reinterpret_cast<uint4*>(img + tile * WT_BYTES + r * 128 + ((c ^ (r & 7)) << 4)) = u.v;
    }
}

struct GemmI8Args {
    const int8_t* img;
    const float* w_scale;
    const int8_t* q;
    long long q_stride;
    const float* scale;
    const int32_t* rows;     // NULL: place p is row p
    const int32_t* offsets;  // NULL: one expert, all places
    void* y;
    long long y_stride;
    int q_rows, places, experts, N, K, n_tiles, k_tiles;
    float alpha;
};

constexpr int SB = 64;  // places and channels of a block

// 64 places x 64 channels a block, 16 x 16 threads of 4 x 4 outputs, four products an instruction on the integer pipe.
template <typename T>
__global__ void __launch_bounds__(256) gemm_i8_simple_kernel(GemmI8Args p) {
    __shared__ uint32_t s_q[SB][33], s_w[SB][33];
    const int e = blockIdx.z, tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    int first = 0, last = p.places;
    if (p.offsets) {
        first = min(max(p.offsets[e], 0), p.places);
        last = min(max(p.offsets[e + 1], first), p.places);
    }
    const int n0 = blockIdx.y * SB;
    for (int m0 = first + blockIdx.x * SB; m0 < last; m0 += gridDim.x * SB) {
        int acc[4][4] = {};
        for (int kt = 0; kt < p.k_tiles; kt++) {
            __syncthreads();
            for (int i = tid; i < SB * 32; i += 256) {
                const int r = i >> 5, c = i & 31, k = kt * WT + c * 4;
                const int place = m0 + r;
                int row = place < last ? (p.rows ? p.rows[place] : place) : -1;
                if (row >= p.q_rows) row = -1;
                uint32_t v = 0;
                if (row >= 0)
                    for (int j = 0; j < 4; j++)
                        if (k + j < p.K) v |= (uint32_t)(uint8_t)p.q[(long long)row * p.q_stride + k + j] << (8 * j);
                s_q[r][c] = v;
                const int n = n0 + r;
                const int8_t* tile = p.img + (((long long)e * p.n_tiles + n / WT) * p.k_tiles + kt) * WT_BYTES;
                s_w[r][c] = *reinterpret_cast<const uint32_t*>(tile + (n % WT) * 128 + (((c >> 2) ^ (n & 7)) << 4) + (c & 3) * 4);
            }
            __syncthreads();
            for (int c = 0; c < 32; c++)
                for (int i = 0; i < 4; i++)
                    for (int j = 0; j < 4; j++) acc[i][j] = __dp4a((int)s_q[ty + 16 * i][c], (int)s_w[tx + 16 * j][c], acc[i][j]);
        }
        for (int i = 0; i < 4; i++) {
            const int place = m0 + ty + 16 * i;
            if (place >= last) continue;
            const int row = p.rows ? p.rows[place] : place;
            const float s = row >= 0 && row < p.q_rows ? p.scale[row] : 0.f;
            for (int j = 0; j < 4; j++) {
                const int n = n0 + tx + 16 * j;
                if (n >= p.N) continue;
                const float v = (float)acc[i][j] * s * p.w_scale[(long long)e * p.n_tiles * WT + n];
                ((T*)p.y)[(long long)place * p.y_stride + n] = from_f32<T>(v > 0 ? v : v * p.alpha);
            }
        }
    }
}

int run_product(tnns_cuda_ctx* ctx, const tnns_cuda_weights_i8* w, const int8_t* d_q, long long q_stride, const float* d_scale, int q_rows,
                const int32_t* d_rows, const int32_t* d_offsets, void* d_y, int dtype, long long y_stride, int places, float alpha, void* stream) {
    if (!tnns_dtype_ok(dtype)) return tnns_fail(TNNS_ERR_INVALID, "unknown element type %d", dtype);
    if (places < 0 || q_rows < 0) return tnns_fail(TNNS_ERR_INVALID, "bad size: %d places, %d rows", places, q_rows);
    if (q_stride < w->K || q_stride % 16 || y_stride < w->N)
        return tnns_fail(TNNS_ERR_INVALID, "rows of %d bytes at a stride of %lld (a multiple of 16), results of %d at %lld", w->K, q_stride, w->N, y_stride);
    if (places == 0) return TNNS_OK;
    if (!d_y || (q_rows && (!d_q || !d_scale))) return tnns_fail(TNNS_ERR_INVALID, "NULL argument");
    if ((uintptr_t)d_q % 16 || (uintptr_t)d_y % tnns_dtype_bytes(dtype) || ((uintptr_t)d_scale | (uintptr_t)d_rows | (uintptr_t)d_offsets) % 4)
        return tnns_fail(TNNS_ERR_INVALID, "unaligned pointer");
    const int rc = tnns_enter(ctx);
    if (rc) return rc;
    if (w->device != ctx->device) return tnns_fail(TNNS_ERR_INVALID, "weights live on device %d, context on %d", w->device, ctx->device);
    GemmI8Args a;
    a.img = w->d_img; a.w_scale = w->d_scale; a.q = d_q; a.q_stride = q_stride; a.scale = d_scale; a.rows = d_rows; a.offsets = d_offsets;
    a.y = d_y; a.y_stride = y_stride; a.q_rows = q_rows; a.places = places; a.experts = w->experts; a.N = w->N; a.K = w->K;
    a.n_tiles = w->n_tiles; a.k_tiles = w->k_tiles; a.alpha = alpha;
    const dim3 grid(std::min((places + SB - 1) / SB, d_offsets ? 64 : 65535), (w->N + SB - 1) / SB, w->experts);
    if (grid.y > 65535u || grid.z > 65535u) return tnns_fail(TNNS_ERR_UNSUPPORTED, "%d channels, %d experts", w->N, w->experts);
    TNNS_FOR_DTYPE(dtype, T, (gemm_i8_simple_kernel<T><<<grid, 256, 0, (cudaStream_t)stream>>>(a)));
    tnns_count_launch();
    TNNS_CUDA_TRY(cudaGetLastError());
    return TNNS_OK;
}

}  // namespace

extern "C" {

int tnns_cuda_upload_weights_i8(tnns_cuda_ctx* ctx, const int8_t* w, const float* scales, int experts, int N, int K,
                                tnns_cuda_weights_i8** out) {
    if (!ctx || !w || !scales || !out) return tnns_fail(TNNS_ERR_INVALID, "NULL argument");
    *out = nullptr;
    if (experts < 1 || experts > 65535 || N < 1 || K < 1 || K > 131071) return tnns_fail(TNNS_ERR_INVALID, "bad weight size: %d kernels of %d x %d (K at most 131071)", experts, N, K);
    int rc = tnns_enter(ctx);
    if (rc) return rc;
    tnns_cuda_weights_i8* h = new (std::nothrow) tnns_cuda_weights_i8();
    if (!h) return tnns_fail(TNNS_ERR_NOMEM, "host allocation failed");
    h->experts = experts; h->N = N; h->K = K; h->device = ctx->device;
    h->n_tiles = N / WT + (N % WT != 0); h->k_tiles = (K + WT - 1) / WT;
    h->d_img = nullptr; h->d_scale = nullptr;
    // a few experts at a time pass through a buffer, so that the transient memory stays below that of the weights themselves
    const size_t one = (size_t)N * K, tile_bytes = (size_t)h->n_tiles * h->k_tiles * WT_BYTES;
    const int step = (int)std::min<size_t>(experts, std::max<size_t>(1, (256u << 20) / one));
    int8_t* tmp = nullptr;
    cudaError_t e = cudaDeviceSynchronize();  // weights in device memory may still be on their way
    if (e == cudaSuccess) e = cudaMalloc(&h->d_img, tile_bytes * experts);
    if (e == cudaSuccess) e = cudaMalloc(&h->d_scale, (size_t)experts * h->n_tiles * WT * sizeof(float));
    if (e == cudaSuccess) e = cudaMalloc(&tmp, one * step);
    if (e == cudaSuccess) e = cudaMemset(h->d_scale, 0, (size_t)experts * h->n_tiles * WT * sizeof(float));
    if (e == cudaSuccess) e = cudaMemcpy2D(h->d_scale, (size_t)h->n_tiles * WT * sizeof(float), scales, (size_t)N * sizeof(float), (size_t)N * sizeof(float), experts, cudaMemcpyDefault);
    for (int i = 0; i < experts && e == cudaSuccess; i += step) {
        const int n = std::min(step, experts - i);
        e = cudaMemcpy(tmp, w + one * i, one * n, cudaMemcpyDefault);
        if (e != cudaSuccess) break;
        const long long pieces = (long long)n * h->n_tiles * h->k_tiles * (WT_BYTES / 16);
        tile_weights_kernel<<<(int)std::min<long long>((pieces + 255) / 256, 32LL * ctx->sm_count), 256>>>(tmp, h->d_img + tile_bytes * i, N, K, h->n_tiles, h->k_tiles, pieces);
        tnns_count_launch();
        e = cudaGetLastError();
    }
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
    if (tmp) cudaFree(tmp);
    if (e != cudaSuccess) {
        tnns_cuda_free_weights_i8(ctx, h);
        return tnns_fail(e == cudaErrorMemoryAllocation ? TNNS_ERR_NOMEM : TNNS_ERR_CUDA, "weight upload failed: %s", cudaGetErrorString(e));
    }
    *out = h;
    return TNNS_OK;
}

void tnns_cuda_free_weights_i8(tnns_cuda_ctx* ctx, tnns_cuda_weights_i8* w) {
    if (!w) return;
    if (ctx) cudaSetDevice(ctx->device);
    if (w->d_img) cudaFree(w->d_img);
    if (w->d_scale) cudaFree(w->d_scale);
    delete w;
}

int tnns_cuda_gemm_i8(tnns_cuda_ctx* ctx, const tnns_cuda_weights_i8* w, const int8_t* d_q, long long q_stride, const float* d_scale,
                      void* d_y, int dtype, long long y_stride, int M, float alpha, void* stream) {
    if (!ctx || !w) return tnns_fail(TNNS_ERR_INVALID, "NULL argument");
    if (w->experts != 1) return tnns_fail(TNNS_ERR_INVALID, "weights of %d experts need tnns_cuda_gemm_i8_experts", w->experts);
    return run_product(ctx, w, d_q, q_stride, d_scale, M, nullptr, nullptr, d_y, dtype, y_stride, M, alpha, stream);
}

int tnns_cuda_gemm_i8_experts(tnns_cuda_ctx* ctx, const tnns_cuda_weights_i8* w, const int8_t* d_q, long long q_stride, const float* d_scale,
                              int q_rows, const int32_t* d_rows, const int32_t* d_offsets, void* d_y, int dtype, long long y_stride, int places,
                              float alpha, void* stream) {
    if (!ctx || !w) return tnns_fail(TNNS_ERR_INVALID, "NULL argument");
    if (places && !d_offsets) return tnns_fail(TNNS_ERR_INVALID, "NULL argument");
    return run_product(ctx, w, d_q, q_stride, d_scale, q_rows, d_rows, d_offsets, d_y, dtype, y_stride, places, alpha, stream);
}

}  // extern "C"
