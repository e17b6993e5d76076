// Routing of tokens to experts: scores, the choice of the best by key, weights, and the pairs (token, slot) in the order
// of their experts.
#include <math.h>

#include "dtype.cuh"
#include "internal.h"

namespace {

struct RouteArgs {
    const void* logits;
    long long stride;
    const float* bias;
    int32_t* experts;
    float* weights;
    int T, E, top_k, sigmoid, groups, group_size, top_groups, group_top, renormalise;
    float scale;
};

// A logit or a bias that bars its expert: -inf and NaN.  +inf counts as the largest finite float.
__device__ __forceinline__ bool barred(float v) { return !(v > -INFINITY); }
__device__ __forceinline__ float bounded(float v) { return fminf(v, 3.402823466e38f); }

constexpr int MAX_E = 1024;

// One warp a token, everything in 64 bits, keys in shared memory.
template <typename T>
__global__ void __launch_bounds__(32) route_kernel(RouteArgs p) {
    __shared__ double s_key[MAX_E];    // -inf: not to be chosen (any more)
    __shared__ double s_score[MAX_E];
    __shared__ double s_worth[32];
    const int lane = threadIdx.x;
    for (int t = blockIdx.x; t < p.T; t += gridDim.x) {
        const T* row = (const T*)p.logits + (long long)t * p.stride;
        double top = -INFINITY;
        for (int e = lane; e < p.E; e += 32) {
            const float l = to_f32(row[e]);
            s_score[e] = barred(l) ? -INFINITY : (double)bounded(l);
            top = fmax(top, s_score[e]);
        }
        for (int d = 16; d; d >>= 1) top = fmax(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
        double sum = 0;
        for (int e = lane; e < p.E; e += 32) {
            const double l = s_score[e];
            const double s = l == -INFINITY ? 0.0 : p.sigmoid ? 1.0 / (1.0 + exp(-l)) : exp(l - top);
            sum += s;
            s_score[e] = s;
            s_key[e] = l;
        }
        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
        __syncwarp();
        for (int e = lane; e < p.E; e += 32) {
            if (!p.sigmoid && sum > 0) s_score[e] /= sum;
            if (p.bias) {
                const float b = p.bias[e];
                s_key[e] = s_key[e] == -INFINITY || barred(b) ? -INFINITY : s_score[e] + (double)bounded(b);
            }
        }
        __syncwarp();
        if (p.top_groups < p.groups) {
            if (lane < p.groups) {
                double a = -INFINITY, b = -INFINITY;  // the two best
                for (int i = 0; i < p.group_size; i++) {
                    const int e = lane * p.group_size + i;
                    if (s_key[e] == -INFINITY) continue;
                    const double v = p.group_top == 2 && !p.bias ? s_score[e] : s_key[e];
                    if (v > a) { b = a; a = v; } else b = fmax(b, v);
                }
                s_worth[lane] = p.group_top == 2 && b != -INFINITY ? a + b : a;
            }
            __syncwarp();
            bool kept = false;
            if (lane < p.groups) {
                int better = 0;
                for (int g = 0; g < p.groups; g++) better += s_worth[g] > s_worth[lane] || (s_worth[g] == s_worth[lane] && g < lane);
                kept = better < p.top_groups;
            }
            const unsigned keep = __ballot_sync(0xFFFFFFFFu, kept);
            for (int e = lane; e < p.E; e += 32)
                if (!((keep >> (e / p.group_size)) & 1)) s_key[e] = -INFINITY;
            __syncwarp();
        }
        double total = 0, mine = 0;
        int my_e = -1;
        for (int j = 0; j < p.top_k; j++) {
            double best = -INFINITY;
            int at = MAX_E;
            for (int e = lane; e < p.E; e += 32)
                if (s_key[e] > best) { best = s_key[e]; at = e; }
            for (int d = 16; d; d >>= 1) {
                const double o = __shfl_xor_sync(0xFFFFFFFFu, best, d);
                const int oe = __shfl_xor_sync(0xFFFFFFFFu, at, d);
                if (o > best || (o == best && oe < at)) { best = o; at = oe; }
            }
            const bool found = best != -INFINITY;
            const double s = found ? s_score[at] : 0;
            total += s;
            if (lane == j) { mine = s; my_e = found ? at : -1; }
            __syncwarp();
            if (found && lane == 0) s_key[at] = -INFINITY;
            __syncwarp();
        }
        if (lane < p.top_k) {
            p.experts[(long long)t * p.top_k + lane] = my_e;
            p.weights[(long long)t * p.top_k + lane] = (float)(p.scale * (p.renormalise ? mine / (total + 1e-20) : mine));
        }
        __syncwarp();
    }
}

constexpr int PLAN_THREADS = 1024;

// One block an expert (and one more for the places behind the last pair): counts the pairs of the experts before it, then
// gives its own pairs their places in order.
__global__ void __launch_bounds__(PLAN_THREADS) plan_kernel(const int32_t* __restrict__ experts, int pairs, int top_k, int E, int32_t* __restrict__ offsets,
                                                            int32_t* __restrict__ rows, int32_t* __restrict__ slots) {
    __shared__ int s_count[PLAN_THREADS / 32];
    __shared__ int s_base;
    const int e = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int before = 0;
    for (int i = tid; i < pairs; i += PLAN_THREADS) {
        const int v = experts[i];
        before += v >= 0 && v < e;
    }
    before = __reduce_add_sync(0xFFFFFFFFu, before);
    if (lane == 0) s_count[warp] = before;
    __syncthreads();
    if (tid == 0) {
        int b = 0;
        for (int i = 0; i < PLAN_THREADS / 32; i++) b += s_count[i];
        s_base = b;
        offsets[e] = b;
    }
    __syncthreads();
    int base = s_base;
    if (e == E) {
        for (int i = base + tid; i < pairs; i += PLAN_THREADS) rows[i] = -1;
        for (int i = tid; i < pairs; i += PLAN_THREADS)
            if (experts[i] < 0) slots[i] = -1;
        return;
    }
    for (int i0 = 0; i0 < pairs; i0 += PLAN_THREADS) {
        const int i = i0 + tid;
        const bool mine = i < pairs && experts[i] == e;
        const unsigned m = __ballot_sync(0xFFFFFFFFu, mine);
        __syncthreads();
        if (lane == 0) s_count[warp] = __popc(m);
        __syncthreads();
        int at = base + __popc(m & ((1u << lane) - 1));
        for (int w = 0; w < warp; w++) at += s_count[w];
        for (int w = 0; w < PLAN_THREADS / 32; w++) base += s_count[w];
        if (mine) {
            rows[at] = i / top_k;
            slots[i] = at;
        }
    }
}

int check_route(const tnns_route_t* r) {
    if (!r) return tnns_fail(TNNS_ERR_INVALID, "route is NULL");
    if (r->experts < 1 || r->experts > MAX_E) return tnns_fail(TNNS_ERR_INVALID, "%d experts (1 .. %d)", r->experts, MAX_E);
    if (r->groups < 1 || r->groups > 32 || r->experts % r->groups) return tnns_fail(TNNS_ERR_INVALID, "%d experts in %d groups", r->experts, r->groups);
    if (r->top_groups < 1 || r->top_groups > r->groups) return tnns_fail(TNNS_ERR_INVALID, "%d of %d groups", r->top_groups, r->groups);
    if (r->top_k < 1 || r->top_k > 32 || r->top_k > r->top_groups * (r->experts / r->groups))
        return tnns_fail(TNNS_ERR_INVALID, "top_k %d of %d groups of %d experts (at most 32)", r->top_k, r->top_groups, r->experts / r->groups);
    if (r->score != TNNS_ROUTE_SOFTMAX && r->score != TNNS_ROUTE_SIGMOID) return tnns_fail(TNNS_ERR_INVALID, "unknown score %d", r->score);
    if (r->group_top != 1 && r->group_top != 2) return tnns_fail(TNNS_ERR_INVALID, "a group's worth is made of 1 or 2 values, not %d", r->group_top);
    return TNNS_OK;
}

}  // namespace

extern "C" {

size_t tnns_route_workspace_bytes(const tnns_route_t* r, int T) {
    (void)T;
    if (check_route(r)) return 0;
    return 0;
}

int tnns_cuda_route(tnns_cuda_ctx* ctx, const tnns_route_t* r, const void* d_logits, int dtype, long long stride, const float* d_bias, int T,
                    int32_t* d_experts, float* d_weights, int32_t* d_offsets, int32_t* d_rows, int32_t* d_slots, void* d_workspace,
                    size_t workspace_bytes, void* stream) {
    if (!ctx) return tnns_fail(TNNS_ERR_INVALID, "ctx is NULL");
    int rc = check_route(r);
    if (rc) return rc;
    if (!tnns_dtype_ok(dtype)) return tnns_fail(TNNS_ERR_INVALID, "unknown element type %d", dtype);
    if (T < 0 || (long long)T * r->top_k > 0x7FFFFFFFLL) return tnns_fail(TNNS_ERR_INVALID, "bad size: %d tokens, top_k %d", T, r->top_k);
    if (stride < r->experts) return tnns_fail(TNNS_ERR_INVALID, "rows of %d logits at a stride of %lld", r->experts, stride);
    const bool plan = d_offsets || d_rows || d_slots;
    if (plan && !d_offsets) return tnns_fail(TNNS_ERR_INVALID, "the order of the pairs needs offsets, rows and slots");
    if (T && (!d_logits || !d_experts || !d_weights)) return tnns_fail(TNNS_ERR_INVALID, "NULL argument");
    if (plan && T && (!d_rows || !d_slots)) return tnns_fail(TNNS_ERR_INVALID, "the order of the pairs needs offsets, rows and slots");
    if ((uintptr_t)d_logits % tnns_dtype_bytes(dtype) || ((uintptr_t)d_bias | (uintptr_t)d_experts | (uintptr_t)d_weights | (uintptr_t)d_offsets | (uintptr_t)d_rows | (uintptr_t)d_slots) % 4)
        return tnns_fail(TNNS_ERR_INVALID, "unaligned pointer");
    (void)d_workspace;
    (void)workspace_bytes;
    if ((rc = tnns_enter(ctx))) return rc;
    RouteArgs a;
    a.logits = d_logits; a.stride = stride; a.bias = d_bias; a.experts = d_experts; a.weights = d_weights;
    a.T = T; a.E = r->experts; a.top_k = r->top_k; a.sigmoid = r->score == TNNS_ROUTE_SIGMOID;
    a.groups = r->groups; a.group_size = r->experts / r->groups; a.top_groups = r->top_groups; a.group_top = r->group_top;
    a.renormalise = r->renormalise; a.scale = r->scale;
    if (T) {
        const int grid = T < 32 * ctx->sm_count ? T : 32 * ctx->sm_count;
        TNNS_FOR_DTYPE(dtype, TI, (route_kernel<TI><<<grid, 32, 0, (cudaStream_t)stream>>>(a)));
        tnns_count_launch();
        TNNS_CUDA_TRY(cudaGetLastError());
    }
    if (plan) {
        plan_kernel<<<r->experts + 1, PLAN_THREADS, 0, (cudaStream_t)stream>>>(d_experts, T * r->top_k, r->top_k, r->experts, d_offsets, d_rows, d_slots);
        tnns_count_launch();
        TNNS_CUDA_TRY(cudaGetLastError());
    }
    return TNNS_OK;
}

}  // extern "C"
