// Routing of tokens to experts: scores, the choice of the best by key, weights, and the pairs (token, slot) in the order
// of their experts.
#include <math.h>

#include <algorithm>

#include "dtype.cuh"
#include "internal.h"
#include "mbar.cuh"

namespace {

struct RouteArgs {
    const void* logits;
    long long stride;
    const float* bias;
    int32_t* experts;
    float* weights;
    int T, E, top_k, sigmoid, groups, group_size, top_groups, group_top, renormalise, glog;
    float scale;
};

// A logit or a bias that bars its expert: -inf and NaN.  +inf counts as the largest finite float.
__device__ __forceinline__ bool barred(float v) { return !(v > -INFINITY); }
__device__ __forceinline__ float bounded(float v) { return fminf(v, 3.402823466e38f); }

constexpr int MAX_E = 1024;
constexpr unsigned FULL = 0xFFFFFFFFu;

struct Choice {
    int mine;       // lane j: the expert of slot j, -1: none
    float top;      // softmax: the largest logit, and the sum of exp(logit - top)
    float sum;
    bool certain;   // false: keys lie closer together than their rounding; nothing else is valid then
};

// A group's experts lie on the 32 / 2^glog lanes of the group, up to NPL a lane: register r holds expert group * group_size +
// r * L + (lane % L).  Without groups that is lane + 32 * r.
struct Lanes {
    int L, group, e0;  // lanes of a group, this lane's group, its first expert
    __device__ __forceinline__ Lanes(const RouteArgs& p, int lane, int glog) : L(32 >> glog), group(lane >> (5 - glog)), e0(group * p.group_size + (lane & (L - 1))) {}
    __device__ __forceinline__ bool there(const RouteArgs& p, int r) const { return group < p.groups && r * L + (e0 - group * p.group_size) < p.group_size; }
};

// A score in fp32 by the fast exponential and quotient, or in 64 bits.
__device__ __forceinline__ float score_of(const RouteArgs& p, float l, float top, float all) {
    return p.sigmoid ? __fdividef(1.0f, 1.0f + __expf(-l)) : __fdividef(__expf(l - top), all);
}
__device__ __forceinline__ double score_of(const RouteArgs& p, double l, double top, double all) {
    return p.sigmoid ? 1.0 / (1.0 + exp(-l)) : exp(l - top) / all;
}
__device__ __forceinline__ float warp_max(float v) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ double warp_max(double v) {
    for (int d = 16; d; d >>= 1) v = fmax(v, __shfl_xor_sync(FULL, v, d));
    return v;
}
// The two best values of a group, (a, b) being those of its lanes, and whether the group is among the best: groups ranked by a, or by
// a + b.  Returns the group's worth.
template <typename Key>
__device__ __forceinline__ Key rank_group(const RouteArgs& p, const Lanes& at, int glog, Key a, Key b, bool& kept) {
    for (int d = 1; d < at.L; d <<= 1) {
        const Key oa = __shfl_xor_sync(FULL, a, d), ob = __shfl_xor_sync(FULL, b, d);
        b = fmax(fmin(a, oa), fmax(b, ob));
        a = fmax(a, oa);
    }
    const Key none = -INFINITY, worth = p.group_top == 2 && b != none ? a + b : a;
    int better = 0;
    for (int g = 0; g < p.groups; g++) {
        const Key o = __shfl_sync(FULL, worth, g << (5 - glog));
        better += o > worth || (o == worth && g < at.group);
    }
    kept = at.group < p.groups && better < p.top_groups;
    return worth;
}

// The choice in 64 bits.
template <typename T, int NPL>
__device__ __noinline__ int choose_exact(const RouteArgs& p, const T* row, int lane, int glog) {
    const Lanes at(p, lane, glog);
    const double none = -INFINITY;
    double key[NPL];
    double top = none;
#pragma unroll
    for (int r = 0; r < NPL; r++) {
        const float l = at.there(p, r) ? to_f32(row[at.e0 + r * at.L]) : -INFINITY;
        key[r] = barred(l) ? none : (double)bounded(l);
        top = fmax(top, key[r]);
    }
    top = warp_max(top);
    double all = 0;
    if (!p.sigmoid && top > none) {
#pragma unroll 1
        for (int r = 0; r < NPL; r++)  // (from memory again: a register array cannot be indexed)
            if (at.there(p, r)) {
                const float l = to_f32(row[at.e0 + r * at.L]);
                if (!barred(l)) all += exp((double)bounded(l) - top);
            }
        for (int d = 16; d; d >>= 1) all += __shfl_xor_sync(FULL, all, d);
    }
    const bool grouped = p.top_groups < p.groups;
    double a = none, b = none;
#pragma unroll
    for (int r = 0; r < NPL; r++) {
        double v = key[r];
        if (v != none && (p.bias || (grouped && p.group_top == 2))) {
            v = score_of(p, v, top, all);
            if (p.bias) {
                const float c = __ldg(p.bias + at.e0 + r * at.L);
                key[r] = v = barred(c) ? none : v + (double)bounded(c);
            }
        }
        b = fmax(b, fmin(a, v));
        a = fmax(a, v);
    }
    if (grouped) {
        bool kept;
        rank_group<double>(p, at, glog, a, b, kept);
        if (!kept) {
#pragma unroll
            for (int r = 0; r < NPL; r++) key[r] = none;
        }
    }
    int mine = -1;
    for (int j = 0; j < p.top_k; j++) {
        double best = none;
        int e = MAX_E;
#pragma unroll
        for (int r = 0; r < NPL; r++)
            if (key[r] > best) { best = key[r]; e = at.e0 + r * at.L; }
        const double m = warp_max(best);
        if (m == none) break;
        e = (int)__reduce_min_sync(FULL, best == m ? (unsigned)e : (unsigned)MAX_E);
        if (lane == j) mine = e;
#pragma unroll
        for (int r = 0; r < NPL; r++)
            if (at.e0 + r * at.L == e) key[r] = none;
    }
    return mine;
}

// The choice for one token by one warp, in fp32.  Every lane sorts its keys, and the warp takes the best of the lanes' first ones,
// top_k times.  A key carries its register's number in its lowest bits (LOG of them), lower registers above higher ones.
//
// The choice is certain unless two keys that have to be told apart are closer than their errors; the token is then chosen in 64
// bits.  A score by the fast functions is off by 2^-22 from the exponential and by the rounding of its argument, of which a score (at
// most 1, and s * d <= 1 / e) keeps 2^-22 together; a softmax's sum adds NPL + 5 roundings of 2^-24, the quotient 2^-22, the bias
// |key| * 2^-24.  A key without a bias is the logit itself.  The register's number takes LOG bits.  Two keys are in order if they
// differ by (NPL + 24) * 2^-23 + |key| * 2^(LOG - 21) (first term: with a bias), or if they are made of the same logit and the same
// bias and come in their experts' order.
template <typename T, int NPL>
__device__ __forceinline__ Choice choose(const RouteArgs& p, const T* row, int lane, int glog) {
    constexpr int LOG = NPL == 2 ? 1 : NPL == 4 ? 2 : NPL == 8 ? 3 : NPL == 16 ? 4 : NPL == 32 ? 5 : 6;
    const Lanes at(p, lane, glog);
    Choice c;
    float key[NPL];
    float top = -INFINITY;
#pragma unroll
    for (int r = 0; r < NPL; r++) {
        float l = -INFINITY;
        if (at.there(p, r)) l = to_f32(row[at.e0 + r * at.L]);
        key[r] = barred(l) ? -INFINITY : bounded(l);
        top = fmaxf(top, key[r]);
    }
    c.top = warp_max(top);
    c.sum = 0.f;
    if (!p.sigmoid && c.top > -INFINITY) {
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < NPL; r++) sum += __expf(key[r] - c.top);  // exp(-inf) = 0
        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(FULL, sum, d);
        c.sum = sum;
    }
    if (p.bias) {
#pragma unroll
        for (int r = 0; r < NPL; r++)
            if (key[r] != -INFINITY) {
                const float b = __ldg(p.bias + at.e0 + r * at.L);
                key[r] = barred(b) ? -INFINITY : score_of(p, key[r], c.top, c.sum) + bounded(b);
            }
    }
    // the register's number: a larger one makes a key smaller, whatever its sign; infinity keeps its bits
#pragma unroll
    for (int r = 0; r < NPL; r++) {
        const uint32_t u = __float_as_uint(key[r]);
        key[r] = key[r] == -INFINITY ? key[r] : __uint_as_float((u & ~(uint32_t)(NPL - 1)) | ((int)u < 0 ? r : NPL - 1 - r));
    }
    auto register_of = [&](float k) { const int v = (int)(__float_as_uint(k) & (NPL - 1)); return (int)__float_as_uint(k) < 0 ? v : NPL - 1 - v; };
    // largest first: Batcher's odd-even merge sort
#pragma unroll
    for (int w = 1; w < NPL; w *= 2)
#pragma unroll
        for (int d = w; d >= 1; d /= 2)
#pragma unroll
            for (int i = d % w; i + d < NPL; i += 2 * d)
#pragma unroll
                for (int j = 0; j < d; j++)
                    if (i + j + d < NPL && (i + j) / (2 * w) == (i + j + d) / (2 * w)) {
                        const float hi = fmaxf(key[i + j], key[i + j + d]), lo = fminf(key[i + j], key[i + j + d]);
                        key[i + j] = hi;
                        key[i + j + d] = lo;
                    }
    const float tol0 = p.bias ? (NPL + 24) * 0x1p-23f : 0.f, tol1 = (1 << LOG) * 0x1p-21f;
    auto near = [&](float hi, float lo) { return hi - lo <= tol0 + fabsf(hi) * tol1 + 1e-30f; };  // (1e-30: around zero)
    bool certain = true;
    if (p.top_groups < p.groups) {
        float a = key[0], b = key[1];
        const bool sums = p.group_top == 2 && !p.bias;
        if (sums) {  // experts are ranked by their logits, groups by scores
            if (a != -INFINITY) a = score_of(p, bounded(to_f32(row[at.e0 + register_of(a) * at.L])), c.top, c.sum);
            if (b != -INFINITY) b = score_of(p, bounded(to_f32(row[at.e0 + register_of(b) * at.L])), c.top, c.sum);
        }
        bool kept;
        const float worth = rank_group<float>(p, at, glog, a, b, kept);
        // the worst group that is kept against the best that is not
        const float best_out = warp_max(kept || at.group >= p.groups ? -INFINITY : worth), worst_in = -warp_max(kept ? -worth : -INFINITY);
        // (a score made of a logit that lost LOG bits is off by |logit| times that; s * |logit| <= s * |top| + 1 / e)
        const float lost = sums ? (1.0f + (p.sigmoid ? 0.f : fabsf(c.top) * fabsf(worst_in))) * tol1 : 0.f;
        const float tol = 4 * ((NPL + 24) * 0x1p-23f * (p.bias || sums) + fmaxf(fabsf(worst_in), fabsf(best_out)) * tol1 + lost) + 1e-30f;
        certain = best_out == -INFINITY || worst_in - best_out > tol;
        if (!kept) key[0] = -INFINITY;
    }
    c.mine = -1;
    float last = 0.f;
    int last_e = -1;
    for (int j = 0; j < MAX_E; j++) {
        const float m = warp_max(key[0]);
        const bool close = j > 0 && near(last, m);
        if (m == -INFINITY || (j >= p.top_k && !close)) break;
        const int mine = at.e0 + register_of(key[0]) * at.L;
        const int e = (int)__reduce_min_sync(FULL, key[0] == m ? (unsigned)mine : (unsigned)MAX_E);
        if (e >= p.E) {
            certain = false;
            break;
        }
        if (close) {
            const bool same = e > last_e && to_f32(row[e]) == to_f32(row[last_e]) && (!p.bias || __ldg(p.bias + e) == __ldg(p.bias + last_e));
            if (!same) {
                certain = false;
                break;
            }
        }
        if (lane == j && j < p.top_k) c.mine = e;
        last = m;
        last_e = e;
        if (key[0] == m && mine == e) {
#pragma unroll
            for (int r = 0; r + 1 < NPL; r++) key[r] = key[r + 1];
            key[NPL - 1] = -INFINITY;
        }
    }
    c.certain = certain;
    return c;
}

// Weights of the chosen, by the full-precision exponential: lane j has slot j.
template <typename T>
__device__ __forceinline__ void finish_token(const RouteArgs& p, const T* row, long long t, int lane, const Choice& c) {
    float s = 0.f;
    if (lane < p.top_k && c.mine >= 0) {
        const float l = bounded(to_f32(row[c.mine]));
        s = p.sigmoid ? 1.0f / (1.0f + expf(-l)) : expf(l - c.top) / c.sum;
    }
    float total = 1.f;
    if (p.renormalise) {
        total = s;
        for (int d = 16; d; d >>= 1) total += __shfl_xor_sync(FULL, total, d);
        total += 1e-20f;
    }
    if (lane < p.top_k) {
        p.experts[t * p.top_k + lane] = c.mine;
        p.weights[t * p.top_k + lane] = p.scale * (s / total);
    }
}

// ---- the order of the pairs: a stable counting sort ----
struct PlanArgs {
    int32_t* offsets;
    int32_t* rows;
    int32_t* slots;
};
// Pairs are cut into one run for each warp.
__device__ __forceinline__ int2 run_of(int pairs, int warp, int warps) {
    const long long each = (((long long)pairs + warps - 1) / warps + 31) & ~31LL;
    const long long a = min(warp * each, (long long)pairs);
    return make_int2((int)a, (int)min(a + each, (long long)pairs));
}
// s_hist[w][e] = pairs of expert e in the run of the block's warp w.  Ends with a barrier.
__device__ __forceinline__ void count_runs(const int32_t* experts, int2 run, int E, int* s_hist, int tid, int threads) {
    const int warp = tid >> 5, lane = tid & 31, warps = threads >> 5;
    for (int i = tid; i < warps * E; i += threads) s_hist[i] = 0;
    __syncthreads();
    for (int i = run.x + lane; i < run.y; i += 32) {
        const int e = experts[i];
        if (e >= 0) atomicAdd(&s_hist[warp * E + e], 1);  // (whole numbers: the order of the additions does not matter)
    }
    __syncthreads();
}
// Places of a warp's pairs, s_hist[w][e] = the first place of warp w's pairs of expert e.
__device__ __forceinline__ void place_runs(const int32_t* experts, int2 run, int top_k, int E, int* s_hist, const PlanArgs& o, int tid) {
    const int warp = tid >> 5, lane = tid & 31;
    for (int base = run.x; base < run.y; base += 32) {
        const int i = base + lane;
        const int e = i < run.y ? experts[i] : -1;
        const unsigned alike = __match_any_sync(FULL, e);
        int at = -1;
        if (e >= 0) at = s_hist[warp * E + e] + __popc(alike & ((1u << lane) - 1));
        __syncwarp();
        if (e >= 0 && (alike >> lane) == 1u) s_hist[warp * E + e] = at + 1;  // the last of the alike
        __syncwarp();
        if (i < run.y) {
            o.slots[i] = at;
            if (e >= 0) o.rows[at] = i / top_k;
        }
    }
}
// Exclusive sums of s_v[0 .. n) by the whole block; s_v[n] = the total.
__device__ __forceinline__ void scan_block(int* s_v, int n, int* s_part, int tid, int threads) {
    const int lane = tid & 31, warp = tid >> 5;
    int carry = 0;
    for (int b = 0; b < n; b += threads) {
        const int v = b + tid < n ? s_v[b + tid] : 0;
        int x = v;
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(FULL, x, d);
            if (lane >= d) x += o;
        }
        if (lane == 31) s_part[warp] = x;
        __syncthreads();
        int before = carry;
        for (int w = 0; w < warp; w++) before += s_part[w];
        int total = carry;
        for (int w = 0; w < (threads >> 5); w++) total += s_part[w];
        if (b + tid < n) s_v[b + tid] = before + x - v;
        carry = total;
        __syncthreads();
    }
    if (tid == 0) s_v[n] = carry;
    __syncthreads();
}

// The order of the pairs by a cluster of RANKS blocks (1: no cluster): every warp counts its run, every block adds up its warps' and
// reads the other blocks' counts from their shared memory, and every warp places its run.  s_hist: [warps][E], [E] counts of the
// block, [E + 1] first places.
template <int RANKS, int THREADS>
__device__ __forceinline__ void plan_pairs(const int32_t* experts, int pairs, int top_k, int E, const PlanArgs& o, int* s_hist, int* s_part, int tid) {
    constexpr int WARPS = THREADS / 32;
    int *s_count = s_hist + WARPS * E, *s_first = s_count + E;
    const int rank = RANKS > 1 ? (int)cluster_ctarank() : 0;
    const int2 run = run_of(pairs, rank * WARPS + (tid >> 5), RANKS * WARPS);
    count_runs(experts, run, E, s_hist, tid, THREADS);
    for (int e = tid; e < E; e += THREADS) {
        int sum = 0;
#pragma unroll
        for (int w = 0; w < WARPS; w++) {
            const int v = s_hist[w * E + e];
            s_hist[w * E + e] = sum;
            sum += v;
        }
        s_count[e] = sum;
    }
    if (RANKS > 1) cluster_sync_all(); else __syncthreads();
    for (int e = tid; e < E; e += THREADS) {
        int all = 0, below = 0;
#pragma unroll
        for (int r = 0; r < RANKS; r++) {
            int v;
            if (RANKS > 1) asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(smem_u32(s_count + e), r)) : "memory");
            else v = s_count[e];
            all += v;
            if (r < rank) below += v;
        }
        s_first[e] = all;
        for (int w = 0; w < WARPS; w++) s_hist[w * E + e] += below;
    }
    __syncthreads();
    scan_block(s_first, E, s_part, tid, THREADS);
    for (int i = tid; i < WARPS * E; i += THREADS) s_hist[i] += s_first[i % E];
    if (rank == 0)
        for (int e = tid; e <= E; e += THREADS) o.offsets[e] = s_first[e];
    __syncthreads();
    place_runs(experts, run, top_k, E, s_hist, o, tid);
    for (int i = s_first[E] + rank * THREADS + tid; i < pairs && i >= 0; i += RANKS * THREADS) o.rows[i] = -1;
    if (RANKS > 1) cluster_sync_all();  // no block leaves while another may read its counts
}

constexpr int ROUTE_WARPS = 16, PLAN_RANKS = 8, PLAN_THREADS = 1024;
constexpr size_t plan_smem(int warps, int E) { return sizeof(int) * ((size_t)(warps + 2) * E + 1); }

// One warp a token.  PLAN: one block takes all tokens and orders the pairs as well.
template <typename T, int NPL, bool PLAN>
__global__ void __launch_bounds__(ROUTE_WARPS * 32, NPL <= 16 ? 2 : 1) route_kernel(RouteArgs p, PlanArgs o) {
    extern __shared__ int s_hist[];
    __shared__ int s_part[32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (long long t = (long long)blockIdx.x * ROUTE_WARPS + warp; t < p.T; t += (long long)gridDim.x * ROUTE_WARPS) {
        const T* row = (const T*)p.logits + t * p.stride;
        Choice c = choose<T, NPL>(p, row, lane, p.glog);
        if (!c.certain) c.mine = choose_exact<T, NPL>(p, row, lane, p.glog);
        finish_token(p, row, t, lane, c);
    }
    if (PLAN) {
        __syncthreads();
        plan_pairs<1, ROUTE_WARPS * 32>(p.experts, p.T * p.top_k, p.top_k, p.E, o, s_hist, s_part, tid);
    }
}

__global__ void __launch_bounds__(PLAN_THREADS, 1) plan_kernel(RouteArgs p, PlanArgs o) {
    extern __shared__ int s_hist[];
    __shared__ int s_part[32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    plan_pairs<PLAN_RANKS, PLAN_THREADS>(p.experts, p.T * p.top_k, p.top_k, p.E, o, s_hist, s_part, threadIdx.x);
}

template <typename... Args>
int launch(void (*kern)(Args...), int grid, int threads, size_t smem, int cluster, cudaStream_t stream, Args... args) {
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
    if (cluster > 1) {
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = cluster;
        attr[1].val.clusterDim.y = 1;
        attr[1].val.clusterDim.z = 1;
        cfg.numAttrs = 2;
    }
    TNNS_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, args...));
    tnns_count_launch();
    TNNS_CUDA_TRY(cudaGetLastError());
    return TNNS_OK;
}

// Tokens that one block chooses and orders in one launch (two for each of its warps); more are chosen by many blocks and ordered by
// a second launch.
constexpr int ONE_BLOCK_TOKENS = 2 * ROUTE_WARPS;

// Dynamic shared memory past 48 KB, once per kernel and device.
template <typename... Args>
int allow_smem(void (*kern)(Args...), size_t bytes, bool (&set)[64], int device) {
    if (!set[device & 63]) {
        TNNS_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
        set[device & 63] = true;
    }
    return TNNS_OK;
}

template <typename T, int NPL>
int launch_route(tnns_cuda_ctx* ctx, const RouteArgs& a, const PlanArgs& o, bool plan, cudaStream_t st) {
    int rc;
    if (plan && a.T <= ONE_BLOCK_TOKENS) {
        static bool set[64] = {false};
        if ((rc = allow_smem(route_kernel<T, NPL, true>, plan_smem(ROUTE_WARPS, MAX_E), set, ctx->device))) return rc;
        return launch<RouteArgs, PlanArgs>(route_kernel<T, NPL, true>, 1, ROUTE_WARPS * 32, plan_smem(ROUTE_WARPS, a.E), 1, st, a, o);
    }
    const int blocks = std::min((a.T + ROUTE_WARPS - 1) / ROUTE_WARPS, (NPL <= 16 ? 2 : 1) * ctx->sm_count);
    if ((rc = launch<RouteArgs, PlanArgs>(route_kernel<T, NPL, false>, blocks, ROUTE_WARPS * 32, 0, 1, st, a, o)) || !plan) return rc;
    static bool set[64] = {false};
    if ((rc = allow_smem(plan_kernel, plan_smem(PLAN_THREADS / 32, MAX_E), set, ctx->device))) return rc;
    return launch<RouteArgs, PlanArgs>(plan_kernel, PLAN_RANKS, PLAN_THREADS, plan_smem(PLAN_THREADS / 32, a.E), PLAN_RANKS, st, a, o);
}
// Registers a lane needs for its share of the experts.
template <typename T>
int launch_route_npl(tnns_cuda_ctx* ctx, const RouteArgs& a, const PlanArgs& o, bool plan, cudaStream_t st) {
    const int lanes = 32 >> a.glog, npl = (a.group_size + lanes - 1) / lanes;
    if (npl <= 2) return launch_route<T, 2>(ctx, a, o, plan, st);
    if (npl <= 4) return launch_route<T, 4>(ctx, a, o, plan, st);
    if (npl <= 8) return launch_route<T, 8>(ctx, a, o, plan, st);
    if (npl <= 16) return launch_route<T, 16>(ctx, a, o, plan, st);
    if (npl <= 32) return launch_route<T, 32>(ctx, a, o, plan, st);
    return launch_route<T, 64>(ctx, a, o, plan, st);
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

int tnns_cuda_route(tnns_cuda_ctx* ctx, const tnns_route_t* r, const void* d_logits, int dtype, long long stride, const float* d_bias, int T,
                    int32_t* d_experts, float* d_weights, int32_t* d_offsets, int32_t* d_rows, int32_t* d_slots, void* stream) {
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
    if ((rc = tnns_enter(ctx))) return rc;
    RouteArgs a;
    a.logits = d_logits; a.stride = stride; a.bias = d_bias; a.experts = d_experts; a.weights = d_weights;
    a.T = T; a.E = r->experts; a.top_k = r->top_k; a.sigmoid = r->score == TNNS_ROUTE_SIGMOID;
    // all groups searched: there is nothing to rank
    a.groups = r->top_groups < r->groups ? r->groups : 1;
    a.top_groups = r->top_groups < r->groups ? r->top_groups : 1;
    a.group_size = r->experts / a.groups; a.group_top = r->group_top;
    for (a.glog = 0; (1 << a.glog) < a.groups;) a.glog++;
    a.renormalise = r->renormalise; a.scale = r->scale;
    const cudaStream_t st = (cudaStream_t)stream;
    if (T == 0) {
        if (plan) TNNS_CUDA_TRY(cudaMemsetAsync(d_offsets, 0, (size_t)(r->experts + 1) * sizeof(int32_t), st));
        return TNNS_OK;
    }
    PlanArgs o;
    o.offsets = d_offsets; o.rows = d_rows; o.slots = d_slots;
    TNNS_FOR_DTYPE(dtype, TI, return launch_route_npl<TI>(ctx, a, o, plan, st));
}

}  // extern "C"
