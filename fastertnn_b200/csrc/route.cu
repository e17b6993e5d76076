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
constexpr unsigned FULL = 0xFFFFFFFFu;

// Keys in fp32, or in 64 bits where fp32 cannot tell the order.
template <typename Key>
struct KeyOps;
template <>
struct KeyOps<float> {
    static __device__ __forceinline__ float none() { return -INFINITY; }
    static __device__ __forceinline__ float warp_max(float v) {
        float r;
        asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
        return r;
    }
    static __device__ __forceinline__ float exponential(float v) { return __expf(v); }
    static __device__ __forceinline__ float quotient(float a, float b) { return __fdividef(a, b); }
};
template <>
struct KeyOps<double> {
    static __device__ __forceinline__ double none() { return -INFINITY; }
    static __device__ __forceinline__ double warp_max(double v) {
        for (int d = 16; d; d >>= 1) v = fmax(v, __shfl_xor_sync(FULL, v, d));
        return v;
    }
    static __device__ __forceinline__ double exponential(double v) { return exp(v); }
    static __device__ __forceinline__ double quotient(double a, double b) { return a / b; }
};

struct Choice {
    int mine;       // lane j: the expert of slot j, -1: none
    float top;      // softmax: the largest logit, and the sum of exp(logit - top)
    float sum;
    bool certain;   // false: keys lie closer together than their rounding; nothing else is valid then
};

// The choice for one token by one warp.  A group's experts lie on the 32 / 2^glog lanes of the group, NPL a lane: a lane's register r
// holds expert group * group_size + r * L + (lane % L), so within a lane, and lane by lane within a register, experts ascend.
//
// Keys in fp32 decide unless two that have to be told apart lie within `tol` of each other.  With a bias a key is score + bias: the
// exponential is off by 2^-22 and by |argument| * 2^-23 for its argument's rounding, of which a score (at most 1, and s * d <= 1/e)
// keeps 2^-22 together; a softmax's sum adds NPL + 5 roundings of 2^-24, quotient and addition add 2^-22 and |key| * 2^-24.  Two
// keys are then in order if they differ by (NPL + 24) * 2^-23 + |key| * 2^-21.  Without a bias keys are the logits themselves: exact.
template <typename T, int NPL, typename Key>
__device__ __forceinline__ Choice choose(const RouteArgs& p, const T* row, int lane, int glog) {
    using Ops = KeyOps<Key>;
    constexpr bool FAST = sizeof(Key) == 4;
    const int L = 32 >> glog, group = lane >> (5 - glog), sub = lane & (L - 1);
    const int e0 = group * p.group_size + sub;
    const bool grouped = p.top_groups < p.groups, sums = grouped && p.group_top == 2 && !p.bias;  // sums: groups by scores, experts by logits
    auto there = [&](int r) { return group < p.groups && r * L + sub < p.group_size; };
    Choice c;
    Key key[NPL];
    float top = -INFINITY;
#pragma unroll
    for (int r = 0; r < NPL; r++) {
        float l = -INFINITY;
        if (there(r)) l = to_f32(row[e0 + r * L]);
        l = barred(l) ? -INFINITY : bounded(l);
        top = fmaxf(top, l);
        key[r] = l;
    }
    top = KeyOps<float>::warp_max(top);
    c.top = top;
    c.sum = 0.f;
    Key all = 1;  // what scores are divided by
    if (!p.sigmoid) {
        Key sum = 0;
        if (top > -INFINITY) {
#pragma unroll
            for (int r = 0; r < NPL; r++) sum += Ops::exponential(key[r] - (Key)top);  // exp(-inf) = 0
        }
        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(FULL, sum, d);
        all = sum;
        c.sum = (float)sum;
    }
    auto score = [&](Key l) -> Key {
        if (l == Ops::none()) return 0;
        return p.sigmoid ? Ops::quotient(1, 1 + Ops::exponential(-l)) : Ops::quotient(Ops::exponential(l - (Key)top), all);
    };
    if (p.bias) {
#pragma unroll
        for (int r = 0; r < NPL; r++) {
            if (key[r] != Ops::none()) {
                const float b = __ldg(p.bias + e0 + r * L);
                key[r] = barred(b) ? Ops::none() : score(key[r]) + (Key)bounded(b);
            }
        }
    }
    auto tolerance = [&](Key k) { return (Key)((NPL + 24) * 0x1p-23f) + (k < 0 ? -k : k) * (Key)0x1p-21f; };
    bool certain = true;
    if (grouped) {
        Key a = Ops::none(), b = Ops::none();  // the group's two best
#pragma unroll
        for (int r = 0; r < NPL; r++) {
            const Key v = sums && key[r] != Ops::none() ? score(key[r]) : key[r];
            b = fmax(b, fmin(a, v));
            a = fmax(a, v);
        }
        for (int d = 1; d < L; d <<= 1) {
            const Key oa = __shfl_xor_sync(FULL, a, d), ob = __shfl_xor_sync(FULL, b, d);
            b = fmax(fmin(a, oa), fmax(b, ob));
            a = fmax(a, oa);
        }
        const Key worth = p.group_top == 2 && b != Ops::none() ? a + b : a;
        int better = 0;
        Key best_out = Ops::none(), worst_in = -Ops::none();
        for (int g = 0; g < p.groups; g++) {
            const Key o = __shfl_sync(FULL, worth, g << (5 - glog));
            better += o > worth || (o == worth && g < group);
        }
        const bool kept = group < p.groups && better < p.top_groups;
        if (FAST && (p.bias || sums)) {
            // the worst group that is kept against the best that is not
            best_out = Ops::warp_max(kept || group >= p.groups ? Ops::none() : worth);
            worst_in = -Ops::warp_max(kept ? -worth : Ops::none());
            certain = best_out == Ops::none() || worst_in - best_out > 4 * tolerance(worst_in);
        }
        if (!kept) {
#pragma unroll
            for (int r = 0; r < NPL; r++) key[r] = Ops::none();
        }
    }
    // The lane's best; ties within a lane stay with the lower expert.
    Key best = Ops::none();
    int at = MAX_E;
    auto look = [&]() {
        best = Ops::none();
        at = MAX_E;
#pragma unroll
        for (int r = 0; r < NPL; r++)
            if (key[r] > best) { best = key[r]; at = e0 + r * L; }
    };
    look();
    c.mine = -1;
    Key last = Ops::none();
    int last_e = -1;
    for (int j = 0;; j++) {
        const Key m = Ops::warp_max(best);
        if (FAST && p.bias && j > 0 && m != Ops::none() && last - m < tolerance(last)) {
            // near the one before: in order only if the two are the same by what they are made of
            const unsigned e = __reduce_min_sync(FULL, best == m ? (unsigned)at : (unsigned)MAX_E);
            const bool same = last == m && to_f32(row[e]) == to_f32(row[last_e]) && __ldg(p.bias + e) == __ldg(p.bias + last_e);
            certain = certain && same;
            if (!certain) break;
        } else if (j >= p.top_k) {
            break;
        }
        if (m == Ops::none()) break;
        const int e = (int)__reduce_min_sync(FULL, best == m ? (unsigned)at : (unsigned)MAX_E);
        if (lane == j && j < p.top_k) c.mine = e;
        last = m;
        last_e = e;
        if (at == e) {
#pragma unroll
            for (int r = 0; r < NPL; r++)
                if (e0 + r * L == e) key[r] = Ops::none();
            look();
        }
        if ((!FAST || !p.bias) && j + 1 >= p.top_k) break;
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

template <typename T, int NPL>
__device__ __noinline__ Choice choose_exact(const RouteArgs& p, const T* row, int lane, int glog) { return choose<T, NPL, double>(p, row, lane, glog); }

// ---- the order of the pairs: a stable counting sort ----
// Pairs [i0, i1) of `warps` warps, each with a run of its own; s_hist[w][e] counts the pairs of warp w.
struct PlanArgs {
    int32_t* offsets;
    int32_t* rows;
    int32_t* slots;
    int32_t* hist;  // [block][experts]
    int tokens_per_block;
};
__device__ __forceinline__ int2 run_of(int i0, int i1, int warp, int warps) {
    const int each = ((i1 - i0 + warps - 1) / warps + 31) & ~31;
    const int a = min(i0 + warp * each, i1);
    return make_int2(a, min(a + each, i1));
}
// Pairs of the block by warp and expert.  Ends with a barrier.
__device__ __forceinline__ void count_runs(const int32_t* experts, int i0, int i1, int E, int* s_hist, int tid, int threads) {
    const int warp = tid >> 5, lane = tid & 31, warps = threads >> 5;
    for (int i = tid; i < warps * E; i += threads) s_hist[i] = 0;
    __syncthreads();
    const int2 run = run_of(i0, i1, warp, warps);
    for (int i = run.x + lane; i < run.y; i += 32) {
        const int e = experts[i];
        if (e >= 0) atomicAdd(&s_hist[warp * E + e], 1);  // (whole numbers: the order of the additions does not matter)
    }
    __syncthreads();
}
// Places of the block's pairs, s_hist[w][e] = the first place of warp w's pairs of expert e.
__device__ __forceinline__ void place_runs(const int32_t* experts, int i0, int i1, int top_k, int E, int* s_hist, const PlanArgs& o, int tid, int threads) {
    const int warp = tid >> 5, lane = tid & 31, warps = threads >> 5;
    const int2 run = run_of(i0, i1, warp, warps);
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

constexpr int ROUTE_WARPS = 16;

// One warp a token; a block the tokens [block * tokens_per_block, ..).  PLAN 0: the choice alone; 1: also the block's pairs by expert,
// for place_kernel; 2: one block, which orders the pairs as well.
template <typename T, int NPL, int PLAN>
__global__ void __launch_bounds__(ROUTE_WARPS * 32) route_kernel(RouteArgs p, PlanArgs o) {
    extern __shared__ int s_hist[];  // [warp][E], PLAN 2: and [E + 1]
    __shared__ int s_part[32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    constexpr int threads = ROUTE_WARPS * 32;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    int glog = 0;
    if (p.top_groups < p.groups)
        while ((1 << glog) < p.groups) glog++;
    else p.groups = p.top_groups = 1, p.group_size = p.E;
    const int t0 = (int)min((long long)blockIdx.x * o.tokens_per_block, (long long)p.T), t1 = (int)min((long long)t0 + o.tokens_per_block, (long long)p.T);
    for (int t = t0 + warp; t < t1; t += ROUTE_WARPS) {
        const T* row = (const T*)p.logits + (long long)t * p.stride;
        Choice c = choose<T, NPL, float>(p, row, lane, glog);
        if (!c.certain) c = choose_exact<T, NPL>(p, row, lane, glog);
        finish_token(p, row, t, lane, c);
    }
    if (PLAN == 0) return;
    __syncthreads();
    const int i0 = t0 * p.top_k, i1 = t1 * p.top_k;
    if (PLAN == 1) {
        for (int e = tid; e < p.E; e += threads) s_hist[e] = 0;
        __syncthreads();
        for (int i = i0 + tid; i < i1; i += threads) {
            const int e = p.experts[i];
            if (e >= 0) atomicAdd(&s_hist[e], 1);
        }
        __syncthreads();
        for (int e = tid; e < p.E; e += threads) o.hist[(long long)blockIdx.x * p.E + e] = s_hist[e];
        return;
    }
    int* s_first = s_hist + ROUTE_WARPS * p.E;
    count_runs(p.experts, i0, i1, p.E, s_hist, tid, threads);
    for (int e = tid; e < p.E; e += threads) {
        int sum = 0;
        for (int w = 0; w < ROUTE_WARPS; w++) {
            const int v = s_hist[w * p.E + e];
            s_hist[w * p.E + e] = sum;
            sum += v;
        }
        s_first[e] = sum;
    }
    __syncthreads();
    scan_block(s_first, p.E, s_part, tid, threads);
    for (int e = tid; e <= p.E; e += threads) o.offsets[e] = s_first[e];
    for (int i = tid; i < ROUTE_WARPS * p.E; i += threads) s_hist[i] += s_first[i % p.E];
    __syncthreads();
    place_runs(p.experts, i0, i1, p.top_k, p.E, s_hist, o, tid, threads);
    for (int i = s_first[p.E] + tid; i < i1; i += threads) o.rows[i] = -1;
}

constexpr int PLACE_WARPS = 8;

// Block b orders the pairs of the tokens that block b of route_kernel<.., 1> counted.
__global__ void __launch_bounds__(PLACE_WARPS * 32) place_kernel(RouteArgs p, PlanArgs o, int blocks) {
    extern __shared__ int s_hist[];  // [warp][E], [E + 1] first places of the experts, [E] of this block's pairs
    __shared__ int s_part[32];
    int *s_first = s_hist + PLACE_WARPS * p.E, *s_below = s_first + p.E + 1;
    const int tid = threadIdx.x;
    constexpr int threads = PLACE_WARPS * 32;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int e = tid; e < 2 * p.E + 1; e += threads) s_first[e] = 0;
    __syncthreads();
    // the counts of all blocks, and of those before this one: threads side by side take neighbouring experts, the rest of the threads
    // other blocks' rows
    const int across = min(p.E, threads), down = threads / across;
    if (tid < across * down)
        for (int e = tid % across; e < p.E; e += across) {
            int all = 0, below = 0;
            int b = tid / across;
            for (; b + 3 * down < blocks; b += 4 * down) {
                int v[4];
#pragma unroll
                for (int u = 0; u < 4; u++) v[u] = o.hist[(long long)(b + u * down) * p.E + e];
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    all += v[u];
                    if (b + u * down < (int)blockIdx.x) below += v[u];
                }
            }
            for (; b < blocks; b += down) {
                const int v = o.hist[(long long)b * p.E + e];
                all += v;
                if (b < (int)blockIdx.x) below += v;
            }
            atomicAdd(&s_first[e], all);
            atomicAdd(&s_below[e], below);
        }
    const int t0 = (int)min((long long)blockIdx.x * o.tokens_per_block, (long long)p.T), t1 = (int)min((long long)t0 + o.tokens_per_block, (long long)p.T);
    const int i0 = t0 * p.top_k, i1 = t1 * p.top_k;
    count_runs(p.experts, i0, i1, p.E, s_hist, tid, threads);
    scan_block(s_first, p.E, s_part, tid, threads);
    if (blockIdx.x == 0)
        for (int e = tid; e <= p.E; e += threads) o.offsets[e] = s_first[e];
    for (int e = tid; e < p.E; e += threads) {
        int sum = s_first[e] + s_below[e];
        for (int w = 0; w < PLACE_WARPS; w++) {
            const int v = s_hist[w * p.E + e];
            s_hist[w * p.E + e] = sum;
            sum += v;
        }
    }
    __syncthreads();
    place_runs(p.experts, i0, i1, p.top_k, p.E, s_hist, o, tid, threads);
    const long long pairs = (long long)p.T * p.top_k;
    for (long long i = s_first[p.E] + blockIdx.x * threads + tid; i < pairs; i += (long long)gridDim.x * threads) o.rows[i] = -1;
}

template <typename... Args>
int launch(void (*kern)(Args...), int grid, int threads, size_t smem, cudaStream_t stream, Args... args) {
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
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

// Up to this many pairs one block chooses and orders; more pairs are chosen by many blocks, which leave their counts in the workspace
// for a second launch.
constexpr int ONE_BLOCK_TOKENS = 2 * ROUTE_WARPS;
constexpr int MAX_BLOCKS = 148;
static inline int tokens_per_block(int T) { return T <= ONE_BLOCK_TOKENS ? T : (T + MAX_BLOCKS - 1) / MAX_BLOCKS; }

template <typename T, int NPL>
int launch_route(tnns_cuda_ctx* ctx, const RouteArgs& a, PlanArgs o, bool plan, cudaStream_t st) {
    const int tpb = o.tokens_per_block;
    const int blocks = (a.T + tpb - 1) / tpb;
    if (!plan) return launch<RouteArgs, PlanArgs>(route_kernel<T, NPL, 0>, blocks, ROUTE_WARPS * 32, 0, st, a, o);
    if (blocks == 1) {
        const size_t smem = 4 * ((size_t)(ROUTE_WARPS + 1) * a.E + 1);
        static bool set[64] = {false};  // the attribute belongs to (function, device)
        if (!set[ctx->device & 63]) {
            TNNS_CUDA_TRY(cudaFuncSetAttribute(route_kernel<T, NPL, 2>, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * ((ROUTE_WARPS + 1) * MAX_E + 1)));
            set[ctx->device & 63] = true;
        }
        return launch<RouteArgs, PlanArgs>(route_kernel<T, NPL, 2>, 1, ROUTE_WARPS * 32, smem, st, a, o);
    }
    const int rc = launch<RouteArgs, PlanArgs>(route_kernel<T, NPL, 1>, blocks, ROUTE_WARPS * 32, 4 * (size_t)a.E, st, a, o);
    if (rc) return rc;
    const size_t smem = 4 * ((size_t)(PLACE_WARPS + 2) * a.E + 1);
    return launch<RouteArgs, PlanArgs, int>(place_kernel, blocks, PLACE_WARPS * 32, smem, st, a, o, blocks);
}
// Registers a lane needs for its share of the experts.
template <typename T>
int launch_route_npl(tnns_cuda_ctx* ctx, const RouteArgs& a, const PlanArgs& o, bool plan, cudaStream_t st) {
    int npl = (a.E + 31) / 32;
    if (a.top_groups < a.groups) {
        int lanes = 32;
        for (int g = 1; g < a.groups; g *= 2) lanes /= 2;
        npl = (a.group_size + lanes - 1) / lanes;
    }
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

size_t tnns_route_workspace_bytes(const tnns_route_t* r, int T) {
    if (check_route(r) || T <= ONE_BLOCK_TOKENS) return 0;
    const int tpb = tokens_per_block(T);
    return (size_t)((T + tpb - 1) / tpb) * r->experts * sizeof(int32_t);
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
    const size_t needed = plan ? tnns_route_workspace_bytes(r, T) : 0;
    if (needed && (!d_workspace || workspace_bytes < needed || (uintptr_t)d_workspace % 16))
        return tnns_fail(TNNS_ERR_INVALID, "a workspace of %zu bytes, 16-byte aligned, is needed (%zu given)", needed, workspace_bytes);
    if ((rc = tnns_enter(ctx))) return rc;
    RouteArgs a;
    a.logits = d_logits; a.stride = stride; a.bias = d_bias; a.experts = d_experts; a.weights = d_weights;
    a.T = T; a.E = r->experts; a.top_k = r->top_k; a.sigmoid = r->score == TNNS_ROUTE_SIGMOID;
    a.groups = r->groups; a.group_size = r->experts / r->groups; a.top_groups = r->top_groups; a.group_top = r->group_top;
    a.renormalise = r->renormalise; a.scale = r->scale;
    const cudaStream_t st = (cudaStream_t)stream;
    if (T == 0) {
        if (plan) TNNS_CUDA_TRY(cudaMemsetAsync(d_offsets, 0, (size_t)(r->experts + 1) * sizeof(int32_t), st));
        return TNNS_OK;
    }
    PlanArgs o;
    o.offsets = d_offsets; o.rows = d_rows; o.slots = d_slots; o.hist = (int32_t*)d_workspace; o.tokens_per_block = tokens_per_block(T);
    TNNS_FOR_DTYPE(dtype, TI, return launch_route_npl<TI>(ctx, a, o, plan, st));
}

}  // extern "C"
