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
    int T, E, top_k, sigmoid, groups, group_size, top_groups, group_top, renormalise, glog, per, vec;
    float scale;
};

// A logit or a bias as it counts: -inf and NaN bar its expert (-inf: a maximum returns the operand that is a number), +inf is the
// largest finite float.
__device__ __forceinline__ float bounded(float v) { return fminf(fmaxf(v, -INFINITY), 3.402823466e38f); }
__device__ __forceinline__ bool barred(float v) { return !(v > -INFINITY); }

constexpr int MAX_E = 1024;
constexpr unsigned FULL = 0xFFFFFFFFu;

struct Choice {
    int mine;       // lane j: the expert of slot j, -1: none
    float top;      // softmax: the largest logit, and the sum of exp(logit - top)
    float sum;
    bool certain;   // false: only the 64-bit form over all experts can tell
};

// A group's experts lie on the 32 / 2^glog lanes of the group, `per` neighbours a lane (at most NPL, in registers 0 ..).
struct Lanes {
    int L, group, e0, have;  // lanes of a group, this lane's group, its first expert, how many it has
    __device__ __forceinline__ Lanes(const RouteArgs& p, int lane) : L(32 >> p.glog), group(lane >> (5 - p.glog)) {
        const int in = (lane & (L - 1)) * p.per;
        e0 = group * p.group_size + in;
        have = group < p.groups ? min(max(p.group_size - in, 0), p.per) : 0;
    }
};
// Values first .. first + NPL - 1 of a row, those past `have` as -inf.  vec: four at a time (rows and `have` allow it).  Plain loads, here
// and wherever these kernels read an input: the launch in front may still write it while the block is resident, so it is no read-only
// data of the kernel.
template <typename T, int NPL>
__device__ __forceinline__ void load_values(const T* at, int have, bool vec, float (&v)[NPL]) {
    if (NPL >= 4 && vec) {
#pragma unroll
        for (int r = 0; r + 3 < NPL; r += 4) {
            v[r] = v[r + 1] = v[r + 2] = v[r + 3] = -INFINITY;
            if (r < have) {
                if constexpr (sizeof(T) == 4) {
                    const float4 f = *reinterpret_cast<const float4*>(at + r);
                    v[r] = f.x; v[r + 1] = f.y; v[r + 2] = f.z; v[r + 3] = f.w;
                } else {
                    const uint2 u = *reinterpret_cast<const uint2*>(at + r);
                    const unsigned short h[4] = {(unsigned short)u.x, (unsigned short)(u.x >> 16), (unsigned short)u.y, (unsigned short)(u.y >> 16)};
#pragma unroll
                    for (int i = 0; i < 4; i++) v[r + i] = to_f32(*reinterpret_cast<const T*>(&h[i]));
                }
            }
        }
    } else {
#pragma unroll
        for (int r = 0; r < NPL; r++) v[r] = r < have ? to_f32(at[r]) : -INFINITY;
    }
}

__device__ __forceinline__ float warp_max(float v) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
// (bits in an order that integers share: first the high words' largest, then the low words' among its lanes)
__device__ __forceinline__ double warp_max(double v) {
    long long b = __double_as_longlong(v + 0.0);  // -0 as +0
    b ^= (b >> 63) & 0x7FFFFFFFFFFFFFFFLL;
    const int hi = (int)(b >> 32), top = __reduce_max_sync(FULL, hi);
    const unsigned low = __reduce_max_sync(FULL, hi == top ? (unsigned)b : 0u);
    b = (long long)top << 32 | low;
    b ^= (b >> 63) & 0x7FFFFFFFFFFFFFFFLL;
    return __longlong_as_double(b);
}
// 2^(v log2 e), off by 2^-22 and by the rounding of the product
__device__ __forceinline__ float exponential(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v * 1.44269504f));
    return r;
}
__device__ __forceinline__ float reciprocal(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// A score in fp32 by the fast exponential and quotient, or in 64 bits.
__device__ __forceinline__ float score_of(const RouteArgs& p, float l, float top, float all) {
    return p.sigmoid ? reciprocal(1.0f + exponential(-l)) : exponential(l - top) * reciprocal(all);
}
__device__ __forceinline__ double score_of(const RouteArgs& p, double l, double top, double all) {
    return p.sigmoid ? 1.0 / (1.0 + exp(-l)) : exp(l - top) / all;
}
// (a, b): the two best values of the lane, on return those of its group; kept: whether the group is among the best, ranked by a, or by
// a + b.  Returns the group's worth: -inf where it has no expert, and there alone (a sum of two finite values that leaves fp32 counts as
// the outermost finite float; in 64 bits none leaves).
template <typename Key>
__device__ __forceinline__ Key rank_group(const RouteArgs& p, const Lanes& at, Key& a, Key& b, bool& kept) {
    for (int d = 1; d < at.L; d <<= 1) {
        const Key oa = __shfl_xor_sync(FULL, a, d), ob = __shfl_xor_sync(FULL, b, d);
        b = fmax(fmin(a, oa), fmax(b, ob));
        a = fmax(a, oa);
    }
    const Key none = -INFINITY;
    Key worth = p.group_top == 2 && b != none ? a + b : a;
    if (sizeof(Key) == 4 && a != none) worth = fmin(fmax(worth, (Key)-3.402823466e38f), (Key)3.402823466e38f);
    int better = 0;
    for (int g = 0; g < p.groups; g++) {
        const Key o = __shfl_sync(FULL, worth, g << (5 - p.glog));
        better += o > worth || (o == worth && g < at.group);
    }
    kept = at.group < p.groups && better < p.top_groups;
    return worth;
}

// The choice in 64 bits.
template <typename T, int NPL>
__device__ __noinline__ int choose_exact(const RouteArgs& p, const T* row, int lane) {
    const Lanes at(p, lane);
    const double none = -INFINITY;
    double key[NPL];
    double top = none;
#pragma unroll
    for (int r = 0; r < NPL; r++) {
        const float l = r < at.have ? to_f32(row[at.e0 + r]) : -INFINITY;
        key[r] = barred(l) ? none : (double)bounded(l);
        top = fmax(top, key[r]);
    }
    top = warp_max(top);
    double all = 0;
    if (!p.sigmoid && top > none) {
#pragma unroll 1
        for (int r = 0; r < at.have; r++) {  // (from memory again: a register array cannot be indexed)
            const float l = to_f32(row[at.e0 + r]);
            if (!barred(l)) all += exp((double)bounded(l) - top);
        }
        __syncwarp();
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
                const float c = p.bias[at.e0 + r];
                key[r] = v = barred(c) ? none : v + (double)bounded(c);
            }
        }
        b = fmax(b, fmin(a, v));
        a = fmax(a, v);
    }
    if (grouped) {
        bool kept;
        rank_group<double>(p, at, a, b, kept);
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
            if (key[r] > best) { best = key[r]; e = at.e0 + r; }
        const double m = warp_max(best);
        if (m == none) break;
        e = (int)__reduce_min_sync(FULL, best == m ? (unsigned)e : (unsigned)MAX_E);
        if (lane == j) mine = e;
#pragma unroll
        for (int r = 0; r < NPL; r++)
            if (at.e0 + r == e) key[r] = none;
    }
    return mine;
}

// A softmax's sum in 64 bits, by the whole warp.
template <typename T>
__device__ __forceinline__ double exact_sum(const RouteArgs& p, const T* row, int lane, double top) {
    double all = 0;
    for (int e = lane; e < p.E; e += 32) {
        const float v = to_f32(row[e]);
        if (!barred(v)) all += exp((double)bounded(v) - top);
    }
    for (int d = 16; d; d >>= 1) all += __shfl_xor_sync(FULL, all, d);
    return all;
}
// The candidates' order in 64 bits: lane j < n has expert `mine` (MAX_E: none) of logit l and bias b.  Returns the expert of place j.
template <typename T>
__device__ __noinline__ int order_exact(const RouteArgs& p, const T* row, int lane, int n, int mine, float l, float b, float top) {
    double key = (double)bounded(l);
    if (p.bias) key = score_of(p, key, (double)top, p.sigmoid ? 1.0 : exact_sum(p, row, lane, (double)top)) + (double)bounded(b);
    int place = 0, result = MAX_E;
    for (int i = 0; i < n; i++) {
        const double o = __shfl_sync(FULL, key, i);
        const int e = __shfl_sync(FULL, mine, i);
        place += e < MAX_E && (o > key || (o == key && e < mine));
    }
    for (int i = 0; i < n; i++) {
        const int at = __shfl_sync(FULL, place, i), e = __shfl_sync(FULL, mine, i);
        if (at == lane && e < MAX_E) result = e;
    }
    return result;
}
// Whether the lane's group is among the best, in 64 bits: ea, eb are the lane's two best experts (MAX_E: none).
template <typename T>
__device__ __noinline__ bool groups_exact(const RouteArgs& p, const T* row, int lane, int ea, int eb, float top) {
    const Lanes at(p, lane);
    const bool by_logit = p.group_top == 1 && !p.bias;
    const double all = p.sigmoid || by_logit ? 1.0 : exact_sum(p, row, lane, (double)top);
    double v[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int e = i ? eb : ea;
        v[i] = -INFINITY;
        if (e < MAX_E) {
            const double l = (double)bounded(to_f32(row[e]));
            v[i] = by_logit ? l : score_of(p, l, (double)top, all) + (p.bias ? (double)bounded(p.bias[e]) : 0.0);
        }
    }
    __syncwarp();
    bool kept;
    double a = fmax(v[0], v[1]), b = fmin(v[0], v[1]);
    rank_group<double>(p, at, a, b, kept);
    return kept;
}

// The choice for one token by one warp, in fp32.  Every lane sorts its keys, and the warp takes the best of the lanes' first ones,
// top_k times.  A key carries its register's number in its lowest bits (LOG of them), lower registers above higher ones.
//
// That is certain unless two keys that have to be told apart are closer than their errors.  Experts, or groups, that are near each other
// are then ordered in 64 bits by themselves; where that is not enough (a lane's third best near its second, more candidates than lanes)
// the token is chosen in 64 bits altogether.  A score by the fast functions is off by 2^-22 from the exponential and by the rounding of its argument, of which a score (at
// most 1, and s * d <= 1 / e) keeps 2^-22 together; a softmax's sum adds NPL + 5 roundings of 2^-24, the quotient 2^-22, the bias
// |key| * 2^-24.  A key without a bias is the logit itself.  The register's number takes LOG bits.  Two keys are in order if they
// differ by (NPL + 24) * 2^-23 + |key| * 2^(LOG - 21) (first term: with a bias), or if they are made of the same logit and the same
// bias and come in their experts' order.
template <typename T, int NPL>
__device__ __forceinline__ Choice choose(const RouteArgs& p, const T* row, int lane) {
    constexpr int LOG = NPL == 2 ? 1 : NPL == 4 ? 2 : NPL == 8 ? 3 : NPL == 16 ? 4 : NPL == 32 ? 5 : 6;
    const Lanes at(p, lane);
    Choice c;
    float key[NPL];
    load_values<T, NPL>(row + at.e0, at.have, p.vec, key);
    float top = -INFINITY;
#pragma unroll
    for (int r = 0; r < NPL; r++) {
        key[r] = bounded(key[r]);
        top = fmaxf(top, key[r]);
    }
    c.top = c.sum = 0.f;
    if (!p.sigmoid) {
        c.top = warp_max(top);
        if (c.top > -INFINITY) {
            float sum = 0.f;
#pragma unroll
            for (int r = 0; r < NPL; r++) sum += exponential(key[r] - c.top);  // exp(-inf) = 0
            for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(FULL, sum, d);
            c.sum = sum;
        }
    }
    if (p.bias) {
        float b[NPL];
        load_values<float, NPL>(p.bias + at.e0, at.have, p.vec, b);
        const float inverse = reciprocal(c.sum);
#pragma unroll
        for (int r = 0; r < NPL; r++) {
            const float s = p.sigmoid ? reciprocal(1.0f + exponential(-key[r])) : exponential(key[r] - c.top) * inverse;
            key[r] = key[r] == -INFINITY ? -INFINITY : s + bounded(b[r]);  // (-inf where the bias is)
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
            if (a != -INFINITY) a = score_of(p, bounded(to_f32(row[at.e0 + register_of(a)])), c.top, c.sum);
            if (b != -INFINITY) b = score_of(p, bounded(to_f32(row[at.e0 + register_of(b)])), c.top, c.sum);
        }
        bool kept;
        const float worth = rank_group<float>(p, at, a, b, kept);
        // A worth is off by what its parts are: each keeps the errors of a score, and |part| times those of its bits (their sum may be far
        // smaller than they are).  A score made of a logit that lost LOG bits is off by |logit| times that; s * |logit| <= s * |top| + 1 / e.
        const bool there = a != -INFINITY;
        const float parts = fabsf(a) + (p.group_top == 2 && b != -INFINITY ? fabsf(b) : 0.f);
        const float lost = sums ? (1.0f + (p.sigmoid ? 0.f : fabsf(c.top) * worth)) * tol1 : 0.f;
        const float off = (NPL + 24) * 0x1p-23f * (p.bias || sums) + parts * (tol1 + 0x1p-22f) + lost + 1e-30f;
        // the least that a kept group can be worth against the most that one can that is not
        const float best_out = warp_max(there && !kept ? worth + off : -INFINITY), worst_in = -warp_max(there && kept ? off - worth : -INFINITY);
        if (!(best_out == -INFINITY || worst_in > best_out)) {
            // the lanes' two best are certain as such unless a third is near them
            const bool third = NPL > 2 && key[1] != -INFINITY && key[NPL > 2 ? 2 : 1] != -INFINITY && near(key[1], key[NPL > 2 ? 2 : 1]);
            if (__any_sync(FULL, third)) certain = false;
            else kept = groups_exact<T>(p, row, lane, key[0] == -INFINITY ? MAX_E : at.e0 + register_of(key[0]), key[1] == -INFINITY ? MAX_E : at.e0 + register_of(key[1]), c.top);
        }
        // every key of the lane, not its first alone: what is taken moves the next one up
#pragma unroll
        for (int r = 0; r < NPL; r++) key[r] = kept ? key[r] : -INFINITY;
    }
    // lane j < n: the j-th best key and its expert
    float mine_key = -INFINITY;
    int mine = MAX_E, n = p.top_k, first = at.e0 + register_of(key[0]);
    auto pop = [&](int j) {
        const float m = warp_max(key[0]);
        if (m == -INFINITY) return false;  // no expert is left
        const int e = (int)__reduce_min_sync(FULL, key[0] == m ? (unsigned)first : (unsigned)MAX_E);
        if (lane == j) {
            mine_key = m;
            mine = e;
        }
        if (key[0] == m && first == e) {
#pragma unroll
            for (int r = 0; r + 1 < NPL; r++) key[r] = key[r + 1];
            key[NPL - 1] = -INFINITY;
            first = at.e0 + register_of(key[0]);
        }
        return true;
    };
    for (int j = 0; j < n && pop(j);) j++;
    // those behind the last slot that are near it, and near each other, are candidates too
    float last = __shfl_sync(FULL, mine_key, n - 1);
    for (;;) {
        const float m = warp_max(key[0]);
        if (m == -INFINITY || !near(last, m)) break;
        if (n == 32) {
            certain = false;
            break;
        }
        pop(n++);
        last = m;
    }
    // in order?  Where two neighbours are near each other, they have to be the same and to come in their experts' order.
    float l = 0.f, b = 0.f;
    if (mine_key != -INFINITY && mine < p.E) {
        l = to_f32(row[mine]);
        if (p.bias) b = p.bias[mine];
    }
    const float prev_key = __shfl_up_sync(FULL, mine_key, 1), prev_l = __shfl_up_sync(FULL, l, 1), prev_b = __shfl_up_sync(FULL, b, 1);
    const int prev = __shfl_up_sync(FULL, mine, 1);
    if (__any_sync(FULL, mine_key != -INFINITY && mine >= p.E)) certain = false;
    const bool odd = lane > 0 && lane < n && mine_key != -INFINITY && near(prev_key, mine_key) && !(mine > prev && l == prev_l && b == prev_b);
    if (__any_sync(FULL, odd) && certain) mine = order_exact<T>(p, row, lane, n, mine_key != -INFINITY ? mine : MAX_E, l, b, c.top);
    c.mine = mine_key != -INFINITY && lane < p.top_k && mine < p.E ? mine : -1;
    c.certain = certain;
    return c;
}

// Weights of the chosen, in fp32: lane j has slot j.  The exponential is the library's; a softmax's sum is the one of fast exponentials that
// the choice made (one more pass over the row for the other would cost as much as the first).  Error against 64 bits over 8191 tokens,
// 8 of 256: 6e-8, the type's own rounding 3e-8.
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
    FastDiv by_k;  // pair -> token
};
// Exclusive sums of s_v[0 .. n) by the whole block; s_v[n] = the total.
template <int THREADS>
__device__ __forceinline__ void scan_block(int* s_v, int n, int* s_part, int tid) {
    const int lane = tid & 31, warp = tid >> 5;
    int carry = 0;
    for (int b = 0; b < n; b += THREADS) {
        const int v = b + tid < n ? s_v[b + tid] : 0;
        int x = v;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(FULL, x, d);
            if (lane >= d) x += o;
        }
        if (lane == 31) s_part[warp] = x;
        __syncthreads();
        // every warp sums the warps' parts for itself
        int part = lane < THREADS / 32 ? s_part[lane] : 0;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(FULL, part, d);
            if (lane >= d) part += o;
        }
        const int before = warp ? __shfl_sync(FULL, part, warp - 1) : 0, total = __shfl_sync(FULL, part, 31);
        if (b + tid < n) s_v[b + tid] = carry + before + x - v;
        carry += total;
        if (b + THREADS < n) __syncthreads();
    }
    if (tid == 0) s_v[n] = carry;
    __syncthreads();
}

// The order of the pairs by a cluster of RANKS blocks (1: no cluster), each with an equal part of the tokens.  A token takes an expert
// at most once, so 32 neighbouring tokens' pairs with an expert are the bits of one word; a pair's place among its expert's is the
// number of bits before its own.  Each block goes over its tokens in slabs of `high` groups of 32; where one slab does not hold them
// all, once to count and once more to place.  Shared memory: masks [high][E], bits before them [high][E], [E] counts of the block,
// [E + 1] first places, [E] pairs of the blocks before.
constexpr size_t plan_smem(int high, int E) { return sizeof(int) * ((size_t)(2 * high + 3) * E + 1); }
template <int RANKS, int THREADS>
__device__ __forceinline__ void plan_pairs(const RouteArgs& p, const PlanArgs& o, int high, int* smem, int* s_part, int tid) {
    const int E = p.E, k = p.top_k;
    unsigned* s_mask = reinterpret_cast<unsigned*>(smem);
    int *s_before = smem + high * E, *s_count = s_before + high * E, *s_first = s_count + E, *s_below = s_first + E + 1;
    const int rank = RANKS > 1 ? (int)cluster_ctarank() : 0;
    const long long groups = ((long long)p.T + 31) / 32, each = (groups + RANKS - 1) / RANKS;
    const long long g0 = min(rank * each, groups), g1 = min(g0 + each, groups);
    const bool once = g1 - g0 <= high;
    for (int x = tid; x < E; x += THREADS) s_count[x] = s_below[x] = 0;
    __syncthreads();
    constexpr int U = 8;  // pairs of a thread whose loads are on their way together
    int e[U];
    for (int pass = 0; pass < 2; pass++) {
        for (long long g = g0; g < g1; g += high) {
            const int here = (int)min((long long)high, g1 - g), t0 = (int)(g * 32), i0 = t0 * k, i1 = (int)min((long long)t0 + here * 32, (long long)p.T) * k;
            const bool kept = once && i1 - i0 <= U * THREADS;  // pass 1 finds the experts in registers
            auto load = [&](int i) {
#pragma unroll
                for (int u = 0; u < U; u++) e[u] = i + u * THREADS < i1 ? p.experts[i + u * THREADS] : -1;
            };
            if (pass == 0 || !once) {
                load(i0 + tid);
                for (int i = tid; i < here * E; i += THREADS) s_mask[i] = 0;
                __syncthreads();
                for (int i = i0 + tid; i < i1; i += U * THREADS) {
                    if (i != i0 + tid) load(i);
#pragma unroll
                    for (int u = 0; u < U; u++)
                        if (e[u] >= 0) {
                            const int t = (int)o.by_k.div((uint32_t)(i + u * THREADS)) - t0;
                            atomicOr(&s_mask[(t >> 5) * E + e[u]], 1u << (t & 31));
                        }
                }
                __syncthreads();
                int* s_run = pass == 0 ? s_count : s_below;
                for (int x = tid; x < E; x += THREADS) {
                    int sum = s_run[x];
#pragma unroll 8
                    for (int h = 0; h < here; h++) {
                        s_before[h * E + x] = sum;
                        sum += __popc(s_mask[h * E + x]);
                    }
                    s_run[x] = sum;
                }
                __syncthreads();
            }
            if (pass == 1)
                for (int i = i0 + tid; i < i1; i += U * THREADS) {
                    if (!kept) load(i);
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        const int j = i + u * THREADS;
                        if (j >= i1) break;
                        int at = -1;
                        if (e[u] >= 0) {
                            const int token = (int)o.by_k.div((uint32_t)j), t = token - t0, m = (t >> 5) * E + e[u];
                            at = s_first[e[u]] + (once ? s_below[e[u]] : 0) + s_before[m] + __popc(s_mask[m] & ((1u << (t & 31)) - 1));
                            o.rows[at] = token;
                        }
                        o.slots[j] = at;
                    }
                }
            __syncthreads();
        }
        if (pass == 1) break;
        if (RANKS > 1) {
            cluster_sync_all();
            for (int e = tid; e < E; e += THREADS) {
                int v[RANKS], all = 0, below = 0;
#pragma unroll
                for (int r = 0; r < RANKS; r++) asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v[r]) : "r"(mapa_shared(smem_u32(s_count + e), r)) : "memory");
#pragma unroll
                for (int r = 0; r < RANKS; r++) {
                    all += v[r];
                    if (r < rank) below += v[r];
                }
                s_first[e] = all;
                s_below[e] = below;
            }
        } else {
            for (int e = tid; e < E; e += THREADS) s_first[e] = s_count[e];
        }
        __syncthreads();
        scan_block<THREADS>(s_first, E, s_part, tid);
        if (rank == 0)
            for (int e = tid; e <= E; e += THREADS) o.offsets[e] = s_first[e];
    }
    const int pairs = p.T * k;
    for (long long i = (long long)s_first[E] + rank * THREADS + tid; i < pairs; i += RANKS * THREADS) o.rows[i] = -1;
    if (RANKS > 1) cluster_sync_all();  // no block leaves while another may read its counts
}

constexpr int ROUTE_WARPS = 16, PLAN_THREADS = 1024;

// One warp a token.  PLAN: one block takes all tokens and orders the pairs as well.
template <typename T, int NPL, bool PLAN>
__global__ void __launch_bounds__(ROUTE_WARPS * 32, NPL <= 16 ? 2 : 1) route_kernel(const __grid_constant__ RouteArgs p, const __grid_constant__ PlanArgs o) {
    extern __shared__ int s_plan[];
    __shared__ int s_part[32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (long long t = (long long)blockIdx.x * ROUTE_WARPS + warp; t < p.T; t += (long long)gridDim.x * ROUTE_WARPS) {
        const T* row = (const T*)p.logits + t * p.stride;
        Choice c = choose<T, NPL>(p, row, lane);
        if (!c.certain) c.mine = choose_exact<T, NPL>(p, row, lane);
        finish_token(p, row, t, lane, c);
    }
    if (PLAN) {
        __syncthreads();
        plan_pairs<1, ROUTE_WARPS * 32>(p, o, 1, s_plan, s_part, tid);
    }
}

template <int RANKS>
__global__ void __launch_bounds__(PLAN_THREADS, 1) plan_kernel(const __grid_constant__ RouteArgs p, const __grid_constant__ PlanArgs o, int high) {
    extern __shared__ int s_plan[];
    __shared__ int s_part[32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    plan_pairs<RANKS, PLAN_THREADS>(p, o, high, s_plan, s_part, threadIdx.x);
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
static_assert(ONE_BLOCK_TOKENS <= 32, "one group of tokens");

// Dynamic shared memory past 48 KB, once per kernel and device.
template <typename... Args>
int allow_smem(void (*kern)(Args...), size_t bytes, bool (&set)[64], int device) {
    if (!set[device & 63]) {
        TNNS_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
        set[device & 63] = true;
    }
    return TNNS_OK;
}

constexpr size_t PLAN_SMEM = 200 * 1024;
template <int RANKS>
int launch_plan_ranks(tnns_cuda_ctx* ctx, const RouteArgs& a, const PlanArgs& o, cudaStream_t st) {
    static bool set[64] = {false};
    const int rc = allow_smem(plan_kernel<RANKS>, PLAN_SMEM, set, ctx->device);
    if (rc) return rc;
    // groups of 32 tokens that a block holds at a time: all of its own, or as many as fit
    const int own = (int)((((long long)a.T + 31) / 32 + RANKS - 1) / RANKS), fit = (int)((PLAN_SMEM / sizeof(int) / a.E - 4) / 2);
    const int high = std::min(own, fit);
    return launch<RouteArgs, PlanArgs, int>(plan_kernel<RANKS>, RANKS, PLAN_THREADS, plan_smem(high, a.E), RANKS, st, a, o, high);
}
// Clusters of sixteen blocks where the device takes them (the blocks' shared-memory counts and scattered stores bound the launch: 8192
// tokens, 8 of 256 experts, eight blocks 12.3 us, sixteen 10.1), else of eight.
int launch_plan(tnns_cuda_ctx* ctx, const RouteArgs& a, const PlanArgs& o, cudaStream_t st) {
    static int ranks[64] = {0};
    int& r = ranks[ctx->device & 63];
    if (r == 0) {
        r = 8;
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute attr[1];
        cfg.gridDim = dim3(16);
        cfg.blockDim = dim3(PLAN_THREADS);
        cfg.dynamicSmemBytes = PLAN_SMEM;
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 16;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int n = 0;
        if (cudaFuncSetAttribute(plan_kernel<16>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
            cudaFuncSetAttribute(plan_kernel<16>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PLAN_SMEM) == cudaSuccess &&
            cudaOccupancyMaxActiveClusters(&n, plan_kernel<16>, &cfg) == cudaSuccess && n > 0)
            r = 16;
        cudaGetLastError();  // a refusal is an answer here
    }
    return r == 16 ? launch_plan_ranks<16>(ctx, a, o, st) : launch_plan_ranks<8>(ctx, a, o, st);
}

template <typename T, int NPL>
int launch_route(tnns_cuda_ctx* ctx, const RouteArgs& a, const PlanArgs& o, bool plan, cudaStream_t st) {
    int rc;
    if (plan && a.T <= ONE_BLOCK_TOKENS) return launch<RouteArgs, PlanArgs>(route_kernel<T, NPL, true>, 1, ROUTE_WARPS * 32, plan_smem(1, a.E), 1, st, a, o);
    const int blocks = std::min((a.T + ROUTE_WARPS - 1) / ROUTE_WARPS, (NPL <= 16 ? 2 : 1) * ctx->sm_count);
    if ((rc = launch<RouteArgs, PlanArgs>(route_kernel<T, NPL, false>, blocks, ROUTE_WARPS * 32, 0, 1, st, a, o)) || !plan) return rc;
    return launch_plan(ctx, a, o, st);
}
// Registers a lane needs for its share of the experts.
template <typename T>
int launch_route_npl(tnns_cuda_ctx* ctx, const RouteArgs& a, const PlanArgs& o, bool plan, cudaStream_t st) {
    const int npl = a.per;
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
    if (T < 0 || (long long)T * r->top_k > 0x7FFF0000LL) return tnns_fail(TNNS_ERR_INVALID, "bad size: %d tokens, top_k %d", T, r->top_k);
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
    // experts of a lane; four at a time where rows, groups and lanes all begin on a multiple of four
    const int lanes = 32 >> a.glog, eb = tnns_dtype_bytes(dtype);
    a.per = (a.group_size + lanes - 1) / lanes;
    a.vec = a.per > 2 && a.group_size % 4 == 0 && stride % 4 == 0 && (uintptr_t)d_logits % (4 * eb) == 0 && (uintptr_t)d_bias % 16 == 0;
    if (a.vec) a.per = (a.per + 3) / 4 * 4;
    a.renormalise = r->renormalise; a.scale = r->scale;
    const cudaStream_t st = (cudaStream_t)stream;
    if (T == 0) {
        if (plan) TNNS_CUDA_TRY(cudaMemsetAsync(d_offsets, 0, (size_t)(r->experts + 1) * sizeof(int32_t), st));
        return TNNS_OK;
    }
    PlanArgs o;
    o.offsets = d_offsets; o.rows = d_rows; o.slots = d_slots; o.by_k = tnns_fastdiv((uint32_t)r->top_k);
    TNNS_FOR_DTYPE(dtype, TI, return launch_route_npl<TI>(ctx, a, o, plan, st));
}

}  // extern "C"
