// Products of quantised rows with 8-bit weights: y = PReLU(row scale * channel scale * sum q w), dense and over the places of
// every expert.
#include <algorithm>
#include <new>

#include "dtype.cuh"
#include "gemm_tc_common.cuh"
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
constexpr int MAX_EXPERTS = 1024;

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
    int dtype;
    bool y_maps;       // results may leave as tensor copies: 16 bytes may be stored at once everywhere in y
    int q_box;         // rows of a tensor copy of q
    float alpha;
    unsigned int* status;
};

// The places of an expert, [first, last).
__device__ __forceinline__ int2 places_of(const GemmI8Args& p, int e) {
    if (!p.offsets) return make_int2(0, p.places);
    const int first = min(max(p.offsets[e], 0), p.places);
    return make_int2(first, min(max(p.offsets[e + 1], first), p.places));
}
// Row of q that a place reads, -1: none (reads as zeros).
__device__ __forceinline__ int row_of(const GemmI8Args& p, int place) {
    const int r = p.rows ? p.rows[place] : place;
    return r >= 0 && r < p.q_rows ? r : -1;
}
__device__ __forceinline__ float prelu(float v, float alpha) { return v * (v > 0 ? 1.0f : alpha); }

// All lanes of a warp wait; none leaves the loop before the others.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, unsigned int* status, unsigned code) {
    return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, abort_flag, status, code));
}

// How a launch's work is dealt out: blocks of TM places of every expert, in the experts' order.  s_first[e] = blocks of the experts
// before e, s_range[e] = the expert's places; called by the whole block, ends with a barrier.  Sums saturate at `limit` (overlapping
// offsets are the caller's mistake), so that what is counted on from them stays an int.
constexpr size_t list_bytes(int experts) { return 8 * (size_t)experts + 4 * ((size_t)experts + 1); }
template <int TM>
__device__ __forceinline__ void list_blocks(const GemmI8Args& p, int2* s_range, int* s_first, unsigned limit, int tid, int threads) {
    for (int e = tid; e < p.experts; e += threads) {
        const int2 r = places_of(p, e);
        s_range[e] = r;
        s_first[e + 1] = (int)min((unsigned)(r.y - r.x) / TM + ((unsigned)(r.y - r.x) % TM != 0), limit);
    }
    if (tid == 0) s_first[0] = 0;
    __syncthreads();
    if (tid < 32) {
        int carry = 0;
        for (int e0 = 0; e0 < p.experts; e0 += 32) {
            const int e = e0 + tid;
            unsigned v = e < p.experts ? (unsigned)s_first[e + 1] : 0u;
            for (int d = 1; d < 32; d <<= 1) {
                const unsigned o = __shfl_up_sync(0xFFFFFFFFu, v, d);
                if (tid >= d) v = min(v + o, limit);
            }
            v = min(v + (unsigned)carry, limit);
            if (e < p.experts) s_first[e + 1] = (int)v;
            carry = (int)__shfl_sync(0xFFFFFFFFu, v, 31);
        }
    }
    __syncthreads();
}
// The expert that block b belongs to: the last e with s_first[e] <= b.
__device__ __forceinline__ int expert_of(const int* s_first, int experts, int b) {
    int lo = 0, hi = experts;  // s_first[lo] <= b < s_first[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_first[mid] <= b) lo = mid; else hi = mid;
    }
    return lo;
}

// ---------------------------------------------------------------------------------------
// Few rows: the weights go straight into the operand registers of the warp-level matrix instruction
// ---------------------------------------------------------------------------------------

constexpr int FEW_WARPS = 8;
__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void load_32b(const int8_t* at, uint4& lo, uint4& hi) {
    asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(lo.x), "=r"(lo.y), "=r"(lo.z), "=r"(lo.w), "=r"(hi.x), "=r"(hi.y), "=r"(hi.z), "=r"(hi.w)
                 : "l"(at));
}
// 16 bytes of a row of q from byte k on; bytes behind K, which need not be readable, as zeros.
__device__ __forceinline__ uint4 load_piece(const int8_t* row, int k, int K) {
    if (k + 16 <= K) return *reinterpret_cast<const uint4*>(row + k);
    uint32_t w[4] = {0, 0, 0, 0};
    for (int j = 0; k + j < K; j++) w[j >> 2] |= (uint32_t)(uint8_t)row[k + j] << (8 * (j & 3));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// 8 * NT places x 16 channels a warp, or S warps that share the K tiles and add up their sums in shared memory; a block holds 8 / S
// such pieces side by side and goes on to others, whose weights it requests before it finishes the present ones.  Bounded by the
// weights' bytes: a lane (g, t) holds the 32 bytes of pieces 2t and 2t + 1 of channels 2g and 2g + 1 (rows g and g + 8 of the
// instruction), so a load takes eight whole lines, four instructions multiply a K tile of 2 KB, and no byte passes through shared
// memory.  The order of K within the tile is the same for weights and rows.  1 x 4096 -> 4096: 5.0 us = 3.4 TB/s (launches
// back to back, weights from memory), of which the launch and the first bytes' way take 2.4.
template <int NT, int U>  // U: K tiles whose loads a warp issues together
__global__ void __launch_bounds__(FEW_WARPS * 32, 2) gemm_i8_few_kernel(const __grid_constant__ GemmI8Args p, int log_s) {
    extern __shared__ int2 s_range[];
    int* s_first = reinterpret_cast<int*>(s_range + p.experts);
    __shared__ int s_sum[FEW_WARPS][NT][16 * 8];
    __shared__ float s_scale[2][8 * NT];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int S = 1 << log_s, ks = warp & (S - 1), log_wide = 7 - log_s, wide = 1 << log_wide;  // this warp's part of K, channels of a block ..
    const int n_mine = (warp >> log_s) * 16, n_out = tid & (wide - 1);                          // .. the first the warp multiplies, the one the thread finishes
    const int n_blocks = (p.N + wide - 1) >> log_wide;
    struct Item {
        int e, m0, last, n0;  // expert, first place, end of the expert's places, first channel of the block
    };
    const int8_t* wt = nullptr;
    uint4 a[U][4], x[U][NT][2];
    int row[NT];     // of q, that the lane's places read; -1: none
    float rs[NT], ws = 0.f;  // scales of those rows, of channel n_out
    auto load_weights = [&](int kt0) {
#pragma unroll
        for (int u = 0; u < U; u++)
            if (kt0 + u * S < p.k_tiles) {
                const int8_t* tile = wt + (long long)(kt0 + u * S) * WT_BYTES;
                load_32b(tile, a[u][0], a[u][1]);        // channel 2g: pieces 2t, 2t + 1
                load_32b(tile + 128, a[u][3], a[u][2]);  // channel 2g + 1: the pattern has the two the other way round
            }
    };
    auto begin_weights = [&](int e, int n0) {
        if (n0 + n_out < p.N) ws = __ldg(p.w_scale + (long long)e * p.n_tiles * WT + n0 + n_out);
        const int n = n0 + n_mine;
        if (n >= p.N) return;
        wt = p.img + ((long long)e * p.n_tiles + n / WT) * p.k_tiles * WT_BYTES + (n % WT + 2 * g) * 128 + ((t ^ (g & 3)) << 5);
        load_weights(ks);
    };
    auto load_x = [&](int kt0) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int k0 = (kt0 + u * S) * WT;
#pragma unroll
            for (int i = 0; i < NT; i++) {
                const int8_t* at = p.q + (long long)max(row[i], 0) * p.q_stride;
                if (k0 + WT <= p.K) {  // a whole tile
                    x[u][i][0] = row[i] >= 0 ? *reinterpret_cast<const uint4*>(at + k0 + t * 32) : make_uint4(0, 0, 0, 0);
                    x[u][i][1] = row[i] >= 0 ? *reinterpret_cast<const uint4*>(at + k0 + t * 32 + 16) : make_uint4(0, 0, 0, 0);
                } else {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int k = k0 + t * 32 + h * 16;
                        x[u][i][h] = row[i] >= 0 && k < p.K ? load_piece(at, k, p.K) : make_uint4(0, 0, 0, 0);
                    }
                }
            }
        }
    };
    auto begin_rows = [&]() {
        load_x(ks);
#pragma unroll
        for (int i = 0; i < NT; i++) rs[i] = row[i] >= 0 ? p.scale[row[i]] : 0.f;
    };
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // one kernel: the weights' way from memory starts before the launch in front has ended
    if (!p.offsets) begin_weights(0, (int)(blockIdx.x % (unsigned)n_blocks) << log_wide);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    list_blocks<8 * NT>(p, s_range, s_first, 0x7FFFFFFFu / n_blocks / 2, tid, FEW_WARPS * 32);
    const int items = s_first[p.experts] * n_blocks;
    auto item_at = [&](int item) {
        Item r;
        const int b = item / n_blocks;
        r.n0 = (item - b * n_blocks) << log_wide;
        r.e = p.experts == 1 ? 0 : expert_of(s_first, p.experts, b);
        const int2 range = s_range[r.e];
        r.m0 = range.x + (b - s_first[r.e]) * 8 * NT;
        r.last = range.y;
        return r;
    };
    auto rows_at = [&](const Item& c) {
#pragma unroll
        for (int i = 0; i < NT; i++) {
            const int place = c.m0 + i * 8 + g;
            row[i] = place < c.last ? row_of(p, place) : -1;
        }
    };
    Item c = {};
    if ((int)blockIdx.x < items) {
        c = item_at(blockIdx.x);
        rows_at(c);
        if (p.offsets) begin_weights(c.e, c.n0);
        begin_rows();
    }
    for (int item = blockIdx.x, turn = 0; item < items; item += gridDim.x, turn ^= 1) {
        const Item now = c;
        const bool more = item + (int)gridDim.x < items;
        int acc[NT][4] = {};
        if (now.n0 + n_mine < p.N) {
            for (int kt0 = ks; kt0 < p.k_tiles; kt0 += S * U) {
                if (kt0 != ks) load_x(kt0);
#pragma unroll
                for (int u = 0; u < U; u++)
                    if (kt0 + u * S < p.k_tiles) {
#pragma unroll
                        for (int i = 0; i < NT; i++) {
                            mma_s8(acc[i], a[u][0].x, a[u][2].x, a[u][1].x, a[u][3].x, x[u][i][0].x, x[u][i][1].x);
                            mma_s8(acc[i], a[u][0].y, a[u][2].y, a[u][1].y, a[u][3].y, x[u][i][0].y, x[u][i][1].y);
                            mma_s8(acc[i], a[u][0].z, a[u][2].z, a[u][1].z, a[u][3].z, x[u][i][0].z, x[u][i][1].z);
                            mma_s8(acc[i], a[u][0].w, a[u][2].w, a[u][1].w, a[u][3].w, x[u][i][0].w, x[u][i][1].w);
                        }
                    }
                load_weights(kt0 + S * U);
            }
        }
        // d[0], d[1]: channel 2g, places 2t, 2t + 1; d[2], d[3]: channel 2g + 1
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) s_sum[warp][i][(2 * t + (j & 1)) * 16 + 2 * g + (j >> 1)] = acc[i][j];
        if (warp == 0 && t == 0) {
#pragma unroll
            for (int i = 0; i < NT; i++) s_scale[turn][i * 8 + g] = rs[i];
        }
        const float ws_now = ws;
        if (more) {
            c = item_at(item + gridDim.x);
            rows_at(c);
            begin_weights(c.e, c.n0);
        }
        __syncthreads();
        // a result for each place and channel of the block, channels side by side
        if (now.n0 + n_out < p.N)
            for (int pl = tid >> log_wide; pl < 8 * NT && now.m0 + pl < now.last; pl += FEW_WARPS * 32 >> log_wide) {
                int sum = 0;
                for (int w = 0; w < S; w++) sum += s_sum[((n_out >> 4) << log_s) + w][pl >> 3][(pl & 7) * 16 + (n_out & 15)];
                const float v = prelu((float)sum * s_scale[turn][pl] * ws_now, p.alpha);
                const long long at = (long long)(now.m0 + pl) * p.y_stride + now.n0 + n_out;
                if (p.dtype == TNNS_F32) ((float*)p.y)[at] = v;
                else if (p.dtype == TNNS_F16) ((__half*)p.y)[at] = __float2half_rn(v);
                else ((__nv_bfloat16*)p.y)[at] = __float2bfloat16_rn(v);
            }
        if (more) begin_rows();
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------------------
// Many rows: 5th-generation tensor cores, accumulators in tensor memory
// ---------------------------------------------------------------------------------------

// Stages of 128 bytes of K: 128 rows of q (one tensor copy, or 16-byte copies by the gather warps where places name their rows) and
// BN / CG channels of weights (contiguous copies of the tiled image).
template <int BN, int CG, bool GATHER, int CS>
struct TcI8 {
    static constexpr int A_STAGE = BM * KCH, B_STAGE = BN / CG * KCH, STAGE = A_STAGE + B_STAGE;
    static constexpr int NSTG = 5 * 32768 / STAGE;
    static constexpr int NBUF = 2;  // accumulator sets
    static constexpr int COLS = NBUF * BN < 32 ? 32 : NBUF * BN;
    static constexpr int GATHER0 = 2, GATHER_WARPS = GATHER ? 6 : 2, EPI0 = GATHER0 + GATHER_WARPS;  // (EPI0: a multiple of four)
    static constexpr int EPI_WARPS = BN == 64 ? 8 : 16, HN = BN / (EPI_WARPS / 4), THREADS = 32 * (EPI0 + EPI_WARPS);  // HN: channels of an epilogue warp
    static constexpr int BARS = 2 * NSTG + 2 * NBUF;
    static constexpr int STAGED = 16;  // words of a row of a warp's buffer for results on their way out
    static constexpr int SHARED_SUMS = (CS - 1) * (BN / CS) * BM;  // words that the cluster's other blocks send
    static constexpr int OUT = EPI_WARPS * 32 * STAGED > SHARED_SUMS ? EPI_WARPS * 32 * STAGED : SHARED_SUMS;
    static constexpr size_t smem(int experts) { return 1024 + (size_t)NSTG * STAGE + 8 * BARS + 16 + (OUT + EPI_WARPS * HN) * 4 + list_bytes(experts); }
    static_assert(CS == 1 || (CG == 1 && !GATHER && HN == 32 && BN % (32 * CS) == 0), "shares: single blocks, whole warps of channels");
    static_assert(!GATHER || NSTG <= GATHER_WARPS, "a gather warp for every slot");
};
struct alignas(64) MapsI8 {
    CUtensorMap q, w, y;
};
__device__ __forceinline__ void tc_mma_i8_lh(uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %2};\n\t"
        "mov.b64 db, {%3, %4};\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], da, db, %5, p;\n\t}"
        ::"r"(d_tmem), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tc_mma_i8_pair_lh(uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %2};\n\t"
        "mov.b64 db, {%3, %4};\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], da, db, %5, p;\n\t}"
        ::"r"(d_tmem), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
        : "memory");
}
// 16 bytes from global to shared memory, of which the first `bytes` are fetched and the rest are zeros.
__device__ __forceinline__ void copy16_async(uint32_t dst_smem, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst_smem), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void tmem_ld_32(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
          "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]),
          "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr));
}
// 64 bytes of each of a warp's rows to y: w = those of the lane's row; they leave through the warp's 32 x 64 bytes of shared memory,
// the 16-byte pieces of a row in the pattern piece ^ (row / 2) % 4 (the copy engine's 64-byte swizzle, free of bank conflicts).
// Whole blocks go out as one tensor copy where y allows it (maps: 16 bytes may be stored at once everywhere in y; a copy that
// ends inside 16 bytes of a row would write all of them).  A store by lanes, each 32 bytes of its own row, took 32 bytes a clock off the
// path that also feeds the tensor core: 65536 x 1024 -> 2048 bf16 in 134 us against 118, fp32 177 against 143.  The rest the warp writes
// along the rows (4096 x 1024 -> 4097: 37 us, by lanes 190).  x, row0: first byte of the row, first row; have: bytes of a row that exist
// (a multiple of `size`, an element's bytes); step: bytes from row to row.
__device__ __forceinline__ void store_rows(const uint32_t (&w)[16], uint32_t* stage, const void* tmap, unsigned char* base, int x, int row0, long long step, int rows,
                                           int have, bool maps, int size, int lane) {
    auto at = [&](int row, int word) { return stage + row * 16 + ((((word >> 2) ^ (row >> 1)) & 3) << 2) + (word & 3); };
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // the copy before has read the buffer
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16; i += 4) *reinterpret_cast<uint4*>(at(lane, i)) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
    if (maps && rows == 32 && have == 64) {
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
            asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(reinterpret_cast<uint64_t>(tmap)), "r"(smem_u32(stage)), "r"(x), "r"(row0)
                         : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
        return;
    }
    __syncwarp();
    // half a warp a row; rows that all start on a word without a neighbour's half (one loop for both kinds: 11364 x 129 -> 2118 39.8 us against 32.9)
    const int col = lane & 15, half = lane >> 4;
    unsigned char* y = base + (long long)(row0 + half) * step + x;
    if (size == 4 || ((reinterpret_cast<uintptr_t>(base) | step) & 2) == 0) {
        for (int r = half; r < rows; r += 2, y += 2 * step) {
            const uint32_t v = *at(r, col);
            if (4 * col + 4 <= have) *reinterpret_cast<uint32_t*>(y + 4 * col) = v;
            else if (4 * col + 2 <= have) *reinterpret_cast<uint16_t*>(y + 4 * col) = (uint16_t)v;
        }
        return;
    }
#pragma unroll 4
    for (int r0 = 0; r0 < 32; r0 += 2, y += 2 * step) {
        const bool there = r0 + half < rows, odd = reinterpret_cast<uintptr_t>(y) & 2;
        const uint32_t v = *at(r0 + half, col), next = __shfl_down_sync(0xFFFFFFFFu, v, 1);
        // a row that starts between two words: the halves of neighbours together, the first and the last by themselves
        const int from = odd ? 2 : 0;  // the lane's word begins so many bytes behind its own column
        const uint32_t w4 = odd ? __funnelshift_r(v, next, 16) : v;
        if (there && 4 * col + 4 + from <= have) *reinterpret_cast<uint32_t*>(y + 4 * col + from) = w4;
        else if (there && 4 * col + 2 + from <= have) *reinterpret_cast<uint16_t*>(y + 4 * col + from) = (uint16_t)w4;
        if (there && odd && col == 0) *reinterpret_cast<uint16_t*>(y) = (uint16_t)v;
    }
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
// Two neighbouring results of a row: the row's scale, the channels' scales, PReLU (slope between 0 and 1: the larger of v and
// alpha * v; mode 0: none, 1: that, 2: any slope).
__device__ __forceinline__ float2 finish_pair(uint32_t a0, uint32_t a1, float rs, float2 ws, float alpha, int mode) {
    float2 f = mul2(mul2(make_float2((float)(int)a0, (float)(int)a1), make_float2(rs, rs)), ws);
    if (mode == 1) {
        const float2 g = mul2(f, make_float2(alpha, alpha));
        f = make_float2(fmaxf(f.x, g.x), fmaxf(f.y, g.y));
    } else if (mode == 2) {
        f = make_float2(prelu(f.x, alpha), prelu(f.y, alpha));
    }
    return f;
}
// C accumulators of the lane's row (64 bytes of results) -> words.
template <int C>
__device__ __forceinline__ void finish_words(int dtype, const uint32_t* v, float rs, const float* ws, float alpha, int mode, uint32_t (&w)[16]) {
#pragma unroll
    for (int j = 0; j < C; j += 4) {
        const float4 w4 = *reinterpret_cast<const float4*>(ws + j);
        const float2 a = finish_pair(v[j], v[j + 1], rs, make_float2(w4.x, w4.y), alpha, mode), b = finish_pair(v[j + 2], v[j + 3], rs, make_float2(w4.z, w4.w), alpha, mode);
        if (C == 16) {
            w[j] = __float_as_uint(a.x);
            w[(j + 1) % 16] = __float_as_uint(a.y);
            w[(j + 2) % 16] = __float_as_uint(b.x);
            w[(j + 3) % 16] = __float_as_uint(b.y);
        } else if (dtype == TNNS_F16) {
            const __half2 x = __floats2half2_rn(a.x, a.y), y = __floats2half2_rn(b.x, b.y);
            w[j / 2] = *reinterpret_cast<const uint32_t*>(&x);
            w[j / 2 + 1] = *reinterpret_cast<const uint32_t*>(&y);
        } else {
            const __nv_bfloat162 x = __floats2bfloat162_rn(a.x, a.y), y = __floats2bfloat162_rn(b.x, b.y);
            w[j / 2] = *reinterpret_cast<const uint32_t*>(&x);
            w[j / 2 + 1] = *reinterpret_cast<const uint32_t*>(&y);
        }
    }
}

// 32 x 32 accumulators of a warp, from place place0 and channel n on: scaled, rounded and stored.
__device__ __forceinline__ void store_chunk(const GemmI8Args& p, const MapsI8& maps, const uint32_t (&v)[32], float rs, const float* ws, int mode, uint32_t* stage, int n,
                                            int place0, int rows, int size, int lane) {
    const int have = (p.N - n) * size, x = n * size;
    if (rows <= 0 || have <= 0) return;
    const long long step = p.y_stride * size;
    unsigned char* base = reinterpret_cast<unsigned char*>(p.y);
    uint32_t w[16];
    if (size == 4) {
        finish_words<16>(p.dtype, v, rs, ws, p.alpha, mode, w);
        store_rows(w, stage, &maps.y, base, x, place0, step, rows, min(have, 64), p.y_maps, 4, lane);
        if (have > 64) {
            finish_words<16>(p.dtype, v + 16, rs, ws + 16, p.alpha, mode, w);
            store_rows(w, stage, &maps.y, base, x + 64, place0, step, rows, min(have - 64, 64), p.y_maps, 4, lane);
        }
    } else {
        finish_words<32>(p.dtype, v, rs, ws, p.alpha, mode, w);
        store_rows(w, stage, &maps.y, base, x, place0, step, rows, min(have, 64), p.y_maps, 2, lane);
    }
}

// One persistent block (CG = 1) or pair of blocks (CG = 2, tcgen05.mma.cta_group::2: 256 rows, each block holds its 128 rows and half
// of the channels) an SM or pair of SMs, over tiles of CG * 128 places x BN channels.  Warp 0 requests the copies, warp 1 issues the
// MMAs, where places name their rows a warp for every slot of the ring gathers them (so that all are on their way at once; of six such
// warps the last stands idle where the ring has five slots), and sixteen
// (tiles of 64 channels: eight) scale, round and store one accumulator while the MMAs fill the other.
// Large products are bound by the tensor pipe at the clock that the power limit leaves: 8192 x 4096 -> 8192 in 170 us, 3.2 POP/s, 0.98 of
// twice the measured bf16 rate (its pipe 75 % active by count: operands come in and go to the pipe at 127 of the shared memory's 128
// bytes a clock).  Short sums are bound by what their results add to that path: 65536 x 1024 -> 2048 118 us, 82 without results.
// Rows by gathering tensor copies, four a request, took 80 clocks a request of 512 bytes: 8192 tokens by 8 of 64 experts, 2048 -> 1024, 360
// us against 128 by the warps.
//
// Where tiles are few and K is long, a cluster of CS blocks shares a tile (one a cluster): each multiplies its part of the K tiles, sends
// the sums of the channels that others finish into their shared memory, adds what comes to its own 1 / CS of the channels and finishes
// those.  Sums of integers: the result is the same whichever blocks form it.  The exchange (a cluster's start, its barrier, 16 KB from
// each block for every 32 channels of another) takes about 2.5 us, a K tile of a lone block 0.2: 128 x 8192 -> 2048 17.7 us alone, 11.0 by four.
template <int BN, int CG, bool GATHER, int CS = 1>
__global__ void __launch_bounds__(TcI8<BN, CG, GATHER, CS>::THREADS, 1) gemm_i8_tc_kernel(const __grid_constant__ GemmI8Args p, const __grid_constant__ MapsI8 maps) {
    using Cfg = TcI8<BN, CG, GATHER, CS>;
    constexpr int NSTG = Cfg::NSTG, NBUF = Cfg::NBUF, TM = CG * BM;
    // s32 accumulators, signed 8-bit operands, both K-major, N >> 3 at bit 17, M >> 4 at bit 24
    constexpr uint32_t IDESC = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(TM >> 4) << 24);
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char *sA = smem, *sB = smem + NSTG * Cfg::A_STAGE;
    uint32_t* s_stage = reinterpret_cast<uint32_t*>(smem + NSTG * Cfg::STAGE);              // [epilogue warp][32][STAGED]
    float* s_ws = reinterpret_cast<float*>(s_stage + Cfg::OUT);                               // [epilogue warp][HN]: its channels' scales
    uint64_t* bars = reinterpret_cast<uint64_t*>(s_ws + Cfg::EPI_WARPS * Cfg::HN);
    const uint32_t bar_full = smem_u32(bars), bar_empty = bar_full + 8 * NSTG, bar_tfull = bar_empty + 8 * NSTG, bar_tempty = bar_tfull + 8 * NBUF;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + Cfg::BARS);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int2* s_range = reinterpret_cast<int2*>(tmem_slot + 4);
    int* s_first = reinterpret_cast<int*>(s_range + p.experts);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = CG == 2 ? cluster_ctarank() : 0u;
    const int unit = blockIdx.x / (CG * CS), units = gridDim.x / (CG * CS);
    const int share = CS > 1 ? (int)cluster_ctarank() : 0, k0 = p.k_tiles * share / CS, k1 = p.k_tiles * (share + 1) / CS;  // the block's K tiles
    float share_rs = 0.f;
    // OWN chunks of 32 channels are the block's to finish.  4 KB for a warp's chunk from each of the other blocks, those of one warp together;
    // 16 bytes a lane, so that a warp's are next to each other.
    constexpr int OWN = BN >= 32 * CS ? BN / 32 / CS : 1;
    auto sums_at = [&](int chunk, int q, int from) {
        return smem_u32(s_stage) + (((chunk % OWN) * 4 + q) * (CS - 1) + (from - chunk / OWN - 1 + CS) % CS) * 4096 + lane * 16;
    };

    if (tid == 0) {
        for (int s = 0; s < NSTG; s++) {
            mbar_init(bar_full + 8 * s, GATHER ? 1 + CG : 1);  // the copies' bytes, and a gather warp of each block
            mbar_init(bar_empty + 8 * s, 1);
        }
        for (int b = 0; b < NBUF; b++) {
            mbar_init(bar_tfull + 8 * b, 1);
            mbar_init(bar_tempty + 8 * b, CG * Cfg::EPI_WARPS);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        prefetch_tensor_map(&maps.q);
        if (CG == 2) prefetch_tensor_map(&maps.w);
    }
    __syncwarp();
    if (warp == WARP_MMA) {
        if (CG == 2) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)Cfg::COLS) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)Cfg::COLS) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    }
    tc_fence_before();
    if (CG * CS > 1) cluster_sync_all(); else __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    // what follows reads and writes tensors that the launch in front may still be working on
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int n_blocks = (p.N + BN - 1) / BN;
    list_blocks<TM>(p, s_range, s_first, 0x7FFFFFFFu / n_blocks / 2, tid, Cfg::THREADS);
    const int tiles = s_first[p.experts] * n_blocks;
    struct Tile {
        int e, m0, last, n;  // expert, first place, end of the expert's places, block of channels
    };
    // within an expert tiles run down RG row blocks before they move one block of channels on: what the SMs hold at one time is then
    // about square, so that rows and weights both come out of L2
    constexpr int RG = 8;
    auto tile_at = [&](int t) {
        const int b = t / n_blocks;
        Tile r;
        r.e = p.experts == 1 ? 0 : expert_of(s_first, p.experts, b);
        const int2 range = s_range[r.e];
        const int before = s_first[r.e], blocks = s_first[r.e + 1] - before, local = t - before * n_blocks;
        const int grp = (b - before) / RG, in = local - grp * RG * n_blocks;
        const int high = min(RG, blocks - grp * RG);
        r.n = in / high;
        r.m0 = range.x + (grp * RG + in - r.n * high) * TM;
        r.last = range.y;
        return r;
    };

    const uint32_t full_lead = CG == 2 ? mapa_shared(bar_full, 0) : bar_full;
    if (warp == WARP_TMA) {
        if (lane == 0) {
            // this thread's instructions stand between a slot that is free and its copies: what does not change from stage to stage is
            // formed once a tile
            constexpr int PARTS = BN / CG < WT ? 1 : BN / CG / WT, HIGH = BN / CG < WT ? BN / CG : WT;  // tiles of weights a stage takes, their channels
            const uint32_t a_smem = smem_u32(sA), b_smem = smem_u32(sB);
            uint32_t s = 0, ph = 1;
            for (int t = unit; t < tiles; t += units) {
                const Tile c = tile_at(t);
                const int n0 = c.n * BN + (int)rank * (BN / CG), m = c.m0 + (int)rank * BM;
                // whole boxes that hold the tile's rows (what else the stage holds is multiplied and not stored); the first block counts both
                auto boxes = [&](int first) { return GATHER ? 0 : min(max((c.last - first + p.q_box - 1) / p.q_box, 0), BM / p.q_box); };
                const int mine = boxes(m), box_bytes = p.q_box * KCH;
                const uint32_t bytes = CG * Cfg::B_STAGE + (uint32_t)((mine + (CG == 2 ? boxes(m + BM) : 0)) * box_bytes);
                // a tile of channels past the last repeats the last one: its results are not stored
                long long tile[PARTS];
#pragma unroll
                for (int n = 0; n < PARTS; n++) tile[n] = ((long long)c.e * p.n_tiles + min((n0 + n * WT) / WT, p.n_tiles - 1)) * p.k_tiles;
                const int8_t* src[PARTS];
                int w_row[PARTS];
#pragma unroll
                for (int n = 0; n < PARTS; n++) {
                    src[n] = p.img + (tile[n] + k0) * WT_BYTES + (n0 % WT) * KCH;
                    w_row[n] = (int)(tile[n] * WT + n0 % WT);
                }
                for (int kt = k0; kt < k1; kt++) {
                    if (!mbar_wait(bar_empty + 8 * s, ph, abort_flag, p.status, 1)) goto done;
                    const uint32_t bar = full_lead + 8 * s, a_dst = a_smem + s * Cfg::A_STAGE, b_dst = b_smem + s * Cfg::B_STAGE;
                    if (rank == 0) mbar_arrive_expect_tx(bar_full + 8 * s, bytes);
#pragma unroll
                    for (int n = 0; n < PARTS; n++) {
                        if (CG == 2) tma_tile2d_g2s_pair(b_dst + n * HIGH * KCH, &maps.w, 0, w_row[n], bar);
                        else bulk_g2s(b_dst + n * HIGH * KCH, src[n], HIGH * KCH, bar);
                        src[n] += WT_BYTES;
                        w_row[n] += WT;
                    }
                    if (!GATHER && mine) {
                        if (CG == 2) tma_tile2d_g2s_pair(a_dst, &maps.q, kt * KCH, m, bar);
                        else tma_tile2d_g2s(a_dst, &maps.q, kt * KCH, m, bar);
                        for (int i = 1; i < mine; i++) {
                            if (CG == 2) tma_tile2d_g2s_pair(a_dst + i * box_bytes, &maps.q, kt * KCH, m + i * p.q_box, bar);
                            else tma_tile2d_g2s(a_dst + i * box_bytes, &maps.q, kt * KCH, m + i * p.q_box, bar);
                        }
                    }
                    if (++s == NSTG) { s = 0; ph ^= 1; }
                }
            }
        }
    } else if (warp == WARP_MMA) {
        if (rank == 0) {
            const bool elected = elect_one();
            const uint64_t da0 = make_desc(smem_u32(sA)), db0 = make_desc(smem_u32(sB));
            const uint32_t a_lo0 = (uint32_t)da0, a_hi = (uint32_t)(da0 >> 32), b_lo0 = (uint32_t)db0, b_hi = (uint32_t)(db0 >> 32);
            uint32_t a_lo = a_lo0, b_lo = b_lo0, s = 0, ph = 0, lt = 0;
            for (int t = unit; t < tiles; t += units, lt++) {
                const uint32_t buf = lt % NBUF;
                if (!warp_wait(bar_tempty + 8 * buf, ((lt / NBUF) & 1) ^ 1, abort_flag, p.status, 2)) goto done;
                tc_fence_after();
                const uint32_t d = tmem_base + buf * BN;
                for (int kt = k0; kt < k1; kt++) {
                    if (!warp_wait(bar_full + 8 * s, ph, abort_flag, p.status, 3)) goto done;
                    tc_fence_after();
                    if (elected) {
#pragma unroll
                        for (int k = 0; k < KCH / 32; k++) {
                            if (CG == 2) tc_mma_i8_pair_lh(d, a_lo + 2 * k, a_hi, b_lo + 2 * k, b_hi, IDESC, (uint32_t)((kt - k0) | k));
                            else tc_mma_i8_lh(d, a_lo + 2 * k, a_hi, b_lo + 2 * k, b_hi, IDESC, (uint32_t)((kt - k0) | k));
                        }
                        if (CG == 2) tc_commit_pair(bar_empty + 8 * s); else tc_commit(bar_empty + 8 * s);
                    }
                    if (++s == NSTG) { s = 0; ph ^= 1; a_lo = a_lo0; b_lo = b_lo0; }
                    else { a_lo += Cfg::A_STAGE >> 4; b_lo += Cfg::B_STAGE >> 4; }
                }
                if (elected) {
                    if (CG == 2) tc_commit_pair(bar_tfull + 8 * buf); else tc_commit(bar_tfull + 8 * buf);
                }
            }
        }
    } else if (warp < Cfg::EPI0) {
        if (GATHER) {
            // Stage i of the block's sequence belongs to gather warp i % NSTG, and so does its slot of the ring: a warp's successive waits on a
            // slot's barrier are then successive phases, which is all that a parity tells apart.  (Six warps on five slots met a slot again
            // one lap early and wrote over a stage that was still to be read; the launch failed.)
            constexpr int GW = NSTG;
            const int own = warp - Cfg::GATHER0;
            uint32_t first = 0;  // stages of the tiles before this one, modulo GW and modulo 2 * NSTG
            uint32_t slot0 = 0;
            const uint32_t step = (uint32_t)p.k_tiles;
            for (int t = unit; t < tiles; t += units, first = (first + step) % GW, slot0 = (slot0 + step) % (2 * NSTG)) {
                int kt = (own + GW - (int)first) % GW;
                if (own >= GW || kt >= p.k_tiles) continue;
                const Tile c = tile_at(t);
                int r[4];  // rows lane, lane + 32, .. of the block's 128; -1: zeros
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int place = c.m0 + (int)rank * BM + 32 * i + lane;
                    r[i] = place < c.last ? row_of(p, place) : -1;
                }
                for (; kt < p.k_tiles; kt += GW) {
                    const uint32_t at = (slot0 + (uint32_t)kt) % (2 * NSTG), s = at % NSTG;
                    if (!warp_wait(bar_empty + 8 * s, at < NSTG ? 1u : 0u, abort_flag, p.status, 5)) goto done;
                    const int sub = lane >> 3, piece = lane & 7;  // of four rows an instruction: the row, and its 16-byte piece
                    const int k = kt * KCH + piece * 16, have = min(max(p.K - k, 0), 16);
                    const uint32_t a_dst = smem_u32(sA + s * Cfg::A_STAGE);
#pragma unroll
                    for (int i = 0; i < 32; i++) {
                        const int row = 4 * i + sub, src = __shfl_sync(0xFFFFFFFFu, r[i >> 3], row & 31);
                        copy16_async(a_dst + row * KCH + ((piece ^ (row & 7)) << 4), p.q + (have ? (long long)max(src, 0) * p.q_stride + k : 0), src >= 0 ? have : 0);
                    }
                    asm volatile("cp.async.wait_all;" ::: "memory");
                    fence_proxy_async();  // what this thread wrote, before the tensor core's reads
                    __syncwarp();
                    if (lane == 0) {
                        if (CG == 2) mbar_arrive_cluster(full_lead + 8 * s); else mbar_arrive(bar_full + 8 * s);
                    }
                }
            }
        }
    } else {
        const int q = warp & 3, part = (warp - Cfg::EPI0) >> 2;
        constexpr int HN = Cfg::HN, NC = HN / 32;  // channels of the part, in chunks of 32
        const uint32_t tempty_lead = CG == 2 ? mapa_shared(bar_tempty, 0) : bar_tempty;
        uint32_t* stage = s_stage + (warp - Cfg::EPI0) * 32 * Cfg::STAGED;
        const int mode = p.alpha == 1.0f ? 0 : p.alpha > 0.0f && p.alpha < 1.0f ? 1 : 2;
        // what a tile's results are scaled with is fetched while the tile before is on its way out
        Tile c = {};
        int row = -1;
        float rs = 0.f, ws[NC];
        float* wsc = s_ws + (warp - Cfg::EPI0) * HN;
        auto fetch = [&](int t) {
            c = tile_at(t);
            const int place = c.m0 + (int)rank * BM + q * 32 + lane, n = c.n * BN + part * HN + lane;
            row = place < c.last ? row_of(p, place) : -1;
#pragma unroll
            for (int i = 0; i < NC; i++) ws[i] = n + 32 * i < p.N ? __ldg(p.w_scale + (long long)c.e * p.n_tiles * WT + n + 32 * i) : 0.f;
        };
        if (unit < tiles) {
            fetch(unit);
            rs = row >= 0 ? p.scale[row] : 0.f;
        }
        uint32_t lt = 0;
        for (int t = unit; t < tiles; t += units, lt++) {
            const uint32_t buf = lt % NBUF;
            __syncwarp();
#pragma unroll
            for (int i = 0; i < NC; i++) wsc[32 * i + lane] = ws[i];
            __syncwarp();
            const Tile now = c;
            const float rs_now = rs;
            const int place0 = now.m0 + (int)rank * BM + q * 32, rows_here = min(32, now.last - place0);
            if (!warp_wait(bar_tfull + 8 * buf, (lt / NBUF) & 1, abort_flag, p.status, 4)) goto done;
            tc_fence_after();
            if (CS > 1) {  // the only tile
                share_rs = rs;
                if (part / OWN != share) {
                    uint32_t v[32];
                    tmem_ld_32(tmem_base + ((uint32_t)(q * 32) << 16) + part * 32, v);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    const uint32_t dst = mapa_shared(sums_at(part, q, share), (uint32_t)(part / OWN));
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + j * 512), "r"(v[4 * j]), "r"(v[4 * j + 1]), "r"(v[4 * j + 2]), "r"(v[4 * j + 3]) : "memory");
                }
                continue;
            }
            if (t + units < tiles) fetch(t + units);
            const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16) + buf * BN + part * HN;
            const int n0 = now.n * BN + part * HN, size = p.dtype == TNNS_F32 ? 4 : 2;
#pragma unroll 1
            for (int i = 0; i < NC; i++) {
                uint32_t v[32];
                tmem_ld_32(taddr + 32 * i, v);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                if (i + 1 == NC) {  // the last columns are in registers: the accumulator may be written again
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        if (CG == 2) mbar_arrive_cluster(tempty_lead + 8 * buf); else mbar_arrive(bar_tempty + 8 * buf);
                    }
                }
                if (i == 0) rs = row >= 0 ? p.scale[row] : 0.f;  // the next tile's
                store_chunk(p, maps, v, rs_now, wsc + 32 * i, mode, stage, n0 + 32 * i, place0, rows_here, size, lane);
                __syncwarp();
            }
        }
    }

done:
    __syncwarp();
    if (*abort_flag && warp == WARP_TMA && lane == 0) {
        // a wait gave up: give the copies already requested time to land before shared memory is released
        for (int i = 0; i < 1000; i++) __nanosleep(1000);
    }
    if (CS > 1) {
        __syncwarp();
        tc_fence_before();
        cluster_sync_all();
        tc_fence_after();
        const int q = warp & 3, chunk = (warp - Cfg::EPI0) >> 2;
        if (warp >= Cfg::EPI0 && chunk / OWN == share && unit < tiles && !*abort_flag) {
            uint32_t v[32];
            tmem_ld_32(tmem_base + ((uint32_t)(q * 32) << 16) + chunk * 32, v);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll 1
            for (int i = 1; i < CS; i++) {
                const uint32_t src = sums_at(chunk, q, (share + i) % CS);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    uint32_t x[4];
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(src + j * 512) : "memory");
#pragma unroll
                    for (int k = 0; k < 4; k++) v[4 * j + k] += x[k];
                }
            }
            __syncwarp();  // the sums are read: their place is the buffer for results
            const Tile c = tile_at(unit);
            const int n0 = c.n * BN + chunk * 32, place0 = c.m0 + q * 32, rows_here = min(32, c.last - place0), size = p.dtype == TNNS_F32 ? 4 : 2;
            const int mode = p.alpha == 1.0f ? 0 : p.alpha > 0.0f && p.alpha < 1.0f ? 1 : 2;
            store_chunk(p, maps, v, share_rs, s_ws + (warp - Cfg::EPI0) * 32, mode, s_stage + ((chunk % OWN) * 4 + q) * (CS - 1) * 1024, n0, place0, rows_here, size, lane);
        }
        __syncwarp();
    }
    if (warp >= Cfg::EPI0 && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");  // results still on their way out of shared memory
    tc_fence_before();
    if (CG == 2) cluster_sync_all(); else __syncthreads();
    if (warp == WARP_MMA) {
        tc_fence_after();
        if (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)Cfg::COLS) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)Cfg::COLS) : "memory");
    }
}

template <typename... Args>
int launch(void (*kern)(Args...), tnns_cuda_ctx* ctx, int grid, int threads, size_t smem, int cluster, cudaStream_t stream, Args... args) {
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

template <int BN, int CG, bool GATHER, int CS = 1>
int launch_tc(tnns_cuda_ctx* ctx, const GemmI8Args& a, cudaStream_t stream) {
    using Cfg = TcI8<BN, CG, GATHER, CS>;
    MapsI8 maps = {};
    int rc = tnns_tensor_map_2d(&maps.q, 1, a.q, (unsigned long long)a.K, (unsigned long long)a.q_rows, (unsigned long long)a.q_stride, KCH, a.q_box, 128);
    if (rc) return rc;
    // the weights' tiles hold the swizzle pattern already: plain rows of 128 bytes
    if (CG == 2 && (rc = tnns_tensor_map_2d(&maps.w, 1, a.img, KCH, (unsigned long long)a.experts * a.n_tiles * a.k_tiles * WT, KCH, KCH, BN / CG))) return rc;
    // y by bytes: boxes of 32 rows x 64 bytes
    if (a.y_maps) {
        const int size = tnns_dtype_bytes(a.dtype);
        if ((rc = tnns_tensor_map_2d(&maps.y, 1, a.y, (unsigned long long)a.N * size, (unsigned long long)a.places, (unsigned long long)a.y_stride * size, 64, 32, 64))) return rc;
    }
    auto kern = gemm_i8_tc_kernel<BN, CG, GATHER, CS>;
    static bool smem_set[64] = {false};  // the attribute belongs to (function, device)
    if (!smem_set[ctx->device & 63]) {
        TNNS_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Cfg::smem(MAX_EXPERTS)));
        smem_set[ctx->device & 63] = true;
    }
    const long long n_blocks = (a.N + BN - 1) / BN;
    const long long most = ((long long)a.places + CG * BM - 1) / (CG * BM) + (a.offsets ? std::min(a.experts, a.places) : 0);
    if (most * n_blocks >= 0x3FFFFFFFLL) return tnns_fail(TNNS_ERR_UNSUPPORTED, "too many tiles: %d places of %d channels", a.places, a.N);
    // shares (CS > 1): a cluster for every tile
    const int grid = CG * CS * (int)(CS > 1 ? most * n_blocks : std::min<long long>(most * n_blocks, ctx->sm_count / CG));
    return launch<GemmI8Args, MapsI8>(kern, ctx, grid, Cfg::THREADS, Cfg::smem(a.experts), CG * CS, stream, a, maps);
}

// Warps that share the K tiles: at least four tiles a warp, so that their loads overlap, unless the pieces do not fill the SMs.
template <int NT>
int launch_few(tnns_cuda_ctx* ctx, const GemmI8Args& a, cudaStream_t stream) {
    const long long high = ((long long)a.places + 8 * NT - 1) / (8 * NT) + (a.offsets ? std::min(a.experts, a.places) : 0);  // at most
    const long long pieces = high * ((a.N + 15) / 16);
    int log_s = 0;
    while (log_s < 3 && (1 << log_s) < a.k_tiles && (a.k_tiles >= 8 << log_s || pieces << log_s < 2LL * FEW_WARPS * ctx->sm_count)) log_s++;
    const int wide = 128 >> log_s;
    const long long items = high * ((a.N + wide - 1) / wide);
    if (items >= 0x3FFFFFFFLL) return tnns_fail(TNNS_ERR_UNSUPPORTED, "too many pieces: %d places of %d channels", a.places, a.N);
    const int grid = (int)std::min<long long>(items, 2LL * ctx->sm_count);  // as many blocks as are resident
    // As many tiles' loads at once as a warp has tiles, four at most (always four / as many: 1 x 1024 -> 1000 3.45 / 2.3 us, 1 x 1024 -> 8192 7.0 /
    // 4.2, 16 x 1024 -> 8192, always two / one, 5.9 / 5.0); experts' few pieces take two (one token, 8 of 64, 4096 -> 1024: four 9.5 / two 7.9).
    const int deep = (a.k_tiles + (1 << log_s) - 1) >> log_s;
    auto go = [&](void (*kern)(GemmI8Args, int)) { return launch<GemmI8Args, int>(kern, ctx, grid, FEW_WARPS * 32, list_bytes(a.experts), 1, stream, a, log_s); };
    if (deep == 1) return go(gemm_i8_few_kernel<NT, 1>);
    return NT == 2 || deep == 2 || a.offsets ? go(gemm_i8_few_kernel<NT, 2>) : go(gemm_i8_few_kernel<1, 4>);
}

int run_product(tnns_cuda_ctx* ctx, const tnns_cuda_weights_i8* w, const int8_t* d_q, long long q_stride, const float* d_scale, int q_rows,
                const int32_t* d_rows, const int32_t* d_offsets, void* d_y, int dtype, long long y_stride, int places, float alpha, void* stream) {
    if (!tnns_dtype_ok(dtype)) return tnns_fail(TNNS_ERR_INVALID, "unknown element type %d", dtype);
    if (places < 0 || places > 0x7FFFF000 || q_rows < 0) return tnns_fail(TNNS_ERR_INVALID, "bad size: %d places, %d rows", places, q_rows);
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
    a.dtype = dtype; a.status = ctx->d_status;
    a.y_maps = ((uintptr_t)d_y | (uintptr_t)(y_stride * tnns_dtype_bytes(dtype))) % 16 == 0;
    const cudaStream_t st = (cudaStream_t)stream;
    // places an expert has on average, experts that may have one, pieces of 64 channels of those
    const long long rows = ((long long)places + w->experts - 1) / w->experts, met = std::min(w->experts, places);
    const long long pieces = met * ((w->N + 63) / 64), sixteens = (rows + 15) / 16 * pieces;
    // Few rows.  One kernel: up to 8 rows; up to 32, or where pieces of 64 channels x 16 rows are no more than SMs, if the pieces' sums are
    // short enough, the more pieces the shorter (few rows' kernel / tensor cores: 16 rows, 4096 -> 4096 6.3 / 10.0 us, 4096 -> 8192 10.6 / 11.5, 8192 ->
    // 8192 18.1 / 16.5; 24 rows 9.4 / 10.4, 16.6 / 12.4, 28.3 / 16.7; 128 x 1024 -> 1024 5.5 / 6.5, 128 x 2048 6.3 / 7.0, 128 x 4096 9.4 / 8.5; 64 x 8192
    // -> 1024 8.5 / 10.1, 64 x 16384 14.2 / 13.8).  Experts: up to 32 rows each, where those that have a row make fewer pieces than SMs (one
    // token, 8 of 64 experts, 2048 -> 1024: 6.0 us, tensor cores 9.2; two tokens 10.8 / 9.9; eight, 1024 -> 2048: 24.8 / 20.5; 352 rows each, 8
    // experts, 1561 -> 226: 27 / 10.6).
    const bool short_sums = (10 * sixteens - 3 * ctx->sm_count) * w->k_tiles <= (rows <= 32 ? 200LL : 100LL) * ctx->sm_count;
    const bool few = !d_offsets ? rows <= 8 || (short_sums && (rows <= 32 || sixteens <= ctx->sm_count)) : pieces < ctx->sm_count && rows <= 32;
    if (q_rows == 0 || few) return rows <= 8 ? launch_few<1>(ctx, a, st) : launch_few<2>(ctx, a, st);
    // Rows of q by boxes of 32 or 64 where most tiles hold no more (8 tokens, 8 of 64 experts: 22.2 / 21.1 us; two boxes instead of a whole
    // one cost 64 x 4096 -> 4096 11.0 / 14.4 us).
    a.q_box = rows <= 16 ? 32 : rows <= 64 ? 64 : BM;
    // Tiles of 256 x 256 on block pairs, of 128 x 128 or of 128 x 64 on single blocks: what takes the fewest clocks, by the waves that the
    // launch's tiles make and the clocks of a K tile in each (measured with every SM at work: about 620, 530 and 410; the large tiles
    // are bound by the shared memory's bandwidth, the small ones by L2's).  1024 x 4096 -> 4096: pairs 17.6 us, 128 x 128 21.5; 512 rows 128 x
    // 128 13.3, 128 x 64 18.6; 1024 x 4096 -> 1024, sums not shared: 128 x 64 11.3, 128 x 128 13.4.
    const long long each = d_offsets ? met : 1;
    auto tiles = [&](int tm, int tn) { return (rows + tm - 1) / tm * each * ((w->N + tn - 1) / tn); };
    auto clocks = [&](int tm, int tn, int units, int per_stage) { return (tiles(tm, tn) + units - 1) / units * per_stage * w->k_tiles; };
    const long long pair = clocks(256, 256, ctx->sm_count / 2, 620), wide = clocks(128, 128, ctx->sm_count, 530), narrow = clocks(128, 64, ctx->sm_count, 410);
    // Fewer tiles than SMs: clusters that share them, where their shorter sums save more than the exchange takes (about 5000 clocks among
    // four, 4400 between two; alone / shared: 256 x 4096 -> 1024 11.1 / 8.7 us, 282 x 14050 -> 1529 31.0 / 19.5, 1024 x 4096 -> 1024 11.2 / 10.2, but 128 x
    // 1024 -> 4096 6.3 / 8.0).  Clusters of four do not find room on every SM.
    if (!d_offsets) {
        const long long best = std::min(std::min(pair, wide), narrow);
        auto shared = [&](int tn, int cs, int units, int per_stage, int exchange) {
            return tiles(BM, tn) <= units && w->k_tiles >= cs ? (long long)(w->k_tiles + cs - 1) / cs * per_stage + exchange : best;
        };
        const long long quarters = shared(128, 4, ctx->sm_count / 4 - 4, 530, 5000), halves = shared(128, 2, ctx->sm_count / 2, 530, 4400), narrow_halves = shared(64, 2, ctx->sm_count / 2, 410, 4400);
        const long long least = std::min(std::min(quarters, halves), narrow_halves);
        if (least < best) {
            if (quarters == least) return launch_tc<128, 1, false, 4>(ctx, a, st);
            if (halves == least) return launch_tc<128, 1, false, 2>(ctx, a, st);
            return launch_tc<64, 1, false, 2>(ctx, a, st);
        }
    }
    if (pair <= wide && pair <= narrow) return d_rows ? launch_tc<256, 2, true>(ctx, a, st) : launch_tc<256, 2, false>(ctx, a, st);
    if (wide <= narrow) return d_rows ? launch_tc<128, 1, true>(ctx, a, st) : launch_tc<128, 1, false>(ctx, a, st);
    return d_rows ? launch_tc<64, 1, true>(ctx, a, st) : launch_tc<64, 1, false>(ctx, a, st);
}

}  // namespace

extern "C" {

int tnns_cuda_upload_weights_i8(tnns_cuda_ctx* ctx, const int8_t* w, const float* scales, int experts, int N, int K,
                                tnns_cuda_weights_i8** out) {
    if (!ctx || !w || !scales || !out) return tnns_fail(TNNS_ERR_INVALID, "NULL argument");
    *out = nullptr;
    if (experts < 1 || experts > MAX_EXPERTS || N < 1 || N > (1 << 28) || K < 1 || K > 131071) return tnns_fail(TNNS_ERR_INVALID, "bad weight size: %d kernels (at most 1024) of %d x %d (K at most 131071)", experts, N, K);
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
