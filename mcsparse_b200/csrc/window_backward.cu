// Windowed attention backward on the tensor cores (fp16 / bf16, rows of 16-byte multiples). With P = exp(S - lse) and
// dS = P * (dP - delta), delta = rowsum(dO * O):
//   keys kernel     one block per 128 keys and key head: S^T = K Q^T, dP^T = V dO^T, dV += P^T dO, dK += dS^T Q over the query
//                   tiles of 64 that see them, for all query heads that share the keys (their sum stays in tensor memory);
//   queries kernel  one block per 128 queries and query head: S = Q K^T, dP = dO V^T, dQ += dS K over the key tiles of 64, and
//                   M += P K, the mean of the keys.
// delta from the rounded O is off by up to half a step of O's type times |dO|, which reaches dQ and dK as much as the rounding of
// dS does. The sum of a row of dS would be 0 with the exact delta; with the other one it is the difference. So the queries kernel,
// which runs first, takes the sum e of its rows of dS (fp32), returns scale * (dQ - e M), and leaves delta + e for the keys kernel.
// Both are one kernel template: 128 stationary rows against a stream of 64-row tiles. S and dP have two buffers in tensor
// memory (three where the sums leave room); two groups of 128 threads, one row each, take the tiles in turn and make P
// and dS of them in place, in 16 bits, while the tensor cores work on the other buffers; P and dS enter the second products
// from tensor memory, P as soon as it is there. (16 bits because the tensor cores take both operands of one such type; with
// fp16 inputs of 1024 x 128, |dO| near 1, dQ's error is 3.0e-4 of it, where rounding dQ alone gives 2.1e-4. P is lifted by
// 2^8 in fp16, dS is not, whose size follows dO: below 2^-14 it loses bits, 4.5e-4 against 2.4e-4 at |dO| near 1e-3, 3.6e-3
// against 1.6e-3 near 1e-4.) Two kernels compute S and dP twice (with M 8
// products instead of 5), which buys sums without atomics: equal inputs give equal bits, and nothing is kept in fp32 in HBM.
//
// A thread block (one per SM) takes over the place of another block of the grid when its loads are out, so that the next work's
// loads and first products run beside the end of this one. 4 x 4096 tokens, 16/4 heads of 128, window 1024 (of a training step
// of 754 us): queries kernel 238 us (272 with blocks of one work), keys kernel 290 (300). What bounds them: a tile's products take
// 1280 clocks (S and dP at 48 clocks per 16 values, the time to read both operands from shared memory, the sums at 64), 1610 are
// measured; the keys kernel's work (72 tiles and more each) comes out at 3.9 rounds of blocks.
//
// The first tokens of a sequence are seen by all its queries. Their key tiles would run far longer than the others: what
// lies past their window is cut into pieces of `chunk` queries, blocks of their own, whose partial sums (fp32) a last kernel
// adds in order.
#include <climits>
#include <type_traits>

#include "launch.h"
#include "tensor_core.h"
#include "window_common.h"
#include "window_maps.h"

namespace mcsp_b200 {
namespace {

using namespace window;
using namespace tc;

constexpr int kRows = 128;  // stationary rows of a block
constexpr int kTile = 64;   // rows of a streamed tile
constexpr int kStages = 4;
constexpr int kElementWarps = 8;  // two buffers x 128 rows
constexpr int kLoadWarp = kElementWarps, kScoreWarp = kElementWarps + 1, kSumWarp = kElementWarps + 2, kClearWarp = kElementWarps + 3;
constexpr int kThreads = 32 * (kElementWarps + 4);
constexpr float kLog2e = 1.4426950408889634f;

template <int DP>
struct Smem {
    static constexpr int kFixed = kRows * DP * 2;   // one stationary operand
    static constexpr int kStream = kTile * DP * 2;  // one streamed operand
    static constexpr int kVectors = 2 * kTile * 4;  // -lse and delta of a streamed tile
    static constexpr int kRing = 2 * kFixed;
    static constexpr int kVec = kRing + kStages * 2 * kStream;
    static constexpr int kBars = kVec + kStages * kVectors;
    static constexpr int kTotal = kBars + 1024 + 1024;  // (the start is aligned to 1024)
    static_assert(kTotal <= 227 * 1024, "shared memory of a block");
};

struct Params {
    Ragged r;
    int window, sinks, q_heads, kv_heads, group, dim, slots;
    int q_mul, k_mul, v_mul, go_mul;
    uint32_t negate;
    float scale, scale_log2;
    const float* lse;
    const float* delta;  // q_heads x total_q; read past L1, which may hold what was there before the launch ahead wrote it
    void *out1, *out2;   // dQ, or dV and dK
    int64_t out1_token, out1_head, out2_token, out2_head;
    // the first tokens' far queries
    int chunk, far_slots, far_tiles;
    float* delta_out;  // queries kernel: the exact delta, the same array
    float* partial;  // [2 * far_slots][far_tiles][kv_heads][2][kRows][DP]: far pieces, then what their own windows hold
    long long limit;
    int* fault;
};

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// How the queries of a key tile (its first key key0) are shared out. [begin, mid): the block's own; pieces of `chunk` queries
// from there when the tile holds first tokens and at least one whole piece is left (the last piece takes the remainder).
struct Split {
    int begin, mid, pieces;
};
__device__ __forceinline__ Split split_of(const Sequence& s, int key0, int window, int sinks, int chunk) {
    const int shift = s.lk - s.lq;
    const int last_key = min(key0 + kRows, s.lk) - 1;
    Split v;
    v.begin = max(key0 - shift, 0);
    v.mid = (int)min((int64_t)s.lq, max((int64_t)last_key + window - shift, (int64_t)0));
    v.pieces = 0;
    if (key0 < sinks) {
        const int left = s.lq - max(v.mid, v.begin);
        if (left >= chunk)
            v.pieces = left / chunk;
        else
            v.mid = s.lq;
        v.mid = max(v.mid, v.begin);
    }
    return v;
}
// The sequence of far slot `number`, and its first number. Numbers start at k_offset / chunk: a sequence with n pieces is at
// least n * chunk keys long, so that the numbers of different sequences differ.
__device__ __forceinline__ RaggedBlock far_block(const Ragged& r, int number, int chunk, int lane) {
    if (r.k_offsets == nullptr) return RaggedBlock{0, number};
    int lo = 0, hi = r.batch;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32;
        const int b = lo + step * lane;
        const bool below = b < hi && clamp_offset(__ldg(r.k_offsets + b), r.total_k) / chunk <= number;
        const unsigned hits = __ballot_sync(0xffffffffu, below);
        lo += step * (hits == 0 ? 0 : 31 - __clz(hits));
        hi = min(lo + step, hi);
    }
    const int start = clamp_offset(__ldg(r.k_offsets + lo), r.total_k) / chunk;
    return RaggedBlock{number >= start ? lo : -1, number - start};
}

// delta = rowsum(dO * O): 16 lanes take four consecutive tokens of a head, 8 values of each row at a time, all eight loads on their
// way together. (Bound by memory, 2 * headDim * 2 bytes per row and head.)
constexpr int kDeltaRows = 4;
template <typename T>
__global__ void __launch_bounds__(256) delta_kernel(AttentionArgs a, float* __restrict__ delta) {
    grid_release();
    const int64_t g = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 4;
    const int part = threadIdx.x & 15, h = (int)(g % a.q_heads);
    const int64_t t0 = g / a.q_heads * kDeltaRows;
    uint4 x[kDeltaRows], y[kDeltaRows];
#pragma unroll
    for (int i = 0; i < kDeltaRows; ++i) {
        x[i] = y[i] = make_uint4(0, 0, 0, 0);
        if (t0 + i < a.total_q && 8 * part < a.dim) {
            x[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.o.p) + (t0 + i) * a.o.token + h * a.o.head + 8 * part);
            y[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.d_o.p) + (t0 + i) * a.d_o.token + h * a.d_o.head + 8 * part);
        }
    }
#pragma unroll
    for (int i = 0; i < kDeltaRows; ++i) {
        const T *xv = reinterpret_cast<const T*>(&x[i]), *yv = reinterpret_cast<const T*>(&y[i]);
        float sum = 0.0f;
#pragma unroll
        for (int c = 0; c < 8; ++c) sum = fmaf(to_float(xv[c]), to_float(yv[c]), sum);
#pragma unroll
        for (int d = 8; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (part == 0 && t0 + i < a.total_q) delta[(int64_t)h * a.total_q + t0 + i] = sum;
    }
}

// Four values of the tile's columns: from shared memory (keys kernel), or the row's own.
template <bool KEYS>
__device__ __forceinline__ void column_values(uint32_t vec, int c, float own, float* v) {
    if (KEYS)
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(vec + 4 * c));
    else
        v[0] = v[1] = v[2] = v[3] = own;
}

// 64 scores of a row -> its weights, in place, and in 16 bits into the first half of the scores' columns. `vec` /
// own_l: -lse (base 2) of the columns / the row. MASK: column c counts iff bit c of `seen` is set.
template <typename T, bool KEYS, bool MASK>
__device__ __forceinline__ void weights(uint32_t* p, uint32_t ts, uint64_t seen, uint32_t vec, float own_l, float scale_log2) {
    const uint64_t scale2 = pair(scale_log2, scale_log2);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t w[16];
        const uint32_t bits = (uint32_t)(seen >> (32 * h));
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
            float l[4];
            column_values<KEYS>(vec, 32 * h + c, own_l, l);
#pragma unroll
            for (int x = 0; x < 4; x += 2) {
                const int at = 32 * h + c + x;
                float p0, p1;
                unpair(fma2(pair(__uint_as_float(p[at]), __uint_as_float(p[at + 1])), scale2, pair(l[x], l[x + 1])), p0, p1);
                p0 = exp2_fast(p0), p1 = exp2_fast(p1);
                if (MASK) {
                    p0 = bits >> (c + x) & 1 ? p0 : 0.0f;
                    p1 = bits >> (c + x + 1) & 1 ? p1 : 0.0f;
                }
                w[(c + x) >> 1] = pack2<T>(p0, p1);
                p[at] = __float_as_uint(p0), p[at + 1] = __float_as_uint(p1);
            }
        }
        tmem_store16(ts + 16 * h, w);
    }
}

// dS = P * (dP - delta) of a row, in 16 bits into the first half of dP's columns. (An unseen pair is 0 also where dP is NaN.)
// Returns the sum of the row's dS in fp32.
template <typename T, bool KEYS, bool MASK>
__device__ __forceinline__ float weight_gradients(const uint32_t* p, const uint32_t* d, uint32_t td, uint64_t seen, uint32_t vec, float own_d) {
    constexpr float kLower = std::is_same<T, __half>::value ? 1.0f / 256.0f : 1.0f;
    const uint64_t lower2 = pair(kLower, kLower);
    uint64_t sum = pair(0.0f, 0.0f);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t w[16];
        const uint32_t bits = (uint32_t)(seen >> (32 * h));
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
            float e[4];
            column_values<KEYS>(vec, 32 * h + c, own_d, e);
#pragma unroll
            for (int x = 0; x < 4; x += 2) {
                const int at = 32 * h + c + x;
                float g0, g1;
                unpair(mul2(pair(__uint_as_float(p[at]), __uint_as_float(p[at + 1])),
                            fma2(pair(__uint_as_float(d[at]), __uint_as_float(d[at + 1])), lower2, pair(e[x], e[x + 1]))), g0, g1);
                if (MASK) {
                    g0 = bits >> (c + x) & 1 ? g0 : 0.0f;
                    g1 = bits >> (c + x + 1) & 1 ? g1 : 0.0f;
                }
                if (!KEYS) sum = add2(sum, pair(g0, g1));
                w[(c + x) >> 1] = pack2<T>(g0, g1);
            }
        }
        tmem_store16(td + 16 * h, w);
    }
    float a, b;
    unpair(sum, a, b);
    return a + b;
}

// What a block number stands for: 128 stationary rows of a head, and the streamed rows [begin, end) (keys kernel).
struct Work {
    Sequence sq;
    int row0, head, begin, end;  // row0 < 0: nothing
    int partial;                 // where the sums go instead of the outputs; -1: to the outputs
};
template <bool KEYS>
__device__ __forceinline__ Work work_of(const Params& a, int number, int lane) {
    const int heads = KEYS ? a.kv_heads : a.q_heads;
    Work w;
    w.sq = Sequence{0, 0, 0, 0};
    w.row0 = -1, w.head = number % heads, w.begin = w.end = 0, w.partial = -1;
    number /= heads;
    const int far_blocks = KEYS ? a.far_slots * a.far_tiles : 0;
    if (KEYS && number < far_blocks) {
        const int far = number / a.far_tiles, tile = number % a.far_tiles;
        const RaggedBlock fb = far_block(a.r, far, a.chunk, lane);
        if (fb.b < 0) return w;
        w.sq = sequence_of(a.r, fb.b);
        if (tile * kRows >= w.sq.lk) return w;
        const Split v = split_of(w.sq, tile * kRows, a.window, a.sinks, a.chunk);
        if (fb.index >= v.pieces) return w;
        w.row0 = tile * kRows;
        w.begin = v.mid + fb.index * a.chunk;
        w.end = fb.index + 1 < v.pieces ? w.begin + a.chunk : w.sq.lq;
        w.partial = (far * a.far_tiles + tile) * a.kv_heads + w.head;
    } else if (KEYS) {
        const RaggedBlock rb = ragged_block(a.r.k_offsets, a.r.batch, a.r.total_k, number - far_blocks, kRows, lane);
        if (rb.b < 0) return w;
        w.sq = sequence_of(a.r, rb.b);
        if ((int64_t)rb.index * kRows >= w.sq.lk) return w;
        w.row0 = rb.index * kRows;
        const Split v = split_of(w.sq, w.row0, a.window, a.sinks, a.chunk);
        w.begin = v.begin, w.end = v.mid;
        if (v.pieces > 0) w.partial = (((a.r.k_offsets == nullptr ? 0 : w.sq.k0 / a.chunk) + a.far_slots) * a.far_tiles + rb.index) * a.kv_heads + w.head;
    } else {
        const RaggedBlock rb = ragged_block(a.r.q_offsets, a.r.batch, a.r.total_q, a.slots - 1 - number, kRows, lane);
        if (rb.b < 0) return w;
        w.sq = sequence_of(a.r, rb.b);
        if ((int64_t)rb.index * kRows < w.sq.lq) w.row0 = rb.index * kRows;
    }
    return w;
}

// KEYS: stationary K, V; streamed Q, dO. Otherwise: stationary Q, dO; streamed K, V.
template <typename T, int DP, bool KEYS>
__global__ void __launch_bounds__(kThreads, 1)
    window_backward_kernel(const __grid_constant__ CUtensorMap map_fixed1, const __grid_constant__ CUtensorMap map_fixed2,
                           const __grid_constant__ CUtensorMap map_stream1, const __grid_constant__ CUtensorMap map_stream2,
                           const Params a) {
    using S = Smem<DP>;
    constexpr bool kHalf = std::is_same<T, __half>::value;
    constexpr int kBlocks = DP / 64;
    constexpr int kBuffers = DP == 128 ? 2 : 3;
    static_assert(kBuffers * 2 * kTile + 2 * DP <= 512, "columns of tensor memory");
    // fp16 P is held 2^8 times too large (at most 256): weights below 2^-14 would lose bits to fp16's subnormal numbers. The
    // factor leaves dS through the other factor of its product and dV at the end.
    constexpr float kLift = kHalf ? 8.0f : 0.0f, kLower = kHalf ? 1.0f / 256.0f : 1.0f;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem = (smem_u32(smem_raw) + 1023) & ~1023u;
    const int warp = uniform((int)(threadIdx.x >> 5)), lane = threadIdx.x & 31;
    // barriers: stationary operands, and their place free again; of every stage: there, clear, done with; of the buffers: S ready, dP
    // ready, P ready, dS ready, S's columns free, dP's columns free; a work's last product done, its sums read; the groups' exchange;
    // of the two places for what a block number stands for: written, read by all other warps; the answer to a request; the ends of
    // the two issuing warps
    const uint32_t bars = smem + S::kBars;
    const uint32_t bar_fixed = bars, bar_fixed_free = bars + 8, bar_full = bars + 16, bar_clear = bar_full + 8 * kStages,
                   bar_empty = bar_clear + 8 * kStages, bar_s = bar_empty + 8 * kStages, bar_dp = bar_s + 8 * kBuffers,
                   bar_p = bar_dp + 8 * kBuffers, bar_ds = bar_p + 8 * kBuffers, bar_free_s = bar_ds + 8 * kBuffers,
                   bar_free_dp = bar_free_s + 8 * kBuffers, bar_last = bar_free_dp + 8 * kBuffers, bar_drained = bar_last + 8,
                   bar_x = bar_drained + 8, bar_work = bar_x + 8, bar_taken = bar_work + 16, bar_asked = bar_taken + 16,
                   bar_end = bar_asked + 8, slot = bar_end + 16;
    const uint32_t answer = bars + 512, works = answer + 16;  // 2 x 48 bytes

    grid_release();
    // (All launches but delta's may come up early: what they read that an earlier one of them wrote is delta, and the partial sums;
    // every block waits for the launch ahead before it ends.)
    Work work;
    if (warp == kSumWarp) {
        tmem_alloc(slot, 512);
    } else if (warp == kLoadWarp) {
        if (lane == 0) {
            tma_prefetch(&map_fixed1), tma_prefetch(&map_fixed2), tma_prefetch(&map_stream1), tma_prefetch(&map_stream2);
            bar_init(bar_fixed, 1), bar_init(bar_fixed_free, 1);
            for (int i = 0; i < 3 * kStages; ++i) bar_init(bar_full + 8 * i, 1);
            for (int i = 0; i < kBuffers; ++i) {
                bar_init(bar_s + 8 * i, 1), bar_init(bar_dp + 8 * i, 1), bar_init(bar_p + 8 * i, kRows), bar_init(bar_ds + 8 * i, kRows);
                bar_init(bar_free_s + 8 * i, 1), bar_init(bar_free_dp + 8 * i, 1);
            }
            bar_init(bar_last, 1), bar_init(bar_drained, 2 * kRows), bar_init(bar_x, 2 * kRows), bar_init(bar_asked, 1);
            for (int i = 0; i < 2; ++i) bar_init(bar_work + 8 * i, 1), bar_init(bar_taken + 8 * i, kThreads / 32 - 1), bar_init(bar_end + 8 * i, 1);
            bar_init_fence();
        }
        __syncwarp();
        work = work_of<KEYS>(a, (int)blockIdx.x, lane);
    }
    fence_before();
    __syncthreads();
    fence_after();
    uint32_t tmem;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(slot));
    tmem = uniform(tmem);
    // tensor memory: the buffers of S and dP, 64 columns each, then the sums (dV and dK, or M and dQ)
    const uint32_t t_s = tmem, t_dp = tmem + kBuffers * kTile, t_out1 = tmem + 2 * kBuffers * kTile, t_out2 = t_out1 + DP;
    bool failed = false;
    // (before any wait that is timed; the load warp has loads to issue first, and waits in publish() if it gets there without any)
    if (warp != kLoadWarp) grid_wait();

    // All warps run through the same work, each with running counts of the barriers' phases: `total` tiles, `turns` works with tiles.
    int turn = 0, total = 0, turns = 0;
    int shift, rows, p_low, p_high;       // (positions: queries kernel)
    int tiles, n, first, low, begin;      // tiles of one head that streams, and of all; queries kernel: key tiles [0, first) and from `low` on
    const auto plan = [&] {
        const int hops = KEYS ? a.group : 1;
        shift = work.sq.lk - work.sq.lq;
        rows = min(kRows, (KEYS ? work.sq.lk : work.sq.lq) - work.row0);
        p_low = shift + work.row0, p_high = p_low + rows - 1;
        tiles = first = low = 0, begin = uniform(work.begin);
        if (KEYS) {
            tiles = work.end > work.begin ? (work.end - work.begin + kTile - 1) / kTile : 0;
        } else if (p_high >= 0) {
            low = max(p_low - a.window + 1, 0) / kTile;
            first = min((min(a.sinks, p_high + 1) + kTile - 1) / kTile, low);
            tiles = first + p_high / kTile - low + 1;
        }
        tiles = uniform(tiles), first = uniform(first), low = uniform(low);
        n = tiles * hops;
        total = uniform(total), turns = uniform(turns);
    };
    // first streamed row of tile i, relative to the sequence
    const auto tile_row = [&](int i) {
        if (KEYS) return begin + (i % tiles) * kTile;
        return (i < first ? i : low + (i - first)) * kTile;
    };
    // Whole warps; false: no more, or `failed`.
    const auto next_work = [&] {
        const int at = turn & 1;
        if (!bar_wait_warp(bar_work + 8 * at, (turn >> 1) & 1, a.limit)) {
            failed = true;
            return false;
        }
        const uint32_t from = works + 48 * at;
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(work.sq.q0), "=r"(work.sq.lq), "=r"(work.sq.k0), "=r"(work.sq.lk) : "r"(from) : "memory");
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(work.row0), "=r"(work.head), "=r"(work.begin), "=r"(work.end) : "r"(from + 16) : "memory");
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(work.partial) : "r"(from + 32) : "memory");
        __syncwarp();
        if (elect()) bar_arrive(bar_taken + 8 * at);
        ++turn;
        if (uniform(work.row0) < 0) return false;
        plan();
        return true;
    };
    const auto work_done = [&] { total += n, turns += n > 0; };

    if (warp == kLoadWarp) {
        // ---- loads, and the order of the work: when a work's last loads are issued, the place of a block of the grid that has not
        // started is taken over (cluster launch control), so that its loads and first products run beside the end of this one.
        int asked = 0;
        const auto publish = [&](int row0) {
            const int at = turn & 1;
            // (the other warps take nothing before the launch ahead is done; works without tiles come here without having waited)
            if (turn >= 2 && turns == 0) grid_wait();
            if (turn >= 2 && !bar_wait_warp(bar_taken + 8 * at, ((turn >> 1) - 1) & 1, a.limit)) {
                failed = true;
                return;
            }
            if (elect()) {
                const uint32_t to = works + 48 * at;
                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(work.sq.q0), "r"(work.sq.lq), "r"(work.sq.k0), "r"(work.sq.lk) : "memory");
                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to + 16), "r"(row0), "r"(work.head), "r"(work.begin), "r"(work.end) : "memory");
                asm volatile("st.shared.u32 [%0], %1;" ::"r"(to + 32), "r"(work.partial) : "memory");
                bar_arrive(bar_work + 8 * at);
            }
            __syncwarp();
            ++turn;
        };
        int issued = 0;  // tiles, of all works
        while (!failed) {
            if (work.row0 >= 0) {
                publish(work.row0);
                plan();
                const Sequence sq = work.sq;
                const int head = work.head, hk = KEYS ? head : head / a.group;
                // -lse (base 2) and delta of the tile's queries, fetched one tile ahead; a row that is none has -lse = -inf: P = 0
                float l[2], d[2];
                const auto fetch = [&](int i) {
                    if (!KEYS || i >= n) return;
                    const int h = head * a.group + i / tiles, row = tile_row(i);
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int q = row + 2 * lane + x;
                        l[x] = -INFINITY, d[x] = 0.0f;
                        if (q < work.end) {
                            const int64_t at = (int64_t)h * a.r.total_q + sq.q0 + q;
                            const float v = __ldg(a.lse + at), w = __ldcg(a.delta + at);  // (both on their way before either is looked at)
                            if (v != -INFINITY) l[x] = kLift - v * kLog2e;
                            d[x] = -kLower * w;
                        }
                    }
                };
                if (n > 0 && !failed) {
                    if (turns > 0) {
                        fetch(0);
                        if (!bar_wait_warp(bar_fixed_free, (turns - 1) & 1, a.limit)) {
                            failed = true;
                            break;
                        }
                    }
                    if (elect()) {
                        bar_expect(bar_fixed, 2 * S::kFixed);
                        const int h1 = head * (KEYS ? a.k_mul : a.q_mul), h2 = head * (KEYS ? a.v_mul : a.go_mul);
                        const int row = (KEYS ? sq.k0 : sq.q0) + work.row0;
                        for (int c = 0; c < kBlocks; ++c) {
                            tma_load_3d(smem + c * (kRows * 128), &map_fixed1, 64 * c, h1, row, bar_fixed);
                            tma_load_3d(smem + S::kFixed + c * (kRows * 128), &map_fixed2, 64 * c, h2, row, bar_fixed);
                        }
                    }
                    if (turns == 0) {
                        grid_wait();  // (the first stationary operands are on their way)
                        fetch(0);
                    }
                    ++turns;
                    for (int i = 0; i < n; ++i) {
                        const int g = total + i, st = g % kStages;
                        if (g >= kStages && !bar_wait_warp(bar_empty + 8 * st, (g / kStages - 1) & 1, a.limit)) {
                            failed = true;
                            break;
                        }
                        if (KEYS) {
                            const uint32_t vec = smem + S::kVec + st * S::kVectors + 8 * lane;
                            asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(vec), "f"(l[0]), "f"(l[1]) : "memory");
                            asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(vec + 4 * kTile), "f"(d[0]), "f"(d[1]) : "memory");
                            fetch(i + 1);
                            __syncwarp();
                        }
                        if (elect()) {
                            bar_expect(bar_full + 8 * st, 2 * S::kStream);
                            const int h = KEYS ? head * a.group + i / tiles : hk;
                            const int h1 = h * (KEYS ? a.q_mul : a.k_mul), h2 = h * (KEYS ? a.go_mul : a.v_mul);
                            const int row = (KEYS ? sq.q0 : sq.k0) + tile_row(i);
                            const uint32_t to = smem + S::kRing + st * 2 * S::kStream;
                            for (int c = 0; c < kBlocks; ++c) {
                                tma_load_3d(to + c * (kTile * 128), &map_stream1, 64 * c, h1, row, bar_full + 8 * st);
                                tma_load_3d(to + S::kStream + c * (kTile * 128), &map_stream2, 64 * c, h2, row, bar_full + 8 * st);
                            }
                        }
                        issued = g + 1;
                    }
                    total += n;
                }
            }
            if (failed) break;
            if (elect()) {
                bar_expect(bar_asked, 16);
                ask_block(answer, bar_asked);
            }
            __syncwarp();
            if (!bar_wait_warp(bar_asked, asked & 1, a.limit)) {
                bar_wait_warp(bar_asked, asked & 1, kDrain);
                failed = true;
                break;
            }
            ++asked;
            const int number = uniform(asked_block(answer));
            fence_async();  // (the next answer is written by another proxy than this one was read by)
            __syncwarp();
            if (number < 0) {
                publish(-1);
                break;
            }
            work = work_of<KEYS>(a, number, lane);
        }
        // nothing of this block's memory is given back while a copy is on its way, whoever gave up
        if (turns > 0) bar_wait_warp(bar_fixed, (turns - 1) & 1, kDrain);
        for (int i = max(0, issued - kStages); i < issued; ++i) bar_wait_warp(bar_full + 8 * (i % kStages), (i / kStages) & 1, kDrain);
    } else if (warp == kScoreWarp) {
        // ---- S and dP, issued by one thread, each once its columns are free
        constexpr uint32_t kDesc = mma_desc(!kHalf, kTile, false);
        const uint64_t f1 = smem_desc(smem), f2 = smem_desc(smem + S::kFixed);
        while (!failed && next_work()) {
            if (n > 0 && elect()) {
                failed = !bar_wait(bar_fixed, turns & 1, a.limit);
                for (int i = 0; i < n && !failed; ++i) {
                    const int g = total + i, st = g % kStages, b = g % kBuffers;
                    const uint32_t before = (g / kBuffers - 1) & 1;  // the phase of the buffer's last use
                    const uint32_t s1 = smem + S::kRing + st * 2 * S::kStream;
                    const uint64_t m1 = smem_desc(s1), m2 = smem_desc(s1 + S::kStream);
                    if (!bar_wait(bar_clear + 8 * st, (g / kStages) & 1, a.limit) || (g >= kBuffers && !bar_wait(bar_free_s + 8 * b, before, a.limit))) {
                        failed = true;
                        break;
                    }
                    fence_after();
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k)
                        mma_ss(t_s + kTile * b, desc_at(f1, (k >> 2) * (kRows * 128) + (k & 3) * 32), desc_at(m1, (k >> 2) * (kTile * 128) + (k & 3) * 32),
                               kDesc | a.negate, k > 0);
                    mma_commit(bar_s + 8 * b);
                    if (g >= kBuffers && !bar_wait(bar_free_dp + 8 * b, before, a.limit)) {
                        failed = true;
                        break;
                    }
                    fence_after();
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k)
                        mma_ss(t_dp + kTile * b, desc_at(f2, (k >> 2) * (kRows * 128) + (k & 3) * 32), desc_at(m2, (k >> 2) * (kTile * 128) + (k & 3) * 32),
                               kDesc, k > 0);
                    mma_commit(bar_dp + 8 * b);
                }
                mma_commit(bar_fixed_free);
            }
            __syncwarp();
            failed = __any_sync(0xffffffffu, failed);
            work_done();
        }
        if (elect()) {
            mma_commit(bar_end);  // the tensor memory is given back only when no product uses it any more
            bar_wait(bar_end, 0, kDrain);
        }
        __syncwarp();
    } else if (warp == kSumWarp) {
        // ---- dV and dK, or M and dQ, issued by one thread
        constexpr uint32_t kDesc = mma_desc(!kHalf, DP, true);
        while (!failed && next_work()) {
            if (n > 0 && elect()) {
                failed = turns > 0 && !bar_wait(bar_drained, (turns - 1) & 1, a.limit);
                for (int i = 0; i < n && !failed; ++i) {
                    const int g = total + i, st = g % kStages, b = g % kBuffers;
                    const uint32_t phase = (g / kBuffers) & 1;
                    const uint32_t s1 = smem + S::kRing + st * 2 * S::kStream;
                    const uint64_t m1 = smem_desc(s1, kTile * 128), m2 = smem_desc(s1 + S::kStream, kTile * 128);
                    if (!bar_wait(bar_clear + 8 * st, (g / kStages) & 1, a.limit) || !bar_wait(bar_p + 8 * b, phase, a.limit)) {
                        failed = true;
                        break;
                    }
                    fence_after();
#pragma unroll
                    for (int k = 0; k < kTile / 16; ++k)
                        mma_ts(t_out1, t_s + kTile * b + 8 * k, desc_at(KEYS ? m2 : m1, k * 2048), kDesc, i > 0 || k > 0);
                    mma_commit(bar_free_s + 8 * b);
                    if (!bar_wait(bar_ds + 8 * b, phase, a.limit)) {
                        failed = true;
                        break;
                    }
                    fence_after();
#pragma unroll
                    for (int k = 0; k < kTile / 16; ++k)
                        mma_ts(t_out2, t_dp + kTile * b + 8 * k, desc_at(m1, k * 2048), kDesc, i > 0 || k > 0);
                    mma_commit(bar_free_dp + 8 * b);
                    mma_commit(bar_empty + 8 * st);
                    if (i == n - 1) mma_commit(bar_last);
                }
            }
            __syncwarp();
            failed = __any_sync(0xffffffffu, failed);
            work_done();
        }
        if (elect()) {
            mma_commit(bar_end + 8);
            bar_wait(bar_end + 8, 0, kDrain);
        }
        __syncwarp();
    } else if (warp == kClearWarp) {
        // ---- rows whose weight is zero for every row here are cleared before they enter a sum: zero times a NaN that lies there
        // would not be zero. Keys kernel: queries behind the last one; queries kernel: keys nobody sees.
        while (!failed && next_work()) {
            const int first_seen = max(p_low - a.window + 1, 0);  // queries kernel: the first key in reach of some row here
            for (int i = 0; i < n; ++i) {
                const int g = total + i, st = g % kStages, row = tile_row(i);
                if (!bar_wait_warp(bar_full + 8 * st, (g / kStages) & 1, a.limit)) {
                    failed = true;
                    break;
                }
                const int clear_low = KEYS ? 0 : min(max(first_seen - row, 0), kTile);
                const int keep = KEYS ? 0 : min(max(a.sinks - row, 0), kTile);
                const int clear_high = min(max((KEYS ? work.end : p_high + 1) - row, 0), kTile);
                if (clear_low > keep || clear_high < kTile) {
                    for (int x = lane; x < (KEYS ? 2 : 1) * kTile * 8 * kBlocks; x += 32) {  // (stream 2 lies behind stream 1)
                        const int at = (x >> 3) & (kTile - 1);
                        if ((at < clear_low && at >= keep) || at >= clear_high)
                            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(smem + S::kRing + st * 2 * S::kStream + x * 16), "r"(0) : "memory");
                    }
                    fence_async();
                    __syncwarp();
                }
                if (elect()) bar_arrive(bar_clear + 8 * st);
                __syncwarp();
            }
            work_done();
        }
    } else {
        // ---- P and dS: thread = stationary row; the two groups take the tiles in turn
        const int group = warp >> 2;
        const int r = threadIdx.x & (kRows - 1);
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;
        while (!failed && next_work()) {
            const int row0 = work.row0;
            const int64_t token = (int64_t)(KEYS ? work.sq.k0 : work.sq.q0) + row0 + r;
            float own_l = -INFINITY, own_d = 0.0f;  // queries kernel: the row's -lse and -delta
            if (!KEYS && r < rows) {
                const int64_t at = (int64_t)work.head * a.r.total_q + token;
                const float v = __ldg(a.lse + at);
                if (v != -INFINITY) own_l = kLift - v * kLog2e;
                own_d = -kLower * __ldcg(a.delta + at);
            }
            float e = 0.0f;  // queries kernel: the sum of the row's dS
            for (int i = (group ^ total) & 1; i < n; i += 2) {
                const int g = total + i, b = g % kBuffers;
                const uint32_t phase = (g / kBuffers) & 1;
                const uint32_t ts = t_s + kTile * b + lanes, td = t_dp + kTile * b + lanes;
                // (the second wait is over by then; it is there for the vectors, which ordinary stores wrote)
                if (!bar_wait_warp(bar_s + 8 * b, phase, a.limit) || (KEYS && !bar_wait_warp(bar_full + 8 * (g % kStages), (g / kStages) & 1, a.limit))) {
                    failed = true;
                    break;
                }
                fence_after();
                uint32_t p[kTile];
                tmem_load32(ts, p);
                tmem_load32(ts + 32, p + 32);
                const int row = tile_row(i);
                uint64_t seen = ~0ull;
                if (KEYS) {
                    // key j = row0 + r, query at position p = shift + row + c: seen iff p >= j and (p < j + window or j < sinks)
                    const int p0 = shift + row, j = row0 + r;  // (positions)
                    if (p0 < row0 + kRows - 1 || (p0 + kTile - 1 >= row0 + a.window && row0 + kRows > a.sinks)) {
                        const int from = min(max(j - p0, 0), 64);
                        const int upto = j < a.sinks ? 64 : min(max(j + a.window - p0, 0), 64);
                        seen = (from < 64 ? ~0ull << from : 0ull) & (upto < 64 ? (1ull << upto) - 1 : ~0ull);
                    }
                } else {
                    // query at p, key j = row + c: seen iff j <= p and (j > p - window or j < sinks)
                    const int at = p_low + r;
                    if (row + kTile - 1 > p_low || (row <= p_low + kRows - 1 - a.window && row + kTile > a.sinks)) {
                        const int upto = min(max(at + 1 - row, 0), 64), from = min(max(at - a.window + 1 - row, 0), 64);
                        const int keep = min(max(a.sinks - row, 0), 64);
                        const uint64_t near = from < 64 ? ~0ull << from : 0ull, kept = keep < 64 ? (1ull << keep) - 1 : ~0ull;
                        seen = (near | kept) & (upto < 64 ? (1ull << upto) - 1 : ~0ull);
                    }
                }
                const uint32_t vec = smem + S::kVec + (g % kStages) * S::kVectors;
                const bool masked = !__all_sync(0xffffffffu, seen == ~0ull);
                wait_loads();
                after_loads32(p), after_loads32(p + 32);
                if (masked)
                    weights<T, KEYS, true>(p, ts, seen, vec, own_l, a.scale_log2);
                else
                    weights<T, KEYS, false>(p, ts, seen, vec, own_l, a.scale_log2);
                wait_stores();
                fence_before();
                bar_arrive(bar_p + 8 * b);
                if (!bar_wait_warp(bar_dp + 8 * b, phase, a.limit)) {
                    failed = true;
                    break;
                }
                fence_after();
                uint32_t d[kTile];
                tmem_load32(td, d);
                tmem_load32(td + 32, d + 32);
                wait_loads();
                after_loads32(d), after_loads32(d + 32);
                if (masked)
                    e += weight_gradients<T, KEYS, true>(p, d, td, seen, vec + 4 * kTile, own_d);
                else
                    e += weight_gradients<T, KEYS, false>(p, d, td, seen, vec + 4 * kTile, own_d);
                wait_stores();
                fence_before();
                bar_arrive(bar_ds + 8 * b);
            }
            // ---- outputs: keys kernel: one group writes dV, the other dK; queries kernel: each half of dQ's columns
            if (n > 0 && !failed) {
                if (!KEYS) {  // the row's sum over the tiles of both groups (two places in turn: a slow reader of the last work's)
                    const uint32_t words = smem + S::kVec + (turns & 1) * (8 * kRows);
                    asm volatile("st.shared.f32 [%0], %1;" ::"r"(words + 4 * (kRows * group + r)), "f"(e) : "memory");
                    bar_arrive(bar_x);
                    failed = !bar_wait_warp(bar_x, turns & 1, a.limit);
                    float e0, e1;
                    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(e0) : "r"(words + 4 * r) : "memory");
                    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(e1) : "r"(words + 4 * (kRows + r)) : "memory");
                    e = e0 + e1;
                    if (group == 0 && r < rows && !failed) a.delta_out[(int64_t)work.head * a.r.total_q + token] = e - own_d / kLower;
                }
                failed = !bar_wait_warp(bar_last, turns & 1, a.limit) || failed;
                fence_after();
            }
            if (failed) break;
            const float less = -e * kLower;
            const float factor = KEYS && group == 0 ? kLower : a.scale;
            T* out = group == 1 && KEYS ? static_cast<T*>(a.out2) + token * a.out2_token + (int64_t)work.head * a.out2_head
                                        : static_cast<T*>(a.out1) + token * a.out1_token + (int64_t)work.head * a.out1_head;
            float* part = work.partial < 0 ? nullptr : a.partial + (((int64_t)work.partial * 2 + group) * kRows + r) * DP;
            const int c0 = KEYS ? 0 : group * (DP / 2), c1 = KEYS ? DP : c0 + DP / 2;
#pragma unroll 1
            for (int c = c0; c < c1; c += 32) {
                uint32_t o[32];
                if (n > 0) {
                    tmem_load32((KEYS && group == 0 ? t_out1 : t_out2) + lanes + c, o);
                    if (!KEYS) {
                        uint32_t m[32];
                        tmem_load32(t_out1 + lanes + c, m);
                        wait_loads();
                        after_loads32(o), after_loads32(m);
#pragma unroll
                        for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(fmaf(less, __uint_as_float(m[x]), __uint_as_float(o[x])));
                    } else {
                        wait_loads();
                        after_loads32(o);
                    }
                    if (c + 32 == c1) {  // the next work's products may overwrite the sums
                        fence_before();
                        bar_arrive(bar_drained);
                    }
                } else {
#pragma unroll
                    for (int x = 0; x < 32; ++x) o[x] = 0u;
                }
                if (part != nullptr) {
#pragma unroll
                    for (int x = 0; x < 32; x += 4) *reinterpret_cast<uint4*>(part + c + x) = make_uint4(o[x], o[x + 1], o[x + 2], o[x + 3]);
                } else if (r < rows) {
#pragma unroll
                    for (int x = 0; x < 32; x += 8) {
                        if (c + x < a.dim) {
                            uint4 w;
                            w.x = pack2<T>(__uint_as_float(o[x]) * factor, __uint_as_float(o[x + 1]) * factor);
                            w.y = pack2<T>(__uint_as_float(o[x + 2]) * factor, __uint_as_float(o[x + 3]) * factor);
                            w.z = pack2<T>(__uint_as_float(o[x + 4]) * factor, __uint_as_float(o[x + 5]) * factor);
                            w.w = pack2<T>(__uint_as_float(o[x + 6]) * factor, __uint_as_float(o[x + 7]) * factor);
                            *reinterpret_cast<uint4*>(out + c + x) = w;
                        }
                    }
                }
            }
            work_done();
        }
        fence_before();
    }
    if (failed && a.fault != nullptr) *reinterpret_cast<volatile int*>(a.fault) = 1;
    grid_wait();
    __syncthreads();
    if (warp == kSumWarp) {
        fence_after();
        tmem_free(tmem, 512);
    }
}

// The sums of a first-tokens tile: what its own window holds, then its far pieces in order. One block per (sequence by its
// first far slot, key tile, key head, which of dV and dK, slice of 16 rows); thread = 4 values.
constexpr int kJoinSlices = 8;
template <typename T, int DP>
__global__ void __launch_bounds__(256) window_backward_join_kernel(const Params a) {
    grid_wait();
    const int lane = threadIdx.x & 31;
    int64_t x = blockIdx.x;
    const int slice = (int)(x % kJoinSlices), which = (int)(x / kJoinSlices & 1), head = (int)((x / kJoinSlices >> 1) % a.kv_heads);
    x = (x / kJoinSlices >> 1) / a.kv_heads;
    const int tile = (int)(x % a.far_tiles), far = (int)(x / a.far_tiles);
    const RaggedBlock fb = far_block(a.r, far, a.chunk, lane);
    if (fb.b < 0 || fb.index != 0) return;
    const Sequence sq = sequence_of(a.r, fb.b);
    const int row0 = tile * kRows;
    if (row0 >= sq.lk) return;
    const Split v = split_of(sq, row0, a.window, a.sinks, a.chunk);
    if (v.pieces == 0) return;
    const float factor = which == 0 ? (std::is_same<T, __half>::value ? 1.0f / 256.0f : 1.0f) : a.scale;
    const auto part = [&](int64_t f) { return a.partial + ((((f * a.far_tiles + tile) * a.kv_heads + head) * 2 + which) * (int64_t)kRows) * DP; };
    constexpr int kSlice = kRows / kJoinSlices * DP;
    for (int i = slice * kSlice + threadIdx.x * 4; i < (slice + 1) * kSlice; i += 256 * 4) {
        const int r = i / DP, c = i % DP;
        if (row0 + r >= sq.lk || c >= a.dim) continue;
        float4 s = *reinterpret_cast<const float4*>(part((int64_t)a.far_slots + far) + i);
        for (int f = 0; f < v.pieces; ++f) {
            const float4 y = *reinterpret_cast<const float4*>(part(far + f) + i);
            s.x += y.x, s.y += y.y, s.z += y.z, s.w += y.w;
        }
        const int64_t token = (int64_t)sq.k0 + row0 + r;
        T* out = which == 0 ? static_cast<T*>(a.out1) + token * a.out1_token + (int64_t)head * a.out1_head
                            : static_cast<T*>(a.out2) + token * a.out2_token + (int64_t)head * a.out2_head;
        uint2 w;
        w.x = pack2<T>(s.x * factor, s.y * factor);
        w.y = pack2<T>(s.z * factor, s.w * factor);
        *reinterpret_cast<uint2*>(out + c) = w;
    }
}

size_t align256(size_t v) { return (v + 255) & ~size_t(255); }

// Key tiles whose far queries are cut into pieces: those of up to 1024 first tokens. (With more of them there are blocks enough,
// and the pieces' partial sums would grow with their square.)
constexpr int kMostFarTiles = 8;
constexpr int kMostPartials = 2048;  // of 128 rows of dV and dK each, for a whole call
// Queries of one piece: about what a key tile's own window holds (the last piece takes the remainder, up to twice as many); at
// least 1024, and no fewer than keep the partial sums in bounds. INT_MAX: nothing is cut.
int far_chunk(const AttentionArgs& a) {
    const int seen = a.sinks < a.total_k ? a.sinks : a.total_k;
    const int64_t tiles = (seen + kRows - 1) / kRows;
    if (tiles == 0 || tiles > kMostFarTiles) return INT_MAX;
    int64_t c = (int64_t)a.window + kRows;
    if (c < 1024) c = 1024;
    const int64_t bound = (int64_t)a.total_k * tiles * a.kv_heads * 2 / kMostPartials + 1;
    if (c < bound) c = bound;
    return c > a.total_k ? INT_MAX : (int)c;  // no sequence reaches past its window by a whole piece when all keys together do not
}
int far_tiles(const AttentionArgs& a) { return far_chunk(a) == INT_MAX ? 0 : ((a.sinks < a.total_k ? a.sinks : a.total_k) + kRows - 1) / kRows; }
int far_slots(const AttentionArgs& a) { return a.total_k / far_chunk(a) + 1; }

template <typename T, int DP>
cudaError_t launch(cudaStream_t s, const AttentionArgs& a, void* buffer) {
    using S = Smem<DP>;
    CUtensorMap q_rows, go_rows, k_rows, v_rows, q_tile, go_tile, k_tile, v_tile;
    if (!head_map(&q_rows, a.q, a.total_q, a.q_heads, a.dim, a.type, kRows) || !head_map(&go_rows, a.d_o, a.total_q, a.q_heads, a.dim, a.type, kRows) ||
        !head_map(&k_rows, a.k, a.total_k, a.kv_heads, a.dim, a.type, kRows) || !head_map(&v_rows, a.v, a.total_k, a.kv_heads, a.dim, a.type, kRows) ||
        !head_map(&q_tile, a.q, a.total_q, a.q_heads, a.dim, a.type, kTile) || !head_map(&go_tile, a.d_o, a.total_q, a.q_heads, a.dim, a.type, kTile) ||
        !head_map(&k_tile, a.k, a.total_k, a.kv_heads, a.dim, a.type, kTile) || !head_map(&v_tile, a.v, a.total_k, a.kv_heads, a.dim, a.type, kTile))
        return cudaErrorNotSupported;
    char* b = static_cast<char*>(align_up_256(buffer));
    float* delta = reinterpret_cast<float*>(b);
    Params p = {};
    p.r = Ragged{a.q_offsets, a.k_offsets, a.batch, a.total_q, a.total_k};
    p.window = a.window, p.sinks = a.sinks, p.q_heads = a.q_heads, p.kv_heads = a.kv_heads, p.group = a.q_heads / a.kv_heads, p.dim = a.dim;
    p.q_mul = a.q.head != 0, p.k_mul = a.k.head != 0, p.v_mul = a.v.head != 0, p.go_mul = a.d_o.head != 0;
    p.negate = a.scale < 0.0f ? kNegateA : 0;
    p.scale = a.scale, p.scale_log2 = fabsf(a.scale) * kLog2e;
    p.lse = a.lse, p.delta = delta;
    p.chunk = far_chunk(a), p.far_tiles = far_tiles(a), p.far_slots = p.far_tiles > 0 ? far_slots(a) : 0;
    p.partial = reinterpret_cast<float*>(b + align256(size_t(a.q_heads) * a.total_q * 4));
    p.limit = window_wait_limit(a), p.fault = a.wait.fault_word;
    const int64_t delta_groups = ((int64_t)a.total_q + kDeltaRows - 1) / kDeltaRows * a.q_heads;
    delta_kernel<T><<<(unsigned)((delta_groups + 15) / 16), 256, 0, s>>>(a, delta);
    cudaError_t e = cudaGetLastError();
    static SharedMemoryOnce once_keys, once_queries;
    if (e == cudaSuccess) e = once_keys.allow(reinterpret_cast<const void*>(window_backward_kernel<T, DP, true>), S::kTotal);
    if (e == cudaSuccess) e = once_queries.allow(reinterpret_cast<const void*>(window_backward_kernel<T, DP, false>), S::kTotal);
    if (e != cudaSuccess) return e;
    Params pk = p;
    pk.out1 = a.dv.p, pk.out1_token = a.dv.token, pk.out1_head = a.dv.head;
    pk.out2 = a.dk.p, pk.out2_token = a.dk.token, pk.out2_head = a.dk.head;
    p.out1 = a.dq.p, p.out1_token = a.dq.token, p.out1_head = a.dq.head;
    p.slots = ragged_slots(a.total_q, a.batch, a.q_offsets != nullptr, kRows);
    p.delta_out = delta;
    e = launch_behind(s, true, window_backward_kernel<T, DP, false>, (unsigned)((int64_t)p.slots * a.q_heads), kThreads, S::kTotal, q_rows, go_rows, k_tile,
                      v_tile, p);
    const int64_t key_blocks = ragged_slots(a.total_k, a.batch, a.k_offsets != nullptr, kRows) + (int64_t)p.far_slots * p.far_tiles;
    if (e == cudaSuccess)
        e = launch_behind(s, true, window_backward_kernel<T, DP, true>, (unsigned)(key_blocks * a.kv_heads), kThreads, S::kTotal, k_rows, v_rows, q_tile,
                          go_tile, pk);
    if (e == cudaSuccess && p.far_tiles > 0)
        e = launch_behind(s, true, window_backward_join_kernel<T, DP>, (unsigned)((int64_t)p.far_slots * p.far_tiles * a.kv_heads * 2 * kJoinSlices), 256, 0, pk);
    return e;
}

}  // namespace

size_t window_backward_mma_bytes(const AttentionArgs& a) {
    const int dp = a.dim <= 64 ? 64 : 128;
    const int tiles = far_tiles(a);
    const size_t partial = tiles > 0 ? size_t(2) * far_slots(a) * tiles * a.kv_heads * 2 * kRows * dp * 4 : 0;
    return align256(size_t(a.q_heads) * a.total_q * 4) + partial + 256;
}

cudaError_t window_backward_mma(cudaStream_t s, const AttentionArgs& a, void* buffer) {
    if (a.type == MACA_R_16BF) return a.dim <= 64 ? launch<__nv_bfloat16, 64>(s, a, buffer) : launch<__nv_bfloat16, 128>(s, a, buffer);
    return a.dim <= 64 ? launch<__half, 64>(s, a, buffer) : launch<__half, 128>(s, a, buffer);
}

}  // namespace mcsp_b200
