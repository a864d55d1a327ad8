// Windowed attention forward on the tensor cores (fp16 / bf16, rows of 16-byte multiples).
//
// One piece of work is 256 consecutive queries of a sequence and one query head: two tiles of 128 rows that share every
// key tile of 64. A thread block (one per SM) takes over the place of another block of the grid when its loads are out, so that the
// loads and first scores of the next work run beside the end of this one (blocks of one work each: 174 us against 159 for 16384
// tokens in 5 sequences, 16/2 heads of 128, window 1024; 1981 against 1874 for 32768 tokens, 32/8 heads, window 4096). S = Q K^T and
// O += P V are tcgen05.mma with S, P and O in tensor memory (P overwrites its S, half as wide); 128 threads per row tile, one row
// each, take maximum, exponentials and sum in registers. S has two buffers per row tile: the next scores are there when a tile's
// weights are done, so the chain scores -> weights -> O -> next scores of a single buffer is cut. Key tiles outside window and
// first tokens are never loaded; a tile needs its mask only at an edge of the pattern.
//
// Bounds at headDim 128, clocks per 64 keys and both row tiles: products 1280 (Q K^T with 64 keys reads 6 KB of shared memory
// per 32 clocks of arithmetic and takes 48; P V reads P from tensor memory: 64), exponentials 1024 (16 per clock). Measured on
// 32768 tokens: 1680, at the 1585 MHz that the power limit leaves. Weights handed over by halves of a tile: no faster.
#include <type_traits>

#include "tensor_core.h"
#include "window_common.h"
#include "window_maps.h"

namespace mcsp_b200 {
namespace {

using namespace window;
using namespace tc;

constexpr int kRows = 128;           // query rows of a tile
constexpr int kKeys = 64;            // keys of a tile
constexpr int kSoftmaxWarps = 8;     // two row tiles
constexpr int kLoadWarp = kSoftmaxWarps, kScoreWarp = kSoftmaxWarps + 1, kValueWarp = kSoftmaxWarps + 2, kClearWarp = kSoftmaxWarps + 3;
constexpr int kThreads = 32 * (kSoftmaxWarps + 4);
constexpr float kLog2e = 1.4426950408889634f;
// The running reference of a row's exponentials is only moved when its maximum has grown past it by more than 2^8: until
// then the weights are at most 256, far from fp16's 65504, and O needs no rescaling. A weight enters the product with V rounded
// to the inputs' type (the tensor cores take both operands of one 16-bit type), and the row's sum as it is in fp32: O differs from
// the exact one by the half step of each weight, by the fp32 sums, and by its own rounding, of which the first is the largest part.
constexpr float kSlack = 8.0f;

template <int DP>
struct Smem {
    static constexpr int kQuery = kRows * DP * 2;        // bytes of a query tile
    static constexpr int kTile = kKeys * DP * 2;          // of a tile of keys, or of values
    static constexpr int kStages = DP == 128 ? 5 : 8;     // of a key tile and a value tile each
    static constexpr int kQ = 0;
    static constexpr int kRing = 2 * kQuery;
    static constexpr int kBars = kRing + kStages * 2 * kTile;
    static constexpr int kTotal = kBars + 1024 + 1024;    // (the start is aligned to 1024)
    static_assert(kTotal <= 227 * 1024, "shared memory of a block");
};

struct Params {
    Ragged r;
    int window, sinks, q_heads, group, dim, total_q, slots;
    int q_mul, k_mul, v_mul;  // 0: the heads of a tensor share one (a head stride of 0)
    uint32_t negate;
    float scale_log2, scale_ln;
    void* o;
    int64_t o_token, o_head;
    float* lse;
    long long limit;
    int* fault;
};

// What one tile of 128 rows has to visit: key tiles [0, first) and [low, high].
struct Visit {
    int rows, p_low, first, low, high;
    __device__ __forceinline__ Visit same() const { return Visit{uniform(rows), uniform(p_low), uniform(first), uniform(low), uniform(high)}; }
    __device__ __forceinline__ bool has(int j) const { return j < first || (j >= low && j <= high); }
    __device__ __forceinline__ int tiles() const { return first + max(high - low + 1, 0); }
};
__device__ __forceinline__ Visit visit_of(const Sequence& s, int row0, int window, int sinks) {
    Visit v;
    v.rows = min(max(s.lq - row0, 0), kRows);
    v.p_low = s.lk - s.lq + row0;
    const int p_high = v.p_low + v.rows - 1;
    if (v.rows == 0 || p_high < 0) {
        v.first = 0, v.low = 1, v.high = 0;
        return v;
    }
    v.low = max(v.p_low - window + 1, 0) / kKeys;
    v.high = p_high / kKeys;
    v.first = min((min(sinks, p_high + 1) + kKeys - 1) / kKeys, v.low);
    return v;
}

// The key tiles of a block in the order they are visited: [0, first), then [low, high].
struct Order {
    int first, low, n;
    __device__ __forceinline__ Order same() const { return Order{uniform(first), uniform(low), uniform(n)}; }
    __device__ __forceinline__ int tile(int i) const { return i < first ? i : low + (i - first); }
};
__device__ __forceinline__ Order order_of(const Visit& a, const Visit& b) {
    Order o;
    const bool ha = a.low <= a.high, hb = b.low <= b.high;
    if (!ha && !hb) return Order{0, 0, 0};
    o.low = ha ? a.low : b.low;
    if (hb) o.low = min(o.low, b.low);
    const int high = max(ha ? a.high : -1, hb ? b.high : -1);
    o.first = min(max(a.first, b.first), o.low);
    o.n = o.first + (high - o.low + 1);
    return o;
}

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

// A thread's running softmax: `ref` is what its exponentials are relative to (base 2), `sum` their sum.
struct Row {
    float ref = -INFINITY, sum = 0.0f;
};

// One tile for one thread: scores from tensor memory, maximum, weights back (16 bits, half the columns). EDGE: column c is seen
// iff c <= above and (c > below or c < keep). `before` waits for the products with the tiles before this one; then O is
// rescaled if the reference moves. False: that wait ran out.
template <typename T, int DP, bool EDGE, typename Before>
__device__ __forceinline__ bool softmax_tile(Row& row, uint32_t t_s, uint32_t t_o, bool rescale, float scale_log2, int above, int below, int keep,
                                             uint32_t ready, Before before) {
    uint32_t s[kKeys];
    float top[2] = {-INFINITY, -INFINITY};
    tmem_load32(t_s, s);
    tmem_load32(t_s + 32, s + 32);
    wait_loads();
#pragma unroll
    for (int c = 0; c < kKeys; c += 32) {
        after_loads32(s + c);
        if (EDGE) {
            // (a mask of bits: with a comparison per column 128 of them took 9000 clocks)
            const uint32_t seen = low_bits(above + 1 - c) & (~low_bits(below + 1 - c) | low_bits(keep - c));
#pragma unroll
            for (int x = 0; x < 32; ++x) s[c + x] = seen >> x & 1 ? s[c + x] : 0xff800000u;
        }
#pragma unroll
        for (int x = 0; x < 32; x += 4) {
            top[0] = max3(top[0], __uint_as_float(s[c + x]), __uint_as_float(s[c + x + 1]));
            top[1] = max3(top[1], __uint_as_float(s[c + x + 2]), __uint_as_float(s[c + x + 3]));
        }
    }
    float m = max3(top[0], top[1], -INFINITY) * scale_log2;
    if (m == INFINITY) m = NAN;  // (a row with an infinite or a NaN score is NaN as a whole)
    const bool move = !(m <= row.ref + kSlack);
    if (__any_sync(0xffffffffu, move)) {
        const float next = move ? m : row.ref;
        const float factor = row.ref == -INFINITY ? 0.0f : exp2_fast(row.ref - next);
        row.sum *= factor;
        if (rescale) {
            if (!before()) return false;
#pragma unroll 1
            for (int c = 0; c < DP; c += 32) {
                uint32_t o[32];
                tmem_load32(t_o + c, o);
                wait_loads();
                after_loads32(o);
#pragma unroll
                for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * factor);
                tmem_store32(t_o + c, o);
            }
        }
        row.ref = next;
    }
    const float minus = row.ref == -INFINITY ? 0.0f : -row.ref;
    const uint64_t minus2 = pair(minus, minus), scale2 = pair(scale_log2, scale_log2);
    uint64_t part[2] = {pair(0.0f, 0.0f), pair(0.0f, 0.0f)};
    uint32_t w[32];
#pragma unroll
    for (int c = 0; c < kKeys; c += 2) {
        float e0, e1;
        unpair(fma2(pair(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), scale2, minus2), e0, e1);
        e0 = exp2_fast(e0), e1 = exp2_fast(e1);
        part[(c / 2) & 1] = add2(part[(c / 2) & 1], pair(e0, e1));
        w[c / 2] = pack2<T>(e0, e1);
    }
    tmem_store32(t_s, w);
    wait_stores();
    fence_before();
    bar_arrive(ready);
    float a, b, c, d;
    unpair(part[0], a, b);
    unpair(part[1], c, d);
    row.sum += (a + b) + (c + d);
    return true;
}

// What a block number stands for.
struct Work {
    Sequence sq;
    int row0, head;  // row0 < 0: nothing
};
__device__ __forceinline__ Work work_of(const Params& a, int number, int lane) {
    Work w;
    w.head = number % a.q_heads;
    const int block = a.slots - 1 - number / a.q_heads;  // the later rows of a sequence have more to do: first
    const RaggedBlock rb = ragged_block(a.r.q_offsets, a.r.batch, a.r.total_q, block, 2 * kRows, lane);
    w.sq = rb.b < 0 ? Sequence{0, 0, 0, 0} : sequence_of(a.r, rb.b);
    w.row0 = rb.b < 0 || (int64_t)rb.index * 2 * kRows >= w.sq.lq ? -1 : rb.index * 2 * kRows;  // (surplus numbers have nothing to do)
    return w;
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
    window_forward_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                          const __grid_constant__ CUtensorMap map_v, const Params a) {
    using S = Smem<DP>;
    constexpr bool kBf16 = sizeof(T) == 2 && !std::is_same<T, __half>::value;
    constexpr int kBlocks = DP / 64;  // 64-value column blocks of an operand
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem = (smem_u32(smem_raw) + 1023) & ~1023u;
    const int warp = uniform((int)(threadIdx.x >> 5)), lane = threadIdx.x & 31;
    // barriers: Q, and its place free again; of every stage: keys there, values there, values clear, stage done with; of the row
    // tiles' two buffers each: S ready, P ready, product with the values done; of the row tiles: O read; of the two places for
    // what a block number stands for: written, read by all other warps; the answer to a request; the ends of the two issuing warps
    const uint32_t bars = smem + S::kBars;
    const uint32_t bar_q = bars, bar_q_free = bars + 8, bar_k = bars + 16, bar_v = bar_k + 8 * S::kStages, bar_clear = bar_v + 8 * S::kStages,
                   bar_done = bar_clear + 8 * S::kStages, bar_s = bar_done + 8 * S::kStages, bar_p = bar_s + 32, bar_o = bar_p + 32,
                   bar_drained = bar_o + 32, bar_work = bar_drained + 16, bar_taken = bar_work + 16, bar_asked = bar_taken + 16,
                   bar_end = bar_asked + 8, slot = bar_end + 16;
    const uint32_t answer = bars + 512, works = answer + 16;  // 2 x 32 bytes

    Work work;
    if (warp == kValueWarp) {
        tmem_alloc(slot, 512);
    } else if (warp == kLoadWarp) {
        if (lane == 0) {
            tma_prefetch(&map_q), tma_prefetch(&map_k), tma_prefetch(&map_v);
            bar_init(bar_q, 1), bar_init(bar_q_free, 1);
            for (int i = 0; i < 4 * S::kStages; ++i) bar_init(bar_k + 8 * i, 1);
            for (int i = 0; i < 4; ++i) bar_init(bar_s + 8 * i, 1), bar_init(bar_p + 8 * i, kRows), bar_init(bar_o + 8 * i, 1);
            for (int i = 0; i < 2; ++i)
                bar_init(bar_drained + 8 * i, kRows), bar_init(bar_work + 8 * i, 1), bar_init(bar_taken + 8 * i, kThreads / 32 - 1), bar_init(bar_end + 8 * i, 1);
            bar_init(bar_asked, 1);
            bar_init_fence();
        }
        __syncwarp();
        work = work_of(a, (int)blockIdx.x, lane);
    }
    fence_before();
    __syncthreads();
    fence_after();
    uint32_t tmem;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(slot));
    tmem = uniform(tmem);
    // tensor memory: S (and P) of the two row tiles, two buffers each; O of the two row tiles
    const uint32_t t_s = tmem, t_o = tmem + 4 * kKeys;
    bool failed = false;

    // All warps run through the same work, each with running counts of the barriers' phases. Whole warps; false: no more, or `failed`.
    int turn = 0;
    Visit va, vb;
    Order order;
    const auto visits = [&] {
        va = visit_of(work.sq, work.row0, a.window, a.sinks).same(), vb = visit_of(work.sq, work.row0 + kRows, a.window, a.sinks).same();
        order = order_of(va, vb).same();
    };
    const auto next_work = [&] {
        const int at = turn & 1;
        if (!bar_wait_warp(bar_work + 8 * at, (turn >> 1) & 1, a.limit)) {
            failed = true;
            return false;
        }
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(work.sq.q0), "=r"(work.sq.lq), "=r"(work.sq.k0), "=r"(work.sq.lk) : "r"(works + 32 * at) : "memory");
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(work.row0), "=r"(work.head) : "r"(works + 32 * at + 16) : "memory");
        __syncwarp();
        if (elect()) bar_arrive(bar_taken + 8 * at);
        ++turn;
        if (uniform(work.row0) < 0) return false;
        visits();
        return true;
    };

    if (warp == kLoadWarp) {
        // ---- loads, and the order of the work: when a block's last loads are issued, the place of a block of the grid that
        // has not started is taken over (cluster launch control), so that its loads and first scores run beside the end of this one.
        int tiles = 0, queries = 0, asked = 0;  // so far: tiles issued, query tiles loaded, requests
        const auto publish = [&](int row0) {
            const int at = turn & 1;
            if (turn >= 2 && !bar_wait_warp(bar_taken + 8 * at, ((turn >> 1) - 1) & 1, a.limit)) {
                failed = true;
                return;
            }
            if (elect()) {
                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(works + 32 * at), "r"(work.sq.q0), "r"(work.sq.lq), "r"(work.sq.k0), "r"(work.sq.lk) : "memory");
                asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(works + 32 * at + 16), "r"(row0), "r"(work.head) : "memory");
                bar_arrive(bar_work + 8 * at);
            }
            __syncwarp();
            ++turn;
        };
        while (!failed) {
            if (work.row0 >= 0) {
                publish(work.row0);
                visits();
                if (order.n > 0 && !failed) {
                    if (queries > 0 && !bar_wait_warp(bar_q_free, (queries - 1) & 1, a.limit)) {
                        failed = true;
                        break;
                    }
                    const int base = uniform(tiles);
                    int issued = 0;
                    if (elect()) {
                        const int hk = work.head / a.group;
                        bar_expect(bar_q, 2 * S::kQuery);
                        for (int t = 0; t < 2; ++t)
                            for (int c = 0; c < kBlocks; ++c)
                                tma_load_3d(smem + S::kQ + t * S::kQuery + c * (kRows * 128), &map_q, 64 * c, work.head * a.q_mul, work.sq.q0 + work.row0 + t * kRows, bar_q);
                        for (int i = 0; i < order.n; ++i) {
                            const int g = base + i, st = g % S::kStages;
                            if (g >= S::kStages && !bar_wait(bar_done + 8 * st, (g / S::kStages - 1) & 1, a.limit)) break;
                            const uint32_t to = smem + S::kRing + st * 2 * S::kTile;
                            const int key = work.sq.k0 + order.tile(i) * kKeys;
                            bar_expect(bar_k + 8 * st, S::kTile);
                            for (int c = 0; c < kBlocks; ++c) tma_load_3d(to + c * (kKeys * 128), &map_k, 64 * c, hk * a.k_mul, key, bar_k + 8 * st);
                            bar_expect(bar_v + 8 * st, S::kTile);
                            for (int c = 0; c < kBlocks; ++c) tma_load_3d(to + S::kTile + c * (kKeys * 128), &map_v, 64 * c, hk * a.v_mul, key, bar_v + 8 * st);
                            issued = i + 1;
                        }
                    }
                    issued = uniform(issued);
                    tiles += issued, ++queries;
                    failed = issued < order.n;
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
            work = work_of(a, number, lane);
        }
        // nothing of this block's memory is given back while a copy is on its way, whoever gave up
        if (queries > 0) bar_wait_warp(bar_q, (queries - 1) & 1, kDrain);
        for (int i = max(0, tiles - S::kStages); i < tiles; ++i) {
            bar_wait_warp(bar_k + 8 * (i % S::kStages), (i / S::kStages) & 1, kDrain);
            bar_wait_warp(bar_v + 8 * (i % S::kStages), (i / S::kStages) & 1, kDrain);
        }
    } else if (warp == kScoreWarp) {
        // ---- scores, issued by one thread: a tile's once the weights that were in its buffer are used up. (Products
        // with the values have a warp of their own: a commit or a wait costs the issuing thread 100 clocks and more, and one
        // thread for both took 2100 clocks a step against 1280 of work.)
        constexpr uint32_t kDesc = mma_desc(kBf16, kKeys, false);
        int tiles = 0, queries = 0, buffers[2] = {0, 0};
        while (!failed && next_work()) {
            if (order.n == 0) continue;
            const int base = uniform(tiles), phase = uniform(queries) & 1;
            int n_s[2] = {uniform(buffers[0]), uniform(buffers[1])};
            if (elect()) {
                failed = !bar_wait(bar_q, phase, a.limit);
                for (int i = 0; i < order.n && !failed; ++i) {
                    const int j = order.tile(i), g = base + i, st = g % S::kStages;
                    if (!bar_wait(bar_k + 8 * st, (g / S::kStages) & 1, a.limit)) {
                        failed = true;
                        break;
                    }
                    const uint64_t k = smem_desc(smem + S::kRing + st * 2 * S::kTile);
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (failed || !(t == 0 ? va : vb).has(j)) continue;
                        const uint64_t q = smem_desc(smem + S::kQ + t * S::kQuery);
                        const int buffer = 2 * t + (n_s[t] & 1);
                        // (each row tile on its own: waiting for both made them run in step, their products in one burst)
                        if (n_s[t] >= 2 && !bar_wait(bar_o + 8 * buffer, ((n_s[t] >> 1) - 1) & 1, a.limit)) {
                            failed = true;
                            continue;
                        }
                        fence_after();
#pragma unroll
                        for (int x = 0; x < DP / 16; ++x)
                            mma_ss(t_s + kKeys * buffer, desc_at(q, (x >> 2) * (kRows * 128) + (x & 3) * 32),
                                   desc_at(k, (x >> 2) * (kKeys * 128) + (x & 3) * 32), kDesc | a.negate, x > 0);
                        mma_commit(bar_s + 8 * buffer);
                        ++n_s[t];
                    }
                }
                mma_commit(bar_q_free);
            }
            __syncwarp();
            failed = __any_sync(0xffffffffu, failed);
            tiles += order.n, ++queries, buffers[0] += va.tiles(), buffers[1] += vb.tiles();
        }
        if (elect()) {
            mma_commit(bar_end);  // the tensor memory is given back only when no product uses it any more
            bar_wait(bar_end, 0, kDrain);
        }
        __syncwarp();
    } else if (warp == kValueWarp) {
        // ---- products of the weights with the values, issued by one thread
        constexpr uint32_t kDesc = mma_desc(kBf16, DP, true);
        int tiles = 0, buffers[2] = {0, 0}, outputs[2] = {0, 0};
        while (!failed && next_work()) {
            const int base = uniform(tiles), out0 = uniform(outputs[0]), out1 = uniform(outputs[1]);
            const int from[2] = {uniform(buffers[0]), uniform(buffers[1])};
            int n_p[2] = {0, 0};
            if (elect()) {
                for (int i = 0; i < order.n && !failed; ++i) {
                    const int j = order.tile(i), g = base + i, st = g % S::kStages;
                    if (!bar_wait(bar_clear + 8 * st, (g / S::kStages) & 1, a.limit)) {
                        failed = true;
                        break;
                    }
                    const uint64_t values = smem_desc(smem + S::kRing + st * 2 * S::kTile + S::kTile, kKeys * 128);
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (failed || !(t == 0 ? va : vb).has(j)) continue;
                        const int n = from[t] + n_p[t], buffer = 2 * t + (n & 1), out = t == 0 ? out0 : out1;
                        if (!bar_wait(bar_p + 8 * buffer, (n >> 1) & 1, a.limit) ||
                            (n_p[t] == 0 && out > 0 && !bar_wait(bar_drained + 8 * t, (out - 1) & 1, a.limit))) {
                            failed = true;
                            continue;
                        }
                        fence_after();
#pragma unroll
                        for (int x = 0; x < kKeys / 16; ++x)
                            mma_ts(t_o + DP * t, t_s + kKeys * buffer + 8 * x, desc_at(values, x * 2048), kDesc, n_p[t] > 0 || x > 0);
                        mma_commit(bar_o + 8 * buffer);
                        ++n_p[t];
                    }
                    if (!failed) mma_commit(bar_done + 8 * st);
                }
            }
            __syncwarp();
            failed = __any_sync(0xffffffffu, failed);
            tiles += order.n;
            buffers[0] += va.tiles(), buffers[1] += vb.tiles();
            outputs[0] += va.tiles() > 0, outputs[1] += vb.tiles() > 0;
        }
        if (elect()) {
            mma_commit(bar_end + 8);
            bar_wait(bar_end + 8, 0, kDrain);
        }
        __syncwarp();
    } else if (warp == kClearWarp) {
        // ---- values nobody here sees (behind the last query, before the first window) have weight zero, but zero times a NaN
        // that lies there would not be zero: such rows are cleared before the products may read the tile.
        int tiles = 0;
        while (!failed && next_work()) {
            const int first_seen = max(va.p_low - a.window + 1, 0);
            const int last_seen = work.sq.lk - work.sq.lq + min(work.row0 + 2 * kRows, work.sq.lq) - 1;
            for (int i = 0; i < order.n; ++i, ++tiles) {
                const int st = tiles % S::kStages, key0 = order.tile(i) * kKeys;
                if (!bar_wait_warp(bar_v + 8 * st, (tiles / S::kStages) & 1, a.limit)) {
                    failed = true;
                    break;
                }
                const int clear_low = min(max(first_seen - key0, 0), kKeys);
                const int clear_high = min(max(last_seen + 1 - key0, 0), kKeys);
                const int keep = min(max(a.sinks - key0, 0), kKeys);  // first tokens stay
                if (clear_low > keep || clear_high < kKeys) {
                    for (int x = lane; x < kKeys * 8 * kBlocks; x += 32) {
                        const int row = (x >> 3) & (kKeys - 1);
                        if ((row < clear_low && row >= keep) || row >= clear_high)
                            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(smem + S::kRing + st * 2 * S::kTile + S::kTile + x * 16), "r"(0)
                                         : "memory");
                    }
                    fence_async();
                    __syncwarp();
                }
                if (elect()) bar_arrive(bar_clear + 8 * st);
                __syncwarp();
            }
        }
    } else {
        // ---- softmax: thread = row
        const int t = warp >> 2;
        const int r = threadIdx.x & (kRows - 1);
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // tensor-memory lane of the warp's first row
        const uint32_t to = t_o + DP * t + lanes;
        int done = 0;  // tiles so far
        // Waits for the product of the last tile's weights. Scores of a tile are issued when the product of the last but one is
        // complete: of the two barriers that the products arrive on in turn, the phase before is over.
        const auto before = [&] {
            const int last = done - 1;
            const bool ok = bar_wait_warp(bar_o + 8 * (2 * t + (last & 1)), (last >> 1) & 1, a.limit);
            fence_after();
            return ok;
        };
        while (!failed && next_work()) {
            const Visit v = t == 0 ? va : vb;
            const int p = v.p_low + r;
            Row row;
            const int start = done;
            for (int i = 0; i < order.n; ++i) {
                const int j = order.tile(i);
                if (!v.has(j)) continue;
                const int buffer = 2 * t + (done & 1);
                if (!bar_wait_warp(bar_s + 8 * buffer, (done >> 1) & 1, a.limit)) {
                    failed = true;
                    break;
                }
                fence_after();
                const int key0 = j * kKeys, last_p = v.p_low + kRows - 1;
                const uint32_t ts = t_s + kKeys * buffer + lanes, ready = bar_p + 8 * buffer;
                const bool edge = key0 + kKeys - 1 > v.p_low || (key0 <= last_p - a.window && key0 + kKeys > a.sinks);
                const bool ok =
                    edge ? softmax_tile<T, DP, true>(row, ts, to, done > start, a.scale_log2, p - key0, p - key0 - a.window, a.sinks - key0, ready, before)
                         : softmax_tile<T, DP, false>(row, ts, to, done > start, a.scale_log2, 0, 0, 0, ready, before);
                if (!ok) {
                    failed = true;
                    break;
                }
                ++done;
            }
            // ---- epilogue
            if (done > start && !failed) failed = !before();
            if (failed) break;
            const float inv = row.sum == 0.0f ? 0.0f : 1.0f / row.sum;
            const int64_t token = (int64_t)work.sq.q0 + work.row0 + t * kRows + r;
            if (a.lse != nullptr && r < v.rows)
                a.lse[(int64_t)work.head * a.total_q + token] = row.sum == 0.0f ? -INFINITY : row.ref * a.scale_ln + logf(row.sum);
            T* out = static_cast<T*>(a.o) + token * a.o_token + (int64_t)work.head * a.o_head;
#pragma unroll 1
            for (int c = 0; c < DP; c += 32) {
                uint32_t o[32];
                if (done > start) {
                    tmem_load32(to + c, o);
                    wait_loads();
                    after_loads32(o);
                    if (c + 32 == DP) {  // the next work's products may overwrite O
                        fence_before();
                        bar_arrive(bar_drained + 8 * t);
                    }
                }
                if (r < v.rows) {
#pragma unroll
                    for (int x = 0; x < 32; x += 8) {
                        if (c + x < a.dim) {
                            uint4 w = make_uint4(0, 0, 0, 0);
                            if (row.sum != 0.0f) {
                                w.x = pack2<T>(__uint_as_float(o[x]) * inv, __uint_as_float(o[x + 1]) * inv);
                                w.y = pack2<T>(__uint_as_float(o[x + 2]) * inv, __uint_as_float(o[x + 3]) * inv);
                                w.z = pack2<T>(__uint_as_float(o[x + 4]) * inv, __uint_as_float(o[x + 5]) * inv);
                                w.w = pack2<T>(__uint_as_float(o[x + 6]) * inv, __uint_as_float(o[x + 7]) * inv);
                            }
                            *reinterpret_cast<uint4*>(out + c + x) = w;
                        }
                    }
                }
            }
        }
        fence_before();
    }
    if (failed && a.fault != nullptr) *reinterpret_cast<volatile int*>(a.fault) = 1;
    __syncthreads();
    if (warp == kValueWarp) {
        fence_after();
        tmem_free(tmem, 512);
    }
}

template <typename T, int DP>
cudaError_t launch(cudaStream_t s, const AttentionArgs& a) {
    using S = Smem<DP>;
    CUtensorMap mq, mk, mv;
    if (!head_map(&mq, a.q, a.total_q, a.q_heads, a.dim, a.type, kRows) || !head_map(&mk, a.k, a.total_k, a.kv_heads, a.dim, a.type, kKeys) ||
        !head_map(&mv, a.v, a.total_k, a.kv_heads, a.dim, a.type, kKeys))
        return cudaErrorNotSupported;
    Params p = {};
    p.r = Ragged{a.q_offsets, a.k_offsets, a.batch, a.total_q, a.total_k};
    p.window = a.window, p.sinks = a.sinks, p.q_heads = a.q_heads, p.group = a.q_heads / a.kv_heads, p.dim = a.dim;
    p.total_q = a.total_q;
    p.slots = ragged_slots(a.total_q, a.batch, a.q_offsets != nullptr, 2 * kRows);
    p.q_mul = a.q.head != 0, p.k_mul = a.k.head != 0, p.v_mul = a.v.head != 0;
    p.negate = a.scale < 0.0f ? kNegateA : 0;
    p.scale_log2 = fabsf(a.scale) * kLog2e, p.scale_ln = 1.0f / kLog2e;
    p.o = a.o.p, p.o_token = a.o.token, p.o_head = a.o.head, p.lse = a.lse;
    p.limit = window_wait_limit(a), p.fault = a.wait.fault_word;
    static SharedMemoryOnce once;
    const cudaError_t e = once.allow(reinterpret_cast<const void*>(window_forward_kernel<T, DP>), S::kTotal);
    if (e != cudaSuccess) return e;
    window_forward_kernel<T, DP><<<(unsigned)((int64_t)p.slots * a.q_heads), kThreads, S::kTotal, s>>>(mq, mk, mv, p);
    return cudaGetLastError();
}

}  // namespace

bool window_tensor_ready(const AttentionTensor& t, int64_t tokens, int heads, int dim) {
    // TMA: 16-byte rows and strides (a head stride of 0 is read as one head; a token stride of 0 has no such form)
    return (reinterpret_cast<uintptr_t>(t.p) & 15) == 0 && dim % 8 == 0 && (t.token % 8 == 0 || tokens <= 1) &&
           (t.head % 8 == 0 || heads <= 1) && (t.token > 0 || tokens <= 1);
}

cudaError_t window_forward_mma(cudaStream_t s, const AttentionArgs& a) {
    if (a.type == MACA_R_16BF) return a.dim <= 64 ? launch<__nv_bfloat16, 64>(s, a) : launch<__nv_bfloat16, 128>(s, a);
    return a.dim <= 64 ? launch<__half, 64>(s, a) : launch<__half, 128>(s, a);
}

}  // namespace mcsp_b200
