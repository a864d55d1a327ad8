// Windowed attention for single tokens over a (paged) cache, fp16 / bf16, rows of 16-byte multiples.
//
// The query heads that share a key head (up to 16) are the rows of one m16n8k16 product, so every key and value is read
// once for all of them; what bounds the call is reading them (2 * headDim * 2 bytes per key and key head), not the products.
// The seen keys (first tokens, then the window) are one compact list, cut into `splits` equal parts, one thread block each;
// inside a block every warp takes tiles of 16 keys in turn through its own ring of asynchronous 16-byte copies and keeps a
// running softmax of its own. Keys that are not seen (behind the list, on a page outside the cache) are copied as zeros and
// masked, so nothing that lies there is read. The warps' results are joined in shared memory, the blocks' of a sequence over
// distributed shared memory (they form a cluster) or, where that many blocks exceed a cluster, through the work buffer.
#include <type_traits>

#include "window_common.h"

namespace mcsp_b200 {
namespace {

using namespace window;

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kKeys = 16;    // keys of a tile
constexpr int kHeads = 16;   // query heads of a block
constexpr int kCluster = 8;  // most blocks of one sequence and key head that join without the work buffer
constexpr float kLog2e = 1.4426950408889634f;
// A row's reference follows its maximum in steps of at least 2^8, so that weights stay below 256, far from fp16's 65504. The product
// with V takes them rounded to the inputs' type (one 16-bit type for both operands), the row's sum in fp32.
constexpr float kSlack = 8.0f;

template <int DP>
struct Ring {
    static constexpr int kStages = DP == 128 ? 3 : 4;
    static constexpr int kOperand = kKeys * DP * 2;     // a tile of keys, or of values
    static constexpr int kWarp = kStages * 2 * kOperand;  // >= kHeads * DP * 4: the warp's sums are left here
    static constexpr int kTotal = kWarps * kWarp;
};

struct Params {
    const int* lengths;
    const int* table;
    int num_pages, max_pages, page_size;
    int64_t room;
    int window, sinks, q_heads, kv_heads, group, head_tiles, dim, splits;
    float scale_log2;
    const void *q, *k, *v;
    int64_t q_token, q_head, k_page, k_token, k_head, v_page, v_token, v_head, o_token, o_head;
    void* o;
    float* lse;
    float* partial;  // null: the blocks of a sequence form a cluster. [item][split][kHeads][DP + 2]: sums, maximum, sum of weights
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
// 16 bytes, or zeros where `bytes` is 0 (then the source is not read).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void load_matrices(uint32_t* r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void load_matrices_t(uint32_t* r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void multiply(float* d, const uint32_t* a, const uint32_t* b) {
    if (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if (std::is_same<T, __half>::value) {
        const __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t remote(uint32_t addr, int rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float load_remote(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 load_remote4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

// Four values of one output row, and its lse: sums joined over `n` parts, part i at (m, l, o) = get(i).
template <typename T, typename Get>
__device__ __forceinline__ void write_joined(const Params& a, int b, int head, int c, int n, Get get) {
    float top = -INFINITY;
    for (int i = 0; i < n; ++i) top = fmaxf(top, get(i, -2).x);
    const float ref = top == -INFINITY ? 0.0f : top;
    float l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int i = 0; i < n; ++i) {
        // (a part whose keys all score NaN has no maximum; its sum carries the NaN)
        const float w = exp2_fast(get(i, -2).x - ref), li = get(i, -1).x;
        const float4 v = get(i, c);
        if (li != 0.0f) {
            const float f = get(i, -2).x == -INFINITY ? 1.0f : w;
            l += f * li, o.x += f * v.x, o.y += f * v.y, o.z += f * v.z, o.w += f * v.w;
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (c < a.dim) {
        uint2 w = make_uint2(0u, 0u);
        if (l != 0.0f) w = make_uint2(pack2<T>(o.x * inv, o.y * inv), pack2<T>(o.z * inv, o.w * inv));
        *reinterpret_cast<uint2*>(static_cast<T*>(a.o) + (int64_t)b * a.o_token + (int64_t)head * a.o_head + c) = w;
    }
    if (c == 0 && a.lse != nullptr) a.lse[(int64_t)b * a.q_heads + head] = l == 0.0f ? -INFINITY : ref / kLog2e + logf(l);
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads) window_decode_kernel(const Params a) {
    using R = Ring<DP>;
    constexpr int kChunks = DP / 8;     // 16-byte chunks of a row
    constexpr int kSteps = DP / 16;     // contraction steps of the scores
    extern __shared__ __align__(128) uint8_t smem_raw[];
    __shared__ float s_m[kWarps][kHeads], s_l[kWarps][kHeads], s_block_m[kHeads], s_block_l[kHeads];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = blockIdx.x % a.splits;
    const int item = blockIdx.x / a.splits;
    const int head_tile = item % a.head_tiles, hk = (item / a.head_tiles) % a.kv_heads, b = item / a.head_tiles / a.kv_heads;
    const int head0 = hk * a.group + head_tile * kHeads, rows = min(kHeads, a.group - head_tile * kHeads);
    const uint32_t ring = smem_u32(smem_raw) + warp * R::kWarp;

    const int len = (int)min((int64_t)max(__ldg(a.lengths + b), 0), a.room);
    const int low = max(len - a.window, 0), first = min(low, a.sinks);
    const int keys = first + len - low;
    const int tiles = (keys + kKeys - 1) / kKeys;
    const int tile0 = (int)((int64_t)tiles * split / a.splits), tile1 = (int)((int64_t)tiles * (split + 1) / a.splits);
    const int mine = tile0 + warp < tile1 ? (tile1 - tile0 - warp + kWarps - 1) / kWarps : 0;

    // Lanes 0 .. 15 look up the place of the tile's key `lane`: page (-1: not seen) and token of the page.
    const auto lookup = [&](int i, int& page, int& at) {
        page = -1, at = 0;
        const int n = (tile0 + warp + i * kWarps) * kKeys + (lane & 15);
        if (i < mine && n < keys) {
            const int j = n < first ? n : low + (n - first);
            const int p = j / a.page_size;
            at = j - p * a.page_size;
            page = a.table != nullptr ? __ldg(a.table + (int64_t)b * a.max_pages + p) : b;
            if (page < 0 || page >= a.num_pages) page = -1;
        }
    };
    // lane: 16-byte chunk lane % kChunks of rows lane / kChunks, + 32 / kChunks, ...
    constexpr int kAside = 32 / kChunks;
    const int chunk = lane % kChunks, aside = lane / kChunks;
    const T* const kbase = static_cast<const T*>(a.k) + (int64_t)hk * a.k_head + 8 * chunk;
    const T* const vbase = static_cast<const T*>(a.v) + (int64_t)hk * a.v_head + 8 * chunk;
    const auto issue = [&](int i, int page, int at) {
        const uint32_t to = ring + (i % R::kStages) * 2 * R::kOperand;
#pragma unroll
        for (int r = 0; r < kKeys; r += kAside) {
            const int row = r + aside;
            const int pg = __shfl_sync(0xffffffffu, page, row), tk = __shfl_sync(0xffffffffu, at, row);
            const int bytes = pg >= 0 && 8 * chunk < a.dim ? 16 : 0;
            const int64_t pz = pg >= 0 ? pg : 0;
            const uint32_t place = row * (2 * DP) + ((chunk ^ (row & 7)) << 4);
            copy16(to + place, bytes ? kbase + pz * a.k_page + (int64_t)tk * a.k_token : a.k, bytes);
            copy16(to + R::kOperand + place, bytes ? vbase + pz * a.v_page + (int64_t)tk * a.v_token : a.v, bytes);
        }
    };

    float o[2 * kSteps][4];
#pragma unroll
    for (int i = 0; i < 2 * kSteps; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[i][x] = 0.0f;
    float ref[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};  // rows lane / 4 and + 8; the lane's part of the sum

    unsigned seen[R::kStages];  // the keys of a stage that are seen (registers: the loop below is unrolled by the stages)
    int page, at;
#pragma unroll
    for (int i = 0; i < R::kStages - 1; ++i) {
        lookup(i, page, at);
        seen[i] = __ballot_sync(0xffffffffu, page >= 0) & 0xffffu;
        if (i < mine) issue(i, page, at);
        commit_copies();
    }
    lookup(R::kStages - 1, page, at);
    // the query heads as the left operand: lane holds rows lane / 4 and + 8, columns 2 * (lane % 4) and + 8 of every step
    uint32_t q[kSteps][4];
    {
        const T* base = static_cast<const T*>(a.q) + (int64_t)b * a.q_token;
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int row = (lane >> 2) + 8 * (x & 1), c = 16 * k + 2 * (lane & 3) + 8 * (x >> 1);
                q[k][x] = row < rows && c < a.dim ? __ldg(reinterpret_cast<const unsigned*>(base + (int64_t)(head0 + row) * a.q_head + c)) : 0u;
            }
    }

    for (int i0 = 0; i0 < mine; i0 += R::kStages) {
#pragma unroll
        for (int s = 0; s < R::kStages; ++s) {
            const int i = i0 + s;
            if (i >= mine) break;
            const int ahead = i + R::kStages - 1;
            seen[(s + R::kStages - 1) % R::kStages] = __ballot_sync(0xffffffffu, page >= 0) & 0xffffu;
            if (ahead < mine) issue(ahead, page, at);
            commit_copies();
            lookup(ahead + 1, page, at);
            wait_copies<R::kStages - 1>();
            __syncwarp();
            const uint32_t kt = ring + s * 2 * R::kOperand, vt = kt + R::kOperand;
            float x[2][4] = {};
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                uint32_t m[4];
                const int row = ((lane >> 4) << 3) + (lane & 7), c = 2 * k + ((lane >> 3) & 1);
                load_matrices(m, kt + row * (2 * DP) + ((c ^ (row & 7)) << 4));
                multiply<T>(x[0], q[k], m);
                multiply<T>(x[1], q[k], m + 2);
            }
            const unsigned bits = seen[s];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    x[h][y] *= a.scale_log2;
                    if (!(bits >> (8 * h + 2 * (lane & 3) + (y & 1)) & 1)) x[h][y] = -INFINITY;
                }
            float top[2];
#pragma unroll
            for (int y = 0; y < 2; ++y) top[y] = fmaxf(fmaxf(x[0][2 * y], x[0][2 * y + 1]), fmaxf(x[1][2 * y], x[1][2 * y + 1]));
            if (__any_sync(0xffffffffu, top[0] > ref[0] + kSlack || top[1] > ref[1] + kSlack)) {
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    float t = fmaxf(top[y], __shfl_xor_sync(0xffffffffu, top[y], 1));
                    t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
                    const float next = fmaxf(ref[y], t);
                    const float f = ref[y] == -INFINITY ? 0.0f : exp2_fast(ref[y] - next);
                    sum[y] *= f;
#pragma unroll
                    for (int d = 0; d < 2 * kSteps; ++d) o[d][2 * y] *= f, o[d][2 * y + 1] *= f;
                    ref[y] = next;
                }
            }
            uint32_t p[4];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const float minus = ref[y] == -INFINITY ? 0.0f : ref[y];
                    const float e0 = exp2_fast(x[h][2 * y] - minus), e1 = exp2_fast(x[h][2 * y + 1] - minus);
                    sum[y] += e0 + e1;
                    p[2 * h + y] = pack2<T>(e0, e1);
                }
#pragma unroll
            for (int d = 0; d < kSteps; ++d) {
                uint32_t m[4];
                const int row = (((lane >> 3) & 1) << 3) + (lane & 7), c = 2 * d + (lane >> 4);
                load_matrices_t(m, vt + row * (2 * DP) + ((c ^ (row & 7)) << 4));
                multiply<T>(o[2 * d], p, m);
                multiply<T>(o[2 * d + 1], p, m + 2);
            }
            __syncwarp();
        }
    }
    wait_copies<0>();
    __syncwarp();
    // ---- the warps' results side by side in shared memory, then one per block
    float* const own = reinterpret_cast<float*>(smem_raw + warp * R::kWarp);
#pragma unroll
    for (int y = 0; y < 2; ++y) {
        sum[y] += __shfl_xor_sync(0xffffffffu, sum[y], 1);
        sum[y] += __shfl_xor_sync(0xffffffffu, sum[y], 2);
        const int row = (lane >> 2) + 8 * y;
        if ((lane & 3) == 0) s_m[warp][row] = ref[y], s_l[warp][row] = sum[y];
#pragma unroll
        for (int d = 0; d < 2 * kSteps; ++d)
            *reinterpret_cast<float2*>(own + row * DP + 8 * d + 2 * (lane & 3)) = make_float2(o[d][2 * y], o[d][2 * y + 1]);
    }
    __syncthreads();
    float* const all = reinterpret_cast<float*>(smem_raw);
    constexpr int kWarpFloats = R::kWarp / 4;
    for (int x = threadIdx.x * 4; x < rows * DP; x += kThreads * 4) {
        const int row = x / DP;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w][row]);
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float l = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float lw = s_l[w][row];
            if (lw != 0.0f) {
                const float f = s_m[w][row] == -INFINITY ? 1.0f : exp2_fast(s_m[w][row] - top);
                const float4 y = *reinterpret_cast<const float4*>(all + w * kWarpFloats + x);
                l += f * lw, v.x += f * y.x, v.y += f * y.y, v.z += f * y.z, v.w += f * y.w;
            }
        }
        *reinterpret_cast<float4*>(all + x) = v;  // (warp 0's place: only this thread reads and writes it)
        if (x % DP == 0) s_block_m[row] = top, s_block_l[row] = l;
    }
    __syncthreads();
    if (a.partial != nullptr) {
        float* to = a.partial + ((int64_t)item * a.splits + split) * kHeads * (DP + 2);
        for (int x = threadIdx.x; x < rows * DP; x += kThreads) to[2 * kHeads + x] = all[x];
        if ((int)threadIdx.x < rows) to[threadIdx.x] = s_block_m[threadIdx.x], to[kHeads + threadIdx.x] = s_block_l[threadIdx.x];
        return;
    }
    if (a.splits == 1) {
        for (int x = threadIdx.x * 4; x < rows * DP; x += kThreads * 4) {
            const int row = x / DP;
            write_joined<T>(a, b, head0 + row, x % DP, 1, [&](int, int c) {
                if (c == -2) return make_float4(s_block_m[row], 0, 0, 0);
                if (c == -1) return make_float4(s_block_l[row], 0, 0, 0);
                return *reinterpret_cast<const float4*>(all + x);
            });
        }
        return;
    }
    // ---- the blocks of a cluster share out the rows' values; block `split` is its rank
    cluster_sync();
    const uint32_t am = smem_u32(s_block_m), al = smem_u32(s_block_l), ao = smem_u32(all);
    for (int x = (split * kThreads + (int)threadIdx.x) * 4; x < rows * DP; x += a.splits * kThreads * 4) {
        const int row = x / DP;
        write_joined<T>(a, b, head0 + row, x % DP, a.splits, [&](int i, int c) {
            if (c == -2) return make_float4(load_remote(remote(am + 4 * row, i)), 0, 0, 0);
            if (c == -1) return make_float4(load_remote(remote(al + 4 * row, i)), 0, 0, 0);
            return load_remote4(remote(ao + 4 * x, i));
        });
    }
    cluster_sync();  // nobody leaves while its shared memory is read
}

// One warp per (item, row): 32 lanes x 4 values.
template <typename T, int DP>
__global__ void __launch_bounds__(256) window_decode_join_kernel(const Params a, int64_t items) {
    const int64_t w = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 5;
    const int64_t item = w / kHeads;
    const int row = (int)(w % kHeads), c = 4 * (threadIdx.x & 31);
    if (item >= items || c >= DP) return;
    const int head_tile = (int)(item % a.head_tiles), hk = (int)((item / a.head_tiles) % a.kv_heads), b = (int)(item / a.head_tiles / a.kv_heads);
    if (row >= min(kHeads, a.group - head_tile * kHeads)) return;
    const float* from = a.partial + item * a.splits * kHeads * (DP + 2);
    write_joined<T>(a, b, hk * a.group + head_tile * kHeads + row, c, a.splits, [&](int i, int x) {
        const float* p = from + (int64_t)i * kHeads * (DP + 2);
        if (x == -2) return make_float4(p[row], 0, 0, 0);
        if (x == -1) return make_float4(p[kHeads + row], 0, 0, 0);
        return *reinterpret_cast<const float4*>(p + 2 * kHeads + row * DP + x);
    });
}

int64_t decode_items(const DecodeArgs& a) {
    const int group = a.q_heads / a.kv_heads;
    return (int64_t)a.batch * a.kv_heads * ((group + kHeads - 1) / kHeads);
}

// Parts per sequence and key head. A part costs its keys and about 250 more (its start, its first loads, the join: fitted to
// 64 sequences x 8 key heads x 4100 keys, where 1, 2, 3 parts took 196, 206, 217 us); with headDim above 64, which it was fitted
// for, two blocks run per SM, so the launch costs its whole rounds of blocks (headDim up to 64: three fit, and the count of rounds
// is too high). At least 64 keys (a tile per warp) each. Up to 8 parts join as a cluster; more take the work buffer
// and a second launch (200 keys' worth) and only come into question when an eighth is still long.
int decode_splits(const DecodeArgs& a) {
    const int64_t room = a.max_pages * a.page_size, items = decode_items(a);
    const int64_t most = (int64_t)a.window + a.sinks < room ? (int64_t)a.window + a.sinks : room;
    const int64_t slots = 2LL * a.sm_count;
    int best = 1;
    int64_t least = INT64_MAX;
    for (int s = 1; s <= 64; s = s < kCluster ? s + 1 : 2 * s) {
        if (s > 1 && (most < 64LL * s || (s > kCluster && most / kCluster < 1024))) break;
        const int64_t cost = (items * s + slots - 1) / slots * (most / s + 250) + (s > kCluster ? 200 : 0);
        if (cost < least) least = cost, best = s;
    }
    return best;
}

template <typename T, int DP>
cudaError_t launch(cudaStream_t s, const DecodeArgs& a, void* buffer) {
    Params p = {};
    p.lengths = a.lengths, p.table = a.page_table;
    p.num_pages = (int)a.num_pages, p.max_pages = (int)a.max_pages, p.page_size = (int)a.page_size, p.room = a.max_pages * a.page_size;
    p.window = a.window, p.sinks = a.sinks, p.q_heads = a.q_heads, p.kv_heads = a.kv_heads, p.group = a.q_heads / a.kv_heads, p.dim = a.dim;
    p.head_tiles = (p.group + kHeads - 1) / kHeads;
    p.splits = decode_splits(a);
    p.scale_log2 = a.scale * kLog2e;
    p.q = a.q.p, p.q_token = a.q.token, p.q_head = a.q.head;
    p.k = a.k.p, p.k_page = a.k_page, p.k_token = a.k.token, p.k_head = a.k.head;
    p.v = a.v.p, p.v_page = a.v_page, p.v_token = a.v.token, p.v_head = a.v.head;
    p.o = a.o.p, p.o_token = a.o.token, p.o_head = a.o.head, p.lse = a.lse;
    const int64_t items = decode_items(a);
    if (items * p.splits > 0x7fffffffLL) return cudaErrorInvalidValue;
    if (p.splits > kCluster) p.partial = static_cast<float*>(align_up_256(buffer));
    static SharedMemoryOnce once;
    cudaError_t e = once.allow(reinterpret_cast<const void*>(window_decode_kernel<T, DP>), Ring<DP>::kTotal);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(items * p.splits));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Ring<DP>::kTotal;
    cfg.stream = s;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = p.partial != nullptr ? 1 : (unsigned)p.splits;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = attr.val.clusterDim.x > 1 ? 1 : 0;
    e = cudaLaunchKernelEx(&cfg, window_decode_kernel<T, DP>, static_cast<const Params>(p));
    if (e != cudaSuccess || p.partial == nullptr) return e;
    window_decode_join_kernel<T, DP><<<(unsigned)((items * kHeads + 7) / 8), 256, 0, s>>>(p, items);
    return cudaGetLastError();
}

}  // namespace

bool window_decode_ready(const DecodeArgs& a) {
    const auto rows = [](const AttentionTensor& t, int64_t page) {
        return (reinterpret_cast<uintptr_t>(t.p) & 15) == 0 && t.token % 8 == 0 && t.head % 8 == 0 && page % 8 == 0;
    };
    return a.type != MACA_R_32F && a.dim % 8 == 0 && rows(a.q, 0) && rows(a.o, 0) && rows(a.k, a.k_page) && rows(a.v, a.v_page);
}

size_t window_decode_mma_bytes(const DecodeArgs& a) {
    const int splits = decode_splits(a);
    if (splits <= kCluster) return 256;
    return size_t(decode_items(a)) * splits * kHeads * ((a.dim <= 64 ? 64 : 128) + 2) * 4 + 256;
}

cudaError_t window_decode_mma(cudaStream_t s, const DecodeArgs& a, void* buffer) {
    if (a.type == MACA_R_16BF) return a.dim <= 64 ? launch<__nv_bfloat16, 64>(s, a, buffer) : launch<__nv_bfloat16, 128>(s, a, buffer);
    return a.dim <= 64 ? launch<__half, 64>(s, a, buffer) : launch<__half, 128>(s, a, buffer);
}

}  // namespace mcsp_b200
