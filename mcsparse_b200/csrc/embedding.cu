// Rows of a table by token ids, Y = alpha * S * E, and the table's gradient, dE = alpha * S^T * dY + beta * dE, for the
// count x rows matrix S with one 1 per row (its column: the token's id). S is never stored.
//
// Lookup: one pass; a warp moves a piece of one row with 16-byte loads and stores. Bound by memory (count * width read,
// unless rows repeat, and written).
//
// Gradient, three launches:
//   1. S^T in CSR form is the tokens sorted by id: a stable radix sort of (id, position) pairs. Up to 131072 tokens one cluster
//      of 8 thread blocks sorts them in two passes or three (ids below 2^18: two 9-bit digits), its digit counts exchanged over
//      distributed shared memory, its barriers the cluster's; more tokens take the multi-launch sort of transpose.cu. The
//      other blocks of the launch meanwhile write the rows no token names (beta = 0: zeros, most of the traffic of a large
//      table); each finds them by marking the ids of its own range of rows in shared memory, so it need not wait for the sort.
//   2. The sorted tokens are cut into chunks of equal size whatever the ids are, so a token that fills half the batch costs no
//      more than any other; a warp owns one chunk and a slab of columns, adds in fp32 and writes every sum that lies inside
//      its chunk. A sum that crosses chunks is left as one partial per chunk.
//   3. Those partials are put together in chunk order.
// No atomics: the order of every addition follows from ids and sizes. Bound by memory: count * width read, rows * width written.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "internal.h"

namespace mcsp_b200 {
namespace {

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// V consecutive values, moved with the widest accesses their size allows (16 bytes).
template <typename T, int V>
struct alignas(sizeof(T) * V >= 16 ? 16 : sizeof(T) * V) Pack {
    T v[V];
};

// How a thread holds its columns: V consecutive ones when every row starts on a 16-byte boundary and the width is a
// multiple of V; otherwise kLoose single columns, 32 apart, so that a warp's accesses stay together.
constexpr int kLoose = 4;
template <int V>
struct Columns {
    static constexpr int kPer = V > 1 ? V : kLoose;
    static constexpr int kSlab = 32 * kPer;
    __device__ static __forceinline__ int64_t at(int lane, int i) { return V > 1 ? lane * V + i : lane + 32 * i; }
};

template <typename T, int V>
__device__ __forceinline__ void load_columns(const T* row, int64_t first, int64_t width, int lane, float* out) {
    if (V > 1) {
        const int64_t c = first + lane * V;
        if (c < width) {
            const Pack<T, V> p = *reinterpret_cast<const Pack<T, V>*>(row + c);
#pragma unroll
            for (int i = 0; i < V; ++i) out[i] = to_float(p.v[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kLoose; ++i) {
            const int64_t c = first + lane + 32 * i;
            if (c < width) out[i] = to_float(row[c]);
        }
    }
}

template <typename T, int V>
__device__ __forceinline__ void store_columns(T* row, int64_t first, int64_t width, int lane, const float* in) {
    if (V > 1) {
        const int64_t c = first + lane * V;
        if (c < width) {
            Pack<T, V> p;
#pragma unroll
            for (int i = 0; i < V; ++i) p.v[i] = from_float<T>(in[i]);
            *reinterpret_cast<Pack<T, V>*>(row + c) = p;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kLoose; ++i) {
            const int64_t c = first + lane + 32 * i;
            if (c < width) row[c] = from_float<T>(in[i]);
        }
    }
}

// ----------------------------------------------------------------------------- lookup

constexpr int kLookupPieces = 4;  // slabs per warp, all loads in flight together

template <typename E, typename Y, typename I, int V>
__global__ void __launch_bounds__(256)
    embedding_lookup_kernel(int64_t count, int64_t rows, int64_t width, const I* __restrict__ ids, int base,
                            const E* __restrict__ table, int64_t ld_e, Y* __restrict__ out, int64_t ld_y,
                            ScalarArg<float> alpha_arg, int64_t pieces) {
    constexpr int kPer = Columns<V>::kPer, kSlab = Columns<V>::kSlab;
    const int64_t warp = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    const int64_t t = warp / pieces;
    if (t >= count) return;
    const int64_t first = (warp - t * pieces) * (kSlab * kLookupPieces);
    const float alpha = alpha_arg.get();
    const int64_t id = (int64_t)__ldg(ids + t) - base;
    float v[kLookupPieces][kPer];
#pragma unroll
    for (int p = 0; p < kLookupPieces; ++p)
#pragma unroll
        for (int i = 0; i < kPer; ++i) v[p][i] = 0.0f;
    const bool live = id >= 0 && id < rows;
    if (live) {
        const E* row = table + id * ld_e;
#pragma unroll
        for (int p = 0; p < kLookupPieces; ++p) load_columns<E, V>(row, first + p * kSlab, width, lane, v[p]);
    }
    Y* dst = out + t * ld_y;
#pragma unroll
    for (int p = 0; p < kLookupPieces; ++p) {
        // (a row without an id is zero even where alpha is not finite)
        if (live) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) v[p][i] *= alpha;
        }
        store_columns<Y, V>(dst, first + p * kSlab, width, lane, v[p]);
    }
}

// ----------------------------------------------------------------------------- gradient

struct GradientArgs {
    int64_t count, rows, width, ld_y, ld_e, chunks;
    int chunk, slabs;
    const int* keys;       // sorted
    const unsigned* perm;  // token of every sorted place
    float* partial;        // [chunk][2][width]: a sum that came in open, a sum that goes out open
};

// dE[r, slab] = beta * dE[r, slab] + alpha * sum
template <typename E, int V>
__device__ __forceinline__ void finish_row(E* table, const GradientArgs& a, int64_t r, int64_t first, int lane, float alpha,
                                           float beta, const float* sum) {
    constexpr int kPer = Columns<V>::kPer;
    E* row = table + r * a.ld_e;
    float out[kPer];
    if (beta != 0.0f) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) out[i] = 0.0f;
        load_columns<E, V>(row, first, a.width, lane, out);
#pragma unroll
        for (int i = 0; i < kPer; ++i) out[i] = fmaf(alpha, sum[i], beta * out[i]);
    } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i) out[i] = alpha * sum[i];
    }
    store_columns<E, V>(row, first, a.width, lane, out);
}

// One warp per (chunk of sorted tokens, slab of columns).
template <typename Y, typename E, int V>
__global__ void __launch_bounds__(256)
    embedding_sum_kernel(GradientArgs a, const Y* __restrict__ dy, E* __restrict__ table, ScalarArg<float> alpha_arg,
                         ScalarArg<float> beta_arg) {
    constexpr int kPer = Columns<V>::kPer, kSlab = Columns<V>::kSlab, kDepth = 8;
    const int64_t warp = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    const float alpha = alpha_arg.get(), beta = beta_arg.get();
    if (warp >= a.chunks * a.slabs) return;
    const int64_t c = warp / a.slabs;
    const int64_t first = (warp - c * a.slabs) * kSlab;
    const int64_t k0 = c * a.chunk, k1 = min(k0 + a.chunk, a.count);
    float sum[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) sum[i] = 0.0f;
    int row = __ldg(a.keys + k0);
    bool open = k0 > 0 && __ldg(a.keys + k0 - 1) == row;  // the first sum began in an earlier chunk
    for (int64_t k = k0; k < k1; k += kDepth) {
        float v[kDepth][kPer];
        int key[kDepth];
#pragma unroll
        for (int j = 0; j < kDepth; ++j) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) v[j][i] = 0.0f;
            key[j] = k + j < k1 ? __ldg(a.keys + k + j) : (int)a.rows;
            if (key[j] < a.rows) load_columns<Y, V>(dy + (int64_t)__ldg(a.perm + k + j) * a.ld_y, first, a.width, lane, v[j]);
        }
#pragma unroll
        for (int j = 0; j < kDepth; ++j) {
            if (k + j < k1) {
                if (key[j] != row) {
                    if (open)
                        store_columns<float, V>(a.partial + (2 * c) * a.width, first, a.width, lane, sum);
                    else
                        finish_row<E, V>(table, a, row, first, lane, alpha, beta, sum);
                    open = false;
                    row = key[j];
#pragma unroll
                    for (int i = 0; i < kPer; ++i) sum[i] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < kPer; ++i) sum[i] += v[j][i];
            }
        }
    }
    if (row >= a.rows) return;
    const bool goes_on = k1 < a.count && __ldg(a.keys + k1) == row;
    if (open)
        store_columns<float, V>(a.partial + (2 * c) * a.width, first, a.width, lane, sum);
    else if (goes_on)
        store_columns<float, V>(a.partial + (2 * c + 1) * a.width, first, a.width, lane, sum);
    else
        finish_row<E, V>(table, a, row, first, lane, alpha, beta, sum);
}

// One warp per (chunk, slab): if a sum starts in this chunk and goes on, its partials are added in chunk order.
template <typename E, int V>
__global__ void __launch_bounds__(256)
    embedding_join_kernel(GradientArgs a, E* __restrict__ table, ScalarArg<float> alpha_arg, ScalarArg<float> beta_arg) {
    constexpr int kPer = Columns<V>::kPer, kSlab = Columns<V>::kSlab, kDepth = 8;
    const int64_t warp = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    const int64_t c = warp / a.slabs;
    if (c + 1 >= a.chunks) return;
    const int64_t first = (warp - c * a.slabs) * kSlab;
    const int64_t k0 = c * a.chunk, k1 = k0 + a.chunk;
    const int row = __ldg(a.keys + k1 - 1);
    if (row >= a.rows || __ldg(a.keys + k1) != row) return;          // nothing goes on
    if (k0 > 0 && __ldg(a.keys + k0 - 1) == row) return;              // it started earlier
    // its last chunk: the keys at the chunks' starts ascend, 32 of them are looked at in one step
    int64_t last = c + 1, beyond = a.chunks;
    while (beyond - last > 1) {
        const int64_t step = (beyond - last + 31) / 32, d = last + step * lane;
        const unsigned same = __ballot_sync(0xffffffffu, d < beyond && __ldg(a.keys + d * a.chunk) == row);
        last += step * (31 - __clz(same));
        beyond = min(last + step, beyond);
    }
    float sum[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) sum[i] = 0.0f;
    load_columns<float, V>(a.partial + (2 * c + 1) * a.width, first, a.width, lane, sum);
    for (int64_t d = c + 1; d <= last; d += kDepth) {
        float v[kDepth][kPer];
#pragma unroll
        for (int j = 0; j < kDepth; ++j) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) v[j][i] = 0.0f;
            if (d + j <= last) load_columns<float, V>(a.partial + (2 * (d + j)) * a.width, first, a.width, lane, v[j]);
        }
#pragma unroll
        for (int j = 0; j < kDepth; ++j)
#pragma unroll
            for (int i = 0; i < kPer; ++i) sum[i] += v[j][i];
    }
    finish_row<E, V>(table, a, row, first, lane, alpha_arg.get(), beta_arg.get(), sum);
}

// ----------------------------------------------------------------------------- sort, and the rows without a token

constexpr int kSortCluster = 8;
constexpr int kSortThreads = 1024;
constexpr int kSortRounds = 16;  // items per thread
constexpr int64_t kSortMost = (int64_t)kSortCluster * kSortThreads * kSortRounds;
constexpr int kMostDigits = 512;

struct SortArgs {
    int64_t count, rows;
    const void* ids;
    bool wide;
    int base;
    int* keys[2];       // ping-pong; the last pass writes the one `passes` says
    unsigned* perm[2];
    int passes, bits;   // digits of `bits` bits, at most 9
    int sorters;        // thread blocks that sort: the first cluster, or none
    // rows without a token
    void* table;
    int64_t ld, width;
    int64_t fill_rows;  // rows a block looks after at a time
};

// key = the row of the table, or `rows` for an id outside it (sorted behind every row and then left out).
__device__ __forceinline__ int key_of(const SortArgs& a, int64_t t) {
    const int64_t id = (a.wide ? __ldg(static_cast<const long long*>(a.ids) + t) : (int64_t)__ldg(static_cast<const int*>(a.ids) + t)) - a.base;
    return (int)(id >= 0 && id < a.rows ? id : a.rows);
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ unsigned load_remote(const unsigned* p, int rank) {
    const uint32_t addr = static_cast<uint32_t>(__cvta_generic_to_shared(p));
    uint32_t r;
    unsigned v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(r) : "memory");
    return v;
}

struct SortShared {
    unsigned short warp[32][kMostDigits];  // digit counts of every warp, then their exclusive sums over the warps
    unsigned total[kMostDigits];           // digit counts of the block, read by the whole cluster
    unsigned base[kMostDigits];            // first place of the block's items with a digit
    unsigned part[32];
};

// Items are owned in ascending order by (block, warp, round, lane), so that equal keys keep their order.
__device__ __forceinline__ void sort_block(const SortArgs& a, SortShared& s) {
    const int rank = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rounds = (int)((a.count + (int64_t)a.sorters * kSortThreads - 1) / ((int64_t)a.sorters * kSortThreads));
    const int64_t begin = ((int64_t)rank * 32 + warp) * rounds * 32 + lane;
    const int digits = 1 << a.bits;
    for (int pass = 0; pass < a.passes; ++pass) {
        const int shift = pass * a.bits, to = pass & 1;
        const int* in_keys = a.keys[to ^ 1];
        const unsigned* in_perm = a.perm[to ^ 1];
        for (int i = threadIdx.x; i < 32 * kMostDigits / 2; i += kSortThreads) reinterpret_cast<unsigned*>(s.warp)[i] = 0u;
        int key[kSortRounds];
        unsigned perm[kSortRounds];
        unsigned short rank_in_warp[kSortRounds];
#pragma unroll
        for (int r = 0; r < kSortRounds; ++r) {
            const int64_t t = begin + 32 * r;
            key[r] = 0, perm[r] = 0;
            if (r < rounds && t < a.count) {
                // (the previous pass's output was written by other blocks of the cluster: read past L1)
                key[r] = pass == 0 ? key_of(a, t) : __ldcg(in_keys + t);
                perm[r] = pass == 0 ? (unsigned)t : __ldcg(in_perm + t);
            }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kSortRounds; ++r) {
            if (r < rounds) {
                const bool live = begin + 32 * r < a.count;
                const unsigned d = live ? ((unsigned)key[r] >> shift) & (digits - 1) : 0xffffu;
                const unsigned peers = __match_any_sync(0xffffffffu, d);
                const unsigned before = live ? s.warp[warp][d] : 0;
                __syncwarp();
                if (live && lane == __ffs(peers) - 1) s.warp[warp][d] = (unsigned short)(before + __popc(peers));
                __syncwarp();
                rank_in_warp[r] = (unsigned short)(before + __popc(peers & ((1u << lane) - 1u)));
            }
        }
        __syncthreads();
        if ((int)threadIdx.x < digits) {  // counts of the warps -> exclusive sums over the warps
            unsigned sum = 0;
            for (int w = 0; w < 32; ++w) {
                const unsigned c = s.warp[w][threadIdx.x];
                s.warp[w][threadIdx.x] = (unsigned short)sum;
                sum += c;
            }
            s.total[threadIdx.x] = sum;
        }
        cluster_sync();
        // places: all smaller digits of the cluster, then the same digit in the blocks before this one
        unsigned all = 0, before = 0;
        if ((int)threadIdx.x < digits) {
            for (int r = 0; r < a.sorters; ++r) {
                const unsigned c = load_remote(&s.total[threadIdx.x], r);
                all += c;
                if (r < rank) before += c;
            }
        }
        unsigned inc = all;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const unsigned o = __shfl_up_sync(0xffffffffu, inc, d);
            if (lane >= d) inc += o;
        }
        if (lane == 31) s.part[warp] = inc;
        __syncthreads();
        unsigned ahead = 0;
        for (int w = 0; w < warp && w < kMostDigits / 32; ++w) ahead += s.part[w];
        if ((int)threadIdx.x < digits) s.base[threadIdx.x] = ahead + inc - all + before;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kSortRounds; ++r) {
            if (r < rounds && begin + 32 * r < a.count) {
                const unsigned d = ((unsigned)key[r] >> shift) & (digits - 1);
                const unsigned at = s.base[d] + s.warp[warp][d] + rank_in_warp[r];
                a.keys[to][at] = key[r];
                a.perm[to][at] = perm[r];
            }
        }
        cluster_sync();  // the pass is in memory, and nobody reads this block's counts any more
    }
}

constexpr int kMostFillRows = 65536;

// The rows [row0, row1) that no id names become beta times what they are (beta = 0: zero). One warp per row.
template <typename E, int V>
__device__ __forceinline__ void fill_block(const SortArgs& a, float beta, unsigned* bits, int64_t row0, int64_t row1) {
    for (int i = threadIdx.x; i < (row1 - row0 + 31) / 32; i += kSortThreads) bits[i] = 0u;
    __syncthreads();
    for (int64_t t = threadIdx.x; t < a.count; t += 4 * kSortThreads) {
        int key[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) key[x] = t + x * kSortThreads < a.count ? key_of(a, t + x * kSortThreads) : -1;
#pragma unroll
        for (int x = 0; x < 4; ++x)
            if (key[x] >= row0 && key[x] < row1) atomicOr(&bits[(key[x] - row0) >> 5], 1u << ((key[x] - row0) & 31));
    }
    __syncthreads();
    const int lane = threadIdx.x & 31;
    for (int64_t r = row0 + (threadIdx.x >> 5); r < row1; r += kSortThreads / 32) {
        if (bits[(r - row0) >> 5] >> ((r - row0) & 31) & 1) continue;
        E* row = static_cast<E*>(a.table) + r * a.ld;
        for (int64_t c = 0; c < a.width; c += Columns<V>::kSlab) {
            float v[Columns<V>::kPer] = {};
            if (beta != 0.0f) {
                load_columns<E, V>(row, c, a.width, lane, v);
#pragma unroll
                for (int i = 0; i < Columns<V>::kPer; ++i) v[i] *= beta;
            }
            store_columns<E, V>(row, c, a.width, lane, v);
        }
    }
    __syncthreads();
}

template <typename E, int V>
__global__ void __launch_bounds__(kSortThreads) embedding_sort_kernel(const SortArgs a, ScalarArg<float> beta_arg) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    if ((int)blockIdx.x < a.sorters) {
        sort_block(a, *reinterpret_cast<SortShared*>(smem_raw));
        return;
    }
    const float beta = beta_arg.get();
    if (beta == 1.0f) return;
    for (int64_t row0 = (blockIdx.x - a.sorters) * a.fill_rows; row0 < a.rows; row0 += (gridDim.x - a.sorters) * a.fill_rows)
        fill_block<E, V>(a, beta, reinterpret_cast<unsigned*>(smem_raw), row0, min(row0 + a.fill_rows, a.rows));
}

template <typename T, int V>
bool wide_rows(const void* p, int64_t ld, int64_t width) {
    return (reinterpret_cast<uintptr_t>(p) & (sizeof(T) * V >= 16 ? 15 : sizeof(T) * V - 1)) == 0 && ld % V == 0 &&
           width % V == 0;
}

// Warps of a launch as a grid of 8-warp blocks; 0 when the grid would be too large.
unsigned warp_blocks(int64_t warps) {
    const int64_t b = (warps + 7) / 8;
    return b > 0x7fffffffLL ? 0u : (unsigned)b;
}

template <typename E, typename Y, typename I, int V>
cudaError_t launch_lookup(cudaStream_t s, const EmbeddingArgs& a, const I* ids) {
    const int64_t span = Columns<V>::kSlab * kLookupPieces;
    const int64_t pieces = (a.width + span - 1) / span;
    const unsigned blocks = warp_blocks(a.count * pieces);
    if (blocks == 0) return cudaErrorInvalidValue;
    embedding_lookup_kernel<E, Y, I, V><<<blocks, 256, 0, s>>>(a.count, a.rows, a.width, ids, a.base, static_cast<const E*>(a.table),
                                                               a.ld_table, static_cast<Y*>(a.tokens), a.ld_tokens, a.alpha, pieces);
    return cudaGetLastError();
}

template <typename E, typename Y>
cudaError_t lookup_typed(cudaStream_t s, const EmbeddingArgs& a) {
    // 16 bytes of the wider of the two types' rows per thread
    constexpr int V = sizeof(E) == 4 && sizeof(Y) == 4 ? 4 : 8;
    const bool wide = wide_rows<E, V>(a.table, a.ld_table, a.width) && wide_rows<Y, V>(a.tokens, a.ld_tokens, a.width);
    if (a.wide_ids) {
        const int64_t* ids = static_cast<const int64_t*>(a.ids);
        return wide ? launch_lookup<E, Y, int64_t, V>(s, a, ids) : launch_lookup<E, Y, int64_t, 1>(s, a, ids);
    }
    const int32_t* ids = static_cast<const int32_t*>(a.ids);
    return wide ? launch_lookup<E, Y, int32_t, V>(s, a, ids) : launch_lookup<E, Y, int32_t, 1>(s, a, ids);
}

size_t align256(size_t v) { return (v + 255) & ~size_t(255); }

// Tokens per chunk: long enough that few sums cross chunks, short enough that the chunks fill the GPU
// (148 SMs x 32 warps) when there are few tokens.
int gradient_chunk(int64_t count, int64_t width) {
    const int64_t slabs = (width + 127) / 128;
    const int64_t want = count * slabs / (148 * 32);
    int chunk = 8;
    while (chunk < 64 && chunk < want) chunk *= 2;
    return chunk;
}

struct GradientLayout {
    bool one_cluster;
    TransposePlan sort;  // more tokens than one cluster sorts
    int chunk;
    int64_t chunks;
    size_t off_raw, off_keys[2], off_perm[2], off_partial, bytes;
};

GradientLayout gradient_layout(int64_t count, int64_t rows, int64_t width) {
    GradientLayout l = {};
    l.one_cluster = count <= kSortMost;
    l.chunk = gradient_chunk(count, width);
    l.chunks = (count + l.chunk - 1) / l.chunk;
    size_t off = 0;
    if (l.one_cluster) {
        for (size_t* p : {&l.off_keys[0], &l.off_keys[1], &l.off_perm[0], &l.off_perm[1]}) {
            *p = off;
            off += align256(size_t(count) * 4);
        }
    } else {
        l.sort = transpose_plan(rows, rows + 1, count, 0);
        for (int i = 0; i < 2; ++i) l.off_keys[i] = l.sort.off_keys[i], l.off_perm[i] = l.sort.off_perm[i];
        off = l.sort.bytes;
        l.off_raw = off;
        off += align256(size_t(count) * 4);
    }
    l.off_partial = off;
    off += align256(size_t(l.chunks) * 2 * size_t(width) * 4);
    l.bytes = off + 256;
    return l;
}

__global__ void __launch_bounds__(256) embedding_keys_kernel(const SortArgs a, int* __restrict__ keys) {
    const int64_t t = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
    if (t < a.count) keys[t] = key_of(a, t);
}

template <typename Y, typename E, int V>
cudaError_t launch_gradient(cudaStream_t s, const EmbeddingArgs& a, char* b) {
    const GradientLayout l = gradient_layout(a.count, a.rows, a.width);
    // ---- sort; rows without a token (none change when beta is 1, which the host may not know)
    SortArgs so = {};
    so.count = a.count, so.rows = a.rows, so.ids = a.ids, so.wide = a.wide_ids, so.base = a.base;
    so.table = a.table, so.ld = a.ld_table, so.width = a.width;
    for (int i = 0; i < 2; ++i)
        so.keys[i] = reinterpret_cast<int*>(b + l.off_keys[i]), so.perm[i] = reinterpret_cast<unsigned*>(b + l.off_perm[i]);
    int need = 1;  // bits of a key, `rows` included
    while (need < 31 && (int64_t(1) << need) <= a.rows) ++need;
    so.passes = (need + 8) / 9;
    so.bits = (need + so.passes - 1) / so.passes;
    const bool fill = a.beta.dev != nullptr || a.beta.host != 1.0f;
    // (few tokens: one block sorts them in two rounds, with a cluster of one)
    const int cluster = l.one_cluster && a.count > 2 * kSortThreads ? kSortCluster : 1;
    so.sorters = l.one_cluster && a.count > 0 ? cluster : 0;
    int last = (so.passes - 1) & 1;
    if (!l.one_cluster) {
        int* raw = reinterpret_cast<int*>(b + l.off_raw);
        embedding_keys_kernel<<<(unsigned)((a.count + 255) / 256), 256, 0, s>>>(so, raw);
        const cudaError_t e = sort_keys(s, a.rows, a.count, raw, l.sort, b);
        if (e != cudaSuccess) return e;
        last = l.sort.final_slot();
    }
    // one block per SM beside the sorting cluster; ranges of rows small enough for their marks to fit in shared memory
    int64_t fillers = fill ? (a.sm_count / cluster) * cluster - (cluster > 1 ? cluster : 0) : 0;
    if (fill) {
        so.fill_rows = (a.rows + fillers - 1) / fillers;
        if (so.fill_rows > kMostFillRows) so.fill_rows = kMostFillRows;
        so.fill_rows = (so.fill_rows + 31) / 32 * 32;
        const int64_t ranges = (a.rows + so.fill_rows - 1) / so.fill_rows;
        if (ranges < fillers) fillers = (ranges + cluster - 1) / cluster * cluster;
    }
    if (so.sorters + fillers > 0) {
        constexpr size_t kShared = sizeof(SortShared) > kMostFillRows / 8 ? sizeof(SortShared) : kMostFillRows / 8;
        static_assert(kShared <= 48 * 1024, "fits without opting in to more");
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(so.sorters + fillers));
        cfg.blockDim = dim3(kSortThreads);
        cfg.dynamicSmemBytes = kShared;
        cfg.stream = s;
        cudaLaunchAttribute attr = {};
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = (unsigned)cluster, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = cluster > 1 ? 1 : 0;
        const cudaError_t e = cudaLaunchKernelEx(&cfg, embedding_sort_kernel<E, V>, static_cast<const SortArgs>(so), a.beta);
        if (e != cudaSuccess) return e;
    }
    if (a.count == 0) return cudaSuccess;
    // ---- sums
    GradientArgs g = {};
    g.count = a.count, g.rows = a.rows, g.width = a.width, g.ld_y = a.ld_tokens, g.ld_e = a.ld_table;
    g.chunk = l.chunk, g.chunks = l.chunks;
    g.keys = so.keys[last], g.perm = so.perm[last];
    g.partial = reinterpret_cast<float*>(b + l.off_partial);
    g.slabs = (int)((a.width + Columns<V>::kSlab - 1) / Columns<V>::kSlab);
    const unsigned blocks = warp_blocks(g.chunks * g.slabs);
    if (blocks == 0) return cudaErrorInvalidValue;
    embedding_sum_kernel<Y, E, V><<<blocks, 256, 0, s>>>(g, static_cast<const Y*>(a.tokens), static_cast<E*>(a.table), a.alpha, a.beta);
    if (g.chunks > 1) embedding_join_kernel<E, V><<<blocks, 256, 0, s>>>(g, static_cast<E*>(a.table), a.alpha, a.beta);
    return cudaGetLastError();
}

template <typename E, typename Y>
cudaError_t gradient_typed(cudaStream_t s, const EmbeddingArgs& a, char* b) {
    constexpr int V = sizeof(E) == 4 && sizeof(Y) == 4 ? 4 : 8;
    const bool wide = wide_rows<E, V>(a.table, a.ld_table, a.width) && wide_rows<Y, V>(a.tokens, a.ld_tokens, a.width);
    return wide ? launch_gradient<Y, E, V>(s, a, b) : launch_gradient<Y, E, 1>(s, a, b);
}

// Calls f<E, Y> for the two value types (they share a type, or one of them is fp32).
#define MCSP_EMBEDDING_TYPES(f, ...)                                                              \
    do {                                                                                          \
        const macaDataType te = a.table_type, ty = a.token_type;                                  \
        if (te == MACA_R_32F && ty == MACA_R_32F) return f<float, float>(__VA_ARGS__);            \
        if (te == MACA_R_16F && ty == MACA_R_16F) return f<__half, __half>(__VA_ARGS__);          \
        if (te == MACA_R_16BF && ty == MACA_R_16BF) return f<__nv_bfloat16, __nv_bfloat16>(__VA_ARGS__); \
        if (te == MACA_R_32F && ty == MACA_R_16F) return f<float, __half>(__VA_ARGS__);           \
        if (te == MACA_R_32F && ty == MACA_R_16BF) return f<float, __nv_bfloat16>(__VA_ARGS__);   \
        if (te == MACA_R_16F && ty == MACA_R_32F) return f<__half, float>(__VA_ARGS__);           \
        if (te == MACA_R_16BF && ty == MACA_R_32F) return f<__nv_bfloat16, float>(__VA_ARGS__);   \
        return cudaErrorInvalidValue;                                                             \
    } while (0)

}  // namespace

cudaError_t embedding_lookup(cudaStream_t s, const EmbeddingArgs& a) {
    if (a.count == 0 || a.width == 0) return cudaSuccess;
    MCSP_EMBEDDING_TYPES(lookup_typed, s, a);
}

size_t embedding_gradient_bytes(int64_t count, int64_t rows, int64_t width) { return gradient_layout(count, rows, width).bytes; }

cudaError_t embedding_gradient(cudaStream_t s, const EmbeddingArgs& a, void* buffer) {
    if (a.rows == 0 || a.width == 0) return cudaSuccess;
    MCSP_EMBEDDING_TYPES(gradient_typed, s, a, static_cast<char*>(align_up_256(buffer)));
}

}  // namespace mcsp_b200
