// Rows of a table by token ids, Y = alpha * S * E, and the table's gradient, dE = alpha * S^T * dY + beta * dE, for the
// count x rows matrix S with one 1 per row (its column: the token's id). S is never stored.
//
// Lookup: one pass; a warp moves a piece of one row with 16-byte loads and stores. Bound by memory (count * width read,
// unless rows repeat, and written).
//
// Gradient, two or three launches, each prepared while the one before it runs (programmatic dependent launch):
//   1. S^T in CSR form is the tokens sorted by id: a stable radix sort of (id, position) pairs. Up to 131072 tokens one cluster
//      of 16 thread blocks sorts them in two passes or three (ids below 2^18: two 9-bit digits), its digit counts exchanged over
//      distributed shared memory, its barriers the cluster's; up to 2048 one block does, as one more block of the next launch. More
//      tokens, or a device that holds no such cluster, take the multi-launch sort of transpose.cu.
//   2. Beside the sort, the rows no token names are written (beta = 0: zeros, most of the traffic of a large table). A block
//      finds those of its rows by marking the ids that are its own in shared memory, so it need not wait for the sort. (As
//      further blocks of the sort's own launch they came up in clusters, few of which the GPU holds at a time: 116 us against 65.)
//   3. The sorted tokens are cut into chunks of equal size whatever the ids are, so a token that fills half the batch, or all
//      of it, costs no more than any other (4194304 rows of 512 bf16 values: 1.31 ms spread, 1.25 with half of them on one row,
//      1.27 with all); a warp owns one chunk and a slab of columns, adds in fp32 and writes every sum that lies inside
//      its chunk. A sum that crosses chunks is left as one partial per chunk; the warp that finds all of a sum's partials there
//      (a counter per sum) adds them, in chunk order, and in groups where there are many.
// The order of every addition follows from ids and sizes alone. Bound by memory: count * width read, rows * width written.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "internal.h"
#include "launch.h"

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

// V consecutive values of one thread, moved in one access of up to 32 bytes.
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
    T v[V];
};
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
    Pack<T, V> r;
    if constexpr (sizeof(r) == 32) {
        float* f = reinterpret_cast<float*>(&r);
        asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3]), "=f"(f[4]), "=f"(f[5]), "=f"(f[6]), "=f"(f[7])
                     : "l"(p));
    } else {
        r = *reinterpret_cast<const Pack<T, V>*>(p);
    }
    return r;
}
// STREAM: written once and not looked at before it has left L2 anyway.
template <typename T, int V, bool STREAM = false>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& r) {
    const float* f = reinterpret_cast<const float*>(&r);
    if constexpr (sizeof(r) == 32 && STREAM) {
        asm volatile("st.global.cs.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]),
                     "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7])
                     : "memory");
    } else if constexpr (sizeof(r) == 16 && STREAM) {
        __stcs(reinterpret_cast<float4*>(p), *reinterpret_cast<const float4*>(f));
    } else if constexpr (sizeof(r) == 32) {
        asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]),
                     "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7])
                     : "memory");
    } else {
        *reinterpret_cast<Pack<T, V>*>(p) = r;
    }
}

// How a thread holds its columns: V consecutive ones when every row starts on a boundary of V values and the width is a
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
            const Pack<T, V> p = load_pack<T, V>(row + c);
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

template <typename T, int V, bool STREAM = false>
__device__ __forceinline__ void store_columns(T* row, int64_t first, int64_t width, int lane, const float* in) {
    if (V > 1) {
        const int64_t c = first + lane * V;
        if (c < width) {
            Pack<T, V> p;
#pragma unroll
            for (int i = 0; i < V; ++i) p.v[i] = from_float<T>(in[i]);
            store_pack<T, V, STREAM>(row + c, p);
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

template <typename E, typename Y, typename I, int V, bool STREAM>
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
        store_columns<Y, V, STREAM>(dst, first + p * kSlab, width, lane, v[p]);
    }
}

// ----------------------------------------------------------------------------- gradient

// The rows of a warp's chunk on their way. Vectors: a ring of asynchronous copies in shared memory, a thread reads back what it
// copied itself; the copies of 8 rows are in flight whatever the warp is doing. (Loads into registers, as many ahead,
// waited for the newest of them at every row: 52 us against 25 for 16384 rows of 2048 bf16 values.)
template <typename T, int V>
struct Rows {
    static constexpr int kBytes = sizeof(Pack<T, V>);      // 16 or 32, per thread and row
    static constexpr int kAhead = 8, kGroup = 4;
    static constexpr int kShared = kAhead * kBytes * 256;  // of a block
    uint32_t ring;
    const T* from;
    int64_t ld;
    bool inside;
    __device__ __forceinline__ Rows(uint8_t* smem, const T* dy, int64_t ld_y, int64_t first, int64_t width, int lane)
        : ring(static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + threadIdx.x * 16), from(dy + first + lane * V), ld(ld_y),
          inside(first + lane * V < width) {}
    // slot of row j: 16-byte pieces of all threads side by side
    __device__ __forceinline__ uint32_t slot(int j) const { return ring + (j % kAhead) * (kBytes * 256); }
    __device__ __forceinline__ void fetch(int j, int, unsigned token) const {
        if (!inside) return;
        const char* src = reinterpret_cast<const char*>(from + (int64_t)token * ld);
#pragma unroll
        for (int b = 0; b < kBytes; b += 16)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(slot(j) + b * 256), "l"(src + b) : "memory");
    }
    __device__ __forceinline__ void commit() const { asm volatile("cp.async.commit_group;" ::: "memory"); }
    __device__ __forceinline__ void wait() const { asm volatile("cp.async.wait_group %0;" ::"n"(kAhead / kGroup - 1) : "memory"); }
    __device__ __forceinline__ void drain() const { asm volatile("cp.async.wait_group 0;" ::: "memory"); }
    __device__ __forceinline__ void add(int j, int, float* sum) const {  // (columns behind the width hold anything and are not stored)
        Pack<T, V> p;
        uint32_t* w = reinterpret_cast<uint32_t*>(&p);
#pragma unroll
        for (int b = 0; b < kBytes; b += 16)
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(w[b / 4]), "=r"(w[b / 4 + 1]), "=r"(w[b / 4 + 2]), "=r"(w[b / 4 + 3])
                         : "r"(slot(j) + b * 256));
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] += to_float(p.v[i]);
    }
};
// Single columns: eight rows at a time in registers.
template <typename T>
struct Rows<T, 1> {
    static constexpr int kAhead = 8, kGroup = 8, kShared = 0;
    T v[kGroup][kLoose];
    const T* from;
    int64_t ld, left;  // columns from the thread's first one on
    __device__ __forceinline__ Rows(uint8_t*, const T* dy, int64_t ld_y, int64_t first, int64_t width, int lane)
        : from(dy + first + lane), ld(ld_y), left(width - first - lane) {}
    __device__ __forceinline__ void fetch(int, int x, unsigned token) {
#pragma unroll
        for (int i = 0; i < kLoose; ++i)
            if (32 * i < left) v[x][i] = from[(int64_t)token * ld + 32 * i];
    }
    __device__ __forceinline__ void commit() const {}
    __device__ __forceinline__ void wait() const {}
    __device__ __forceinline__ void drain() const {}
    __device__ __forceinline__ void add(int, int x, float* sum) const {
#pragma unroll
        for (int i = 0; i < kLoose; ++i) sum[i] += to_float(v[x][i]);
    }
};

struct GradientArgs {
    int64_t count, rows, width, ld_y, ld_e, chunks;
    int chunk, slabs;
    const uint2* sorted;  // (row, token) by row, then token; row = rows: none
    float* partial;       // [chunk][2][width]: a sum that came in open, a sum that goes out open
    unsigned* arrived;    // [chunk][slab]: partials that are there of the sum that goes out of a chunk; zero before the launch
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

// Called by the warp that has written chunk c's partial of a sum over several chunks. The one that comes last of them puts the
// partials together, in chunk order whoever it is. More than 64 of them are put together in groups of about the square root of
// their number, each by its own last warp, and the groups' sums by the last warp of those. (One warp for all the partials of a
// sum: 14.4 ms against 1.27 for 4194304 tokens of one id, width 512.)
template <typename E, int V>
__device__ __forceinline__ void join_partials(E* table, const GradientArgs& a, int c, bool came_in, int slab, int row, int64_t first, int lane,
                                              float alpha, float beta) {
    constexpr int kPer = Columns<V>::kPer, kDepth = 3;  // (4 at a time went past 64 registers: 396 us against 390, two passes of 65536 tokens)
    // (there are fewer than 2^28 chunks, so that `extent` below steps at most 2^25 of them: its places are int32)
    const auto starts_with = [&](int d) { return d >= 0 && d < a.chunks && (int)__ldcg(&a.sorted[(int64_t)d * a.chunk].x) == row; };
    // The run of chunks around c that start with the row: its last one in a direction. Rows ascend, so a step looks at 32 chunks,
    // the next ones first, then 32 times as far apart as long as all 32 belong to it, and back to single chunks: two steps for
    // each factor of 32. (One chunk after the other, 32 in a step, the warps of a run of n chunks took n * n / 32 looks: 48 ms
    // against 14 for 4194304 tokens of one id, width 512.)
    const auto extent = [&](int at, int way) {
        int step = 1;
        for (bool wider = true;;) {
            const int n = __popc(__ballot_sync(0xffffffffu, starts_with(at + way * step * (lane + 1))));
            at += way * step * n;
            wider = wider && n == 32;
            if (!wider && step == 1) return at;
            step = wider ? step * 32 : step / 32;
        }
    };
    int begin = came_in ? extent(c, -1) : c;
    const int last = extent(c, 1);
    // the sum began in the chunk before the first of them, unless it began right with it
    if (came_in && begin > 0 && (int)__ldcg(&a.sorted[(int64_t)begin * a.chunk - 1].x) == row) --begin;
    const int parts = last - begin + 1;
    int shift = 6;  // groups of 2^shift chunks
    if (parts > 64)
        for (shift = 4; (int64_t(1) << (2 * shift)) < parts; ++shift) {}
    // Whether this warp is the last of n that arrive at a chunk's counter.
    const auto last_of = [&](int d, int n) {
        __threadfence();
        __syncwarp();
        unsigned before = 0;
        if (lane == 0) before = atomicAdd(a.arrived + (int64_t)d * a.slabs + slab, 1u);
        before = __shfl_sync(0xffffffffu, before, 0);
        __threadfence();
        return before == (unsigned)(n - 1);
    };
    const int groups = ((parts - 1) >> shift) + 1, head = begin + ((c - begin) >> shift << shift);
    int d0 = head, d1 = min(head + (1 << shift) - 1, last), step = 1;
    // Counters: a group's is that of the chunk before it, the first group's that of its first chunk. No other sum goes out of these
    // chunks: the row fills every chunk between the first and the last. The second chunk's counts the groups (of 16 chunks or more).
    if (!last_of(head == begin ? begin : head - 1, d1 - d0 + 1)) return;
    const auto place = [&](int d) { return a.partial + (2 * (int64_t)d + (d == begin)) * a.width; };
    const auto load = [&](int d, float* v) {
        const float* from = place(d) + first;
#pragma unroll
        for (int i = 0; i < kPer; i += V > 1 ? 4 : 1) {
            const int64_t x = Columns<V>::at(lane, i);
            if (V > 1) {
                const float4 f = first + x < a.width ? __ldcg(reinterpret_cast<const float4*>(from + x)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                v[i] = f.x, v[(i + 1) % kPer] = f.y, v[(i + 2) % kPer] = f.z, v[(i + 3) % kPer] = f.w;
            } else {
                v[i] = first + x < a.width ? __ldcg(from + x) : 0.0f;
            }
        }
    };
    float sum[kPer];
    while (true) {
        load(d0, sum);
        for (int d = d0 + step; d <= d1; d += kDepth * step) {
            float v[kDepth][kPer];
#pragma unroll
            for (int j = 0; j < kDepth; ++j) {
#pragma unroll
                for (int i = 0; i < kPer; ++i) v[j][i] = 0.0f;
                if (d + j * step <= d1) load(d + j * step, v[j]);
            }
#pragma unroll
            for (int j = 0; j < kDepth; ++j)
#pragma unroll
                for (int i = 0; i < kPer; ++i) sum[i] += v[j][i];
        }
        if (step > 1 || groups == 1) break;
        store_columns<float, V>(place(head), first, a.width, lane, sum);  // (nobody else reads this partial any more)
        if (!last_of(begin + 1, groups)) return;
        d0 = begin, d1 = last, step = 1 << shift;
    }
    finish_row<E, V>(table, a, row, first, lane, alpha, beta, sum);
}

// One warp per (chunk of sorted tokens, slab of columns).
template <typename Y, typename E, int V>
__global__ void __launch_bounds__(256, 4)  // (64 registers: 389 us against 401 with 76, two passes of 65536 tokens)
    embedding_sum_kernel(GradientArgs a, const Y* __restrict__ dy, E* __restrict__ table, ScalarArg<float> alpha_arg,
                         ScalarArg<float> beta_arg) {
    constexpr int kPer = Columns<V>::kPer, kSlab = Columns<V>::kSlab;
    const int64_t warp = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    const float alpha = alpha_arg.get(), beta = beta_arg.get();
    if (warp >= a.chunks * a.slabs) {
        grid_wait();
        return;
    }
    const int64_t c = warp / a.slabs;
    const int slab = (int)(warp - c * a.slabs);
    const int64_t first = (int64_t)slab * kSlab;
    const int64_t k0 = c * a.chunk, k1 = min(k0 + a.chunk, a.count);
    grid_wait();  // the sort
    float sum[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) sum[i] = 0.0f;
    int row = (int)__ldcg(&a.sorted[k0].x);
    bool open = k0 > 0 && (int)__ldcg(&a.sorted[k0 - 1].x) == row;  // the first sum began in an earlier chunk
    int came_in = -1;                                               // its row, once its partial is written
    extern __shared__ __align__(16) uint8_t smem_raw[];
    Rows<Y, V> rows(smem_raw, dy, a.ld_y, first, a.width, lane);
    for (int64_t k = k0; k < k1; k += 32) {
        // lane l holds token k + l
        const uint2 token = k + lane < k1 ? __ldcg(a.sorted + k + lane) : make_uint2((unsigned)a.rows, 0u);
        const int n = (int)min(k1 - k, (int64_t)32);
        const auto fetch = [&](int j) {  // the next kGroup tokens
#pragma unroll
            for (int x = 0; x < Rows<Y, V>::kGroup; ++x) {
                const unsigned key = __shfl_sync(0xffffffffu, token.x, (j + x) & 31), t = __shfl_sync(0xffffffffu, token.y, (j + x) & 31);
                const unsigned last = __shfl_sync(0xffffffffu, token.x, (j + x - 1) & 31);
                if (j + x < n && key < (unsigned)a.rows) {
                    rows.fetch(j + x, x, t);
                    // (a row of the table that will be read when its sum is done)
                    if (V > 1 && beta != 0.0f && (j + x == 0 || key != last) && first + lane * V < a.width)
                        asm volatile("prefetch.global.L2 [%0];" ::"l"(table + (int64_t)key * a.ld_e + first + lane * V));
                }
            }
            rows.commit();
        };
#pragma unroll
        for (int j = 0; j < Rows<Y, V>::kAhead; j += Rows<Y, V>::kGroup) fetch(j);
        for (int j0 = 0; j0 < n; j0 += Rows<Y, V>::kGroup) {
            rows.wait();
#pragma unroll
            for (int x = 0; x < Rows<Y, V>::kGroup; ++x) {
                const int key = (int)__shfl_sync(0xffffffffu, token.x, (j0 + x) & 31);
                if (j0 + x < n) {
                    if (key != row) {
                        if (open) {
                            store_columns<float, V>(a.partial + (2 * c) * a.width, first, a.width, lane, sum);
                            came_in = row;
                        } else {
                            finish_row<E, V>(table, a, row, first, lane, alpha, beta, sum);
                        }
                        open = false;
                        row = key;
#pragma unroll
                        for (int i = 0; i < kPer; ++i) sum[i] = 0.0f;
                    }
                    if (key < a.rows) rows.add(j0 + x, x, sum);
                }
            }
            fetch(j0 + Rows<Y, V>::kAhead);
        }
        rows.drain();
    }
    bool goes_on = false;
    if (row < a.rows) {
        goes_on = k1 < a.count && (int)__ldcg(&a.sorted[k1].x) == row;
        if (open) {
            store_columns<float, V>(a.partial + (2 * c) * a.width, first, a.width, lane, sum);
            came_in = row;
            goes_on = false;  // (the same sum)
        } else if (goes_on) {
            store_columns<float, V>(a.partial + (2 * c + 1) * a.width, first, a.width, lane, sum);
        } else {
            finish_row<E, V>(table, a, row, first, lane, alpha, beta, sum);
        }
    }
    for (int part = 0; part < 2; ++part) {
        if (part == 0 ? came_in < 0 : !goes_on) continue;
        join_partials<E, V>(table, a, (int)c, part == 0, slab, part == 0 ? came_in : row, first, lane, alpha, beta);
    }
}

// ----------------------------------------------------------------------------- sort, and the rows without a token

constexpr int kSortCluster = 16;  // (8, the most that every device must hold, took 36 us against 24 for 65536 tokens)
constexpr int kSortThreads = 1024;
constexpr int kSortRounds = 8;  // items per thread, at most
constexpr int kFewRounds = 2;   // the same, of the kernel for few tokens (room for more costs it registers and time)
constexpr int64_t kSortAlone = kSortThreads * kFewRounds;  // tokens that one block sorts
constexpr int64_t kSortMost = (int64_t)kSortCluster * kSortThreads * kSortRounds;
constexpr int kMostDigits = 512;

struct SortArgs {
    int64_t count, rows;
    const void* ids;
    bool wide;
    int base;
    uint2* sorted[2];   // (key, token); the passes write them in turn
    int passes, bits;   // digits of `bits` bits, at most 9
    int sorters;        // thread blocks that sort (one cluster)
    unsigned* arrived;  // set to zero on the way, `counters` of them
    int64_t counters;
    // rows without a token
    void* table;
    int64_t ld, width;
    int fill_shift;     // 2^fill_shift thread blocks look after them: row r belongs to block r % 2^fill_shift
    int fill_rows;      // rows of a block that are marked at a time
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
    unsigned quarter[4][kMostDigits / 2];  // sums over 8 warps each, two digits to a word
    unsigned total[kMostDigits];           // digit counts of the block, read by the whole cluster
    unsigned base[kMostDigits];            // first place of the block's items with a digit
    unsigned part[32];
};

// Lanes with the same digit as the calling one (a lane that is not live: nobody's). One vote per bit:
// __match_any_sync took four times as long on ids as text has them.
__device__ __forceinline__ unsigned same_digit(unsigned d, bool live, int bits) {
    unsigned peers = __ballot_sync(0xffffffffu, live);
#pragma unroll
    for (int b = 0; b < 9; ++b) {
        if (b < bits) {
            const unsigned votes = __ballot_sync(0xffffffffu, d >> b & 1);
            peers &= d >> b & 1 ? votes : ~votes;
        }
    }
    return peers;
}

// Items are owned in ascending order by (block, warp, round, lane), so that equal keys keep their order. At most R rounds.
template <int R>
__device__ __forceinline__ void sort_block(const SortArgs& a, SortShared& s, int rank) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rounds = (int)((a.count + (int64_t)a.sorters * kSortThreads - 1) / ((int64_t)a.sorters * kSortThreads));
    const int64_t begin = ((int64_t)rank * 32 + warp) * rounds * 32 + lane;
    const int digits = 1 << a.bits;
    for (int64_t i = rank * kSortThreads + (int)threadIdx.x; i < a.counters; i += (int64_t)a.sorters * kSortThreads) a.arrived[i] = 0u;
    for (int pass = 0; pass < a.passes; ++pass) {
        const int shift = pass * a.bits, to = pass & 1;
        const uint2* in = to ? a.sorted[0] : a.sorted[1];
        uint2* const out = to ? a.sorted[1] : a.sorted[0];
        for (int i = threadIdx.x; i < 32 * kMostDigits / 2; i += kSortThreads) reinterpret_cast<unsigned*>(s.warp)[i] = 0u;
        uint2 pair[R];
        unsigned ranks[(R + 1) / 2];  // place of an item among its warp's items with the same digit, two to a word
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t t = begin + 32 * r;
            pair[r] = make_uint2(0u, 0u);
            // (the previous pass's output was written by other blocks of the cluster: read past L1)
            if (r < rounds && t < a.count) pair[r] = pass == 0 ? make_uint2((unsigned)key_of(a, t), (unsigned)t) : __ldcg(in + t);
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (r < rounds) {
                const bool live = begin + 32 * r < a.count;
                const unsigned d = (pair[r].x >> shift) & (digits - 1);
                const unsigned peers = same_digit(d, live, a.bits);
                const unsigned before = live ? s.warp[warp][d] : 0;
                __syncwarp();
                if (live && lane == __ffs(peers) - 1) s.warp[warp][d] = (unsigned short)(before + __popc(peers));
                __syncwarp();
                const unsigned rank_here = before + __popc(peers & ((1u << lane) - 1u));
                ranks[r / 2] = r & 1 ? ranks[r / 2] | rank_here << 16 : rank_here;
            }
        }
        __syncthreads();
        {  // counts of the warps -> exclusive sums over the warps: a thread takes two digits (one word) of 8 warps
            const int word = threadIdx.x & (kMostDigits / 2 - 1), q = threadIdx.x / (kMostDigits / 2);
            unsigned* const col = reinterpret_cast<unsigned*>(s.warp[8 * q]) + word;
            unsigned c[8], sum = 0;
#pragma unroll
            for (int w = 0; w < 8; ++w) c[w] = col[w * (kMostDigits / 2)];
#pragma unroll
            for (int w = 0; w < 8; ++w) {  // (a block has at most 2^14 items: the halves of a word do not meet)
                const unsigned x = c[w];
                c[w] = sum;
                sum += x;
            }
            s.quarter[q][word] = sum;
            __syncthreads();
            unsigned ahead = 0;
            for (int x = 0; x < q; ++x) ahead += s.quarter[x][word];
#pragma unroll
            for (int w = 0; w < 8; ++w) col[w * (kMostDigits / 2)] = ahead + c[w];
            if (q == 3) {
                const unsigned all = ahead + sum;
                s.total[2 * word] = all & 0xffffu, s.total[2 * word + 1] = all >> 16;
            }
        }
        cluster_sync();
        // places: all smaller digits of the cluster, then the same digit in the blocks before this one
        unsigned all = 0, before = 0;
        if ((int)threadIdx.x < digits) {
            unsigned c[kSortCluster];
#pragma unroll
            for (int r = 0; r < kSortCluster; ++r) c[r] = r < a.sorters ? load_remote(&s.total[threadIdx.x], r) : 0u;
#pragma unroll
            for (int r = 0; r < kSortCluster; ++r) {
                all += c[r];
                if (r < rank) before += c[r];
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
        for (int r = 0; r < R; ++r) {
            if (r < rounds && begin + 32 * r < a.count) {
                const unsigned d = (pair[r].x >> shift) & (digits - 1);
                const unsigned at = s.base[d] + s.warp[warp][d] + (r & 1 ? ranks[r / 2] >> 16 : ranks[r / 2] & 0xffffu);
                out[at] = pair[r];
            }
        }
        cluster_sync();  // the pass is in memory, and nobody reads this block's counts any more
    }
}

constexpr int kMostFillRows = 65536;      // 8 KB of marks
constexpr int kZeroBytes = 16384;         // behind them: zeros to copy from
constexpr int kFillShared = kMostFillRows / 8 + kZeroBytes;

// Of the rows `block`, block + fillers, ..., those that no id names become beta times what they are (beta = 0: zero). Their
// marks are set from all ids, for fill_rows of them at a time; one warp per row then. Zeros leave as bulk copies of shared
// memory: one instruction per row keeps HBM's write path full (ordinary 32-byte stores reached 3.1 TB/s, these 6).
template <typename E, int V>
__device__ __forceinline__ void fill_block(const SortArgs& a, float beta, uint8_t* smem, int block) {
    unsigned* const bits = reinterpret_cast<unsigned*>(smem);
    const uint32_t zeros = static_cast<uint32_t>(__cvta_generic_to_shared(smem + kMostFillRows / 8));
    const bool bulk = V > 1 && beta == 0.0f;
    if (bulk) {
        for (int i = threadIdx.x; i < kZeroBytes / 16; i += kSortThreads)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(zeros + 16 * i), "r"(0) : "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    const int fillers = 1 << a.fill_shift;
    const int64_t mine = (a.rows - block + fillers - 1) >> a.fill_shift;
    for (int64_t from = 0; from < mine; from += a.fill_rows) {
        const int n = (int)min((int64_t)a.fill_rows, mine - from);
        for (int i = threadIdx.x; i < (n + 31) / 32; i += kSortThreads) bits[i] = 0u;
        __syncthreads();
        for (int64_t t = threadIdx.x; t < a.count; t += 8 * kSortThreads) {
            int key[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) key[x] = t + x * kSortThreads < a.count ? key_of(a, t + x * kSortThreads) : (int)a.rows;
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                const int64_t i = (key[x] >> a.fill_shift) - from;
                if (key[x] < a.rows && (key[x] & (fillers - 1)) == block && i >= 0 && i < n) atomicOr(&bits[i >> 5], 1u << (i & 31));
            }
        }
        __syncthreads();
        const int lane = threadIdx.x & 31;
        for (int i = threadIdx.x >> 5; i < n; i += kSortThreads / 32) {
            if (bits[i >> 5] >> (i & 31) & 1) continue;
            E* row = static_cast<E*>(a.table) + (((from + i) << a.fill_shift) + block) * a.ld;
            if (bulk) {
                const int64_t bytes = a.width * (int64_t)sizeof(E);
                if (lane == 0)
                    for (int64_t x = 0; x < bytes; x += kZeroBytes)
                        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(reinterpret_cast<char*>(row) + x),
                                     "r"(zeros), "r"((int)min(bytes - x, (int64_t)kZeroBytes))
                                     : "memory");
                continue;
            }
            for (int64_t c = 0; c < a.width; c += Columns<V>::kSlab) {
                float v[Columns<V>::kPer] = {};
                if (beta != 0.0f) {
                    load_columns<E, V>(row, c, a.width, lane, v);
#pragma unroll
                    for (int x = 0; x < Columns<V>::kPer; ++x) v[x] *= beta;
                }
                store_columns<E, V>(row, c, a.width, lane, v);
            }
        }
        __syncthreads();
    }
    if (bulk) asm volatile("cp.async.bulk.commit_group;\ncp.async.bulk.wait_group 0;" ::: "memory");
}

template <int R>
__global__ void __launch_bounds__(kSortThreads) embedding_sort_kernel(const SortArgs a) {
    __shared__ SortShared s;
    grid_release();
    sort_block<R>(a, s, (int)blockIdx.x);
}

// Runs beside the sort, which lets it start at once; it ends no earlier than the sort does, so that what waits for this launch
// waits for both. A sort by one block is its last block.
template <typename E, int V>
__global__ void __launch_bounds__(kSortThreads) embedding_fill_kernel(const SortArgs a, ScalarArg<float> beta_arg) {
    constexpr size_t kShared = sizeof(SortShared) > kFillShared ? sizeof(SortShared) : kFillShared;
    __shared__ __align__(16) uint8_t smem[kShared];
    grid_release();
    if ((int)blockIdx.x == 1 << a.fill_shift) {
        sort_block<kFewRounds>(a, *reinterpret_cast<SortShared*>(smem), 0);
        return;
    }
    const float beta = beta_arg.get();
    if (beta != 1.0f && (int64_t)blockIdx.x < a.rows) fill_block<E, V>(a, beta, smem, (int)blockIdx.x);
    grid_wait();
}

template <typename T, int V>
bool wide_rows(const void* p, int64_t ld, int64_t width) {
    return (reinterpret_cast<uintptr_t>(p) & (sizeof(T) * V - 1)) == 0 && ld % V == 0 && width % V == 0;
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
    // Rows of the result that cannot stay in L2 (126 MB) leave it first, so that rows of the table which come again are still there.
    const bool stream = V > 1 && a.count * a.width * (int64_t)sizeof(Y) > (int64_t(64) << 20);
    const auto kernel = stream ? embedding_lookup_kernel<E, Y, I, V, (V > 1)> : embedding_lookup_kernel<E, Y, I, V, false>;
    kernel<<<blocks, 256, 0, s>>>(a.count, a.rows, a.width, ids, a.base, static_cast<const E*>(a.table), a.ld_table, static_cast<Y*>(a.tokens),
                                  a.ld_tokens, a.alpha, pieces);
    return cudaGetLastError();
}

template <typename E, typename Y>
cudaError_t lookup_typed(cudaStream_t s, const EmbeddingArgs& a) {
    // 8 values per thread (16 or 32 bytes); fp32 on both sides: 4, so that narrow tables still fill a warp
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
// (148 SMs x 16 warps) when there are few tokens.
int gradient_chunk(int64_t count, int64_t width) {
    const int64_t slabs = (width + 255) / 256;
    const int64_t want = count * slabs / (148 * 16);
    int chunk = 8;
    while (chunk < 64 && 2 * chunk <= want) chunk *= 2;
    return chunk;
}

struct GradientLayout {
    TransposePlan sort;  // for tokens that one cluster does not sort
    int chunk;
    int64_t chunks;
    size_t off_raw, off_sorted[2], off_partial, off_arrived, bytes;
};

GradientLayout gradient_layout(int64_t count, int64_t rows, int64_t width) {
    GradientLayout l = {};
    l.chunk = gradient_chunk(count, width);
    l.chunks = (count + l.chunk - 1) / l.chunk;
    size_t off = 0;
    if (count > kSortAlone) {  // (room for it whatever the device holds: the size is asked for without one)
        l.sort = sort_plan(rows + 1, count);
        off = l.sort.bytes;
        l.off_raw = off;
        off += align256(size_t(count) * 4);
    }
    for (int i = 0; i < (count <= kSortMost ? 2 : 1); ++i) {
        l.off_sorted[i] = off;
        off += align256(size_t(count) * 8);
    }
    l.off_partial = off;
    off += align256(size_t(l.chunks) * 2 * size_t(width) * 4);
    l.off_arrived = off;
    off += align256(size_t(l.chunks) * ((width + 127) / 128) * 4);  // (a slab is 128 columns at least)
    l.bytes = off + 256;
    return l;
}

__global__ void __launch_bounds__(256) embedding_keys_kernel(const SortArgs a, int* __restrict__ keys) {
    const int64_t t = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
    if (t < a.count) keys[t] = key_of(a, t);
    for (int64_t i = t; i < a.counters; i += (int64_t)gridDim.x * blockDim.x) a.arrived[i] = 0u;
}
__global__ void __launch_bounds__(256)
    embedding_pairs_kernel(int64_t count, const int* __restrict__ keys, const unsigned* __restrict__ perm, uint2* __restrict__ sorted) {
    const int64_t t = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
    if (t < count) sorted[t] = make_uint2((unsigned)keys[t], perm[t]);
}

cudaLaunchConfig_t cluster_config(cudaStream_t s, unsigned blocks, cudaLaunchAttribute& attr) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(kSortThreads);
    cfg.stream = s;
    attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = blocks, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cfg;
}

// Whether the current device holds a cluster of kSortCluster blocks (a part of a partitioned one may not). Asked once per device.
bool sort_cluster_fits() {
    static std::atomic<int> known[64];  // 0: not asked, 1: no, 2: yes
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return false;
    if (device < 64 && known[device].load(std::memory_order_relaxed) != 0) return known[device].load(std::memory_order_relaxed) == 2;
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = cluster_config(nullptr, kSortCluster, attr);
    const auto allow = [&](auto kernel) {
        int clusters = 0;
        return cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel), cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
               cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) == cudaSuccess && clusters > 0;
    };
    const bool fits = allow(embedding_sort_kernel<kFewRounds>) && allow(embedding_sort_kernel<kSortRounds>);
    if (!fits) cudaGetLastError();
    if (device < 64) known[device].store(fits ? 2 : 1, std::memory_order_relaxed);
    return fits;
}

template <typename Y, typename E, int V>
cudaError_t launch_gradient(cudaStream_t s, const EmbeddingArgs& a, char* b) {
    const GradientLayout l = gradient_layout(a.count, a.rows, a.width);
    // ---- sort; rows without a token (none change when beta is 1, which the host may not know)
    SortArgs so = {};
    so.count = a.count, so.rows = a.rows, so.ids = a.ids, so.wide = a.wide_ids, so.base = a.base;
    so.table = a.table, so.ld = a.ld_table, so.width = a.width;
    for (int i = 0; i < 2; ++i) so.sorted[i] = reinterpret_cast<uint2*>(b + l.off_sorted[i]);
    const int slabs = (int)((a.width + Columns<V>::kSlab - 1) / Columns<V>::kSlab);
    so.arrived = reinterpret_cast<unsigned*>(b + l.off_arrived), so.counters = l.chunks * slabs;
    int need = 1;  // bits of a key, `rows` included
    while (need < 31 && (int64_t(1) << need) <= a.rows) ++need;
    so.passes = (need + 8) / 9;
    so.bits = (need + so.passes - 1) / so.passes;
    const bool fill = a.beta.dev != nullptr || a.beta.host != 1.0f;
    int last = (so.passes - 1) & 1;
    // few tokens: one block sorts them in two rounds, as a further block of the other launch where there is one
    so.sorters = a.count == 0 ? 0 : a.count <= kSortAlone ? 1 : a.count <= kSortMost && sort_cluster_fits() ? kSortCluster : 0;
    const bool together = fill && so.sorters == 1;
    if (so.sorters > 0 && !together) {
        cudaLaunchAttribute attr;
        const cudaLaunchConfig_t cfg = cluster_config(s, (unsigned)so.sorters, attr);
        const bool few = a.count <= (int64_t)so.sorters * kSortThreads * kFewRounds;
        const cudaError_t e = few ? cudaLaunchKernelEx(&cfg, embedding_sort_kernel<kFewRounds>, static_cast<const SortArgs>(so))
                                  : cudaLaunchKernelEx(&cfg, embedding_sort_kernel<kSortRounds>, static_cast<const SortArgs>(so));
        if (e != cudaSuccess) return e;
    }
    if (a.count > 0 && so.sorters == 0) {
        int* raw = reinterpret_cast<int*>(b + l.off_raw);
        embedding_keys_kernel<<<(unsigned)((a.count + 255) / 256), 256, 0, s>>>(so, raw);
        const cudaError_t e = sort_keys(s, a.count, raw, l.sort, b);
        if (e != cudaSuccess) return e;
        const int slot = l.sort.final_slot();
        last = 0;
        embedding_pairs_kernel<<<(unsigned)((a.count + 255) / 256), 256, 0, s>>>(
            a.count, reinterpret_cast<const int*>(b + l.sort.off_keys[slot]), reinterpret_cast<const unsigned*>(b + l.sort.off_perm[slot]), so.sorted[0]);
    }
    if (fill) {  // a power of two of blocks, at most one per SM
        while ((2 << so.fill_shift) <= a.sm_count && (int64_t(1) << so.fill_shift) < a.rows) ++so.fill_shift;
        const int64_t each = (a.rows >> so.fill_shift) + 1;
        so.fill_rows = (int)(each < kMostFillRows ? each : kMostFillRows);
        const cudaError_t e = launch_behind(s, so.sorters == kSortCluster, embedding_fill_kernel<E, V>, (1u << so.fill_shift) + (together ? 1u : 0u), kSortThreads, 0, so, a.beta);
        if (e != cudaSuccess) return e;
    }
    if (a.count == 0) return cudaSuccess;
    // ---- sums
    GradientArgs g = {};
    g.count = a.count, g.rows = a.rows, g.width = a.width, g.ld_y = a.ld_tokens, g.ld_e = a.ld_table;
    g.chunk = l.chunk, g.chunks = l.chunks;
    g.sorted = so.sorted[last];
    g.partial = reinterpret_cast<float*>(b + l.off_partial);
    g.slabs = slabs, g.arrived = so.arrived;
    const unsigned blocks = warp_blocks(g.chunks * g.slabs);
    if (blocks == 0) return cudaErrorInvalidValue;
    constexpr int kShared = Rows<Y, V>::kShared;
    cudaError_t e = cudaSuccess;
    static SharedMemoryOnce once;
    if (kShared > 48 * 1024) e = once.allow(reinterpret_cast<const void*>(embedding_sum_kernel<Y, E, V>), kShared);
    if (e == cudaSuccess) e = launch_behind(s, true, embedding_sum_kernel<Y, E, V>, blocks, 256, kShared, g, static_cast<const Y*>(a.tokens), static_cast<E*>(a.table), a.alpha, a.beta);
    return e;
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
