// Rows of a table by token ids, Y = alpha * S * E, and the table's gradient, dE = alpha * S^T * dY + beta * dE, for the
// count x rows matrix S with one 1 per row (its column: the token's id). S is never stored.
//
// Lookup: one pass; a warp moves a piece of one row with 16-byte loads and stores. Bound by memory (count * width read,
// unless rows repeat, and written).
//
// Gradient: S^T in CSR form is the tokens sorted by id, so the ids are sorted (stable radix sort of (id, position) pairs)
// and the rows of dY summed in that order. The sorted tokens are cut into chunks of equal size whatever the ids are, so a
// token that fills half the batch costs no more than any other; a warp owns one chunk and a slab of columns, adds in fp32
// and writes every sum that lies inside its chunk. A sum that crosses chunks is left as one partial per chunk and put
// together, in chunk order, by a second kernel. No atomics: the order of every addition follows from ids and sizes.
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

// key = the row of the table, or `rows` for an id outside it (sorted behind every row and then left out).
template <typename I>
__global__ void __launch_bounds__(256)
    embedding_keys_kernel(int64_t count, int64_t rows, const I* __restrict__ ids, int base, int* __restrict__ keys) {
    const int64_t t = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
    if (t >= count) return;
    const int64_t id = (int64_t)ids[t] - base;
    keys[t] = (int)(id >= 0 && id < rows ? id : rows);
}

struct GradientArgs {
    int64_t count, rows, width, ld_y, ld_e, chunks;
    int chunk, slabs;
    const int* keys;       // sorted
    const unsigned* perm;  // token of every sorted place
    const int* offsets;    // rows + 1: where a row's tokens start
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

// One warp per (chunk of sorted tokens, slab of columns); behind those, one warp per (row, slab) for the rows that have
// no token and still change (beta != 1).
template <typename Y, typename E, int V>
__global__ void __launch_bounds__(256)
    embedding_sum_kernel(GradientArgs a, const Y* __restrict__ dy, E* __restrict__ table, ScalarArg<float> alpha_arg,
                         ScalarArg<float> beta_arg) {
    constexpr int kPer = Columns<V>::kPer, kSlab = Columns<V>::kSlab, kDepth = 8;
    const int64_t warp = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    const float alpha = alpha_arg.get(), beta = beta_arg.get();
    if (warp >= a.chunks * a.slabs) {
        const int64_t w = warp - a.chunks * a.slabs;
        const int64_t r = w / a.slabs;
        if (r >= a.rows || beta == 1.0f) return;
        if (__ldg(a.offsets + r) != __ldg(a.offsets + r + 1)) return;
        const int64_t first = (w - r * a.slabs) * kSlab;
        float none[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) none[i] = 0.0f;
        finish_row<E, V>(table, a, r, first, lane, 0.0f, beta, none);
        return;
    }
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
    const int64_t end = __ldg(a.offsets + row + 1);                   // its last token is at end - 1
    const int64_t last = (end - 1) / a.chunk;
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
    TransposePlan sort;
    int chunk;
    int64_t chunks;
    size_t off_keys, off_partial, bytes;
};

GradientLayout gradient_layout(int64_t count, int64_t rows, int64_t width) {
    GradientLayout l;
    l.sort = transpose_plan(rows, rows + 1, count, 0);
    l.chunk = gradient_chunk(count, width);
    l.chunks = (count + l.chunk - 1) / l.chunk;
    size_t off = l.sort.bytes;
    l.off_keys = off;
    off += align256(size_t(count) * 4);
    l.off_partial = off;
    off += align256(size_t(l.chunks) * 2 * size_t(width) * 4);
    l.bytes = off + 256;
    return l;
}

template <typename Y, typename E, int V>
cudaError_t launch_gradient(cudaStream_t s, const EmbeddingArgs& a, GradientArgs g) {
    g.slabs = (int)((a.width + Columns<V>::kSlab - 1) / Columns<V>::kSlab);
    // beta == 1 on the host's side needs no warps for the rows without tokens
    const bool all_rows = a.beta.dev != nullptr || a.beta.host != 1.0f;
    const int64_t warps = (g.chunks + (all_rows ? a.rows : 0)) * g.slabs;
    if (warps == 0) return cudaSuccess;
    const unsigned blocks = warp_blocks(warps);
    if (blocks == 0) return cudaErrorInvalidValue;
    embedding_sum_kernel<Y, E, V><<<blocks, 256, 0, s>>>(g, static_cast<const Y*>(a.tokens), static_cast<E*>(a.table), a.alpha, a.beta);
    if (g.chunks > 1)
        embedding_join_kernel<E, V><<<warp_blocks(g.chunks * g.slabs), 256, 0, s>>>(g, static_cast<E*>(a.table), a.alpha, a.beta);
    return cudaGetLastError();
}

template <typename E, typename Y>
cudaError_t gradient_typed(cudaStream_t s, const EmbeddingArgs& a, const GradientArgs& g) {
    constexpr int V = sizeof(E) == 4 && sizeof(Y) == 4 ? 4 : 8;
    const bool wide = wide_rows<E, V>(a.table, a.ld_table, a.width) && wide_rows<Y, V>(a.tokens, a.ld_tokens, a.width);
    return wide ? launch_gradient<Y, E, V>(s, a, g) : launch_gradient<Y, E, 1>(s, a, g);
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
    const GradientLayout l = gradient_layout(a.count, a.rows, a.width);
    char* b = static_cast<char*>(align_up_256(buffer));
    int* keys = reinterpret_cast<int*>(b + l.off_keys);
    if (a.count > 0) {
        const unsigned blocks = (unsigned)((a.count + 255) / 256);
        if (a.wide_ids)
            embedding_keys_kernel<<<blocks, 256, 0, s>>>(a.count, a.rows, static_cast<const int64_t*>(a.ids), a.base, keys);
        else
            embedding_keys_kernel<<<blocks, 256, 0, s>>>(a.count, a.rows, static_cast<const int32_t*>(a.ids), a.base, keys);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return e;
    }
    const cudaError_t e = sort_keys(s, a.rows, a.count, keys, l.sort, b);
    if (e != cudaSuccess) return e;
    GradientArgs g = {};
    g.count = a.count, g.rows = a.rows, g.width = a.width, g.ld_y = a.ld_tokens, g.ld_e = a.ld_table;
    g.chunk = l.chunk, g.chunks = l.chunks;
    g.keys = reinterpret_cast<const int*>(b + l.sort.off_keys[l.sort.final_slot()]);
    g.perm = reinterpret_cast<const unsigned*>(b + l.sort.off_perm[l.sort.final_slot()]);
    g.offsets = reinterpret_cast<const int*>(b + l.sort.off_ptr);
    g.partial = reinterpret_cast<float*>(b + l.off_partial);
    MCSP_EMBEDDING_TYPES(gradient_typed, s, a, g);
}

}  // namespace mcsp_b200
