// Tensor maps of tokens x heads x dim tensors for tiled TMA loads, and the cutting of a ragged batch into blocks.
#ifndef MCSPARSE_B200_WINDOW_MAPS_H_
#define MCSPARSE_B200_WINDOW_MAPS_H_

#include <cuda.h>

#include "internal.h"

namespace mcsp_b200 {

// A map whose box is 64 values of one head of `rows` tokens, written to shared memory in the 128-byte swizzle; values
// behind the tensor's last dimension, head or token read as zero. Coordinates: {value, head, token}; with a head stride of 0
// the tensor has one head. False: the tensor has no such map.
bool head_map(CUtensorMap* map, const AttentionTensor& t, int64_t tokens, int heads, int dim, macaDataType type, int rows);

// Blocks of `size` rows of every sequence, numbered without knowing the lengths on the host: sequence b owns the numbers
// [offset[b] / size + b, offset[b + 1] / size + b + 1), which are at least as many as its blocks; the surplus does nothing.
inline int ragged_slots(int total, int batch, bool offsets, int size) { return offsets ? total / size + batch : (total + size - 1) / size; }

// SM clocks a wait may take: 64 times the handle's limit (20 ms), so that a process that was switched off the GPU for a while
// does not look like one whose copies never arrive.
inline long long window_wait_limit(const AttentionArgs& a) { return a.wait.limit_cycles > (1LL << 50) ? (1LL << 56) : a.wait.limit_cycles * 64; }

struct RaggedBlock {
    int b, index;  // sequence (-1: none), block inside it
};

#ifdef __CUDACC__
// Called by whole warps; `number` is the same in all lanes. The search takes 32 samples at a time.
__device__ __forceinline__ RaggedBlock ragged_block(const int* offsets, int batch, int total, int number, int size, int lane) {
    if (offsets == nullptr) return RaggedBlock{0, number};
    // the last b in [0, batch) with start(b) <= number, start(b) = offset[b] / size + b
    int lo = 0, hi = batch;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32;
        const int b = lo + step * lane;
        bool below = false;
        if (b < hi) below = min(max(__ldg(offsets + b), 0), total) / size + b <= number;
        const unsigned hits = __ballot_sync(0xffffffffu, below);
        const int last = hits == 0 ? 0 : 31 - __clz(hits);
        lo += step * last;
        hi = min(lo + step, hi);
    }
    const int start = min(max(__ldg(offsets + lo), 0), total) / size + lo;
    return RaggedBlock{number >= start ? lo : -1, number - start};
}
#endif

}  // namespace mcsp_b200

#endif  // MCSPARSE_B200_WINDOW_MAPS_H_
