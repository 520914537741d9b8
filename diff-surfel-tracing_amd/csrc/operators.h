// What the label and attention operators share on the host: errors, sizes, the choice of a split.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dst_api.h"

// dst_api.hip: the message of dst_op_error(), a fixed array of the calling thread (nothing is allocated, nothing throws).
int dst_op_fail(int code, const char *format, ...) __attribute__((format(printf, 2, 3)));

#define DST_OP_LAUNCH(name)                                                                                     \
    do {                                                                                                        \
        hipError_t e_ = hipGetLastError();                                                                      \
        if (e_ != hipSuccess) return dst_op_fail(DST_E_DEVICE, "%s: launch failed: %s", name, hipGetErrorString(e_)); \
    } while (0)

namespace {

inline int value_size(int dtype) { return dtype == DST_DTYPE_F32 ? 4 : 2; }
// 64-byte fragments of a row, as the kernels are instantiated: 1, 2, 4, 8 or 16
inline int fragments_of(int channels, int dtype) {
    const int bytes = channels * value_size(dtype);
    int nk = 1;
    while (nk * 64 < bytes) nk *= 2;
    return nk;
}
inline bool words_align(const void *p, int64_t stride, int channels, int size) {
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (stride * size) % 16 == 0 && (channels * size) % 16 == 0;
}
inline int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline uint64_t align_up(uint64_t bytes) { return (bytes + 255u) & ~(uint64_t)255u; }

// How many parts the streamed tiles are cut into. 256 compute units want about two workgroups each; every part costs a
// write and a read of the own rows' sums, so a part has at least four tiles while there are any.
constexpr int kMostSplits = 512;
struct Split {
    int splits, per_split;
};
inline Split split_tiles(int64_t own_tiles, int64_t stream_tiles) {
    if (stream_tiles < 1) return Split{1, 1};
    int64_t want = div_up(kMostSplits, own_tiles > 0 ? own_tiles : 1);
    const int64_t most = stream_tiles >= 8 ? stream_tiles / 4 : 1;
    if (want > most) want = most;
    if (want < 1) want = 1;
    const int64_t per = div_up(stream_tiles, want);
    return Split{(int)div_up(stream_tiles, per), (int)per};
}

// Whether the own rows are few: blocks of 16 * QB rows a wave would leave compute units without a workgroup, however the streamed
// rows are split; one block of 16 a wave then makes more, shorter ones.
inline bool few_rows(int64_t rows, int own, int64_t stream_tiles) {
    const int64_t most = stream_tiles >= 8 ? stream_tiles / 4 : 1;
    return div_up(rows, own) * most < 256;
}

// Pieces of a workspace, in order.
struct Carve {
    char *base;
    uint64_t used;
    template <class T> T *take(uint64_t n) {
        T *p = reinterpret_cast<T *>(base + used);
        used += align_up(n * sizeof(T));
        return p;
    }
};

// out[i] = sum of part[s][i], always in the same order. Two arrays in one launch (the second may be empty): a launch costs more than
// either sum. kLanes parts are added side by side where there are many (a few thousand sums of 450 parts: 6 us with 8 lanes,
// 115 with one, whose loads wait for each other).
template <class E, class E2, int kLanes>
__global__ __launch_bounds__(256) void k_sum_parts(const float *part, E *out, int64_t n, const float *part2, E2 *out2, int64_t n2, int splits) {
    constexpr int kColumns = 256 / kLanes;
    __shared__ float lds[256];
    const int column = threadIdx.x % kColumns, lane = threadIdx.x / kColumns;
    const int64_t blocks = (n + kColumns - 1) / kColumns, all = blocks + (n2 + kColumns - 1) / kColumns;
    for (int64_t b = blockIdx.x; b < all; b += gridDim.x) {
        const bool second = b >= blocks;
        const int64_t i = (second ? b - blocks : b) * kColumns + column, size = second ? n2 : n;
        const float *from = (second ? part2 : part) + i;
        float s = 0.0f;
        if (i < size)
#pragma unroll 4
            for (int k = lane; k < splits; k += kLanes) s += from[(int64_t)k * size];
        if constexpr (kLanes > 1) {
            __syncthreads();
            lds[threadIdx.x] = s;
            __syncthreads();
            if (lane != 0) continue;
#pragma unroll
            for (int k = 1; k < kLanes; ++k) s += lds[k * kColumns + column];
        }
        if (i < size) {
            if (second) out2[i] = (E2)s;
            else out[i] = (E)s;
        }
    }
}
template <class E, class E2>
inline void sum_parts(const float *part, E *out, int64_t n, const float *part2, E2 *out2, int64_t n2, int splits, hipStream_t s) {
    if (!out) n = 0;
    if (!out2) n2 = 0;
    if (n + n2 == 0) return;
    const int columns = splits >= 16 ? 32 : 256;
    const int64_t blocks = div_up(n, columns) + div_up(n2, columns);
    const dim3 grid((uint32_t)(blocks < 8192 ? blocks : 8192));
    if (splits >= 16) k_sum_parts<E, E2, 8><<<grid, 256, 0, s>>>(part, out, n, part2, out2, n2, splits);
    else k_sum_parts<E, E2, 1><<<grid, 256, 0, s>>>(part, out, n, part2, out2, n2, splits);
}

}  // namespace
