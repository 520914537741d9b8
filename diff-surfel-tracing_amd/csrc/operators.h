// What the label and attention operators share on the host: errors, sizes, the choice of a split.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dst_api.h"
#include "tiles.inc"

// dst_api.hip: the message of dst_op_error(), a fixed array of the calling thread (nothing is allocated, nothing throws).
int dst_op_fail(int code, const char *format, ...) __attribute__((format(printf, 2, 3)));

#define DST_OP_LAUNCH(name)                                                                                     \
    do {                                                                                                        \
        hipError_t e_ = hipGetLastError();                                                                      \
        if (e_ != hipSuccess) return dst_op_fail(DST_E_DEVICE, "%s: launch failed: %s", name, hipGetErrorString(e_)); \
    } while (0)

namespace {

inline int value_size(int dtype) { return dtype == DST_DTYPE_F32 ? 4 : 2; }
// 64-byte fragments of a row, as the kernels are instantiated: 0 (half a one), 1, 2, 4, 8 or 16
inline int fragments_of(int channels, int dtype) {
    const int bytes = channels * value_size(dtype);
    if (dtype == DST_DTYPE_F32 && bytes <= 32) return 0;
    int nk = 1;
    while (nk * 64 < bytes) nk *= 2;
    return nk;
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

// Rows that the kernels cannot read where they lie, copied: (batches, heads, rows) of whole words, zeros behind the channels.
struct RowCopy {
    const char *from;
    int64_t batch, row, in_group;   // bytes; a head is `group` steps of in_group
    int32_t heads, group, size, channels, words;
    int64_t rows, all_words;
    uint4 *to;
};
__global__ __launch_bounds__(256) void k_copy_rows(RowCopy c) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= c.all_words) return;
    const int64_t at = i / c.words, r = at % c.rows, head = at / c.rows % c.heads, batch = at / c.rows / c.heads;
    const int w = (int)(i - at * c.words);
    const char *from = c.from + batch * c.batch + r / c.group * c.row + (head * c.group + r % c.group) * c.in_group;
    uint32_t word[4] = {0u, 0u, 0u, 0u};
    if (c.size == 4) {
        for (int k = 0; k < 4; ++k)
            if (4 * w + k < c.channels) word[k] = reinterpret_cast<const uint32_t *>(from)[4 * w + k];
    } else {
        for (int k = 0; k < 8; ++k)
            if (8 * w + k < c.channels) word[k / 2] |= (uint32_t) reinterpret_cast<const uint16_t *>(from)[8 * w + k] << (16 * (k & 1));
    }
    c.to[i] = uint4{word[0], word[1], word[2], word[3]};
}

// A set of rows for the kernels: as it lies, or a copy that `prepare` makes in the workspace first. Strides in values: from batch to batch,
// row to row (of `group` heads) and head to head; `stride`: a step in rows that has to be of whole groups.
struct RowSet {
    Rows rows;
    RowCopy copy;
    bool copied;
};
inline RowSet row_set(const void *p, int64_t batch, int64_t row, int64_t head, int64_t batches, int heads, int group, int64_t n, int channels,
                      int dtype, int stride, Carve &c) {
    const int size = value_size(dtype), words = (channels * size + 15) / 16;
    RowSet s = {};
    s.rows = Rows{(const char *)p, batch * size, head * size * group, row * size, (int32_t)(head * size), group, words};
    const int64_t widest = (256 / group + 1) * s.rows.row + (int64_t)group * head * size + 4096;   // within 256 rows
    s.copied = (channels * size) % 16 != 0 || (reinterpret_cast<uintptr_t>(p) & 3u) != 0 || (batch * size) % 4 != 0 || (row * size) % 4 != 0 ||
               (head * size) % 4 != 0 || stride % group != 0 || widest > 0x7fffffff || head * size > 0x7fffffff;
    if (s.copied) {
        const int64_t all = batches * heads * n * words;
        s.copy = RowCopy{(const char *)p, batch * size, row * size, head * size, heads, group, size, channels, words, n, all, c.take<uint4>(all)};
        s.rows = Rows{(const char *)s.copy.to, (int64_t)heads * n * words * 16, n * words * 16, words * 16, 0, 1, words};
    }
    return s;
}
inline void prepare(const RowSet &s, hipStream_t stream) {
    if (s.copied && s.copy.all_words > 0) k_copy_rows<<<dim3((uint32_t)div_up(s.copy.all_words, 256)), 256, 0, stream>>>(s.copy);
}

}  // namespace
