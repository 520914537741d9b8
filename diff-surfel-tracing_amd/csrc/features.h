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
struct Split {
    int splits, per_split;
};
inline Split split_tiles(int64_t own_tiles, int64_t stream_tiles) {
    if (stream_tiles < 1) return Split{1, 1};
    int64_t want = div_up(512, own_tiles > 0 ? own_tiles : 1);
    const int64_t most = stream_tiles >= 8 ? stream_tiles / 4 : 1;
    if (want > most) want = most;
    if (want < 1) want = 1;
    const int64_t per = div_up(stream_tiles, want);
    return Split{(int)div_up(stream_tiles, per), (int)per};
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

// out[i] = sum of part[s][i]: the parts in their order.
template <class E> __global__ __launch_bounds__(256) void k_sum_parts(const float *part, E *out, int64_t n, int splits) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        float s = 0.0f;
        for (int k = 0; k < splits; ++k) s += part[(int64_t)k * n + i];
        out[i] = (E)s;
    }
}
inline uint32_t sum_blocks(int64_t n) { return (uint32_t)(div_up(n, 256) < 4096 ? div_up(n, 256) : 4096); }

}  // namespace
