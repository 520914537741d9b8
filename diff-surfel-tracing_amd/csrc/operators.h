// What the label and attention operators share on the host: errors, sizes, the choice of a split.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <initializer_list>
#include <type_traits>

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

constexpr int64_t kLongestStride = (int64_t)1 << 44;   // values; offsets of 256 rows in bytes are far from 64 bits' end
inline int value_size(int dtype) { return dtype == DST_DTYPE_F32 ? 4 : 2; }
// 32-bit rows longer than this are split into planes of 16 bits (tiles.inc).
constexpr int kLongest32 = 16;
// 64-byte fragments of a row (of its planes, where it is split), as the kernels are instantiated: 0 (half a one), 1, 2, 4 or 8
inline int fragments_of(int channels, int dtype) {
    if (dtype == DST_DTYPE_F32 && channels <= kLongest32) return channels <= 8 ? 0 : 1;
    int nk = 1;
    while (nk * 32 < channels) nk *= 2;
    return nk;
}
// f(type, integral constant of the fragments) of a call
template <class TY, class F> int with_fragments(int nk, F f) {
    if constexpr (std::is_same_v<TY, F32>) {
        return nk == 0 ? f(TY{}, std::integral_constant<int, 0>{}) : f(TY{}, std::integral_constant<int, 1>{});
    } else {
        switch (nk) {
            case 1: return f(TY{}, std::integral_constant<int, 1>{});
            case 2: return f(TY{}, std::integral_constant<int, 2>{});
            case 4: return f(TY{}, std::integral_constant<int, 4>{});
            default: return f(TY{}, std::integral_constant<int, 8>{});
        }
    }
}
// (SHORT: for products with a table, whose rows of up to eight values have a type of their own)
template <bool SHORT, class F> int with_floats(int channels, F f) {
    const int nk = fragments_of(channels, DST_DTYPE_F32);
    if constexpr (SHORT) {
        if (channels <= 8) return f(Short32{}, std::integral_constant<int, 0>{});
        if (channels <= kLongest32) return f(F32{}, std::integral_constant<int, 1>{});
    } else {
        if (channels <= kLongest32) return with_fragments<F32>(nk, f);
    }
    return with_fragments<Split32>(nk, f);
}
inline int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline uint64_t align_up(uint64_t bytes) { return (bytes + 255u) & ~(uint64_t)255u; }

// Who does what. A workgroup takes a tile of own rows against all streamed tiles; the device holds `slots` workgroups at once, and own
// tiles that do not fill its last round (or are fewer than it holds) are cut into parts of the streamed tiles, whose sums a
// closing kernel adds: 513 tiles on 512 places would take two rounds. Tiles below `whole` are not cut.
constexpr int kMostSplits = 512;
constexpr int64_t kMostBlocks = 0xffffff;   // workgroups of a launch, whose threads are counted in 32 bits
struct Cut {
    int32_t tiles, whole, splits, per_split;   // per_split: streamed tiles of a part
    __host__ __device__ int64_t parted() const { return tiles - whole; }
    int64_t blocks() const { return whole + parted() * splits; }
};
struct Turn {   // a workgroup's
    int tile, split;
    bool part;
};
__device__ inline Turn turn_of(const Cut &c) {
    const int b = (int)blockIdx.x - c.whole;
    if (b < 0) return Turn{(int)blockIdx.x, 0, false};
    return Turn{c.whole + b / c.splits, b % c.splits, c.splits > 1};
}
// Where a part's row lies among the parts: `own` rows a tile.
__device__ inline int64_t part_row(const Cut &c, const Turn &t, int own, int row) {
    return ((int64_t)(t.tile - c.whole) * c.splits + t.split) * own + row;
}

// `tile_us`: what a streamed tile takes a workgroup, about; `own_bytes`: what a part writes and the closing kernel reads. The parts are those
// of the shortest time by this count: rounds of workgroups, each of its part's tiles and two tiles' worth of beginning and
// end; then the closing kernel, 4 us and the parts' bytes at 4 TB/s.
inline Cut cut_tiles(int64_t own_tiles, int64_t stream_tiles, int slots, double tile_us, double own_bytes, bool ragged = false) {
    Cut c = {(int)own_tiles, (int)own_tiles, 1, (int)(stream_tiles > 0 ? stream_tiles : 1)};
    // (of ragged rows about half is there: tiles that fill the places once even out by themselves, fewer are cut finer)
    if (ragged && own_tiles >= slots) return c;
    if (ragged) slots *= 2;
    const int64_t rest = own_tiles % slots;
    if (rest == 0 || stream_tiles < 4) return c;
    double best = (stream_tiles + 2) * tile_us;
    for (int rounds = 1; rounds <= 8; ++rounds) {
        int64_t want = rounds * (int64_t)slots / rest;
        if (want > kMostSplits) want = kMostSplits;
        if (want > stream_tiles / 2) want = stream_tiles / 2;
        if (want < 2) continue;
        const int64_t per = div_up(stream_tiles, want), splits = div_up(stream_tiles, per);
        const double us = div_up(rest * splits, slots) * (per + 2) * tile_us + 4.0 + 2.0 * rest * splits * own_bytes / 4e6;
        if (splits > 1 && us < best) best = us, c.whole = (int)(own_tiles - rest), c.splits = (int)splits, c.per_split = (int)per;
    }
    return c;
}
// Workgroups of a kernel that the current device runs side by side: one or two on a compute unit. (A third hides some latency but has
// no more of the matrix units: counted as a place of its own it made the parts smaller and the kernels 6 % slower.)
inline int slots_of(const void *kernel) {
    int each = 0, units = 0, device = 0;
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&each, kernel, 256, 0) != hipSuccess || each < 1 || hipGetDevice(&device) != hipSuccess ||
        hipDeviceGetAttribute(&units, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || units < 1) {
        (void)hipGetLastError();
        return 512;
    }
    return (each < 2 ? each : 2) * units;
}
// What a streamed tile takes a workgroup, about: `products` of own x tile x depth at 40 % of a compute unit's rate, shared by two
// workgroups, and the exponentials.
template <class TY, int NK> double tile_time(int own, int products) {
    const double flops = 2.0 * own * Shape<TY, NK>::kRows * (NK ? NK * TY::kDepth : 8) * products;
    return 2.0 * (flops / (TY::kPlanes == 3 ? 0.7e6 : TY::kRounds ? 4e6 : 0.4e6) + own * Shape<TY, NK>::kRows * 1.6e-5);
}

// Whether the own rows are few: blocks of 16 * QB rows a wave would leave compute units without a workgroup, however the streamed
// rows are cut; one block of 16 a wave then makes more, shorter ones.
inline bool few_rows(int64_t own_tiles, int64_t stream_tiles) {
    return own_tiles * (stream_tiles >= 8 ? stream_tiles / 4 : 1) < 256;
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

// The sums of parts, always in the same order. Two arrays of rows in one launch (a launch costs more than either sum): `width`
// values a row, out[to(i)] of the i-th parted row; to(i) < 0: no such row. kLanes parts are added side by side where there are many
// (a few thousand sums of 450 parts: 7 us with 8 lanes, 115 with one, whose loads wait for each other).
template <class E> struct Parts {
    const float *part;
    E *out;       // nullptr: not wanted
    int32_t width;
};
template <class E, class E2, int kLanes, class To>
__global__ __launch_bounds__(256) void k_sum_parts(Parts<E> a, Parts<E2> b, Cut cut, int own, To to) {
    constexpr int kColumns = 256 / kLanes;
    __shared__ float lds[256];
    const int column = threadIdx.x % kColumns, lane = threadIdx.x / kColumns;
    const uint32_t rows = (uint32_t)cut.parted() * own;
    const uint32_t n = a.out ? rows * a.width : 0u, n2 = b.out ? rows * b.width : 0u;
    const uint32_t blocks = (n + kColumns - 1) / kColumns, all = blocks + (n2 + kColumns - 1) / kColumns;
    for (uint32_t at = blockIdx.x; at < all; at += gridDim.x) {
        const bool second = at >= blocks;
        const uint32_t i = (second ? at - blocks : at) * kColumns + column, width = second ? b.width : a.width;
        const uint32_t row = i / width, tile = row / (uint32_t)own, size = own * width;
        const bool there = i < (second ? n2 : n);
        const float *from = (second ? b.part : a.part) + (uint64_t)tile * cut.splits * size + (i - tile * size);
        float s = 0.0f;
        if (there)
#pragma unroll 4
            for (int k = lane; k < cut.splits; k += kLanes) s += from[(uint64_t)k * size];
        if constexpr (kLanes > 1) {
            __syncthreads();
            lds[threadIdx.x] = s;
            __syncthreads();
            if (lane != 0) continue;
#pragma unroll
            for (int k = 1; k < kLanes; ++k) s += lds[k * kColumns + column];
        }
        if (!there) continue;
        const int64_t where = to((int)tile, (int)(row - tile * own));
        if (where < 0) continue;
        if (second) b.out[where * width + (i - row * width)] = (E2)s;
        else a.out[where * width + (i - row * width)] = (E)s;
    }
}
// f(a value of the type that gradients of E rows are written in)
template <class E, class F> inline void with_output(bool half, F f) {
    if constexpr (sizeof(E) == 4)
        if (half) return f((_Float16)0.0f);
    f(E{});
}
template <class E, class E2, class To> inline void sum_parts(Parts<E> a, Parts<E2> b, const Cut &cut, int own, To to, hipStream_t s) {
    if (cut.splits < 2 || (!a.out && !b.out)) return;
    const int columns = cut.splits >= 16 ? 32 : 256;
    const int64_t rows = cut.parted() * own, blocks = div_up(a.out ? rows * a.width : 0, columns) + div_up(b.out ? rows * b.width : 0, columns);
    const dim3 grid((uint32_t)(blocks < 8192 ? blocks : 8192));
    if (cut.splits >= 16) k_sum_parts<E, E2, 8><<<grid, 256, 0, s>>>(a, b, cut, own, to);
    else k_sum_parts<E, E2, 1><<<grid, 256, 0, s>>>(a, b, cut, own, to);
}

// Rows that the kernels cannot read where they lie, copied: (batches, heads, rows) of whole words, zeros behind the channels; 32-bit
// values split into planes where `split`, binary16 values widened to 32 bits where `half`; `low`: 0, or rows like `from` that are added.
struct RowCopy {
    const char *from, *low;
    int64_t batch, row, in_group;   // bytes; a head is `group` steps of in_group
    int32_t heads, group, size, channels, words, split, half;
    int64_t rows, all_words;
    uint4 *to;
};
constexpr int kMostSets = 6;
struct CopyList {   // in one launch: set s has the blocks first[s] .. first[s + 1] - 1
    RowCopy set[kMostSets];
    uint32_t first[kMostSets + 1];
};
__global__ __launch_bounds__(256) void k_copy_rows(CopyList list) {
    int s = 0;
#pragma unroll
    for (int k = 1; k < kMostSets; ++k) s = blockIdx.x >= list.first[k] ? k : s;
    const RowCopy c = list.set[s];
    const int64_t i = (int64_t)(blockIdx.x - list.first[s]) * 256 + threadIdx.x;
    if (i >= c.all_words) return;
    const int64_t at = i / c.words, r = at % c.rows, head = at / c.rows % c.heads, batch = at / c.rows / c.heads;
    const int w = (int)(i - at * c.words);
    const int64_t offset = batch * c.batch + r / c.group * c.row + (head * c.group + r % c.group) * c.in_group;
    const char *from = c.from + offset;
    auto value = [&](int k) {   // in 32 bits
        if (k >= c.channels) return 0.0f;
        if (!c.half) return reinterpret_cast<const float *>(from)[k];
        const float v = (float)reinterpret_cast<const _Float16 *>(from)[k];
        return c.low ? v + (float)reinterpret_cast<const _Float16 *>(c.low + offset)[k] : v;
    };
    if (c.split) {
        f4 v[2];
        for (int h = 0; h < 2; ++h)
            if (!c.half && 8 * w + 4 * h + 4 <= c.channels) __builtin_memcpy(&v[h], from + 32 * w + 16 * h, 16);
            else v[h] = f4{value(8 * w + 4 * h), value(8 * w + 4 * h + 1), value(8 * w + 4 * h + 2), value(8 * w + 4 * h + 3)};
        u4 planes[3];
        Split32::pack(v[0], v[1], planes);
        for (int p = 0; p < 3; ++p) reinterpret_cast<u4 *>(c.to)[(at * 3 + p) * c.words + w] = planes[p];
        return;
    }
    uint32_t word[4] = {0u, 0u, 0u, 0u};
    if (c.size == 4 || c.half) {
        for (int k = 0; k < 4; ++k) word[k] = __builtin_bit_cast(uint32_t, value(4 * w + k));
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
template <class TY>
RowSet row_set(const void *p, int dtype, int64_t batch, int64_t row, int64_t head, int64_t batches, int heads, int group, int64_t n, int channels, int stride,
               Carve &c, const void *low = nullptr) {
    constexpr bool split = TY::kPlanes == 3;
    const bool half = dtype == DST_DTYPE_F16 && sizeof(typename TY::E) == 4;   // gradients of binary16 rows are formed in 32 bits
    const int size = value_size(dtype), words = split ? (channels + 7) / 8 : (channels * (int)sizeof(typename TY::E) + 15) / 16;
    RowSet s = {};
    s.rows = Rows{(const char *)p, batch * size, head * size * group, row * size, head * size > 0x7fffffff ? 0 : (int32_t)(head * size), group, words};
    const int64_t widest = (256 / group + 1) * s.rows.row + (int64_t)group * head * size + 4096;   // within 256 rows
    s.copied = split || half || (channels * size) % 16 != 0 || (reinterpret_cast<uintptr_t>(p) & 3u) != 0 || (batch * size) % 4 != 0 ||
               (row * size) % 4 != 0 || (head * size) % 4 != 0 || stride % group != 0 || widest > 0x7fffffff || head * size > 0x7fffffff;
    if (s.copied) {
        const int64_t all = batches * heads * n * words, line = words * TY::kPlanes * 16;
        s.copy = RowCopy{(const char *)p, half ? (const char *)low : nullptr, batch * size, row * size, head * size, heads, group, size, channels, words,
                         split, half, n, all, c.take<uint4>(all * TY::kPlanes)};
        s.rows = Rows{(const char *)s.copy.to, (int64_t)heads * n * line, n * line, line, 0, 1, words};
    }
    return s;
}
// Workgroups of the launch that makes the copies.
inline int64_t copy_blocks(std::initializer_list<const RowSet *> sets) {
    int64_t blocks = 0;
    for (const RowSet *s : sets)
        if (s->copied) blocks += div_up(s->copy.all_words, 256);
    return blocks;
}
// Makes the copies of the sets that have any.
inline void prepare(std::initializer_list<const RowSet *> sets, hipStream_t stream) {
    CopyList list = {};
    int n = 0;
    uint32_t blocks = 0;
    for (const RowSet *s : sets)
        if (s->copied && s->copy.all_words > 0) {
            list.set[n] = s->copy, list.first[n++] = blocks;
            blocks += (uint32_t)div_up(s->copy.all_words, 256);
        }
    for (int k = n; k <= kMostSets; ++k) list.first[k] = blocks;
    if (blocks > 0) k_copy_rows<<<dim3(blocks), 256, 0, stream>>>(list);
}

}  // namespace
