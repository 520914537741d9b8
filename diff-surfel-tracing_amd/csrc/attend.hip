// Attention of rays' queries to a memory of another length, forward and backward.
//
//     s_ij = c q_i . k_j,   p = softmax_j over j < length,   o_i = sum_j p_ij v_j,   lse_i = log sum_j exp s_ij
//     delta_i = do_i . o_i,   ds_ij = p_ij (do_i . v_j - delta_i),   dq = c ds k,   dk = c ds^T q,   dv = p^T do
//
// Rows: the queries of all heads that share a kv head (row = query * group + head of the group), so that a memory's tile is
// read once for all of them, and a shared head's gradient is one sum. The forward kernel and the kernel of dq own rows and
// stream the memory; the kernel of dk and dv owns the memory's rows and streams the queries; both form p again from the
// saved lse. No atomics. Own tiles that do not fill the device's last round, or are too few to fill it at all (one ray that asks
// a long memory), are cut into parts of the streamed rows, which a closing kernel joins.
#include <type_traits>

#include "operators.h"

namespace {

struct AttendArgs {
    Rows q, k, v, o, low, up;      // o, low: out as the backward pass reads it, and what its rounding left; up: its gradient
    const int32_t *lengths;
    int32_t queries, memory, heads, kv_heads, group, rows;   // rows = queries * group
    int32_t d, dv;
    Cut cut;
    int32_t own, tiles;            // own rows of a workgroup; tiles of them of one kv head of one batch
    float scale, c;                // c: what brings a product of rows to a score in units of log 2, but for what own rows carry
    float own_scale;               // 32-bit rows
    int32_t flip;                  // 16-bit rows
    void *out, *out_low;           // out_low: of 16-bit rows, what out's rounding leaves, rounded to the same type; or nullptr
    int32_t half;                  // gradients are written in binary16 though rows are in 32 bits
    float *lse2, *delta;
    void *dq, *dk, *dvalue;        // contiguous
    float2 *part;                  // of a part's rows: maximum and sum
    float *out_part, *out_part2;   // of a part's rows: sums
    int64_t all_rows;              // batch * kv_heads * rows
};

// Own blocks of 16 rows a wave. More of them read a streamed tile fewer times from LDS, fewer leave registers for a second wave on a
// SIMD, which counts for more: the waits of one are the other's work (16384 x 8192, 8 heads of 128, bf16: forward 802 us with 4
// blocks, 685 with 2; dk and dv 1619 with 2, 1317 with 1).
template <class TY, int NK> constexpr int forward_blocks() { return NK * TY::kPlanes <= 8 ? 2 : 1; }
template <class TY, int NK> constexpr int dq_blocks() { return NK * TY::kPlanes <= 6 ? 2 : 1; }
template <class TY, int NK> constexpr int dkv_blocks() { return NK * TY::kPlanes <= 3 ? 2 : 1; }

struct Place {   // which own tile, batch and kv head a workgroup has
    int tile, batch, kv, length;
};
__device__ inline Place place_of(const AttendArgs &a, uint32_t i) {
    Place p;
    p.tile = i % (uint32_t)a.tiles, i /= (uint32_t)a.tiles;
    p.kv = i % (uint32_t)a.kv_heads, p.batch = i / (uint32_t)a.kv_heads;
    p.length = a.lengths ? min(max(a.lengths[p.batch], 0), a.memory) : a.memory;
    return p;
}

// Where a row of out and dq is written (contiguous: batch, query, head): the offset in rows.
__device__ inline int64_t out_row(const AttendArgs &a, const Place &p, int row) {
    const int query = a.group == 1 ? row : (int)((uint32_t)row / (uint32_t)a.group), head = p.kv * a.group + row - query * a.group;
    return ((int64_t)p.batch * a.queries + query) * a.heads + head;
}
// Row of lse, delta and the parts
__device__ inline int64_t stat_row(const AttendArgs &a, const Place &p, int row) { return ((int64_t)p.batch * a.kv_heads + p.kv) * a.rows + row; }

// What own rows carry of the scores' factor: rows in 32 bits all of it, rows of 16 bits or planes the sign.
template <class TY, int NK, int QB> __device__ inline void carry_scale(Own<TY, NK, QB> &own, const AttendArgs &a) {
#pragma unroll
    for (int q = 0; q < QB; ++q)
#pragma unroll
        for (int k = 0; k < fragments<NK>(); ++k)
#pragma unroll
            for (int p = 0; p < TY::kPlanes; ++p) {
                u4 &w = own.f[q][k].w[p];
                if constexpr (TY::kDepth == 16) w = __builtin_bit_cast(u4, __builtin_bit_cast(f4, w) * a.own_scale);
                else if (a.flip) w ^= u4{0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u};
            }
}
// The weight of a product of rows, `less` its row's maximum or lse. The score is rounded before the difference is formed (no fused
// multiply-add): both are then rounded alike, however large, and a row with one weight gets exactly 1, its value and, in the backward
// pass, scores without a gradient. (With a fused one a score of 1.7e7 had weights of up to 2, and one of 1e10 had none: the exact score
// lies that far from the rounded one. It saved 4 % of 131,072 rows x 1024 in 4 heads of 64.)
// Weights of binary16 rows come 2^kLift larger: they are rounded to binary16 for the product with the values, where less than 2^-14 loses bits
// and less than 2^-25 everything, while the sum of weights, in 32 bits, counts it. (A row with one strong score and 65,535 of weights
// just below 2^-25 lost 0.2 % of its mass.) With kSlack the weights stay at or below 2^15.
template <class TY> constexpr float kLift = std::is_same_v<TY, F16> ? 7.0f : 0.0f;
template <class TY> constexpr float kLiftBack = std::is_same_v<TY, F16> ? 1.0f / 128.0f : 1.0f;
template <class TY> __device__ inline float weight_of(const AttendArgs &a, float s, float less) {
    if constexpr (TY::kDepth == 16) return exp2_of(s - less);
    else if constexpr (std::is_same_v<TY, F16>) return exp2_of(s * a.c - less + kLift<TY>);   // (less - kLift would round)
    else return exp2_of(s * a.c - less);
}

// A row of out, and of what its rounding leaves: delta, a difference of what cancels, is formed of both.
template <class E> __device__ inline void store_out(const AttendArgs &a, int64_t row, int at, f4 v, bool four) {
    store_four(reinterpret_cast<E *>(a.out) + row * a.dv, at, a.dv, v, four);
    if constexpr (sizeof(E) == 2)
        if (a.out_low) {
            f4 rest;
#pragma unroll
            for (int i = 0; i < 4; ++i) rest[i] = v[i] - (float)(E)v[i];
            store_four(reinterpret_cast<E *>(a.out_low) + row * a.dv, at, a.dv, rest, four);
        }
}

// ---- forward --------------------------------------------------------------------------------------------------------
// The running maximum is raised (and the sums scaled) only when a value is more than 2^kSlack above it: the weights then
// stay below 2^kSlack, which every type holds (binary16 with kLift too), and most tiles need no exchange between lanes.
constexpr float kSlack = 8.0f;

// Bound by vector and matrix instructions together, which two waves on a SIMD overlap in part: 131,072 rows x 1024 in 4 heads of 64, bf16,
// 185 us, 743 TFLOP/s, vector instructions 83 % of the cycles and matrix ones 38 %; 16384 x 8192 in 8 heads of 128, 656 us,
// 838 TFLOP/s, 49 % and 42 %. One ray that asks a long memory is bound by reading it: 65,536 rows of 8 heads of 128, 46 us, 5.8 TB/s
// (a kernel that only reads gets 5.95 out of 4 GiB), in 64 parts a head, and 7 us to join them.
template <class TY, int NK, int QB> __global__ __launch_bounds__(kThreads) void k_attend_forward(AttendArgs a) {
    typedef Shape<TY, NK> T;
    typedef typename TY::E E;
    constexpr int NM = depth_blocks<TY, NK>();
    __shared__ alignas(16) char tile_k[T::kTile], tile_v[T::kTile];
    __shared__ alignas(16) float tile_mask[T::kRows];   // 0, or -inf of a row behind the length, which takes it out of every sum
    const int lane = threadIdx.x & 63, g = lane >> 4, wave = wave_number();
    const Turn turn = turn_of(a.cut);
    const Place p = place_of(a, turn.tile);
    const int row0 = p.tile * (kWaves * 16 * QB) + wave * 16 * QB;
    const int first = turn.split * a.cut.per_split * T::kRows;
    const int last = turn.part ? min(p.length, first + a.cut.per_split * T::kRows) : p.length;

    Stage<TY, NK> stage_k, stage_v;
    stage_k.begin(a.k, tile_base(a.k, first, p.batch, p.kv));
    stage_v.begin(a.v, tile_base(a.v, first, p.batch, p.kv));
    auto fetch = [&](int at) {
        stage_k.load(last - at);
        stage_v.load(last - at);
    };
    if (first < last) fetch(first);
    Own<TY, NK, QB> own;
    own.load(a.q, tile_base<true>(a.q, row0, p.batch, p.kv), a.rows - row0);
    carry_scale(own, a);
    float m[QB], l[QB];
    f4 out[QB][NM];
#pragma unroll
    for (int q = 0; q < QB; ++q) {
        m[q] = -kInf, l[q] = 0.0f;
#pragma unroll
        for (int i = 0; i < NM; ++i) out[q][i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    rows_are_here(own);
    for (int at = first; at < last; at += T::kRows) {
        stage_k.store(tile_k);
        stage_v.store(tile_v);
        if ((int)threadIdx.x < T::kRows) tile_mask[threadIdx.x] = at + (int)threadIdx.x < last ? 0.0f : -kInf;
        __syncthreads();
        if (at + T::kRows < last) fetch(at + T::kRows);
#pragma unroll
        for (int pair = 0; pair < T::kBlocks; pair += 2) {
            if constexpr (TY::kRounds)
                if (pair == 0) loads_between_products();
            f4 s[2][QB];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const f4 mask = *reinterpret_cast<const f4 *>(tile_mask + (pair + j) * 16 + 4 * g);
#pragma unroll
                for (int q = 0; q < QB; ++q) s[j][q] = mask;
                product<TY, NK, QB>(tile_k, pair + j, own, s[j]);
            }
            float top[QB];
            bool raise = false;
#pragma unroll
            for (int q = 0; q < QB; ++q) {
                const f4 u = s[0][q], v = s[1][q];
                top[q] = a.c * larger(largest(u), largest(v));
                raise |= top[q] > m[q] + kSlack;
            }
            if (__any(raise)) {
#pragma unroll
                for (int q = 0; q < QB; ++q) {
                    const float to = larger(m[q], max_group(top[q])), by = exp2_of(m[q] - finite_or_zero(to));
                    m[q] = to;
                    l[q] *= by;
#pragma unroll
                    for (int i = 0; i < NM; ++i) out[q][i] *= by;
                }
            }
#pragma unroll
            for (int q = 0; q < QB; ++q) {
                const float use = finite_or_zero(m[q]);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[j][q][r] = weight_of<TY>(a, s[j][q][r], use);
                const f4 u = s[0][q], v = s[1][q];
                l[q] += ((u[0] + u[1]) + (u[2] + u[3])) + ((v[0] + v[1]) + (v[2] + v[3]));
            }
            accumulate<TY, NK, QB, NM>(tile_v, pair, s[0], s[1], out);
        }
        __syncthreads();
    }
    const bool four = (a.dv & 3) == 0;
#pragma unroll
    for (int q = 0; q < QB; ++q) {
        const int row = row0 + q * 16 + (lane & 15);
        const float sum = sum_group(l[q]) * kLiftBack<TY>;
        if (row >= a.rows) continue;
        const int64_t at = stat_row(a, p, row);
        if (turn.part) {
            const int64_t part = part_row(a.cut, turn, kWaves * 16 * QB, wave * 16 * QB + q * 16 + (lane & 15));
            if (g == 0) a.part[part] = float2{m[q], sum};
            if (first < last)
#pragma unroll
                for (int i = 0; i < NM; ++i) store_four(a.out_part + part * a.dv, i * 16 + 4 * g, a.dv, out[q][i] * kLiftBack<TY>, four);
            continue;
        }
        const float by = p.length > 0 ? kLiftBack<TY> / sum : 0.0f;
        if (g == 0 && a.lse2) a.lse2[at] = p.length > 0 ? m[q] + log2_of(sum) : kInf;
        const int64_t to = out_row(a, p, row);
#pragma unroll
        for (int i = 0; i < NM; ++i) store_out<E>(a, to, i * 16 + 4 * g, out[q][i] * by, four);
    }
}

// The parts of a split forward pass, a workgroup a row: for many parts of few rows (one ray that asks a long memory), which the
// kernel below would go through one after another (8 rows of 256 parts: 5 us, 45 with that one).
template <class E> __global__ __launch_bounds__(kThreads) void k_attend_join_row(AttendArgs a, int rows_per_part, int rows_per_tile) {
    __shared__ float weight[kMostSplits], wave_top[kWaves], wave_sum[kWaves];
    __shared__ f4 sums[kThreads];
    const int tile = blockIdx.x / rows_per_tile, r = blockIdx.x % rows_per_tile, tid = threadIdx.x;
    const Place p = place_of(a, a.cut.whole + tile);
    const int row = p.tile * a.own + r, length = p.length;
    if (row >= a.rows) return;
    const int64_t from = (int64_t)tile * a.cut.splits * a.own + r;   // the row's first part; the next: own rows on
    const int64_t at = stat_row(a, p, row);
    const int used = (length + rows_per_part - 1) / rows_per_part;   // (parts behind the length left no sums)
    float top = -kInf;
    for (int s = tid; s < used; s += kThreads) top = fmaxf(top, a.part[from + (int64_t)s * a.own].x);
    for (int step = 32; step > 0; step >>= 1) top = fmaxf(top, __shfl_xor(top, step));
    if ((tid & 63) == 0) wave_top[tid >> 6] = top;
    __syncthreads();
    const float m = fmaxf(fmaxf(wave_top[0], wave_top[1]), fmaxf(wave_top[2], wave_top[3])), use = finite_or_zero(m);
    float l = 0.0f;
    for (int s = tid; s < used; s += kThreads) {
        const float2 ml = a.part[from + (int64_t)s * a.own];
        const float by = exp2_of(ml.x - use);
        weight[s] = by;
        l += ml.y * by;
    }
    for (int step = 32; step > 0; step >>= 1) l += __shfl_xor(l, step);
    if ((tid & 63) == 0) wave_sum[tid >> 6] = l;
    __syncthreads();
    l = (wave_sum[0] + wave_sum[1]) + (wave_sum[2] + wave_sum[3]);
    const int words = (a.dv + 3) / 4;   // at most 64
    int wide = 1;
    while (wide < words) wide *= 2;
    const int word = tid & (wide - 1), lane = tid / wide, lanes = kThreads / wide;
    const bool four = (a.dv & 3) == 0;
    f4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    if (word < words) {
#pragma unroll 4
        for (int s = lane; s < used; s += lanes) {
            const float *part = a.out_part + (from + (int64_t)s * a.own) * a.dv + 4 * word;
            if (four) {
                o += *reinterpret_cast<const f4 *>(part) * weight[s];
            } else {
                for (int i = 0; i < 4; ++i)
                    if (4 * word + i < a.dv) o[i] += part[i] * weight[s];
            }
        }
    }
    sums[tid] = o;
    for (int step = lanes / 2; step > 0; step >>= 1) {
        __syncthreads();
        if (lane < step) sums[tid] += sums[tid + step * wide];
    }
    if (tid == 0 && a.lse2) a.lse2[at] = length > 0 ? m + log2_of(l) : kInf;
    if (lane == 0 && word < words)
        store_out<E>(a, out_row(a, p, row), 4 * word, length > 0 ? sums[tid] * (1.0f / l) : sums[tid], four);
}

// The same, a thread for four channels of a row.
template <class E> __global__ __launch_bounds__(kThreads) void k_attend_join(AttendArgs a, int rows_per_part) {
    const int words = (a.dv + 3) / 4;
    const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x, i = id / words;
    const int c = (int)(id - i * words) * 4, tile = (int)(i / a.own);
    if (i >= a.cut.parted() * a.own) return;
    const Place p = place_of(a, a.cut.whole + tile);
    const int row = p.tile * a.own + (int)(i % a.own), length = p.length;
    if (row >= a.rows) return;
    const int64_t first = (int64_t)tile * a.cut.splits * a.own + i % a.own, at = stat_row(a, p, row);
    const int used = (length + rows_per_part - 1) / rows_per_part;   // (parts behind the length left no sums)
    float m = -kInf;
    for (int s = 0; s < used; ++s) m = fmaxf(m, a.part[first + (int64_t)s * a.own].x);
    const float use = finite_or_zero(m);
    const bool four = (a.dv & 3) == 0;
    float l = 0.0f;
    f4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = 0; s < used; ++s) {
        const int64_t part = first + (int64_t)s * a.own;
        const float2 ml = a.part[part];
        const float by = exp2_of(ml.x - use);
        l += ml.y * by;
        const float *from = a.out_part + part * a.dv + c;
        if (four) {
            o += *reinterpret_cast<const f4 *>(from) * by;
        } else {
            for (int i = 0; i < 4; ++i)
                if (c + i < a.dv) o[i] += from[i] * by;
        }
    }
    if (c == 0 && a.lse2) a.lse2[at] = length > 0 ? m + log2_of(l) : kInf;
    store_out<E>(a, out_row(a, p, row), c, length > 0 ? o * (1.0f / l) : o, four);
}

// ---- backward -------------------------------------------------------------------------------------------------------
// delta of the wave's rows, from fragments: by the matrix instruction that also forms do . v, so that where a row's weight is
// on one value alone (o = v) the two are the same number and its ds is 0, not a rounding error.
template <class TY, int NK, int QB>
__device__ inline void deltas(const Own<TY, NK, QB> &o, const Own<TY, NK, QB> &low, const Own<TY, NK, QB> &up, float (&delta)[QB]) {
    const int lane = threadIdx.x & 63, g = lane >> 4, l = lane & 15;
#pragma unroll
    for (int q = 0; q < QB; ++q) {
        f4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < fragments<NK>(); ++k) s = fragment_product<TY, NK>(o.f[q][k], up.f[q][k], s);
        if constexpr (TY::kRounds)
#pragma unroll
            for (int k = 0; k < fragments<NK>(); ++k) s = fragment_product<TY, NK>(low.f[q][k], up.f[q][k], s);
        const float mine = (l & 2) ? ((l & 1) ? s[3] : s[2]) : ((l & 1) ? s[1] : s[0]);
        delta[q] = sum_group(g == (l >> 2) ? mine : 0.0f);   // (the diagonal's one value)
    }
}

// dq, and delta for the other kernel: queries as own rows, the memory streamed. 16384 x 8192 in 8 heads of 128, bf16: 842 us,
// 979 TFLOP/s, matrix instructions 49 % of the cycles.
template <class TY, int NK, int QB> __global__ __launch_bounds__(kThreads) void k_attend_dq(AttendArgs a) {
    typedef Shape<TY, NK> T;
    typedef typename TY::E E;
    constexpr int NM = depth_blocks<TY, NK>();
    __shared__ alignas(16) char tile_k[T::kTile], tile_v[T::kTile];
    __shared__ alignas(16) float tile_mask[T::kRows];   // 0, or -inf of a row behind the length, which takes it out of every sum
    const int lane = threadIdx.x & 63, g = lane >> 4, wave = wave_number();
    const Turn turn = turn_of(a.cut);
    const Place p = place_of(a, turn.tile);
    const int row0 = p.tile * (kWaves * 16 * QB) + wave * 16 * QB;
    const int first = turn.split * a.cut.per_split * T::kRows;
    const int last = !a.dq ? 0 : turn.part ? min(p.length, first + a.cut.per_split * T::kRows) : p.length;

    Stage<TY, NK> stage_k, stage_v;
    stage_k.begin(a.k, tile_base(a.k, first, p.batch, p.kv));
    stage_v.begin(a.v, tile_base(a.v, first, p.batch, p.kv));
    auto fetch = [&](int at) {
        stage_k.load(last - at);
        stage_v.load(last - at);
    };
    if (first < last) fetch(first);
    Own<TY, NK, QB> own, up;
    float delta[QB], lse2[QB];
    up.load(a.up, tile_base<true>(a.up, row0, p.batch, p.kv), a.rows - row0);
    own.load(a.o, tile_base<true>(a.o, row0, p.batch, p.kv), a.rows - row0);
    {
        Own<TY, NK, QB> low;
        if constexpr (TY::kRounds) low.load(a.low, tile_base<true>(a.low, row0, p.batch, p.kv), a.rows - row0);
        deltas<TY, NK, QB>(own, low, up, delta);
    }
    own.load(a.q, tile_base<true>(a.q, row0, p.batch, p.kv), a.rows - row0);
    carry_scale(own, a);
    f4 out[QB][NM];
#pragma unroll
    for (int q = 0; q < QB; ++q) {
        const int row = row0 + q * 16 + (lane & 15);
        lse2[q] = row < a.rows ? a.lse2[stat_row(a, p, row)] : kInf;
        if (row < a.rows && g == 0 && turn.split == 0) a.delta[stat_row(a, p, row)] = delta[q];
#pragma unroll
        for (int i = 0; i < NM; ++i) out[q][i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    rows_are_here(own), rows_are_here(up);
    for (int at = first; at < last; at += T::kRows) {
        stage_k.store(tile_k);
        stage_v.store(tile_v);
        if ((int)threadIdx.x < T::kRows) tile_mask[threadIdx.x] = at + (int)threadIdx.x < last ? 0.0f : -kInf;
        __syncthreads();
        if (at + T::kRows < last) fetch(at + T::kRows);
#pragma unroll
        for (int pair = 0; pair < T::kBlocks; pair += 2) {
            f4 s[2][QB];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                f4 dp[QB];
                const f4 mask = *reinterpret_cast<const f4 *>(tile_mask + (pair + j) * 16 + 4 * g);
#pragma unroll
                for (int q = 0; q < QB; ++q) s[j][q] = mask, dp[q] = f4{0.0f, 0.0f, 0.0f, 0.0f};
                product<TY, NK, QB>(tile_k, pair + j, own, s[j]);
                product<TY, NK, QB>(tile_v, pair + j, up, dp);
#pragma unroll
                for (int q = 0; q < QB; ++q)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        s[j][q][r] = weight_of<TY>(a, s[j][q][r], lse2[q]) * (dp[q][r] - delta[q]);
            }
            accumulate<TY, NK, QB, NM>(tile_k, pair, s[0], s[1], out);
        }
        __syncthreads();
    }
    if (!a.dq) return;
    const bool four = (a.d & 3) == 0;
#pragma unroll
    for (int q = 0; q < QB; ++q) {
        const int row = row0 + q * 16 + (lane & 15);
        if (row >= a.rows) continue;
        const int64_t to = out_row(a, p, row);
#pragma unroll
        for (int i = 0; i < NM; ++i) {
            const f4 v = out[q][i] * a.scale;
            if (turn.part) store_four(a.out_part + part_row(a.cut, turn, kWaves * 16 * QB, wave * 16 * QB + q * 16 + (lane & 15)) * a.d, i * 16 + 4 * g, a.d, v, four);
            else store_sums<E>(a.dq, to, i * 16 + 4 * g, a.d, v, four, a.half);
        }
    }
}

// dk and dv: the memory's rows as own rows, the queries streamed. Four products of a tile with one own block a wave (two would leave one
// wave on a SIMD): 16384 x 8192 in 8 heads of 128, bf16: 1271 us, 865 TFLOP/s, LDS reads 59 % of the cycles.
template <class TY, int NK, int QB> __global__ __launch_bounds__(kThreads) void k_attend_dkv(AttendArgs a) {
    typedef Shape<TY, NK> T;
    typedef typename TY::E E;
    constexpr int NM = depth_blocks<TY, NK>();
    __shared__ alignas(16) char tile_q[T::kTile], tile_o[T::kTile];
    __shared__ alignas(16) float tile_lse2[T::kRows], tile_delta[T::kRows];
    const int lane = threadIdx.x & 63, g = lane >> 4, wave = wave_number();
    const Turn turn = turn_of(a.cut);
    const Place p = place_of(a, turn.tile);
    const int tile0 = p.tile * (kWaves * 16 * QB), row0 = tile0 + wave * 16 * QB;
    const int first = turn.split * a.cut.per_split * T::kRows;
    const int last = tile0 >= p.length ? 0 : turn.part ? min(a.rows, first + a.cut.per_split * T::kRows) : a.rows;

    Stage<TY, NK> stage_q, stage_o;
    stage_q.begin(a.q, tile_base<true>(a.q, first, p.batch, p.kv));
    stage_o.begin(a.up, tile_base<true>(a.up, first, p.batch, p.kv));
    float stage_lse2 = kInf, stage_delta = 0.0f;
    auto fetch = [&](int at) {
        stage_q.load(last - at);
        stage_o.load(last - at);
        if ((int)threadIdx.x < T::kRows) {
            const int row = at + threadIdx.x;
            stage_lse2 = row < last ? a.lse2[stat_row(a, p, row)] : kInf;
            stage_delta = row < last ? a.delta[stat_row(a, p, row)] : 0.0f;
        }
    };
    if (first < last) fetch(first);
    Own<TY, NK, QB> own_k, own_v;
    const int own_rows = first < last ? p.length - row0 : 0;   // (without queries the memory need not be there)
    own_k.load(a.k, tile_base(a.k, row0, p.batch, p.kv), own_rows);
    own_v.load(a.v, tile_base(a.v, row0, p.batch, p.kv), own_rows);
    carry_scale(own_k, a);
    f4 dk[QB][NM], dv[QB][NM];
#pragma unroll
    for (int q = 0; q < QB; ++q)
#pragma unroll
        for (int i = 0; i < NM; ++i) dk[q][i] = dv[q][i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    rows_are_here(own_k), rows_are_here(own_v);
    for (int at = first; at < last; at += T::kRows) {
        stage_q.store(tile_q);
        stage_o.store(tile_o);
        if ((int)threadIdx.x < T::kRows) tile_lse2[threadIdx.x] = stage_lse2, tile_delta[threadIdx.x] = stage_delta;
        __syncthreads();
        if (at + T::kRows < last) fetch(at + T::kRows);
#pragma unroll
        for (int pair = 0; pair < T::kBlocks; pair += 2) {
            f4 s[2][QB], dp[2][QB];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int q = 0; q < QB; ++q) s[j][q] = dp[j][q] = f4{0.0f, 0.0f, 0.0f, 0.0f};
                product<TY, NK, QB, true>(tile_q, pair + j, own_k, s[j]);
                product<TY, NK, QB, true>(tile_o, pair + j, own_v, dp[j]);
                const int at4 = (pair + j) * 16 + 4 * g;
                const f4 lse2 = *reinterpret_cast<const f4 *>(tile_lse2 + at4), delta = *reinterpret_cast<const f4 *>(tile_delta + at4);
#pragma unroll
                for (int q = 0; q < QB; ++q)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float e = weight_of<TY>(a, s[j][q][r], lse2[r]);
                        s[j][q][r] = e;
                        dp[j][q][r] = e * (dp[j][q][r] - delta[r]);
                    }
            }
            accumulate<TY, NK, QB, NM>(tile_o, pair, s[0], s[1], dv);
            accumulate<TY, NK, QB, NM>(tile_q, pair, dp[0], dp[1], dk);
        }
        __syncthreads();
    }
    const bool four_k = (a.d & 3) == 0, four_v = (a.dv & 3) == 0;
    const f4 none = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int q = 0; q < QB; ++q) {
        const int row = row0 + q * 16 + (lane & 15);
        if (row >= a.memory) continue;
        const int64_t to = ((int64_t)p.batch * a.memory + row) * a.kv_heads + p.kv;
        const bool there = row < p.length;   // (a row behind the length has products of zeros with anything)
        const int64_t part = part_row(a.cut, turn, kWaves * 16 * QB, wave * 16 * QB + q * 16 + (lane & 15));
#pragma unroll
        for (int i = 0; i < NM; ++i) {
            const f4 k = there ? dk[q][i] * a.scale : none, v = there ? dv[q][i] : none;
            if (turn.part) {
                store_four(a.out_part + part * a.d, i * 16 + 4 * g, a.d, k, four_k);
                store_four(a.out_part2 + part * a.dv, i * 16 + 4 * g, a.dv, v, four_v);
            } else {
                if (a.dk) store_sums<E>(a.dk, to, i * 16 + 4 * g, a.d, k, four_k, a.half);
                if (a.dvalue) store_sums<E>(a.dvalue, to, i * 16 + 4 * g, a.dv, v, four_v, a.half);
            }
        }
    }
}

}  // namespace

// ---- host -----------------------------------------------------------------------------------------------------------
namespace {

int check(const DstAttendParams *p) {
    if (!p) return dst_op_fail(DST_E_INVALID, "params is null");
    if (p->dtype != DST_DTYPE_F32 && p->dtype != DST_DTYPE_BF16 && p->dtype != DST_DTYPE_F16)
        return dst_op_fail(DST_E_UNSUPPORTED, "dtype must be float32, bfloat16 or float16");
    if (p->batch < 0 || p->queries < 0 || p->memory < 0) return dst_op_fail(DST_E_INVALID, "negative size");
    if (p->heads < 1 || p->kv_heads < 1 || p->heads % p->kv_heads != 0)
        return dst_op_fail(DST_E_INVALID, "heads must be a multiple of kv_heads");
    if (p->channels < 1 || p->channels > DST_MAX_CHANNELS || p->value_channels < 1 || p->value_channels > DST_MAX_CHANNELS)
        return dst_op_fail(DST_E_UNSUPPORTED, "channels must be in 1..%d", DST_MAX_CHANNELS);
    if (!(p->scale == p->scale) || p->scale - p->scale != 0.0f) return dst_op_fail(DST_E_INVALID, "scale must be finite");
    const int64_t rows = (int64_t)p->queries * (p->heads / p->kv_heads), most = 0x3fffffff;
    if (rows > most || p->memory > most || (int64_t)p->batch * p->kv_heads > most ||
        (int64_t)p->batch * p->kv_heads * (div_up(rows, 16) > div_up(p->memory, 16) ? div_up(rows, 16) : div_up(p->memory, 16)) > most)
        return dst_op_fail(DST_E_UNSUPPORTED, "too many rows");
    for (const int64_t *strides : {p->q_strides, p->k_strides, p->v_strides})
        for (int i = 0; i < 3; ++i)
            if (strides[i] < 0 || strides[i] > kLongestStride) return dst_op_fail(DST_E_INVALID, "strides must be in 0..2^44");
    const bool any = p->batch > 0 && p->queries > 0;
    if (any && (!p->q || !p->out || (p->memory > 0 && (!p->k || !p->v)))) return dst_op_fail(DST_E_INVALID, "q, k, v and out are required");
    return DST_OK;
}

int longest(const DstAttendParams *p) { return p->channels > p->value_channels ? p->channels : p->value_channels; }

template <class TY> AttendArgs arguments(const DstAttendParams *p) {
    AttendArgs a = {};
    a.lengths = p->lengths;
    a.queries = p->queries, a.memory = p->memory, a.heads = p->heads, a.kv_heads = p->kv_heads;
    a.group = p->heads / p->kv_heads, a.rows = p->queries * a.group;
    a.d = p->channels, a.dv = p->value_channels;
    a.scale = p->scale, a.flip = p->scale < 0.0f;
    // (a scale of 0 stands for all scores equal: the smallest normal number says that of any score that is finite, and leaves
    // -inf what it is)
    a.c = __builtin_fabsf(p->scale) * kLog2E;
    if (a.c < 1.1754944e-38f) a.c = 1.1754944e-38f;
    if (std::is_same_v<TY, F32>) a.own_scale = a.flip ? -a.c : a.c, a.c = 1.0f;
    a.out = p->out, a.out_low = p->out_low, a.lse2 = p->lse;
    a.half = p->dtype == DST_DTYPE_F16 && sizeof(typename TY::E) == 4;
    a.all_rows = (int64_t)p->batch * p->kv_heads * a.rows;
    return a;
}

// f(type, integral constant of the fragments) for the call's type and channels
template <class F> int with_type(const DstAttendParams *p, F f) {
    const int nk = fragments_of(longest(p), p->dtype);
    if (p->dtype == DST_DTYPE_F32) return with_floats<false>(longest(p), f);
    return p->dtype == DST_DTYPE_BF16 ? with_fragments<BF16>(nk, f) : with_fragments<F16>(nk, f);
}
// Gradients of binary16 rows are formed in 32 bits.
template <class F> int with_gradients(const DstAttendParams *p, F f) {
    return p->dtype == DST_DTYPE_BF16 ? with_fragments<BF16>(fragments_of(longest(p), p->dtype), f) : with_floats<false>(longest(p), f);
}

// The rows of all sets, copied into the workspace's front where the kernels cannot read them where they lie.
struct Sets {
    RowSet q, k, v, o, low, up;
};
template <class TY, int NK> Sets row_sets(const DstAttendParams *p, AttendArgs &a, bool backward, Carve &c) {
    // (a group has to fit whole into the steps between a thread's words, and into the blocks of 16 own rows)
    const int stride = Shape<TY, NK>::kStride < 16 ? Shape<TY, NK>::kStride : 16, group = a.group;
    auto memory = [&](const void *t, const int64_t (&s)[3], int channels) {
        return row_set<TY>(t, p->dtype, s[0], s[1], s[2], p->batch, p->kv_heads, 1, p->memory, channels, stride, c);
    };
    auto queries = [&](const void *t, int64_t batch, int64_t row, int64_t head, int channels, const void *low = nullptr) {
        return row_set<TY>(t, p->dtype, batch, row, head, p->batch, p->kv_heads, group, a.rows, channels, stride, c, low);
    };
    const int64_t row = (int64_t)p->heads * p->value_channels;
    Sets s = {};
    s.q = queries(p->q, p->q_strides[0], p->q_strides[1], p->q_strides[2], p->channels);
    s.k = memory(p->k, p->k_strides, p->channels);
    s.v = memory(p->v, p->v_strides, p->value_channels);
    if (backward) {
        s.o = queries(p->out, p->queries * row, row, p->value_channels, p->value_channels, p->out_low);
        if (TY::kRounds) s.low = queries(p->out_low, p->queries * row, row, p->value_channels, p->value_channels);
        s.up = queries(p->upstream, p->queries * row, row, p->value_channels, p->value_channels);
    }
    a.q = s.q.rows, a.k = s.k.rows, a.v = s.v.rows, a.o = s.o.rows, a.low = s.low.rows, a.up = s.up.rows;
    return s;
}
void prepare(const Sets &s, hipStream_t stream) { prepare({&s.q, &s.k, &s.v, &s.o, &s.low, &s.up}, stream); }
int64_t copy_blocks(const Sets &s) { return copy_blocks({&s.q, &s.k, &s.v, &s.o, &s.low, &s.up}); }

// DST_OK, or the refusal of rows that need more workgroups than a launch holds.
int check_blocks(const Sets &s, const Cut &cut) {
    return cut.blocks() <= kMostBlocks && copy_blocks(s) <= kMostBlocks ? (int)DST_OK : dst_op_fail(DST_E_UNSUPPORTED, "too many rows");
}

// Cuts a pass's own tiles; whether its rows are few. `kernel(few)`: the pass's kernel; `own_bytes`: of a part's row.
template <class TY, int NK, class K>
bool plan_cut(AttendArgs &a, int most, int64_t own_rows, int64_t streamed_rows, int64_t heads, int products, double row_bytes, K kernel) {
    constexpr int tile = Shape<TY, NK>::kRows;
    const int64_t streamed = div_up(streamed_rows, tile);
    const bool few = own_rows <= kWaves * 16 || few_rows(div_up(own_rows, kWaves * 16 * most) * heads, streamed);
    a.own = kWaves * 16 * (few ? 1 : most);
    a.tiles = (int)div_up(own_rows, a.own);
    a.cut = cut_tiles(a.tiles * heads, streamed, slots_of(kernel(few)), tile_time<TY, NK>(a.own, products),
                      a.own * row_bytes, a.lengths != nullptr);
    return few;
}
uint64_t parted_rows(const AttendArgs &a) { return a.cut.splits > 1 ? (uint64_t)a.cut.parted() * a.own * a.cut.splits : 0; }

struct Plan {
    bool few;
    uint64_t bytes;
};
template <class TY, int NK> Plan plan_forward(AttendArgs &a, int64_t heads, Carve c) {
    Plan p;
    p.few = plan_cut<TY, NK>(a, forward_blocks<TY, NK>(), a.rows, a.memory, heads, 2, a.dv * 4.0 + 8.0, [](bool few) {
        return few ? (const void *)&k_attend_forward<TY, NK, 1> : (const void *)&k_attend_forward<TY, NK, forward_blocks<TY, NK>()>;
    });
    if (const uint64_t rows = parted_rows(a)) {
        a.part = c.take<float2>(rows);
        a.out_part = c.take<float>(rows * a.dv);
    }
    p.bytes = c.used;
    return p;
}
template <class TY, int NK> Plan plan_dq(AttendArgs &a, int64_t heads, Carve c) {
    Plan p;
    p.few = plan_cut<TY, NK>(a, dq_blocks<TY, NK>(), a.rows, a.dq ? a.memory : 0, heads, 3, a.d * 4.0, [](bool few) {
        return few ? (const void *)&k_attend_dq<TY, NK, 1> : (const void *)&k_attend_dq<TY, NK, dq_blocks<TY, NK>()>;
    });
    a.delta = c.take<float>(a.all_rows);
    if (const uint64_t rows = parted_rows(a)) a.out_part = c.take<float>(rows * a.d);
    p.bytes = c.used;
    return p;
}
template <class TY, int NK> Plan plan_dkv(AttendArgs &a, int64_t heads, Carve c) {
    Plan p;
    p.few = plan_cut<TY, NK>(a, dkv_blocks<TY, NK>(), a.memory, a.rows, heads, 4, (a.d + a.dv) * 4.0, [](bool few) {
        return few ? (const void *)&k_attend_dkv<TY, NK, 1> : (const void *)&k_attend_dkv<TY, NK, dkv_blocks<TY, NK>()>;
    });
    a.delta = c.take<float>(a.all_rows);
    if (const uint64_t rows = parted_rows(a)) {
        a.out_part = c.take<float>(rows * a.d);
        a.out_part2 = c.take<float>(rows * a.dv);
    }
    p.bytes = c.used;
    return p;
}

// The output row of a parted row: of dq, of dk and dv
struct QueryRow {
    int whole, tiles, own, rows, kv_heads, group, queries;
    __device__ int64_t operator()(int tile, int row) const {
        const int t = whole + tile, r = t % tiles * own + row, head = t / tiles % kv_heads, batch = t / tiles / kv_heads;
        if (r >= rows) return -1;
        return ((int64_t)batch * queries + r / group) * (kv_heads * group) + head * group + r % group;
    }
};
struct MemoryRow {
    int whole, tiles, own, memory, kv_heads;
    __device__ int64_t operator()(int tile, int row) const {
        const int t = whole + tile, r = t % tiles * own + row, head = t / tiles % kv_heads, batch = t / tiles / kv_heads;
        return r < memory ? ((int64_t)batch * memory + r) * kv_heads + head : -1;
    }
};

int check_workspace(const DstAttendParams *p, uint64_t need) {
    if (need == 0) return DST_OK;
    if (!p->workspace || p->workspace_bytes < need)
        return dst_op_fail(DST_E_INVALID, "workspace of %llu bytes is needed", (unsigned long long)need);
    if (reinterpret_cast<uintptr_t>(p->workspace) & 255u) return dst_op_fail(DST_E_INVALID, "workspace must be aligned to 256 bytes");
    return DST_OK;
}

}  // namespace

extern "C" {

uint64_t dst_attend_workspace_bytes(const DstAttendParams *p, int pass) {
    if (check(p) != DST_OK) return 0;
    uint64_t bytes = 0;
    const int64_t heads = (int64_t)p->batch * p->kv_heads;
    if (pass == DST_PASS_FORWARD) {
        with_type(p, [&](auto ty, auto nk) {
            typedef decltype(ty) TY;
            constexpr int NK = decltype(nk)::value;
            AttendArgs a = arguments<TY>(p);
            if (a.all_rows == 0) return (int)DST_OK;
            Carve c = {nullptr, 0};
            const Sets sets = row_sets<TY, NK>(p, a, false, c);
            const uint64_t need = plan_forward<TY, NK>(a, heads, c).bytes;
            if (int rc = check_blocks(sets, a.cut)) return rc;
            bytes = need;
            return (int)DST_OK;
        });
    } else {
        with_gradients(p, [&](auto ty, auto nk) {
            typedef decltype(ty) TY;
            constexpr int NK = decltype(nk)::value;
            AttendArgs a = arguments<TY>(p);
            Carve c = {nullptr, 0};
            const Sets sets = row_sets<TY, NK>(p, a, true, c);
            a.dq = p->grad_q;
            uint64_t need = plan_dq<TY, NK>(a, heads, c).bytes;
            if (int rc = check_blocks(sets, a.cut)) return rc;
            if (p->grad_k || p->grad_v) {
                const uint64_t more = plan_dkv<TY, NK>(a, heads, c).bytes;
                if (int rc = check_blocks(sets, a.cut)) return rc;
                need = more > need ? more : need;
            }
            bytes = need;
            return (int)DST_OK;
        });
    }
    return bytes;
}

int dst_attend_forward(const DstAttendParams *p, void *stream) {
    if (int rc = check(p)) return rc;
    return with_type(p, [&](auto ty, auto nk) {
        typedef decltype(ty) TY;
        typedef typename TY::E E;
        constexpr int NK = decltype(nk)::value, QB = forward_blocks<TY, NK>();
        AttendArgs a = arguments<TY>(p);
        if (a.all_rows == 0) return (int)DST_OK;
        const int64_t heads = (int64_t)p->batch * p->kv_heads;
        Carve c = {(char *)p->workspace, 0};
        const Sets sets = row_sets<TY, NK>(p, a, false, c);
        const Plan plan = plan_forward<TY, NK>(a, heads, c);
        if (int rc = check_blocks(sets, a.cut)) return rc;
        if (int rc = check_workspace(p, plan.bytes)) return rc;
        const hipStream_t s = (hipStream_t)stream;
        prepare(sets, s);
        const dim3 grid((uint32_t)a.cut.blocks());
        if (plan.few) k_attend_forward<TY, NK, 1><<<grid, kThreads, 0, s>>>(a);
        else k_attend_forward<TY, NK, QB><<<grid, kThreads, 0, s>>>(a);
        DST_OP_LAUNCH("attention");
        if (a.cut.splits > 1) {
            const int64_t rows = a.cut.parted() * a.own;
            const int part = a.cut.per_split * Shape<TY, NK>::kRows;
            const int some = a.own < a.rows ? a.own : a.rows;   // rows of a tile that are there
            if (a.cut.splits >= 16) k_attend_join_row<E><<<dim3((uint32_t)(a.cut.parted() * some)), kThreads, 0, s>>>(a, part, some);
            else k_attend_join<E><<<dim3((uint32_t)div_up(rows * ((a.dv + 3) / 4), kThreads)), kThreads, 0, s>>>(a, part);
            DST_OP_LAUNCH("attention, joining");
        }
        return (int)DST_OK;
    });
}

int dst_attend_backward(const DstAttendParams *p, void *stream) {
    if (int rc = check(p)) return rc;
    if (!p->grad_q && !p->grad_k && !p->grad_v) return DST_OK;
    if (p->batch > 0 && p->queries > 0 && (!p->lse || !p->upstream)) return dst_op_fail(DST_E_INVALID, "lse and upstream are required");
    if (p->batch > 0 && p->queries > 0 && p->dtype != DST_DTYPE_F32 && !p->out_low)
        return dst_op_fail(DST_E_INVALID, "out_low is required of 16-bit rows");
    if ((reinterpret_cast<uintptr_t>(p->grad_q) | reinterpret_cast<uintptr_t>(p->grad_k) | reinterpret_cast<uintptr_t>(p->grad_v)) & 15u)
        return dst_op_fail(DST_E_INVALID, "gradients must be aligned to 16 bytes");
    return with_gradients(p, [&](auto ty, auto nk) {
        typedef decltype(ty) TY;
        typedef typename TY::E E;
        constexpr int NK = decltype(nk)::value;
        const hipStream_t s = (hipStream_t)stream;
        const int64_t heads = (int64_t)p->batch * p->kv_heads;
        AttendArgs a = arguments<TY>(p);
        Carve c = {(char *)p->workspace, 0};
        const Sets sets = row_sets<TY, NK>(p, a, true, c);
        a.dq = p->grad_q, a.dk = p->grad_k, a.dvalue = p->grad_v;
        // (both passes are looked at before either runs)
        const bool queries = a.all_rows > 0, memory = (a.dk || a.dvalue) && heads * a.memory > 0;
        AttendArgs m = a;
        Plan plan = {}, plan_m = {};
        if (queries) {
            plan = plan_dq<TY, NK>(a, heads, c);
            if (int rc = check_blocks(sets, a.cut)) return rc;
        }
        if (memory) {
            plan_m = plan_dkv<TY, NK>(m, heads, c);
            if (int rc = check_blocks(sets, m.cut)) return rc;
        }
        if (int rc = check_workspace(p, plan.bytes > plan_m.bytes ? plan.bytes : plan_m.bytes)) return rc;
        if (queries) {
            prepare(sets, s);
            const dim3 grid((uint32_t)a.cut.blocks());
            if (plan.few) k_attend_dq<TY, NK, 1><<<grid, kThreads, 0, s>>>(a);
            else k_attend_dq<TY, NK, dq_blocks<TY, NK>()><<<grid, kThreads, 0, s>>>(a);
            DST_OP_LAUNCH("attention gradient, queries");
            const QueryRow to = {a.cut.whole, a.tiles, a.own, a.rows, a.kv_heads, a.group, a.queries};
            with_output<E>(a.half, [&](auto one) {
                typedef decltype(one) To;
                sum_parts(Parts<To>{a.out_part, (To *)a.dq, a.d}, Parts<To>{nullptr, nullptr, 1}, a.cut, a.own, to, s);
            });
            DST_OP_LAUNCH("attention gradient, summing");
        }
        if (memory) {
            const dim3 grid((uint32_t)m.cut.blocks());
            if (plan_m.few) k_attend_dkv<TY, NK, 1><<<grid, kThreads, 0, s>>>(m);
            else k_attend_dkv<TY, NK, dkv_blocks<TY, NK>()><<<grid, kThreads, 0, s>>>(m);
            DST_OP_LAUNCH("attention gradient, memory");
            const MemoryRow to = {m.cut.whole, m.tiles, m.own, m.memory, m.kv_heads};
            with_output<E>(m.half, [&](auto one) {
                typedef decltype(one) To;
                sum_parts(Parts<To>{m.out_part, (To *)m.dk, m.d}, Parts<To>{m.out_part2, (To *)m.dvalue, m.dv}, m.cut, m.own, to, s);
            });
            DST_OP_LAUNCH("attention gradient, summing");
        }
        return (int)DST_OK;
    });
}

}  // extern "C"
