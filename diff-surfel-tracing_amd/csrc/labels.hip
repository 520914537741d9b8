// Labels of rays: softmax cross entropy of a ray's channels against a table of labels, its gradients, and the best label.
//
//     s_rv = x_r . w_v + b_v,   lse_r = log sum_v exp s_rv,   loss_r = lse_r - s_{r,t_r}
//     ds_rv = g_r (exp(s_rv - lse_r) - [v = t_r]),   dx = ds w,   dw = ds^T x,   db = sum_r ds
//
// The (rays, labels) matrix is never stored: the forward kernel goes over the table in tiles and keeps a running maximum
// and sum for every ray; each of the two backward kernels forms the tiles again from the saved lse, one with the rays
// as own rows (dx), one with the labels (dw, db). The weight of the label itself, less one, is not formed again: near a weight of 1 it
// would be a difference of two rounded logits. The forward kernel leaves it, formed of the loss. Every sum has one owner and one order: no atomics, the same bits every
// time. Own tiles that do not fill the device's last round, or are too few to fill it at all, are cut into parts of the streamed
// rows, which a closing kernel adds.
#include <type_traits>

#include "operators.h"

namespace {

// ---- launch parameters as the kernels take them -------------------------------------------------------------------
struct LabelArgs {
    Rows x, w;
    const float *bias;              // (labels) or nullptr
    const int64_t *target;          // (rays)
    int64_t rays, ignore;
    int32_t d, labels;
    Cut cut;
    int32_t own;                    // own rows of a workgroup
    // forward
    float2 *part;                   // of a part's rays: maximum and sum
    float *target_logit;            // of the parted rays
    float *lse2;                    // (rays): log2 of the sum of exponentials; +inf where the ray is ignored
    float *top, *log_sum, *hit;     // (rays): largest logit, log2 of the sum relative to it (+inf where the ray is ignored), the weight of the
                                    // ray's label less one; forward: or nullptr
    float *rows;                    // (rays) losses, or nullptr
    double *sums;                   // (blocks): sums of losses ...
    uint32_t *counts;               // ... and rays counted in them
    // the best label
    const float *bounds;            // (kBoundBlocks, 3): largest row norm of the table, |bias| and bias
    float margin;                   // what a logit may be off by, of the norms and the |bias|
    int4 *best;                     // of a part's rays: bits of the best logit, its label, bits of the second best, -
    int64_t *label;                 // (rays)
    float *log_prob;                // (rays)
    uint32_t *near_count;           // rays whose two best labels 32 bits cannot tell apart ...
    uint32_t *near_list;            // ... which ...
    float *near_floor;              // ... and what a label's logit has to come to to be the best
    // backward
    const float *upstream;          // (rays) or one value
    const float *inverse;           // one value that multiplies a single upstream value, or nullptr
    int32_t upstream_rows;
    int32_t half;                   // gradients are written in binary16 though rows are in 32 bits
    void *out;                      // (rays, d) or (labels, d), of the inputs' type
    float *out_part;                // of a part's rows: d values
    float *bias_out, *bias_part;    // (labels); of a part's rows
};

constexpr int kBoundBlocks = 64;

// Own blocks of 16 rows of a wave. More of them read a streamed tile fewer times from LDS, fewer leave registers for a second wave
// on a SIMD, which counts for more (32768 rays x 32771 labels, 256 channels, bf16: dx with 2 blocks and one wave 1661 us, with
// 1 and two 1237, with 2 and two, which its registers just hold, 1042).
template <class TY, int NK> constexpr int forward_blocks() { return NK <= 1 ? 4 : NK * TY::kPlanes <= 12 ? 2 : 1; }
template <class TY, int NK> constexpr int dx_blocks() { return NK <= 1 ? (TY::kDepth == 32 ? 2 : 4) : NK * TY::kPlanes <= 8 ? 2 : 1; }
template <class TY, int NK> constexpr int dw_blocks() { return NK <= 1 ? (TY::kDepth == 32 ? 2 : 4) : NK * TY::kPlanes <= 6 ? 2 : 1; }

// Whether a block's products go before the other waves' instructions, in the forward kernels and in that of dx (32768 rays x 32771 labels of 256
// channels in 16 bits: forward 692 us, 573 with it, dx 1094 and 1057; best label of 65,536 rays among 4096, eight channels in 32 bits:
// 137 us and 128). Short rows of 16 bits, planes, dw and the attention gain nothing by it, or lose.
template <class TY, int NK> constexpr bool goes_first() { return TY::kPlanes == 1 && (!TY::kRounds || NK >= 4); }

// The one value that the rays share
__device__ inline float upstream_value(const LabelArgs &a) { return a.upstream[0] * a.inverse[0]; }
// The upstream gradient of a ray's loss: 0 where it is ignored, NaN where its label is none.
__device__ inline float upstream_of(const LabelArgs &a, int64_t row, int64_t t) {
    if (t == a.ignore) return 0.0f;
    if (t < 0 || t >= a.labels) return __builtin_nanf("");
    return a.upstream_rows ? a.upstream[row] : upstream_value(a);
}

// ---- forward --------------------------------------------------------------------------------------------------------
// What a logit lies below the logarithm of the sum. The sum is 1 or more and relative to the maximum, and the logit is taken relative to the maximum
// too, so of what both have in common nothing is rounded: a label with almost all of the weight keeps the digits of what it
// lacks. (A term near 1 is taken as the sum has it, rounded: a label alone lacks nothing.)
__device__ inline float below_sum(Running r, float logit) {
    const float at = logit - r.m, log_sum = log2_of(r.l);
    return at > -1.0f ? larger(log_sum - log2_of(exp_of(at)), 0.0f) * kLn2 : log_sum * kLn2 - at;
}
// Whether there is a logit above -inf and none is +inf.
__device__ inline bool has_sum(Running r) { return r.l > 0.0f; }
// The logit of each own row's own label, by the instructions that formed it among the others: the same bits.
template <class TY, int NK> __device__ inline float logit_of(const Fragment<TY> (&own)[fragments<NK>()], const char *label_row, int words, float bias) {
    const int lane = threadIdx.x & 63, g = lane >> 4, l = lane & 15;
    f4 s = {bias, bias, bias, bias};
#pragma unroll
    for (int k = 0; k < fragments<NK>(); ++k) s = fragment_product<TY, NK>(own_word<TY, NK>(label_row, k, words), own[k], s);
    const float mine = (l & 2) ? ((l & 1) ? s[3] : s[2]) : ((l & 1) ? s[1] : s[0]);
    return sum_group(g == (l >> 2) ? mine : 0.0f);   // (the diagonal's one value)
}

// A ray's loss from its maximum and sum; adds it to the thread's sums.
__device__ inline void finish_row(const LabelArgs &a, int64_t row, Running r, float target_logit, double &sum, uint32_t &count) {
    const int64_t t = a.target[row];
    const bool ignored = t == a.ignore;
    const float log_sum = log2_of(r.l);
    float loss = below_sum(r, target_logit);
    if (!has_sum(r) || t < 0 || t >= a.labels) loss = __builtin_nanf("");
    if (ignored) loss = 0.0f;
    a.lse2[row] = ignored ? kInf : r.m * kLog2E + log_sum;
    if (a.hit) a.top[row] = ignored ? 0.0f : r.m, a.log_sum[row] = ignored ? kInf : log_sum, a.hit[row] = expm1f(-loss);
    if (a.rows) a.rows[row] = loss;
    sum += (double)loss;
    count += ignored ? 0u : 1u;
}

// The workgroup's sum of losses and count of rays, in an order of its own.
__device__ inline void block_sums(const LabelArgs &a, int at, double sum, uint32_t count, char *lds) {
    if (!a.sums) return;
    double *s = reinterpret_cast<double *>(lds);
    uint32_t *c = reinterpret_cast<uint32_t *>(lds + sizeof(double) * kThreads);
    __syncthreads();
    s[threadIdx.x] = sum, c[threadIdx.x] = count;
    for (int step = kThreads / 2; step > 0; step >>= 1) {
        __syncthreads();
        if ((int)threadIdx.x < step) s[threadIdx.x] += s[threadIdx.x + step], c[threadIdx.x] += c[threadIdx.x + step];
    }
    if (threadIdx.x == 0) a.sums[at] = s[0], a.counts[at] = c[0];
}

// A norm is at least what its squares' sum says, and more by what squares below 2^-126 lost: sqrt(256) 2^-63 at most.
constexpr float kNormLost = 2e-18f;

// The best label of a ray, or a place on the list of those that 32 bits cannot decide. A logit starts as its label's bias and takes d
// products (six a channel, in planes); the tile product rounds at most once a product and once a block, each time by at most 2^-23 of the
// norms and the |bias|: it is off by less than (d + 16) 2^-22 of them, (3 d + 32) 2^-22 in planes (and by products too small for 32
// bits), twice that between two. A ray without channels (norm 0)
// has the biases themselves. Of the biases those count that can be the best label's: one more than 2 norms below the largest cannot, so a
// label that is masked by the lowest value of its type does not bring every ray onto the list. (Full-HD rays, 8 channels, 151 labels, a third
// of them so masked: 3767 us with all biases counted, 173 with these, when both were tried.)
__device__ inline void finish_best(const LabelArgs &a, int64_t row, Running r, float best, int label, float second, float norm, float3 bound) {
    const float reach = norm * bound.x, tall = fminf(bound.y, __builtin_fabsf(bound.z) + 2.1f * reach);
    const float off = norm > 0.0f ? a.margin * (reach + tall) + 1e-35f : 0.0f;
    a.label[row] = label == 0x7fffffff ? 0 : label;
    a.log_prob[row] = has_sum(r) ? -below_sum(r, best) : __builtin_nanf("");   // (no label left: there is no probability)
    if (best - second < 2.0f * off) {
        const uint32_t i = atomicAdd(a.near_count, 1u);
        a.near_list[i] = (uint32_t)row;
        a.near_floor[i] = best - 3.0f * off;   // (the best label's logit is best - off at least, and another sum of it off by as much)
    }
}
// The largest norm, |bias| and bias over the blocks that looked for them: every lane of a wave takes one.
__device__ inline float3 table_bound(const LabelArgs &a) {
    const float *from = a.bounds + 3 * (threadIdx.x & 63);
    float3 b = {from[0], from[1], from[2]};
    for (int step = 32; step > 0; step >>= 1)
        b.x = fmaxf(b.x, __shfl_xor(b.x, step)), b.y = fmaxf(b.y, __shfl_xor(b.y, step)), b.z = fmaxf(b.z, __shfl_xor(b.z, step));
    return b;
}
static_assert(kBoundBlocks == 64, "a lane each");

// (best, label) of two lanes or parts: the larger, the lower label where they are equal; `second`: the largest of the others.
__device__ inline void merge_best(float &best, int &label, float &second, float b, int l, float s) {
    const bool theirs = b > best || (b == best && l < label);
    second = fmaxf(fmaxf(second, s), theirs ? best : b);
    best = theirs ? b : best;
    label = theirs ? l : label;
}

// Rays as own rows, the table streamed. BEST: the best label instead of the loss.
// A lane keeps the maximum and sum of its own quarter of the table (its group's rows of every block), so nothing is exchanged until the
// end. Short rows are bound by the vector unit, not by the products: a difference, its scaling, an exponential, half a maximum and an
// addition for a logit, and four instructions more for the best label (full-HD, 8 channels, 151 labels: 167 us, vector
// instructions 88 % of the cycles). Long ones by vector and matrix instructions, 56 % and 46 % of the cycles, which overlap in part (32768 rays x
// 32771 labels of 256 channels, bf16: 583 us, 943 TFLOP/s, of the 1119 to 1206 that a large library product reaches).
template <class TY, int NK, int QB, bool BEST> __global__ __launch_bounds__(kThreads) void k_label_forward(LabelArgs a) {
    typedef Shape<TY, NK> T;
    __shared__ alignas(16) char tile[T::kTile > kThreads * 12 ? T::kTile : kThreads * 12];
    __shared__ alignas(16) float tile_bias[T::kRows];
    const int lane = threadIdx.x & 63, g = lane >> 4, wave = wave_number();
    const Turn turn = turn_of(a.cut);
    const int64_t row0 = (int64_t)turn.tile * (kWaves * 16 * QB) + wave * 16 * QB;
    const int first = turn.part ? turn.split * a.cut.per_split * T::kRows : 0;
    const int last = turn.part ? min(a.labels, first + a.cut.per_split * T::kRows) : a.labels;   // (the host keeps labels below 2^30)

    Stage<TY, NK> stage;
    stage.begin(a.w, tile_base(a.w, first));
    float stage_bias = 0.0f;   // of a row behind the table's end: -inf, which takes it out of every sum
    auto fetch = [&](int at) {
        stage.load(last - at);
        if ((int)threadIdx.x < T::kRows) stage_bias = at + (int)threadIdx.x >= last ? -kInf : a.bias ? a.bias[at + threadIdx.x] : 0.0f;
    };
    fetch(first);
    Own<TY, NK, QB> own;
    own.load(a.x, tile_base(a.x, row0), (int)min(a.rays - row0, (int64_t)(16 * QB)));

    Running run[QB];
    float low[QB];   // what the running sum's additions added too much
    float best[QB], second[QB];
    int label[QB];
#pragma unroll
    for (int q = 0; q < QB; ++q) run[q] = Running{-kInf, 0.0f}, low[q] = 0.0f, best[q] = second[q] = -kInf, label[q] = 0x7fffffff;
    rows_are_here(own);
    for (int at = first; at < last; at += T::kRows) {
        stage.store(tile);
        if ((int)threadIdx.x < T::kRows) tile_bias[threadIdx.x] = stage_bias;
        __syncthreads();
        if (at + T::kRows < last) fetch(at + T::kRows);
        float before[QB];   // the best up to this tile
        int place[QB];      // of the best in this tile, less 4 g
#pragma unroll
        for (int q = 0; q < QB; ++q) before[q] = best[q], place[q] = 0;
#pragma unroll
        for (int pair = 0; pair < T::kBlocks; pair += 2) {
            if constexpr (TY::kRounds)
                if (pair == 0) loads_between_products();
            if (NK <= 2 && at + pair * 16 >= last) break;   // (short rows: the work on a logit is most of all work)
            f4 s[2][QB];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const f4 b = *reinterpret_cast<const f4 *>(tile_bias + (pair + j) * 16 + 4 * g);
#pragma unroll
                for (int q = 0; q < QB; ++q) s[j][q] = b;
                product<TY, NK, QB, false, goes_first<TY, NK>()>(tile, pair + j, own, s[j]);
            }
#pragma unroll
            for (int q = 0; q < QB; ++q) {
                float top;
                if constexpr (BEST) {
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float v = s[j][q][r];
                            second[q] = __builtin_amdgcn_fmed3f(v, best[q], second[q]);
                            place[q] = v > best[q] ? (pair + j) * 16 + r : place[q];
                            best[q] = larger(best[q], v);
                        }
                    top = best[q];
                } else {
                    top = larger(larger(largest(s[0][q]), largest(s[1][q])), run[q].m);
                }
                // (a difference and its scaling are an instruction more than a fused product less the scaled maximum; that compared exact
                // products with a rounded one, and gave a lane that had met nothing but labels masked by -1e10 a sum of +inf)
                // (eight at a time, added in pairs: the running sum sees an eighth of the additions)
                const float use = finite_or_zero(top);
                f4 e[2];
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) e[j][r] = exp_of(s[j][q][r] - use);
                const float sum = ((e[0][0] + e[0][1]) + (e[0][2] + e[0][3])) + ((e[1][0] + e[1][1]) + (e[1][2] + e[1][3]));
                const float by = exp_of(run[q].m - use), l = run[q].l * by;
                // (a label near weight 1 would take a long tail's small terms in one by one, and lose them)
                const float more = sum - low[q] * by;
                run[q].l = l + more;
                low[q] = (run[q].l - l) - more;
                run[q].m = top;
            }
        }
        if constexpr (BEST)
#pragma unroll
            for (int q = 0; q < QB; ++q) label[q] = best[q] > before[q] ? at + 4 * g + place[q] : label[q];
        __syncthreads();
    }

    double sum = 0.0;
    uint32_t count = 0;
    float3 bound = {0.0f, 0.0f, 0.0f};
    if constexpr (BEST) bound = table_bound(a);
#pragma unroll
    for (int q = 0; q < QB; ++q) {
        const int64_t row = row0 + q * 16 + (lane & 15);
        const Running r = merge_group(Running{run[q].m, run[q].l - low[q]});
        if constexpr (BEST) {
            float norm = 0.0f;
            uint32_t any = 0u;   // of the bits but the signs
#pragma unroll
            for (int k = 0; k < fragments<NK>(); ++k) {
                norm += fragment_dot<TY>(own.f[q][k], own.f[q][k]);
#pragma unroll
                for (int p = 0; p < TY::kPlanes; ++p) {
                    const u4 w = own.f[q][k].w[p] & (TY::kDepth == 16 ? 0x7fffffffu : 0x7fff7fffu);
                    any |= (w[0] | w[1]) | (w[2] | w[3]);
                }
            }
            any |= __shfl_xor(any, 16), any |= __shfl_xor(any, 32);
            norm = sqrtf(sum_group(norm));
            norm = any ? norm + kNormLost : 0.0f;
#pragma unroll
            for (int step = 16; step <= 32; step <<= 1)
                merge_best(best[q], label[q], second[q], __shfl_xor(best[q], step), __shfl_xor(label[q], step), __shfl_xor(second[q], step));
            if (row < a.rays && g == 0) {
                if (turn.part) {
                    const int64_t part = part_row(a.cut, turn, kWaves * 16 * QB, wave * 16 * QB + q * 16 + (lane & 15));
                    a.part[part] = float2{r.m, r.l};
                    a.best[part] = int4{__builtin_bit_cast(int, best[q]), label[q], __builtin_bit_cast(int, second[q]),
                                                                 __builtin_bit_cast(int, norm)};
                } else {
                    finish_best(a, row, r, best[q], label[q], second[q], norm, bound);
                }
            }
        } else {
            float logit = 0.0f;
            if (turn.split == 0) {
                const int64_t t = row < a.rays ? a.target[row] : -1;
                const bool there = t >= 0 && t < a.labels;
                logit = logit_of<TY, NK>(own.f[q], there ? tile_base(a.w, t) : nullptr, a.w.words, there && a.bias ? a.bias[t] : 0.0f);
            }
            if (row < a.rays && g == 0) {
                if (turn.part) {
                    a.part[part_row(a.cut, turn, kWaves * 16 * QB, wave * 16 * QB + q * 16 + (lane & 15))] = float2{r.m, r.l};
                    if (turn.split == 0) a.target_logit[row - (int64_t)a.cut.whole * (kWaves * 16 * QB)] = logit;
                } else {
                    finish_row(a, row, r, logit, sum, count);
                }
            }
        }
    }
    if constexpr (!BEST)
        if (!turn.part) block_sums(a, turn.tile, sum, count, tile);
}

// The parts of a split forward pass, a thread a ray.
template <bool BEST> __global__ __launch_bounds__(kThreads) void k_label_join(LabelArgs a) {
    __shared__ alignas(16) char lds[kThreads * 12];
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x, row = (int64_t)a.cut.whole * a.own + i;
    double sum = 0.0;
    uint32_t count = 0;
    float3 bound = {0.0f, 0.0f, 0.0f};
    if constexpr (BEST) bound = table_bound(a);
    if (row < a.rays) {
        float m = -kInf;
        double l = 0.0;   // (hundreds of parts, of which one may have almost all of the sum)
        float best = -kInf, second = -kInf, norm = 0.0f;
        int label = 0x7fffffff;
        const int64_t from = i / a.own * a.cut.splits * a.own + i % a.own;
        for (int s = 0; s < a.cut.splits; ++s) {
            const float2 p = a.part[from + (int64_t)s * a.own];
            const float top = larger(m, p.x), use = finite_or_zero(top);
            l = l * (double)exp_of(m - use) + (double)p.y * (double)exp_of(p.x - use);
            m = top;
            if constexpr (BEST) {
                const int4 b = a.best[from + (int64_t)s * a.own];
                merge_best(best, label, second, __builtin_bit_cast(float, b.x), b.y, __builtin_bit_cast(float, b.z));
                norm = __builtin_bit_cast(float, b.w);
            }
        }
        const Running r = {m, (float)l};
        if constexpr (BEST) finish_best(a, row, r, best, label, second, norm, bound);
        else finish_row(a, row, r, a.target_logit[i], sum, count);
    }
    if constexpr (!BEST) block_sums(a, a.cut.whole + blockIdx.x, sum, count, lds);
}

// The sum of the blocks' losses, or their mean over the rays counted (none counted: 0 / 0), and what an upstream gradient
// of it is multiplied by for one ray.
__global__ __launch_bounds__(kThreads) void k_label_mean(const double *sums, const uint32_t *counts, uint32_t blocks, int mean, float *loss, float *inverse) {
    __shared__ double s[kThreads];
    __shared__ unsigned long long c[kThreads];
    double sum = 0.0;
    unsigned long long count = 0;
    for (uint32_t i = threadIdx.x; i < blocks; i += kThreads) sum += sums[i], count += counts[i];
    s[threadIdx.x] = sum, c[threadIdx.x] = count;
    for (int step = kThreads / 2; step > 0; step >>= 1) {
        __syncthreads();
        if ((int)threadIdx.x < step) s[threadIdx.x] += s[threadIdx.x + step], c[threadIdx.x] += c[threadIdx.x + step];
    }
    if (threadIdx.x == 0) {
        *loss = (float)(mean ? s[0] / (double)c[0] : s[0]);
        *inverse = !mean ? 1.0f : c[0] != 0 ? (float)(1.0 / (double)c[0]) : 0.0f;   // (of nothing: a loss of NaN, and no gradient)
    }
}

// ---- the best label where 32 bits do not decide ---------------------------------------------------------------------
// Largest norm of a row of the table, largest |bias| and bias, for every block; empties the list of near rays.
template <class TY> __global__ __launch_bounds__(kThreads) void k_label_bounds(LabelArgs a, float *bounds) {
    __shared__ float s[3 * kThreads];
    const int lane = threadIdx.x & 63;
    float wide = 0.0f, tall = 0.0f, most = a.bias ? -kInf : 0.0f;
    for (int64_t v = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6); v < a.labels; v += (int64_t)kBoundBlocks * kWaves) {
        float n = 0.0f;
        for (int k = lane; k < a.w.words; k += 64) {
            float w[kWordValues<TY>];
            row_values<TY>(tile_base(a.w, v), k, a.w.words, w);
            for (int j = 0; j < kWordValues<TY>; ++j) n = __builtin_fmaf(w[j], w[j], n);
        }
        for (int step = 32; step > 0; step >>= 1) n += __shfl_xor(n, step);
        wide = fmaxf(wide, n);
        if (a.bias) {   // (a label switched off by an infinite bias bounds nothing)
            const float b = __builtin_fabsf(a.bias[v]);
            tall = fmaxf(tall, b == kInf ? 0.0f : b);
            most = fmaxf(most, b == kInf ? -kInf : a.bias[v]);
        }
    }
    s[threadIdx.x] = wide, s[kThreads + threadIdx.x] = tall, s[2 * kThreads + threadIdx.x] = most;
    for (int step = kThreads / 2; step > 0; step >>= 1) {
        __syncthreads();
        if ((int)threadIdx.x < step) {
            s[threadIdx.x] = fmaxf(s[threadIdx.x], s[threadIdx.x + step]);
            s[kThreads + threadIdx.x] = fmaxf(s[kThreads + threadIdx.x], s[kThreads + threadIdx.x + step]);
            s[2 * kThreads + threadIdx.x] = fmaxf(s[2 * kThreads + threadIdx.x], s[2 * kThreads + threadIdx.x + step]);
        }
    }
    if (threadIdx.x == 0) {
        bounds[3 * blockIdx.x] = sqrtf(s[0]) * 1.0001f + kNormLost, bounds[3 * blockIdx.x + 1] = s[kThreads], bounds[3 * blockIdx.x + 2] = s[2 * kThreads];
        if (blockIdx.x == 0) *a.near_count = 0u;
    }
}

// The rays on the list, a workgroup each: every label's logit again in 32 bits, and in 64 where it can be the best.
template <class TY> __global__ __launch_bounds__(kThreads) void k_label_near(LabelArgs a) {
    constexpr int per = kWordValues<TY>;
    __shared__ alignas(16) float x[DST_MAX_CHANNELS];
    __shared__ double top[kThreads];
    __shared__ int at[kThreads];
    const uint32_t n = *a.near_count;
    for (uint32_t i = blockIdx.x; i < n; i += gridDim.x) {
        const int64_t row = a.near_list[i];
        const float floor = a.near_floor[i];
        __syncthreads();
        if ((int)threadIdx.x < a.x.words) {
            float v[per];
            row_values<TY>(tile_base(a.x, row), threadIdx.x, a.x.words, v);
            for (int j = 0; j < per; ++j) x[threadIdx.x * per + j] = v[j];
        }
        __syncthreads();
        double best = -__builtin_huge_val();
        int label = 0x7fffffff;
        for (int v = threadIdx.x; v < a.labels; v += kThreads) {
            const char *w = tile_base(a.w, v);
            float s = a.bias ? a.bias[v] : 0.0f;
#pragma unroll 4
            for (int k = 0; k < a.w.words; ++k) {
                float word[per];
                row_values<TY>(w, k, a.w.words, word);
#pragma unroll
                for (int j = 0; j < per; ++j) s = __builtin_fmaf(x[k * per + j], word[j], s);
            }
            if (!(s >= floor)) continue;
            double exact = 0.0;
            for (int k = 0; k < a.w.words; ++k) {
                float word[per];
                row_values<TY>(w, k, a.w.words, word);
                for (int j = 0; j < per; ++j) exact = __builtin_fma((double)x[k * per + j], (double)word[j], exact);
            }
            if (a.bias) exact += (double)a.bias[v];
            if (exact > best) best = exact, label = v;
        }
        top[threadIdx.x] = best, at[threadIdx.x] = label;
        for (int step = kThreads / 2; step > 0; step >>= 1) {
            __syncthreads();
            if ((int)threadIdx.x < step) {
                const double b = top[threadIdx.x + step];
                const int l = at[threadIdx.x + step];
                if (b > top[threadIdx.x] || (b == top[threadIdx.x] && l < at[threadIdx.x])) top[threadIdx.x] = b, at[threadIdx.x] = l;
            }
        }
        if (threadIdx.x == 0 && at[0] != 0x7fffffff) a.label[row] = at[0];
    }
}
// ---- backward -------------------------------------------------------------------------------------------------------
// dx: rays as own rows, the table streamed; the tile is read twice from LDS, by rows for the logits and turned for the sums.
// 921,600 rays x 256 labels of 8 channels: 125 us, vector instructions 88 % of the cycles; 131,072 x 4096 of 64 channels
// in planes: 641 us, matrix instructions 68 %; 32768 x 32771 of 256 channels, bf16: 1044 us, 1053 TFLOP/s, matrix instructions 49 %.
template <class TY, int NK, int QB> __global__ __launch_bounds__(kThreads, TY::kPlanes == 1 ? 2 : 1) void k_label_dx(LabelArgs a) {
    typedef Shape<TY, NK> T;
    constexpr int NM = depth_blocks<TY, NK>();
    __shared__ alignas(16) char tile[T::kTile];
    __shared__ alignas(16) float tile_bias[T::kRows];
    const int lane = threadIdx.x & 63, g = lane >> 4, wave = wave_number();
    const Turn turn = turn_of(a.cut);
    const int64_t row0 = (int64_t)turn.tile * (kWaves * 16 * QB) + wave * 16 * QB;
    const int first = turn.part ? turn.split * a.cut.per_split * T::kRows : 0;
    const int last = turn.part ? min(a.labels, first + a.cut.per_split * T::kRows) : a.labels;

    Stage<TY, NK> stage;
    stage.begin(a.w, tile_base(a.w, first));
    float stage_bias = 0.0f;   // of a row behind the table's end: -inf, which takes it out of every sum
    auto fetch = [&](int at) {
        stage.load(last - at);
        if ((int)threadIdx.x < T::kRows) stage_bias = at + (int)threadIdx.x >= last ? -kInf : a.bias ? a.bias[at + threadIdx.x] : 0.0f;
    };
    fetch(first);
    Own<TY, NK, QB> own;
    own.load(a.x, tile_base(a.x, row0), (int)min(a.rays - row0, (int64_t)(16 * QB)));
    float top[QB], log_sum[QB], up[QB], hit[QB];
    int label[QB];   // relative to the lane's first row of a tile
    f4 out[QB][NM];
#pragma unroll
    for (int q = 0; q < QB; ++q) {
        const int64_t row = row0 + q * 16 + (lane & 15);
        const int64_t t = row < a.rays ? a.target[row] : a.ignore;
        top[q] = row < a.rays ? a.top[row] : 0.0f;
        log_sum[q] = row < a.rays ? a.log_sum[row] : kInf;
        up[q] = row < a.rays ? upstream_of(a, row, t) : 0.0f;
        hit[q] = row < a.rays ? a.hit[row] : 0.0f;
        label[q] = (t >= 0 && t < a.labels ? (int)t : -0x40000000) - 4 * g;
#pragma unroll
        for (int m = 0; m < NM; ++m) out[q][m] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    rows_are_here(own);
    for (int at = first; at < last; at += T::kRows) {
        stage.store(tile);
        if ((int)threadIdx.x < T::kRows) tile_bias[threadIdx.x] = stage_bias;
        __syncthreads();
        if (at + T::kRows < last) fetch(at + T::kRows);
#pragma unroll
        for (int pair = 0; pair < T::kBlocks; pair += 2) {
            f4 p[2][QB];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const f4 b = *reinterpret_cast<const f4 *>(tile_bias + (pair + j) * 16 + 4 * g);
#pragma unroll
                for (int q = 0; q < QB; ++q) p[j][q] = b;
                product<TY, NK, QB, false, goes_first<TY, NK>()>(tile, pair + j, own, p[j]);
#pragma unroll
                for (int q = 0; q < QB; ++q)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float e = exp2_of(__builtin_fmaf(p[j][q][r] - top[q], kLog2E, -log_sum[q]));
                        p[j][q][r] = label[q] - at == (pair + j) * 16 + r ? hit[q] : e;
                    }
            }
            accumulate<TY, NK, QB, NM>(tile, pair, p[0], p[1], out);
        }
        __syncthreads();
    }
    typedef typename TY::E E;
    const bool four = (a.d & 3) == 0;
#pragma unroll
    for (int q = 0; q < QB; ++q) {
        const int64_t row = row0 + q * 16 + (lane & 15);
        whole_sums<TY>(out[q]);
        if (row >= a.rays) continue;
#pragma unroll
        for (int m = 0; m < NM; ++m) {
            f4 v = out[q][m] * up[q];
            if (up[q] == 0.0f) v = f4{0.0f, 0.0f, 0.0f, 0.0f};   // (an ignored ray's channels may hold anything)
            if (turn.part) store_four(a.out_part + part_row(a.cut, turn, kWaves * 16 * QB, wave * 16 * QB + q * 16 + (lane & 15)) * a.d, m * 16 + 4 * g, a.d, v, four);
            else store_sums<E>(a.out, row, m * 16 + 4 * g, a.d, v, four, a.half);
        }
    }
}

// dw and db: labels as own rows, the rays streamed, with their lse, upstream gradient and label in LDS. Few labels are cut into as many
// parts of the rays as fill the device. 921,600 rays x 256 labels of 8 channels: 130 us, vector instructions 80 % of the cycles; 131,072 x
// 4096 of 64 channels in planes: 742 us, matrix instructions 58 % (one wave on a SIMD, of four registers too many: 907); 32768 x 32771 of 256
// channels, bf16: 1529 us, 719 TFLOP/s, LDS reads 52 %.
// ONE: the rays share one upstream gradient, which multiplies the sums at the end; else each ray's weights have its own.
template <class TY, int NK, int QB, bool ONE> __global__ __launch_bounds__(kThreads, NK * TY::kPlanes <= 12 ? 2 : 1) void k_label_dw(LabelArgs a) {
    typedef Shape<TY, NK> T;
    constexpr int NM = depth_blocks<TY, NK>();
    __shared__ alignas(16) char tile[T::kTile];
    __shared__ alignas(16) float tile_top[2][T::kRows], tile_log_sum[2][T::kRows], tile_up[2][T::kRows], tile_hit[2][T::kRows];
    __shared__ alignas(16) int tile_label[2][T::kRows];
    const int lane = threadIdx.x & 63, g = lane >> 4, wave = wave_number();
    const Turn turn = turn_of(a.cut);
    const int row0 = turn.tile * (kWaves * 16 * QB) + wave * 16 * QB;   // (the host keeps labels below 2^30)
    const int64_t first = turn.part ? (int64_t)turn.split * a.cut.per_split * T::kRows : 0;
    const int64_t last = turn.part ? min(a.rays, first + (int64_t)a.cut.per_split * T::kRows) : a.rays;

    Stage<TY, NK> stage;
    stage.begin(a.x, tile_base(a.x, first));
    // Of every ray: maximum and sum (+inf where it is ignored or behind the end, which makes its weights 0), upstream gradient, label and its weight. They are a tile
    // ahead of the channels, which are read only of rays that are not ignored: those of the others may hold anything.
    float stage_top = 0.0f, stage_log_sum = kInf, stage_up = 0.0f, stage_hit = 0.0f;
    int64_t stage_target = a.ignore;
    auto fetch_stats = [&](int64_t at) {   // (as they lie: what is made of them waits for them)
        const int64_t row = at + threadIdx.x;
        stage_target = a.ignore, stage_top = 0.0f, stage_log_sum = kInf;
        if ((int)threadIdx.x < T::kRows && row < last) {
            stage_target = a.target[row], stage_top = a.top[row], stage_log_sum = a.log_sum[row], stage_hit = a.hit[row];
            if (!ONE) stage_up = a.upstream[row];
        }
    };
    auto store_stats = [&](int at) {
        if ((int)threadIdx.x >= T::kRows) return;
        const bool ignored = stage_target == a.ignore, none = !ignored && (stage_target < 0 || stage_target >= a.labels);
        tile_top[at][threadIdx.x] = stage_top;
        tile_log_sum[at][threadIdx.x] = none ? __builtin_nanf("") : stage_log_sum;
        tile_label[at][threadIdx.x] = ignored || none ? -1 : (int)stage_target;
        tile_hit[at][threadIdx.x] = stage_hit;
        if (!ONE) tile_up[at][threadIdx.x] = ignored ? 0.0f : stage_up;
    };
    auto fetch = [&](int64_t at, int half) {
        stage.template load<true>((int)min(last - at, (int64_t)T::kRows), tile_log_sum[half]);
    };
    fetch_stats(first);
    Own<TY, NK, QB> own;
    own.load(a.w, tile_base(a.w, row0), min(a.labels - row0, 16 * QB));
    store_stats(0);
    __syncthreads();
    if (first < last) fetch(first, 0);
    fetch_stats(first + T::kRows);
    float bias[QB], db[QB], db_low[QB];   // (a sum over all rays: with what its additions lost)
    f4 out[QB][NM];
#pragma unroll
    for (int q = 0; q < QB; ++q) {
        const int v = row0 + q * 16 + (lane & 15);
        bias[q] = a.bias && v < a.labels ? a.bias[v] : 0.0f;
        db[q] = db_low[q] = 0.0f;
#pragma unroll
        for (int m = 0; m < NM; ++m) out[q][m] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    int half = 0;
    rows_are_here(own);
    for (int64_t at = first; at < last; at += T::kRows, half ^= 1) {
        stage.store(tile);
        store_stats(half ^ 1);
        __syncthreads();
        if (at + T::kRows < last) {
            fetch(at + T::kRows, half ^ 1);
            fetch_stats(at + 2 * T::kRows);
        }
#pragma unroll
        for (int pair = 0; pair < T::kBlocks; pair += 2) {
            f4 p[2][QB];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int q = 0; q < QB; ++q) p[j][q] = f4{bias[q], bias[q], bias[q], bias[q]};
                product<TY, NK, QB>(tile, pair + j, own, p[j]);
                const int at4 = (pair + j) * 16 + 4 * g;
                const f4 top = *reinterpret_cast<const f4 *>(tile_top[half] + at4), log_sum = *reinterpret_cast<const f4 *>(tile_log_sum[half] + at4);
                const f4 up = ONE ? f4{} : *reinterpret_cast<const f4 *>(tile_up[half] + at4);
                const f4 hit = *reinterpret_cast<const f4 *>(tile_hit[half] + at4);
                const int4 label = *reinterpret_cast<const int4 *>(tile_label[half] + at4);
                const int labels[4] = {label.x, label.y, label.z, label.w};
#pragma unroll
                for (int q = 0; q < QB; ++q) {
                    const int v = row0 + q * 16 + (lane & 15);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        float e = exp2_of(__builtin_fmaf(p[j][q][r] - top[r], kLog2E, -log_sum[r]));
                        e = labels[r] == v ? hit[r] : e;
                        if constexpr (!ONE) e *= up[r];
                        p[j][q][r] = e;
                    }
                }
            }
#pragma unroll
            for (int q = 0; q < QB; ++q) {
                const f4 e = p[0][q] + p[1][q];
                const float more = ((e[0] + e[1]) + (e[2] + e[3])) - db_low[q], to = db[q] + more;
                db_low[q] = (to - db[q]) - more;
                db[q] = to;
            }
            accumulate<TY, NK, QB, NM>(tile, pair, p[0], p[1], out);
        }
        __syncthreads();
    }
    typedef typename TY::E E;
    const bool four = (a.d & 3) == 0;
#pragma unroll
    for (int q = 0; q < QB; ++q) {
        const int v = row0 + q * 16 + (lane & 15);
        const float by = ONE ? (a.rays > 0 ? upstream_value(a) : 0.0f) : 1.0f;
        const float b = sum_group(db[q]) * by;
        whole_sums<TY>(out[q]);
        if (v >= a.labels) continue;
        const int64_t part = part_row(a.cut, turn, kWaves * 16 * QB, wave * 16 * QB + q * 16 + (lane & 15));
        if (g == 0 && a.bias_out) *(turn.part ? a.bias_part + part : a.bias_out + v) = b;
#pragma unroll
        for (int m = 0; m < NM; ++m) {
            if (turn.part) store_four(a.out_part + part * a.d, m * 16 + 4 * g, a.d, out[q][m] * by, four);
            else if (a.out) store_sums<E>(a.out, v, m * 16 + 4 * g, a.d, out[q][m] * by, four, a.half);
        }
    }
}
}  // namespace

// ---- host -----------------------------------------------------------------------------------------------------------
namespace {

int check(const DstLabelParams *p) {
    if (!p) return dst_op_fail(DST_E_INVALID, "params is null");
    if (p->dtype != DST_DTYPE_F32 && p->dtype != DST_DTYPE_BF16 && p->dtype != DST_DTYPE_F16)
        return dst_op_fail(DST_E_UNSUPPORTED, "dtype must be float32, bfloat16 or float16");
    if (p->rays < 0 || p->rays > 0x7fffffff) return dst_op_fail(DST_E_INVALID, "rays must be in 0..2^31-1");
    if (p->labels < 1 || p->labels > DST_MAX_LABELS) return dst_op_fail(DST_E_UNSUPPORTED, "labels must be in 1..%d", DST_MAX_LABELS);
    if (p->channels < 1 || p->channels > DST_MAX_CHANNELS)
        return dst_op_fail(DST_E_UNSUPPORTED, "channels must be in 1..%d", DST_MAX_CHANNELS);
    if (p->features_stride < p->channels || p->weight_stride < p->channels)
        return dst_op_fail(DST_E_INVALID, "rows of features and weight must not overlap");
    if (p->features_stride > kLongestStride || p->weight_stride > kLongestStride) return dst_op_fail(DST_E_INVALID, "strides must be in 0..2^44");
    if (p->reduction < DST_REDUCE_NONE || p->reduction > DST_REDUCE_MEAN) return dst_op_fail(DST_E_INVALID, "unknown reduction");
    if ((p->rays > 0 && !p->features) || !p->weight) return dst_op_fail(DST_E_INVALID, "features and weight are required");
    return DST_OK;
}

LabelArgs arguments(const DstLabelParams *p) {
    LabelArgs a = {};
    a.bias = p->bias, a.target = p->targets;
    a.rays = p->rays, a.ignore = p->ignore_index, a.d = p->channels, a.labels = p->labels;
    a.lse2 = p->lse;
    if (p->stats) a.top = p->stats, a.log_sum = p->stats + p->rays, a.hit = p->stats + 2 * p->rays;
    return a;
}

// The rows of both sets, copied into the workspace's front where the kernels cannot read them where they lie.
struct Sets {
    RowSet x, w;
};
template <class TY> Sets row_sets(const DstLabelParams *p, Carve &c) {
    Sets s;
    s.x = row_set<TY>(p->features, p->dtype, 0, p->features_stride, 0, 1, 1, 1, p->rays, p->channels, 1, c);
    s.w = row_set<TY>(p->weight, p->dtype, 0, p->weight_stride, 0, 1, 1, 1, p->labels, p->channels, 1, c);
    return s;
}

template <class TY, int NK> struct Shapes {   // own rows of a workgroup, rows of a tile
    static constexpr int kForward = kWaves * 16 * forward_blocks<TY, NK>(), kDx = kWaves * 16 * dx_blocks<TY, NK>(),
                         kDw = kWaves * 16 * dw_blocks<TY, NK>();
    static constexpr int kTile = Shape<TY, NK>::kRows;
};

// f(type, integral constant of the fragments) for the call's type and channels. The backward kernels take 32-bit rows of up to eight values
// in planes (Short32), the forward ones, which have half the products, in 32 bits (921,600 rays x 256 labels: dx 111 us for 131,
// dw 128 for 155, forward 96 for 89). Gradients of binary16 rows are formed in 32 bits.
template <class F> int with_type(const DstLabelParams *p, F f) {
    const int nk = fragments_of(p->channels, p->dtype);
    if (p->dtype == DST_DTYPE_F32) return with_floats<false>(p->channels, f);
    return p->dtype == DST_DTYPE_BF16 ? with_fragments<BF16>(nk, f) : with_fragments<F16>(nk, f);
}
template <class F> int with_gradients(const DstLabelParams *p, F f) {
    return p->dtype == DST_DTYPE_BF16 ? with_fragments<BF16>(fragments_of(p->channels, p->dtype), f) : with_floats<true>(p->channels, f);
}

struct ForwardPlan {
    Sets sets;
    bool few;
    uint32_t sums;    // blocks that leave a sum
    uint64_t bytes;
};
template <class TY, int NK, bool BEST> const void *forward_kernel(bool few) {
    return few ? (const void *)&k_label_forward<TY, NK, 1, BEST> : (const void *)&k_label_forward<TY, NK, forward_blocks<TY, NK>(), BEST>;
}
template <class TY, int NK, bool BEST> ForwardPlan forward_plan(const DstLabelParams *p, LabelArgs &a, char *base) {
    typedef Shapes<TY, NK> S;
    ForwardPlan f;
    const int64_t streamed = div_up(p->labels, S::kTile);
    f.few = few_rows(div_up(p->rays, S::kForward), streamed);
    a.own = f.few ? kWaves * 16 : S::kForward;
    a.cut = cut_tiles(div_up(p->rays, a.own), streamed, slots_of(forward_kernel<TY, NK, BEST>(f.few)),
                      tile_time<TY, NK>(a.own, 1), a.own * (BEST ? 24.0 : 8.0));
    const uint64_t rest = a.cut.splits > 1 ? (uint64_t)a.cut.parted() * a.own : 0, parts = rest * a.cut.splits;
    f.sums = (uint32_t)(a.cut.splits > 1 ? a.cut.whole + div_up(rest, kThreads) : a.cut.tiles);
    Carve c = {base, 0};
    f.sets = row_sets<TY>(p, c);
    a.x = f.sets.x.rows, a.w = f.sets.w.rows;
    if (parts) {
        a.part = c.take<float2>(parts);
        if (BEST) a.best = c.take<int4>(parts);
        else a.target_logit = c.take<float>(rest);
    }
    if (BEST) {
        a.margin = 2.3841858e-7f * (float)(TY::kPlanes == 3 ? 3 * p->channels + 32 : p->channels + 16);
        a.bounds = c.take<float>(3 * kBoundBlocks);
        a.near_count = c.take<uint32_t>(1);
        a.near_list = c.take<uint32_t>(p->rays);
        a.near_floor = c.take<float>(p->rays);
    } else if (p->reduction != DST_REDUCE_NONE) {
        a.sums = c.take<double>(f.sums);
        a.counts = c.take<uint32_t>(f.sums);
    }
    f.bytes = c.used;
    return f;
}

struct BackwardPlan {
    Sets sets;
    bool few;
    uint64_t bytes;
};
// DX: the rays are the own rows; else the labels
template <class TY, int NK, bool DX> BackwardPlan backward_plan(const DstLabelParams *p, LabelArgs &a, char *base) {
    typedef Shapes<TY, NK> S;
    constexpr int QB = DX ? dx_blocks<TY, NK>() : dw_blocks<TY, NK>();
    const int64_t own = DX ? p->rays : p->labels, streamed = div_up(DX ? p->labels : p->rays, S::kTile);
    BackwardPlan b;
    constexpr int whole = DX ? S::kDx : S::kDw;
    b.few = few_rows(div_up(own, whole), streamed);
    a.own = b.few ? kWaves * 16 : whole;
    const void *kernel;
    if constexpr (DX) kernel = b.few ? (const void *)&k_label_dx<TY, NK, 1> : (const void *)&k_label_dx<TY, NK, QB>;
    else if (p->reduction == DST_REDUCE_NONE) kernel = b.few ? (const void *)&k_label_dw<TY, NK, 1, false> : (const void *)&k_label_dw<TY, NK, QB, false>;
    else kernel = b.few ? (const void *)&k_label_dw<TY, NK, 1, true> : (const void *)&k_label_dw<TY, NK, QB, true>;
    a.cut = cut_tiles(div_up(own, a.own), streamed, slots_of(kernel), tile_time<TY, NK>(a.own, 2),
                      a.own * (p->channels + 1) * 4.0);
    const uint64_t parts = a.cut.splits > 1 ? (uint64_t)a.cut.parted() * a.own * a.cut.splits : 0;
    Carve c = {base, 0};
    b.sets = row_sets<TY>(p, c);
    a.x = b.sets.x.rows, a.w = b.sets.w.rows;
    if (parts) {
        a.out_part = c.take<float>(parts * p->channels);
        if (!DX) a.bias_part = c.take<float>(parts);
    }
    b.bytes = c.used;
    return b;
}

// The output row of a parted row
struct LabelRow {
    int64_t first, rows;
    int own;
    __device__ int64_t operator()(int tile, int row) const {
        const int64_t r = first + (int64_t)tile * own + row;
        return r < rows ? r : -1;
    }
};

// DST_OK, or the refusal of rows that need more workgroups than a launch holds.
int check_blocks(const Sets &s, const Cut &cut) {
    return cut.blocks() <= kMostBlocks && copy_blocks({&s.x, &s.w}) <= kMostBlocks ? (int)DST_OK
                                                                                  : dst_op_fail(DST_E_UNSUPPORTED, "too many rays or labels");
}

int check_workspace(const DstLabelParams *p, uint64_t need) {
    if (need == 0) return DST_OK;
    if (!p->workspace || p->workspace_bytes < need)
        return dst_op_fail(DST_E_INVALID, "workspace of %llu bytes is needed", (unsigned long long)need);
    if (reinterpret_cast<uintptr_t>(p->workspace) & 255u) return dst_op_fail(DST_E_INVALID, "workspace must be aligned to 256 bytes");
    return DST_OK;
}

}  // namespace

extern "C" {

uint64_t dst_label_workspace_bytes(const DstLabelParams *p, int pass) {
    if (check(p) != DST_OK) return 0;
    uint64_t bytes = 0;
    LabelArgs a = {};
    if (pass == DST_PASS_BACKWARD) {
        with_gradients(p, [&](auto ty, auto nk) {
            typedef decltype(ty) TY;
            constexpr int NK = decltype(nk)::value;
            uint64_t need = 0;
            for (int dx = 1; dx >= 0; --dx) {
                if (dx ? !p->grad_features : !p->grad_weight && !p->grad_bias) continue;
                const BackwardPlan b = dx ? backward_plan<TY, NK, true>(p, a, nullptr) : backward_plan<TY, NK, false>(p, a, nullptr);
                if (int rc = check_blocks(b.sets, a.cut)) return rc;
                need = b.bytes > need ? b.bytes : need;
            }
            bytes = need;
            return (int)DST_OK;
        });
    } else {
        with_type(p, [&](auto ty, auto nk) {
            typedef decltype(ty) TY;
            constexpr int NK = decltype(nk)::value;
            const ForwardPlan f = pass == DST_PASS_BEST ? forward_plan<TY, NK, true>(p, a, nullptr) : forward_plan<TY, NK, false>(p, a, nullptr);
            if (int rc = check_blocks(f.sets, a.cut)) return rc;
            bytes = f.bytes;
            return (int)DST_OK;
        });
    }
    return bytes;
}

int dst_label_loss_forward(const DstLabelParams *p, void *stream) {
    if (int rc = check(p)) return rc;
    if (p->rays > 0 && (!p->targets || !p->lse)) return dst_op_fail(DST_E_INVALID, "targets and lse are required");
    if (!p->loss && (p->rays > 0 || p->reduction != DST_REDUCE_NONE)) return dst_op_fail(DST_E_INVALID, "loss is required");
    if (p->reduction != DST_REDUCE_NONE && !p->inverse) return dst_op_fail(DST_E_INVALID, "a reduced loss needs inverse");
    return with_type(p, [&](auto ty, auto nk) {
        typedef decltype(ty) TY;
        constexpr int NK = decltype(nk)::value;
        LabelArgs a = arguments(p);
        const ForwardPlan f = forward_plan<TY, NK, false>(p, a, (char *)p->workspace);
        if (int rc = check_blocks(f.sets, a.cut)) return rc;
        if (int rc = check_workspace(p, f.bytes)) return rc;
        if (p->reduction == DST_REDUCE_NONE) a.rows = p->loss;
        const hipStream_t s = (hipStream_t)stream;
        if (a.cut.tiles > 0) {
            prepare({&f.sets.x, &f.sets.w}, s);
            const dim3 grid((uint32_t)a.cut.blocks());
            if (f.few) k_label_forward<TY, NK, 1, false><<<grid, kThreads, 0, s>>>(a);
            else k_label_forward<TY, NK, forward_blocks<TY, NK>(), false><<<grid, kThreads, 0, s>>>(a);
            DST_OP_LAUNCH("label loss");
            if (a.cut.splits > 1) {
                k_label_join<false><<<dim3(f.sums - (uint32_t)a.cut.whole), kThreads, 0, s>>>(a);
                DST_OP_LAUNCH("label loss, joining");
            }
        }
        if (p->reduction != DST_REDUCE_NONE) {
            k_label_mean<<<1, kThreads, 0, s>>>(a.sums, a.counts, f.sums, p->reduction == DST_REDUCE_MEAN,
                                               p->loss, p->inverse);
            DST_OP_LAUNCH("label loss, summing");
        }
        return (int)DST_OK;
    });
}

int dst_label_loss_backward(const DstLabelParams *p, void *stream) {
    if (int rc = check(p)) return rc;
    if (p->rays > 0 && (!p->targets || !p->lse || !p->upstream)) return dst_op_fail(DST_E_INVALID, "targets, lse and upstream are required");
    if (p->reduction != DST_REDUCE_NONE && !p->inverse) return dst_op_fail(DST_E_INVALID, "a reduced loss needs inverse");
    if ((reinterpret_cast<uintptr_t>(p->grad_features) | reinterpret_cast<uintptr_t>(p->grad_weight)) & 15u)
        return dst_op_fail(DST_E_INVALID, "gradients must be aligned to 16 bytes");
    if (p->rays > 0 && !p->stats) return dst_op_fail(DST_E_INVALID, "stats are required");
    return with_gradients(p, [&](auto ty, auto nk) {
        typedef decltype(ty) TY;
        typedef typename TY::E E;
        constexpr int NK = decltype(nk)::value, QB = dw_blocks<TY, NK>();
        const hipStream_t s = (hipStream_t)stream;
        const bool wanted[2] = {p->grad_features && p->rays > 0, p->grad_weight || p->grad_bias};   // dx, dw
        LabelArgs args[2] = {arguments(p), arguments(p)};
        BackwardPlan plans[2];
        uint64_t need = 0;
        for (int pass = 0; pass < 2; ++pass) {   // (both are looked at before either runs)
            if (!wanted[pass]) continue;
            plans[pass] = pass == 0 ? backward_plan<TY, NK, true>(p, args[0], (char *)p->workspace)
                                    : backward_plan<TY, NK, false>(p, args[1], (char *)p->workspace);
            if (int rc = check_blocks(plans[pass].sets, args[pass].cut)) return rc;
            need = plans[pass].bytes > need ? plans[pass].bytes : need;
        }
        if (int rc = check_workspace(p, need)) return rc;
        bool copied = false;
        for (int pass = 0; pass < 2; ++pass) {
            if (!wanted[pass]) continue;
            const bool dx = pass == 0;
            LabelArgs &a = args[pass];
            const BackwardPlan &b = plans[pass];
            a.half = p->dtype == DST_DTYPE_F16;
            a.upstream = p->upstream, a.upstream_rows = p->reduction == DST_REDUCE_NONE;
            a.inverse = a.upstream_rows ? nullptr : p->inverse;
            a.out = dx ? p->grad_features : p->grad_weight, a.bias_out = p->grad_bias;
            const dim3 grid((uint32_t)a.cut.blocks());
            if (!copied) prepare({&b.sets.x, &b.sets.w}, s);   // (both passes have the copies in the same place)
            copied = true;
            if (dx && b.few) k_label_dx<TY, NK, 1><<<grid, kThreads, 0, s>>>(a);
            else if (dx) k_label_dx<TY, NK, dx_blocks<TY, NK>()><<<grid, kThreads, 0, s>>>(a);
            else if (b.few && a.upstream_rows) k_label_dw<TY, NK, 1, false><<<grid, kThreads, 0, s>>>(a);
            else if (b.few) k_label_dw<TY, NK, 1, true><<<grid, kThreads, 0, s>>>(a);
            else if (a.upstream_rows) k_label_dw<TY, NK, QB, false><<<grid, kThreads, 0, s>>>(a);
            else k_label_dw<TY, NK, QB, true><<<grid, kThreads, 0, s>>>(a);
            DST_OP_LAUNCH("label gradient");
            const LabelRow to = {(int64_t)a.cut.whole * a.own, dx ? p->rays : (int64_t)p->labels, a.own};
            with_output<E>(a.half, [&](auto one) {
                typedef decltype(one) To;
                sum_parts(Parts<To>{a.out_part, (To *)a.out, p->channels}, Parts<float>{a.bias_part, dx ? nullptr : p->grad_bias, 1}, a.cut, a.own, to, s);
            });
            DST_OP_LAUNCH("label gradient, summing");
        }
        return (int)DST_OK;
    });
}

int dst_label_best(const DstLabelParams *p, void *stream) {
    if (int rc = check(p)) return rc;
    if (p->rays == 0) return DST_OK;
    if (!p->best || !p->log_prob) return dst_op_fail(DST_E_INVALID, "best and log_prob are required");
    return with_type(p, [&](auto ty, auto nk) {
        typedef decltype(ty) TY;
        constexpr int NK = decltype(nk)::value;
        LabelArgs a = arguments(p);
        const ForwardPlan f = forward_plan<TY, NK, true>(p, a, (char *)p->workspace);
        if (int rc = check_blocks(f.sets, a.cut)) return rc;
        if (int rc = check_workspace(p, f.bytes)) return rc;
        a.label = p->best, a.log_prob = p->log_prob;
        const hipStream_t s = (hipStream_t)stream;
        prepare({&f.sets.x, &f.sets.w}, s);
        k_label_bounds<TY><<<kBoundBlocks, kThreads, 0, s>>>(a, const_cast<float *>(a.bounds));
        const dim3 grid((uint32_t)a.cut.blocks());
        if (f.few) k_label_forward<TY, NK, 1, true><<<grid, kThreads, 0, s>>>(a);
        else k_label_forward<TY, NK, forward_blocks<TY, NK>(), true><<<grid, kThreads, 0, s>>>(a);
        DST_OP_LAUNCH("best label");
        if (a.cut.splits > 1) k_label_join<true><<<dim3(f.sums - (uint32_t)a.cut.whole), kThreads, 0, s>>>(a);
        // (as many workgroups as the device holds; each takes rays off the list until there are no more)
        k_label_near<TY><<<dim3((uint32_t)(p->rays < 2048 ? p->rays : 2048)), kThreads, 0, s>>>(a);
        DST_OP_LAUNCH("best label, near rays");
        return (int)DST_OK;
    });
}

}  // extern "C"
