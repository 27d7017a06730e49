// Attention of the rows of a batch over the 4-bit paged cache: o = softmax(scale q k^T) v over the positions a row sees.
//
// A key is k[d] = m_g + s_g c[d] with one (s, m) per group g of 32 dims, so a score is
//   q . k = sum_g s_g (sum_{d in g} q[d] c[d]) + m_g (sum_{d in g} q[d]),
// and the matrix cores multiply q with the bare codes: a 4-bit field that a mask leaves in place IS an fp16 number, the
// subnormal c * 2^-24 (bits 0-3) or c * 2^-20 (bits 4-7), and v_mfma_f32_16x16x32_f16 takes subnormals as they are. 32 dims
// are the depth of one such instruction, so one instruction sums one group; s and m are applied to its fp32 result. The
// same holds for the values: sum_t p_t (m_tg + s_tg c_td) = sum_t (p_t s_tg) c_td + sum_t p_t m_tg with bare codes as one
// operand and p s as the other. p s is taken in two fp16 pieces (the second is what the first's rounding left), so the only
// roundings to fewer than 32 bits are 2^-22 of p s, and the result's.
#include "kv4.h"

namespace tllm {
namespace {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef uint32_t uint4_t __attribute__((ext_vector_type(4)));
typedef uint32_t uint2_t __attribute__((ext_vector_type(2)));

constexpr int kWaves = 4, kThreads = kWaves * kWave;
constexpr float kEmpty = -1e30f;  // below every score (|q.k| < 2^40, |scale| <= 2^40): no position yet
constexpr int kHeadroom = 6;      // powers of two that a weight may outgrow its base by before everything is rescaled
constexpr int kTopPower = 8;      // a base puts the largest weight seen (times its step) at 2^kTopPower
constexpr int kMostSplits = 128;
constexpr uint32_t kEvenCodes = 0x000F000Fu, kOddCodes = 0x00F000F0u;
// The values' codes are brought to c - 8 in ordinary fp16 first: 1024 + c (or 64 + c, from bits 4-7) with one ternary
// instruction, minus the rest with a packed one. Bare codes would be cheaper by that one, but the matrix unit lines products
// up by their operands' exponents, of which a subnormal has the smallest however few bits it fills, and cuts what falls off:
// sums of up to 2^-22 too low, which positive codes add up to 2 sqrt(positions) times what is left of the values in the end
// (4e-4 of the result at 131072 positions). Scores, sums of 128 products with their signs, do not feel it.
constexpr uint32_t kEvenBits = 0x64006400u, kOddBits = 0x54005400u;

__device__ __forceinline__ float low_half(uint32_t w) { return h2f((uint16_t)w); }
__device__ __forceinline__ float high_half(uint32_t w) { return h2f((uint16_t)(w >> 16)); }

// What the host and both kernels have to agree on.
struct SplitPlan {
    int splits;      // most parts that a row tile's positions are shared out to
    int row_tiles;   // of max_query rows
};

// The positions [lo, hi) that some row of a tile sees, and its parts in steps of `step` positions.
struct Span {
    int first, steps, per, used;  // first step, steps, steps per part, parts that have any
    __device__ Span(int lo, int hi, int step, int splits) {
        first = lo / step;
        steps = hi > lo ? (hi + step - 1) / step - first : 0;
        per = (steps + splits - 1) / splits;
        per = per < kWaves ? kWaves : (per + kWaves - 1) & ~(kWaves - 1);
        used = (steps + per - 1) / per;
    }
};

// Rows of a sequence, in range whatever the arrays hold.
struct Sequence {
    int row0, rows, pos0;  // first row, rows, position of the first row
    __device__ Sequence(const AttentionKv4Args &a, int seq) {
        const int s0 = a.batch.starts[seq], s1 = a.batch.starts[seq + 1];
        row0 = s0;
        rows = min(min(s1, a.batch.n_tokens) - s0, a.max_query);
        if (s0 < 0) rows = 0;
        const long long p = (long long)a.batch.lengths[seq] - s1 + s0;
        pos0 = (int)max(min(p, (long long)INT32_MAX - (1 << 25)), -(1ll << 25));
    }
};
__device__ __forceinline__ int position_limit(const AttentionKv4Args &a) { return min(a.batch.width << a.cache.page_shift, a.max_length); }
__device__ __forceinline__ int window_begin(const AttentionKv4Args &a, int pos) { return a.window > 0 ? max(0, pos - a.window + 1) : 0; }

// ------------------------------------------------------------------------------------------------- few rows: decode
//
// A workgroup takes up to kRows rows (query rows times the heads that share a kv head; kRows 4, 8 or 16) and a part of the
// positions; its four waves take steps of kStep positions in turn and are joined through LDS at the end, parts through the
// workspace. Bound: HBM, the cache's 5 bits per value; the work per position has to stay small beside it, above all the
// work on scores, of which 16 x 16 come out of every matrix instruction however few rows there are. So the row operand
// repeats its kRows rows, and of kPack = 16 / kRows tiles of 16 positions each quad of lanes keeps the results of its own
// tile: each of the 64 lanes then has ONE position and four rows of its own (lane = (position t, quad)), steps and minima
// are one coalesced word per lane and group, and softmax runs on four registers. For the values, weights p s go through LDS ([position][group][row], fp16) and come
// back transposed (ds_read_b64_tr_b16) with (group, row) pairs as the 16 columns of the operand: one instruction multiplies
// a row tile's weights of all groups in the set, of which each dim uses its own group's.
template <int kDim, int kRows>
struct Decode {
    static constexpr int kGroups = kDim / kKvGroup, kWords = kDim / 8;
    static constexpr int kPack = 16 / kRows;
    static constexpr int kTiles = kRows == 16 ? 2 : 4, kStep = 16 * kTiles, kPasses = kTiles / kPack;
    static constexpr int kColumns = kGroups * kRows < 16 ? 16 : kGroups * kRows;  // of the weights: (group, row)
    static constexpr int kSets = kColumns / 16, kSetGroups = kGroups / kSets;
    static constexpr int kSetWords = 4 * kSetGroups, kLanesPerWord = 16 / kSetWords, kNibbles = 8 / kLanesPerWord;
    static constexpr int kRowBytes = 4 * kColumns + 16;  // of a position's weights in LDS: both pieces, 16 bytes off a power of two
    static constexpr int kWaveBytes = kStep * kRowBytes;
    static constexpr int kJoinBytes = kWaves * kRows * kDim * 4;
    static constexpr int kLds = kWaves * kWaveBytes > kJoinBytes ? kWaves * kWaveBytes : kJoinBytes;
    static_assert(kWaveBytes >= 64 * (kGroups * 4 + 4) * 4 / 4, "the sums of the minima");
    using KeyWords = typename std::conditional<kGroups == 4, uint4_t, uint2_t>::type;
    struct Places {
        int block[kTiles], slot[kTiles];  // of each tile of 16 positions: page * n_kv_heads + head, first slot
        uint32_t there;                   // bit i: tile i has a page
    };
    struct Keys {
        KeyWords k[kTiles];
        uint32_t km[kPasses][kGroups], vm[kPasses][kGroups];  // step | minimum << 16 of this lane's position, keys and values
    };
    struct Values {
        uint4_t v[kTiles][kSets];
    };
};

template <int kDim, int kRows>
__global__ __launch_bounds__(kThreads, 2) void attention_decode_kernel(const AttentionKv4Args a, const SplitPlan plan) {
    using D = Decode<kDim, kRows>;
    constexpr int G = D::kGroups;
    __shared__ __align__(16) unsigned char lds[D::kLds];
    __shared__ float join_base[kWaves][kRows], join_sum[kWaves][kRows];
    const Kv4Cache &c = a.cache;
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int quad = lane >> 4, t16 = lane & 15;
    const int kv = blockIdx.x % c.n_kv_heads;  // fastest: a kv head's parts and tiles fall on the same XCDs
    const int part = blockIdx.x / c.n_kv_heads % plan.splits, tile = blockIdx.x / c.n_kv_heads / plan.splits;
    const int seq = blockIdx.y, heads = a.n_heads / c.n_kv_heads;

    const Sequence s(a, seq);
    const int first_row = tile * kRows, rows_left = s.rows * heads - first_row;  // rows are (query row, head), heads fastest
    if (rows_left <= 0) return;
    const int last_row = first_row + min(rows_left, kRows) - 1;
    const int pos_low = s.pos0 + first_row / heads, pos_high = s.pos0 + last_row / heads;
    const Span span(window_begin(a, pos_low), min(pos_high + 1, position_limit(a)), D::kStep, plan.splits);
    if (plan.splits > 1 && part >= span.used) return;  // (one part: it writes the zeros of rows that see nothing)

    // row operands: this lane's row and its 8 dims of each group
    // (rows that are not there are zeros; what they see shows in their own columns only)
    half8_t q[G];
    float own_sum[G];
    {
        const int row = t16 % kRows, at = first_row + row;
        const bool real = row < rows_left;
        const uint16_t *src = a.q + (size_t)(s.row0 + (real ? at / heads : 0)) * a.q_stride + (size_t)(kv * heads + (real ? at % heads : 0)) * kDim + quad * 8;
#pragma unroll
        for (int g = 0; g < G; g++) {
            half8_t x = real ? *(const half8_t *)(src + g * 32) : half8_t{};
            own_sum[g] = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) own_sum[g] += (float)x[j];
            own_sum[g] += __shfl_xor(own_sum[g], 16, kWave);
            own_sum[g] += __shfl_xor(own_sum[g], 32, kWave);
            q[g] = x;
        }
    }
    // the four rows that this lane has results of: 4 * row_quad + r
    const int row_quad = quad % (kRows / 4), pack = quad / (kRows / 4);
    float q_sum[G][4];
    int pos[4];
#pragma unroll
    for (int r = 0; r < 4; r++) {
#pragma unroll
        for (int g = 0; g < G; g++) q_sum[g][r] = __shfl(own_sum[g], 4 * quad + r, kWave);
        const int row = 4 * row_quad + r;
        pos[r] = row < rows_left ? s.pos0 + (first_row + row) / heads : -1;
    }

    const size_t code_words = kv4_code_words(1 << c.page_shift, kDim), scale_words = kv4_scale_words(1 << c.page_shift, kDim);
    const int *table = a.batch.table + (size_t)seq * a.batch.width;
    const uint32_t key_offset = (uint32_t)(t16 * D::kWords + quad * G);
    const uint32_t value_offset = (uint32_t)(quad * (D::kWords * 4) + (t16 / D::kLanesPerWord) * 4);

    auto find = [&](int step) {
        typename D::Places x;
        const int at = step * D::kStep;
        x.there = 0;
#pragma unroll
        for (int i = 0; i < D::kTiles; i++) {
            const int index = (at + 16 * i) >> c.page_shift;
            const int page = index < a.batch.width ? table[index] : -1;
            const bool there = page >= 0 && page < c.n_pages;
            x.there |= (uint32_t)there << i;
            x.block[i] = (there ? page : 0) * c.n_kv_heads + kv;
            x.slot[i] = (at + 16 * i) & ((1 << c.page_shift) - 1);
        }
        return x;
    };
    auto load_keys = [&](typename D::Keys &x, const typename D::Places &at) {
#pragma unroll
        for (int i = 0; i < D::kTiles; i++)
            x.k[i] = *(const typename D::KeyWords *)(c.k_codes + (size_t)at.block[i] * code_words + (size_t)at.slot[i] * D::kWords + key_offset);
#pragma unroll
        for (int p = 0; p < D::kPasses; p++) {
            int b = at.block[p * D::kPack], sl = at.slot[p * D::kPack];
#pragma unroll
            for (int u = 1; u < D::kPack; u++)
                if (pack == u) b = at.block[p * D::kPack + u], sl = at.slot[p * D::kPack + u];
            const size_t word = (size_t)b * scale_words + sl + t16;
#pragma unroll
            for (int g = 0; g < G; g++) {
                x.km[p][g] = c.k_scales[word + ((size_t)g << c.page_shift)];
                x.vm[p][g] = c.v_scales[word + ((size_t)g << c.page_shift)];
            }
        }
    };
    auto load_values = [&](typename D::Values &x, const typename D::Places &at) {
#pragma unroll
        for (int i = 0; i < D::kTiles; i++)
#pragma unroll
            for (int e = 0; e < D::kSets; e++)
                x.v[i][e] = *(const uint4_t *)(c.v_codes + (size_t)at.block[i] * code_words + (size_t)at.slot[i] * D::kWords + value_offset + e * D::kSetWords * 4);
    };

    const int limit = position_limit(a);
    float4_t acc[D::kSets][D::kNibbles] = {};
    float acc_min[G][4] = {}, sum[4] = {}, top[4], base[4];
#pragma unroll
    for (int r = 0; r < 4; r++) top[r] = base[r] = kEmpty;
    int power = -24;            // 2^power is at least every step of the values seen so far
    uint32_t power_bits = 0;    // ... as fp16 bits (steps are positive: their bits compare as the numbers do)
    const float c_min = a.scale * 1.44269504088896f, c_even = c_min * 16777216.0f, c_odd = c_min * 1048576.0f;
    unsigned char *mine = lds + wave * D::kWaveBytes;

    auto work = [&](const typename D::Keys &x, const typename D::Values &y, uint32_t pages, int step, bool whole) {
        float raw[D::kPasses][4], most = -INFINITY;
        uint32_t vm[D::kPasses][G], largest = 0, sees = ~0u;  // sees: bit 4 p + r
#pragma unroll
        for (int p = 0; p < D::kPasses; p++) {
            float4_t d[G];
#pragma unroll
            for (int pair = 0; pair < G / 2; pair++)
#pragma unroll
                for (int u = 0; u < D::kPack; u++) {
                    const uint32_t w0 = x.k[p * D::kPack + u][2 * pair], w1 = x.k[p * D::kPack + u][2 * pair + 1];
                    const uint4_t even = {w0 & kEvenCodes, w0 >> 8 & kEvenCodes, w1 & kEvenCodes, w1 >> 8 & kEvenCodes};
                    const uint4_t odd = {w0 & kOddCodes, w0 >> 8 & kOddCodes, w1 & kOddCodes, w1 >> 8 & kOddCodes};
                    const float4_t d0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(q[2 * pair], __builtin_bit_cast(half8_t, even), float4_t{}, 0, 0, 0);
                    const float4_t d1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(q[2 * pair + 1], __builtin_bit_cast(half8_t, odd), float4_t{}, 0, 0, 0);
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        d[2 * pair][r] = u == 0 || pack == u ? d0[r] : d[2 * pair][r];
                        d[2 * pair + 1][r] = u == 0 || pack == u ? d1[r] : d[2 * pair + 1][r];
                    }
                    if (u & 1) __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
            for (int g = 0; g < G; g++) vm[p][g] = x.vm[p][g];
            if (!whole) {
                const int at = step * D::kStep + 16 * (p * D::kPack + pack) + t16;
                const bool there = (pages >> (p * D::kPack + pack) & 1) && at < limit;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const bool one = there && at <= pos[r] && (a.window == 0 || at > pos[r] - a.window);
                    sees &= ~((uint32_t)!one << (4 * p + r));
                }
#pragma unroll
                for (int g = 0; g < G; g++) vm[p][g] = sees >> (4 * p) & 15 ? vm[p][g] : 0;  // what lies there must not reach the powers below
            }
#pragma unroll
            for (int r = 0; r < 4; r++) {
                float even = 0, odd = 0, low = 0;
#pragma unroll
                for (int g = 0; g < G; g++) {
                    if (g & 1) odd = __builtin_fmaf(low_half(x.km[p][g]), d[g][r], odd);
                    else even = __builtin_fmaf(low_half(x.km[p][g]), d[g][r], even);
                    low = __builtin_fmaf(high_half(x.km[p][g]), q_sum[g][r], low);
                }
                raw[p][r] = __builtin_fmaf(even, c_even, __builtin_fmaf(odd, c_odd, low * c_min));
                raw[p][r] = sees >> (4 * p + r) & 1 ? raw[p][r] : -INFINITY;
                most = fmaxf(most, raw[p][r] - base[r]);
            }
#pragma unroll
            for (int g = 0; g < G; g++) largest = max(largest, vm[p][g] & 0xFFFFu);
        }
        const bool grown = most > (float)(kHeadroom + kTopPower - power) || largest > power_bits;
            if (__ballot(grown)) {
                // rare after the first steps: new bases (a base is the row's largest score so far, moved by the powers)
                int bits = (int)largest;
#pragma unroll
                for (int off = 1; off < kWave; off <<= 1) bits = max(bits, __shfl_xor(bits, off, kWave));
                if ((uint32_t)bits > power_bits) {
                    if (bits > 0x7BFF) bits = 0x7BFF;  // (infinite or NaN: the weights carry it on)
                    int e;
                    frexpf(h2f((uint16_t)bits), &e);  // steps <= 2^e
                    power = e;
                    power_bits = e > 15 ? 0x7BFFu : f2h(ldexpf(1.0f, e));
                }
                float keep[4];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    float m = raw[0][r];
#pragma unroll
                    for (int p = 1; p < D::kPasses; p++) m = fmaxf(m, raw[p][r]);
#pragma unroll
                    for (int off = 1; off < 16; off <<= 1) m = fmaxf(m, __shfl_xor(m, off, kWave));
#pragma unroll
                    for (int off = 4 * kRows; off < kWave; off <<= 1) m = fmaxf(m, __shfl_xor(m, off, kWave));
                    top[r] = fmaxf(top[r], m);
                    const float now = top[r] + (float)(power - kTopPower);
                    keep[r] = __builtin_amdgcn_exp2f(base[r] - now);
                    base[r] = now;
                    sum[r] *= keep[r];
#pragma unroll
                    for (int g = 0; g < G; g++) acc_min[g][r] *= keep[r];
                }
                const int row = t16 % kRows;
                float column = 0;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float k = __shfl(keep[r], (row >> 2) * 16, kWave);
                    column = (row & 3) == r ? k : column;
                }
#pragma unroll
                for (int e = 0; e < D::kSets; e++)
#pragma unroll
                    for (int i = 0; i < D::kNibbles; i++) acc[e][i] *= column;
            }
#pragma unroll
        for (int p = 0; p < D::kPasses; p++) {
            float w[4];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                w[r] = __builtin_amdgcn_exp2f(raw[p][r] - base[r]);
                sum[r] += w[r];
            }
            unsigned char *at = mine + (16 * (p * D::kPack + pack) + t16) * D::kRowBytes + row_quad * 8;
            auto weigh = [&](auto keep) {
#pragma unroll
                for (int g = 0; g < G; g++) {
                    const float low = __builtin_fmaf(low_half(vm[p][g]), 8.0f, high_half(vm[p][g]));  // of code 8
                    float ws[4];
                    uint32_t hi[2], lo[2];
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        ws[r] = keep(r, w[r] * low_half(vm[p][g]), 0.0f);
                        acc_min[g][r] = keep(r, __builtin_fmaf(w[r], low, acc_min[g][r]), acc_min[g][r]);
                    }
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        // (both to nearest: the codes are all positive, so a bias of 2^-22 would add up over a long context
                        // to more than what is left of the values' average, 2^-22 * 2 sqrt(positions))
                        const half2_t h = {(_Float16)ws[2 * j], (_Float16)ws[2 * j + 1]};
                        const half2_t l = {(_Float16)(ws[2 * j] - (float)h[0]), (_Float16)(ws[2 * j + 1] - (float)h[1])};
                        hi[j] = __builtin_bit_cast(uint32_t, h);
                        lo[j] = __builtin_bit_cast(uint32_t, l);
                    }
                    *(uint2_t *)(at + g * kRows * 2) = uint2_t{hi[0], hi[1]};
                    *(uint2_t *)(at + D::kColumns * 2 + g * kRows * 2) = uint2_t{lo[0], lo[1]};
                }
            };
            // (what a row does not see may be anything, NaN too, also where another row sees it: taken out by choice, not by a zero)
            if (whole) weigh([](int, float x, float) { return x; });
            else weigh([&](int r, float x, float other) { return sees >> (4 * p + r) & 1 ? x : other; });
        }
        // (the lanes read each other's weights: the wave's LDS accesses run in order, the compiler has to keep it)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int half = 0; half < D::kTiles / 2; half++) {
            half8_t weights[D::kSets][2];
#pragma unroll
            for (int e = 0; e < D::kSets; e++)
#pragma unroll
                for (int piece = 0; piece < 2; piece++) {
                    short4_t two[2];
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        unsigned char *from = mine + (16 * (2 * half + i) + 4 * quad + (lane >> 2 & 3)) * D::kRowBytes + piece * D::kColumns * 2 + e * 32 + (lane & 3) * 8;
                        two[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t *)from);
                    }
                    struct Both { short4_t x[2]; } both = {{two[0], two[1]}};
                    weights[e][piece] = __builtin_bit_cast(half8_t, both);
                }
#pragma unroll
            for (int e = 0; e < D::kSets; e++) {
                const uint4_t va = y.v[2 * half][e], vb = y.v[2 * half + 1][e];
                constexpr int kPieces = D::kNibbles == 8 ? 2 : 1;
#pragma unroll
                for (int piece = 0; piece < kPieces; piece++) {
                    // one 16-bit piece of two positions' words side by side (a byte where four lanes share a word)
                    uint32_t select;
                    if constexpr (D::kNibbles == 8) select = piece ? 0x07060302u : 0x05040100u;
                    else if constexpr (D::kNibbles == 4) select = t16 & 1 ? 0x07060302u : 0x05040100u;
                    else select = 0x0C000C00u | (uint32_t)((t16 & 3) + 4) << 16 | (uint32_t)(t16 & 3);
                    const uint32_t pairs[4] = {__builtin_amdgcn_perm(va[1], va[0], select), __builtin_amdgcn_perm(va[3], va[2], select),
                                               __builtin_amdgcn_perm(vb[1], vb[0], select), __builtin_amdgcn_perm(vb[3], vb[2], select)};
#pragma unroll
                    for (int i = 0; i < (D::kNibbles < 4 ? D::kNibbles : 4); i++) {
                        half8_t codes;
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const uint32_t field = i & 2 ? pairs[j] >> 8 : pairs[j];
                            const half2_t two = __builtin_bit_cast(half2_t, i & 1 ? (field & kOddCodes) | kOddBits : (field & kEvenCodes) | kEvenBits) -
                                                (i & 1 ? half2_t{72, 72} : half2_t{1032, 1032});
                            codes[2 * j] = two[0];
                            codes[2 * j + 1] = two[1];
                        }
                        float4_t &into = acc[e][piece * 4 + i];
                        into = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes, weights[e][0], into, 0, 0, 0);
                        into = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes, weights[e][1], into, 0, 0, 0);
                        if (i & 1) __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };

    const int end = min(span.first + span.steps, span.first + (part + 1) * span.per);
    int step = span.first + part * span.per + wave;
    for (; step < end; step += kWaves) {
        const typename D::Places at = find(step);
        typename D::Keys keys;
        typename D::Values values;
        load_keys(keys, at);
        load_values(values, at);
        const int first = step * D::kStep;
        const bool whole = at.there == (1u << D::kTiles) - 1 && first + D::kStep - 1 <= pos_low && first + D::kStep <= limit &&
                           (a.window == 0 || first > pos_high - a.window);
        work(keys, values, at.there, step, whole);
    }

    // ---- the wave's sums over its lanes
#pragma unroll
    for (int r = 0; r < 4; r++) {
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) {
            sum[r] += __shfl_xor(sum[r], off, kWave);
#pragma unroll
            for (int g = 0; g < G; g++) acc_min[g][r] += __shfl_xor(acc_min[g][r], off, kWave);
        }
#pragma unroll
        for (int off = 4 * kRows; off < kWave; off <<= 1) {
            sum[r] += __shfl_xor(sum[r], off, kWave);
#pragma unroll
            for (int g = 0; g < G; g++) acc_min[g][r] += __shfl_xor(acc_min[g][r], off, kWave);
        }
    }
    if (t16 == 0 && pack == 0) {
#pragma unroll
        for (int r = 0; r < 4; r++) {
            join_base[wave][4 * row_quad + r] = base[r];
            join_sum[wave][4 * row_quad + r] = sum[r];
        }
    }
    // this lane's column is (group in the set, row): the minima's share of each set's group
    const int row = t16 % kRows, in_set = t16 / kRows;
    float low[D::kSets];
#pragma unroll
    for (int e = 0; e < D::kSets; e++) {
        low[e] = 0;
#pragma unroll
        for (int g = 0; g < D::kSetGroups; g++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float v = __shfl(acc_min[e * D::kSetGroups + g][r], (row >> 2) * 16, kWave);
                if (in_set == g && (row & 3) == r) low[e] = v;
            }
    }
    __syncthreads();  // (also: every wave is through with its weights in LDS)
    float highest = kEmpty;
#pragma unroll
    for (int w = 0; w < kWaves; w++) highest = fmaxf(highest, join_base[w][row]);
    const float mine_keep = __builtin_amdgcn_exp2f(join_base[wave][row] - highest);
    float *out = (float *)lds + (size_t)wave * kRows * kDim + row * kDim;
#pragma unroll
    for (int e = 0; e < D::kSets; e++)
#pragma unroll
        for (int i = 0; i < D::kNibbles; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int n = 4 * quad + r;  // the operand's row: word n / kLanesPerWord of the set, nibble part n % kLanesPerWord
                const int dim = (e * D::kSetWords + n / D::kLanesPerWord) * 8 + n % D::kLanesPerWord * D::kNibbles + i;
                const float v = acc[e][i][r] + low[e];
                if (in_set < D::kSetGroups && dim / 32 - e * D::kSetGroups == in_set) out[dim] = v * mine_keep;
            }
    __syncthreads();
    constexpr int kParts = kDim / 4;  // float4s of a row
    for (int j = threadIdx.x; j < kRows * kParts; j += kThreads) {
        const int r = j / kParts, d = j % kParts * 4;
        if (r >= rows_left) break;
        float4_t o = {};
        float m = kEmpty, total = 0;
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            o += *(const float4_t *)((const float *)lds + (size_t)w * kRows * kDim + r * kDim + d);
            m = fmaxf(m, join_base[w][r]);
        }
#pragma unroll
        for (int w = 0; w < kWaves; w++) total += join_sum[w][r] * __builtin_amdgcn_exp2f(join_base[w][r] - m);
        const int at = first_row + r;
        const size_t query = (size_t)(s.row0 + at / heads);
        const int head = kv * heads + at % heads;
        if (plan.splits == 1) {
            const float inv = total == 0.0f ? 0.0f : 1.0f / total;  // nothing seen: 0
            const uint2_t packed = {(uint32_t)f2h(o[0] * inv) | (uint32_t)f2h(o[1] * inv) << 16, (uint32_t)f2h(o[2] * inv) | (uint32_t)f2h(o[3] * inv) << 16};
            *(uint2_t *)(a.output + query * a.output_stride + (size_t)head * kDim + d) = packed;
        } else {
            const size_t slot = (query * a.n_heads + head) * plan.splits + part;
            float *base_sum = (float *)a.workspace + (size_t)a.batch.n_tokens * a.n_heads * plan.splits * kDim + slot * 2;
            if (d == 0) base_sum[0] = m, base_sum[1] = total;
            *(float4_t *)((float *)a.workspace + slot * kDim + d) = o;
        }
    }
}

// Joins the parts of one (query row, head): a workgroup each, 16 bytes per lane, kDim / 4 lanes per part.
template <int kDim>
__global__ __launch_bounds__(kThreads) void attention_join_kernel(const AttentionKv4Args a, const SplitPlan plan, int rows_per_tile, int step) {
    constexpr int kLanes = kDim / 4, kAtOnce = kThreads / kLanes;
    __shared__ float weight[kMostSplits];
    __shared__ float4_t sums[kAtOnce][kLanes];
    const int row = blockIdx.x, head = blockIdx.y;
    const int seq = kv4_find_sequence(a.batch.starts, a.batch.batch, row);
    if (seq >= a.batch.batch) return;
    const Sequence s(a, seq);
    const int i = row - s.row0;
    if (i < 0 || i >= s.rows) return;
    const int heads = a.n_heads / a.cache.n_kv_heads;
    const int first_row = (i * heads + head % heads) / rows_per_tile * rows_per_tile, last_row = min(first_row + rows_per_tile, s.rows * heads) - 1;
    const Span span(window_begin(a, s.pos0 + first_row / heads), min(s.pos0 + last_row / heads + 1, position_limit(a)), step, plan.splits);
    const size_t slot = ((size_t)row * a.n_heads + head) * plan.splits;
    const float *base_sum = (const float *)a.workspace + (size_t)a.batch.n_tokens * a.n_heads * plan.splits * kDim + slot * 2;
    float m = kEmpty, total = 0;
    for (int p = 0; p < span.used; p++) m = fmaxf(m, base_sum[2 * p]);
    for (int p = 0; p < span.used; p++) total += base_sum[2 * p + 1] * __builtin_amdgcn_exp2f(base_sum[2 * p] - m);
    if (threadIdx.x < span.used) weight[threadIdx.x] = __builtin_amdgcn_exp2f(base_sum[2 * threadIdx.x] - m);
    __syncthreads();
    const int at = threadIdx.x / kLanes, d = threadIdx.x % kLanes;
    const float4_t *parts = (const float4_t *)((const float *)a.workspace + slot * kDim);
    float4_t o = {};
    for (int p = at; p < span.used; p += kAtOnce) o += parts[(size_t)p * kLanes + d] * weight[p];
    sums[at][d] = o;
    __syncthreads();
    if (at) return;
#pragma unroll
    for (int j = 1; j < kAtOnce; j++) o += sums[j][d];
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    const uint2_t packed = {(uint32_t)f2h(o[0] * inv) | (uint32_t)f2h(o[1] * inv) << 16, (uint32_t)f2h(o[2] * inv) | (uint32_t)f2h(o[3] * inv) << 16};
    *(uint2_t *)(a.output + (size_t)row * a.output_stride + (size_t)head * kDim + d * 4) = packed;
}

int decode_rows(const AttentionKv4Args &a) {
    const long long rows = (long long)a.max_query * (a.n_heads / a.cache.n_kv_heads);
    return rows <= 4 ? 4 : rows <= 8 ? 8 : 16;
}

SplitPlan decode_plan(const AttentionKv4Args &a) {
    const int rows = decode_rows(a), step = rows == 16 ? 32 : 64;
    const long long heads = a.n_heads / a.cache.n_kv_heads;
    SplitPlan p;
    p.row_tiles = (int)((a.max_query * heads + rows - 1) / rows);
    long long reach = a.max_length;
    if (a.window > 0 && (long long)a.window + a.max_query + step < reach) reach = (long long)a.window + a.max_query + step;
    const long long groups = (long long)p.row_tiles * a.cache.n_kv_heads * a.batch.batch;
    const long long want = (4ll * current_device_cus() + groups - 1) / groups, most = (reach + kWaves * step - 1) / (kWaves * step);
    long long n = want < most ? want : most;
    p.splits = (int)(n < 1 ? 1 : n > kMostSplits ? kMostSplits : n);
    return p;
}

template <int kDim>
hipError_t launch_decode(const AttentionKv4Args &a, hipStream_t s) {
    const SplitPlan plan = decode_plan(a);
    const int rows = decode_rows(a);
    const dim3 grid((unsigned)(a.cache.n_kv_heads * plan.splits) * (unsigned)plan.row_tiles, (unsigned)a.batch.batch);
    if (rows == 4) attention_decode_kernel<kDim, 4><<<grid, kThreads, 0, s>>>(a, plan);
    else if (rows == 8) attention_decode_kernel<kDim, 8><<<grid, kThreads, 0, s>>>(a, plan);
    else attention_decode_kernel<kDim, 16><<<grid, kThreads, 0, s>>>(a, plan);
    if (hipError_t e = hipGetLastError()) return e;
    if (plan.splits > 1) {
        attention_join_kernel<kDim><<<dim3((unsigned)a.batch.n_tokens, (unsigned)a.n_heads), kThreads, 0, s>>>(a, plan, rows, rows == 16 ? 32 : 64);
        return hipGetLastError();
    }
    return hipSuccess;
}

}  // namespace

size_t attention_kv4_workspace(const AttentionKv4Args &a) {
    const SplitPlan plan = decode_plan(a);
    return plan.splits == 1 ? 0 : (size_t)a.batch.n_tokens * a.n_heads * plan.splits * (a.cache.head_dim + 2) * 4;
}

hipError_t launch_attention_kv4(const AttentionKv4Args &a, hipStream_t s) {
    return a.cache.head_dim == 64 ? launch_decode<64>(a, s) : launch_decode<128>(a, s);
}

}  // namespace tllm
