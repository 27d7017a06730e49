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
#include <algorithm>

#include "kv4.h"

namespace tllm {
namespace {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef uint32_t uint4_t __attribute__((ext_vector_type(4)));
typedef uint32_t uint2_t __attribute__((ext_vector_type(2)));

constexpr float kEmpty = -1e30f;  // below every score (|q.k| < 2^40, |scale| <= 2^40): no position yet
constexpr int kHeadroom = 6;      // powers of two that a weight may outgrow its base by before everything is rescaled
constexpr int kTopPower = 8;      // a base puts the largest weight seen (times its step) at 2^kTopPower
constexpr uint32_t kEvenCodes = 0x000F000Fu, kOddCodes = 0x00F000F0u;
// The values' codes are all brought to bits 4-7, and every second position's enter as 15 - c with a negative weight (15 p s
// goes to the minima's sum). The matrix unit lines products up by their operands' exponents, of which a subnormal has the
// smallest however few bits it fills, and cuts what falls off: with codes in bits 0-3 sums come out 2^-22 too low, which
// positive codes add up to 2 sqrt(positions) times what is left of the values in the end (4e-4 of the result at 131072
// positions). Scores, sums of 128 products with their signs, do not feel it.
constexpr uint32_t kSecondFlipped = 0xFFFF0000u;

__device__ __forceinline__ float low_half(uint32_t w) { return h2f((uint16_t)w); }
__device__ __forceinline__ float high_half(uint32_t w) { return h2f((uint16_t)(w >> 16)); }

// Sums and maxima over the 16 lanes of a quad, in every lane (rotations inside the quad), and over all lanes.
template <int kBy>
__device__ __forceinline__ float rotated(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 + kBy, 0xF, 0xF, false));
}
__device__ __forceinline__ float quad_sum(float v) {
    v += rotated<8>(v);
    v += rotated<4>(v);
    v += rotated<2>(v);
    return v + rotated<1>(v);
}
// Sum over the lanes up to and including this one.
template <int kControl, int kRows>
__device__ __forceinline__ int shifted(int v) {
    return __builtin_amdgcn_update_dpp(0, v, kControl, kRows, 0xF, false);
}
__device__ __forceinline__ int running_sum(int v) {
    v += shifted<0x111, 0xF>(v);  // by 1, 2, 4, 8 lanes inside each quad
    v += shifted<0x112, 0xF>(v);
    v += shifted<0x114, 0xF>(v);
    v += shifted<0x118, 0xF>(v);
    v += shifted<0x142, 0xA>(v);  // the last lane of quads 0 and 2 to quads 1 and 3
    return v + shifted<0x143, 0xC>(v);  // lane 31 to quads 2 and 3
}
__device__ __forceinline__ float quad_max(float v) {
    v = fmaxf(v, rotated<8>(v));
    v = fmaxf(v, rotated<4>(v));
    v = fmaxf(v, rotated<2>(v));
    return fmaxf(v, rotated<1>(v));
}

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
// Bound: HBM, the cache's 5 bits per value; the work per position has to stay small beside it, above all the work on scores,
// of which 16 x 16 come out of every matrix instruction however few rows there are. So the row operand repeats its kRows
// rows (query rows times the heads that share a kv head: 4, 8 or 16), and of kPack = 16 / kRows tiles of 16 positions each
// quad of lanes keeps the results of its own tile: each of the 64 lanes then has ONE position and four rows of its own (lane
// = (position t, quad)), steps and minima are one coalesced word per lane and group, and softmax runs on four registers. For
// the values, weights p s go through LDS ([position][group][row], fp16) and come back transposed (ds_read_b64_tr_b16) with
// (group, row) pairs as the 16 columns of the operand: one instruction multiplies a row tile's weights of all groups in the
// set, of which each dim uses its own group's.
//
// The positions of all sequences are one line of steps, cut into equal pieces, one per wave (each kv head its own line):
// however ragged the batch, all waves end together. A piece may end inside a sequence and begin inside another; its stretch
// of a sequence is a segment. A sequence that lies in one piece is stored at once, the segments of others are joined by a
// second launch. A wave is a workgroup of its own: nothing waits for another wave. Short contexts (at most kAloneSteps steps)
// take the other form: a workgroup of kAloneWaves waves has a whole row tile, the waves take its steps in turn and meet in
// LDS, and there is no second launch (517 positions, 8 kv heads: 11 us and 8 + 4 us).
constexpr int kAloneWaves = 8, kAloneSteps = 16;
struct DecodePlan {
    int workers;  // waves per kv head
    int tiles;    // row tiles per sequence; row tile t of sequence b is number b * tiles + t of the line
    int least;    // steps that a piece has at least
    int alone;    // every workgroup has a whole row tile (no second launch)
};

template <int kDim, int kRows>
struct Decode {
    static constexpr int kGroups = kDim / kKvGroup, kWords = kDim / 8;
    static constexpr int kPack = 16 / kRows;
    static constexpr int kTiles = kRows == 4 ? 4 : 2, kStep = 16 * kTiles, kPasses = kTiles / kPack;
    static constexpr int kColumns = kGroups * kRows < 16 ? 16 : kGroups * kRows;  // of the weights: (group, row)
    static constexpr int kSets = kColumns / 16, kSetGroups = kGroups / kSets;
    static constexpr int kSetWords = 4 * kSetGroups, kLanesPerWord = 16 / kSetWords, kNibbles = 8 / kLanesPerWord;
    static constexpr int kRowBytes = 4 * kColumns + 16;  // of a position's weights in LDS: both pieces, 16 bytes off a power of two
    static constexpr int kLds = kStep * kRowBytes;
    static_assert(kLds >= 4 * (kGroups * 4 + 8) * 4, "the sums of four quads");
    using KeyWords = typename std::conditional<kGroups == 4, uint4_t, uint2_t>::type;
    struct Places {
        uint32_t block[kTiles], slot[kTiles];  // of each tile of 16 positions: page * n_kv_heads + head, first slot
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

// One row tile: its rows and the steps of positions that some row of it sees.
struct RowTile {
    int row0, rows_left, first_row, pos0, pos_low, pos_high, first_step, steps;
    __device__ RowTile(const AttentionKv4Args &a, const DecodePlan &plan, int number, int rows_per_tile, int step) {
        const int seq = plan.tiles == 1 ? number : number / plan.tiles, tile = plan.tiles == 1 ? 0 : number - seq * plan.tiles;
        const int heads = a.n_heads / a.cache.n_kv_heads;
        const Sequence s(a, seq);
        row0 = s.row0;
        pos0 = s.pos0;
        first_row = tile * rows_per_tile;
        rows_left = s.rows * heads - first_row;
        pos_low = s.pos0 + first_row / heads;
        pos_high = s.pos0 + (first_row + min(rows_left, rows_per_tile) - 1) / heads;
        const int lo = window_begin(a, pos_low), hi = min(pos_high + 1, position_limit(a));
        first_step = lo / step;
        steps = rows_left > 0 && hi > lo ? (hi + step - 1) / step - first_step : 0;
    }
    RowTile() = default;
    __device__ RowTile of_lane(int lane) const {
        RowTile t;
        t.row0 = __builtin_amdgcn_readlane(row0, lane);
        t.rows_left = __builtin_amdgcn_readlane(rows_left, lane);
        t.first_row = __builtin_amdgcn_readlane(first_row, lane);
        t.pos0 = __builtin_amdgcn_readlane(pos0, lane);
        t.pos_low = __builtin_amdgcn_readlane(pos_low, lane);
        t.pos_high = __builtin_amdgcn_readlane(pos_high, lane);
        t.first_step = __builtin_amdgcn_readlane(first_step, lane);
        t.steps = __builtin_amdgcn_readlane(steps, lane);
        return t;
    }
};

// Where segments and what joins them lie in the workspace. A segment has the number worker + row tile (unique: from one
// segment to the next of a line one of the two grows): kRows rows of kDim sums, then their (base, sum).
struct Segments {
    float *sums, *bases;
    int2 *parts;  // of each row tile: first worker, and how many (0: it sees nothing)
    int per_head;
    __host__ __device__ Segments(const AttentionKv4Args &a, const DecodePlan &plan, int rows) {
        const int numbers = a.batch.batch * plan.tiles;
        per_head = plan.workers + numbers;
        const size_t all = (size_t)a.cache.n_kv_heads * per_head * rows;
        sums = (float *)a.workspace;
        bases = sums + all * a.cache.head_dim;
        parts = (int2 *)(bases + all * 2);
    }
    __host__ __device__ static size_t bytes(const AttentionKv4Args &a, const DecodePlan &plan, int rows) {
        const size_t numbers = (size_t)a.batch.batch * plan.tiles;
        return (size_t)a.cache.n_kv_heads * (plan.workers + numbers) * rows * (a.cache.head_dim + 2) * 4 + numbers * 8;
    }
};

__device__ __forceinline__ void store_row(const AttentionKv4Args &a, size_t query, int head, int d, float4_t o, float total) {
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;  // nothing seen: 0
    const uint2_t packed = {(uint32_t)f2h(o[0] * inv) | (uint32_t)f2h(o[1] * inv) << 16, (uint32_t)f2h(o[2] * inv) | (uint32_t)f2h(o[3] * inv) << 16};
    *(uint2_t *)(a.output + query * a.output_stride + (size_t)head * a.cache.head_dim + d) = packed;
}

template <int kDim, int kRows, int kWaves>
__global__ __launch_bounds__(kWaves *kWave, 2) void attention_decode_kernel(const AttentionKv4Args a, const DecodePlan plan) {
    using D = Decode<kDim, kRows>;
    constexpr int G = D::kGroups;
    constexpr bool kAlone = kWaves > 1;
    constexpr int kJoin = kAlone ? kWaves * kRows * kDim * 4 : 0;
    __shared__ __align__(16) unsigned char lds_all[kWaves * D::kLds > kJoin ? kWaves * D::kLds : kJoin];
    __shared__ float2 join_bases[kAlone ? kWaves : 1][kRows];
    const Kv4Cache &c = a.cache;
    const int lane = threadIdx.x % kWave, quad = lane >> 4, t16 = lane & 15;
    const int wave = kAlone ? __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) : 0;
    unsigned char *lds = lds_all + wave * D::kLds;
    const int kv = blockIdx.x, worker = blockIdx.y + blockIdx.z * gridDim.y;  // kv fastest: a head's pieces fall on the same XCDs
    if (worker >= plan.workers) return;
    const int heads = a.n_heads / c.n_kv_heads, numbers = a.batch.batch * plan.tiles;

    // this wave's piece of the line, and the row tile that it begins in
    int number = worker, offset = 0, left = INT32_MAX;
    RowTile tile;
    if constexpr (kAlone) {
        tile = RowTile(a, plan, number, kRows, D::kStep);
        if (tile.rows_left <= 0) return;
    } else {
        int total = 0;
        RowTile own;
        const auto running = [&](int base) {
            own.steps = 0;
            if (base + lane < numbers) own = RowTile(a, plan, base + lane, kRows, D::kStep);
            return running_sum(own.steps);
        };
        int upto = 0;
        for (int base = 0; base < numbers; base += kWave) {
            upto = running(base);
            total += __builtin_amdgcn_readlane(upto, kWave - 1);
        }
        const int per = max(plan.least, (total + plan.workers - 1) / plan.workers);
        const long long begin = (long long)worker * per;
        const bool scribe = kv == 0 && worker == 0;
        left = (int)min((long long)per, total - begin);
        if (left <= 0 && !scribe) return;
        const Segments segments(a, plan, kRows);
        int before = 0, at = -1;
        for (int base = 0; base < numbers && (at < 0 || scribe); base += kWave) {
            if (numbers > kWave) upto = running(base);
            const int from = before + upto - own.steps;
            if (scribe && base + lane < numbers)
                segments.parts[base + lane] = make_int2(from / per, own.steps ? (from + own.steps - 1) / per - from / per + 1 : 0);
            const unsigned long long here = __ballot(at < 0 && own.steps > 0 && begin >= from && begin < from + own.steps);
            if (here) {
                const int l = __builtin_amdgcn_readfirstlane(__ffsll(here) - 1);
                at = base + l;
                offset = (int)begin - __builtin_amdgcn_readlane(from, l);
                tile = own.of_lane(l);
            }
            before += __builtin_amdgcn_readlane(upto, kWave - 1);
        }
        if (left <= 0) return;  // (nothing at all to see)
        number = __builtin_amdgcn_readfirstlane(at);
        left = __builtin_amdgcn_readfirstlane(left);
    }

    const int limit = position_limit(a);
    const int row_quad = quad % (kRows / 4), pack = quad / (kRows / 4);  // this lane's results: rows 4 * row_quad + r of tile `pack`
    const size_t code_words = kv4_code_words(1 << c.page_shift, kDim), scale_words = kv4_scale_words(1 << c.page_shift, kDim);
    // this lane's bytes in a tile: its position's words of its depth, four positions of its word, its position's step and minimum
    const uint32_t key_offset = (uint32_t)(t16 * D::kWords + quad * G) * 4;
    const uint32_t value_offset = (uint32_t)(quad * (D::kWords * 4) + (t16 / D::kLanesPerWord) * 4) * 4;
    const uint32_t scale_offset = (uint32_t)(16 * pack + t16) * 4;
    const float sign = t16 & 1 ? -1.0f : 1.0f, flipped = t16 & 1 ? 15.0f : 0.0f;  // of this lane's positions
    float minus_one = -1.0f;  // (a variable: the product with it is folded into a mixed-precision instruction, a difference is not)
    asm("" : "+v"(minus_one));
    const float c_low = a.scale * 1.44269504088896f, c_even = c_low * 16777216.0f, c_odd = c_low * 1048576.0f;

    while (true) {
        const int count = min(tile.steps - offset, left);
        const bool entire = kAlone || (offset == 0 && count == tile.steps);
        const int *table = a.batch.table + (size_t)(plan.tiles == 1 ? number : number / plan.tiles) * a.batch.width;

        // 64 entries of the page table at a time, one per lane: a step's pages are then a lane read away (a load of their own
        // would stand in front of every step's loads)
        int held_from = (tile.first_step + offset) * D::kStep >> c.page_shift, held = table[min(held_from + lane, a.batch.width - 1)];
        auto find = [&](int step) {
            typename D::Places x;
            const int at = step * D::kStep, last = (at + 16 * (D::kTiles - 1)) >> c.page_shift;
            if (last >= held_from + kWave) {
                held_from = at >> c.page_shift;
                held = table[min(held_from + lane, a.batch.width - 1)];
            }
            x.there = 0;
#pragma unroll
            for (int i = 0; i < D::kTiles; i++) {
                const int index = (at + 16 * i) >> c.page_shift;
                const int page = __builtin_amdgcn_readlane(held, index - held_from);
                const bool there = index < a.batch.width && page >= 0 && page < c.n_pages;
                x.there |= (uint32_t)there << i;
                x.block[i] = (there ? page : 0) * c.n_kv_heads + kv;
                x.slot[i] = (at + 16 * i) & ((1 << c.page_shift) - 1);
            }
            return x;
        };
        const bool one_page = 1 << c.page_shift >= D::kStep;  // a step's positions lie in one page
        const auto bytes = [](const void *at, size_t words) { return (const unsigned char *)at + words * 4; };
        auto load_keys = [&](typename D::Keys &x, const typename D::Places &at) {
#pragma unroll
            for (int i = 0; i < D::kTiles; i++)
                x.k[i] = *(const typename D::KeyWords *)(bytes(c.k_codes, at.block[i] * code_words + (size_t)at.slot[i] * D::kWords) + key_offset);
            if (one_page) {
                const size_t word = at.block[0] * scale_words + at.slot[0];
#pragma unroll
                for (int g = 0; g < G; g++)
#pragma unroll
                    for (int p = 0; p < D::kPasses; p++) {
                        x.km[p][g] = *(const uint32_t *)(bytes(c.k_scales, word + ((size_t)g << c.page_shift)) + scale_offset + p * D::kPack * 64);
                        x.vm[p][g] = *(const uint32_t *)(bytes(c.v_scales, word + ((size_t)g << c.page_shift)) + scale_offset + p * D::kPack * 64);
                    }
            } else {
#pragma unroll
                for (int p = 0; p < D::kPasses; p++) {
                    uint32_t b = at.block[p * D::kPack], sl = at.slot[p * D::kPack];
#pragma unroll
                    for (int u = 1; u < D::kPack; u++)
                        if (pack == u) b = at.block[p * D::kPack + u], sl = at.slot[p * D::kPack + u];
                    const size_t word = b * scale_words + sl + t16;
#pragma unroll
                    for (int g = 0; g < G; g++) {
                        x.km[p][g] = c.k_scales[word + ((size_t)g << c.page_shift)];
                        x.vm[p][g] = c.v_scales[word + ((size_t)g << c.page_shift)];
                    }
                }
            }
        };
        auto load_values = [&](typename D::Values &x, const typename D::Places &at) {
#pragma unroll
            for (int i = 0; i < D::kTiles; i++)
#pragma unroll
                for (int e = 0; e < D::kSets; e++)
                    x.v[i][e] = *(const uint4_t *)(bytes(c.v_codes, at.block[i] * code_words + (size_t)at.slot[i] * D::kWords + e * D::kSetWords * 4) + value_offset);
        };

        int step = tile.first_step + offset + wave;
        const int end = tile.first_step + offset + count;
        // row operands: this lane's row and its 8 dims of each group; and the groups' sums, which the minima multiply, as one
        // more operand: first and second fp16 piece of sum / 32 at the depth of the quad that holds the minima of the row's tile
        // (rows that are not there are zeros; what they see shows in their own columns only)
        half8_t q[G], q_sums = {};
        {
            const int row = t16 % kRows, at_row = tile.first_row + row;
            const bool real = row < tile.rows_left;
            const uint16_t *src = a.q + (size_t)(tile.row0 + (real ? at_row / heads : 0)) * a.q_stride + (size_t)(kv * heads + (real ? at_row % heads : 0)) * kDim + quad * 8;
#pragma unroll
            for (int g = 0; g < G; g++) {
                q[g] = real ? *(const half8_t *)(src + g * 32) : half8_t{};
            }
        }
        typename D::Places at;
        typename D::Keys now;
        if (step < end) {
            at = find(step);
            load_keys(now, at);
        }
        {
#pragma unroll
            for (int g = 0; g < G; g++) {
                float sum = 0;
#pragma unroll
                for (int j = 0; j < 8; j++) sum += (float)q[g][j];
                sum += __shfl_xor(sum, 16, kWave);
                sum += __shfl_xor(sum, 32, kWave);
                sum *= 0.03125f;
                if (quad == t16 / kRows * (kRows / 4)) {
                    q_sums[g] = (_Float16)sum;
                    q_sums[G + g] = (_Float16)(sum - (float)q_sums[g]);
                }
            }
        }

        float4_t acc[D::kSets][D::kNibbles] = {};
        float acc_min[G][4] = {}, sum[4] = {}, base[4] = {kEmpty, kEmpty, kEmpty, kEmpty};
        int power = -24;          // 2^power is at least every step of the values seen so far
        uint32_t power_bits = 0;  // ... as fp16 bits (steps are positive: their bits compare as the numbers do)

        // this step's values, which the work on the scores covers, then the next step's keys
        while (step < end) {
            typename D::Values values;
            load_values(values, at);
            const uint32_t pages = at.there;
            const int first = step * D::kStep;
            typename D::Keys next;
            step += kWaves;
            if (step < end) {
                at = find(step);
                load_keys(next, at);
            }
            // whole: every row sees all of the step's positions
            const bool whole = pages == (1u << D::kTiles) - 1 && first + D::kStep - 1 <= tile.pos_low && first + D::kStep <= limit &&
                               (a.window == 0 || first > tile.pos_high - a.window);
            float raw[D::kPasses][4], most = -INFINITY;
            uint32_t largest = 0, sees = ~0u;  // sees: bit 4 p + r
#pragma unroll
            for (int p = 0; p < D::kPasses; p++) {
                float4_t d[G];
#pragma unroll
                for (int pair = 0; pair < G / 2; pair++)
#pragma unroll
                    for (int u = 0; u < D::kPack; u++) {
                        const uint32_t w0 = now.k[p * D::kPack + u][2 * pair], w1 = now.k[p * D::kPack + u][2 * pair + 1];
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
                bool unsound = false;
                if (!whole) {
                    asm volatile("");  // (a branch: not worked out and chosen from in every step)
                    const int t = first + 16 * (p * D::kPack + pack) + t16;
                    const bool there = (pages >> (p * D::kPack + pack) & 1) && t < limit;
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const int row = 4 * row_quad + r, pos = tile.pos0 + (tile.first_row + row) / heads;
                        const bool one = there && row < tile.rows_left && t <= pos && (a.window == 0 || t > pos - a.window);
                        sees &= ~((uint32_t)!one << (4 * p + r));
                    }
                    // What no row sees may be anything, and must reach neither the powers below nor, in the product of the
                    // minima, the other tiles' positions. Nor must what is not finite and only some rows see reach the others:
                    // a key's rows get their NaN in the scores below, a value's in the sum of its group's minima.
                    const bool any = there && t <= tile.pos_high && (a.window == 0 || t > tile.pos_low - a.window);
#pragma unroll
                    for (int g = 0; g < G; g++) {
                        unsound |= any && (now.km[p][g] & 0x7C000000u) == 0x7C000000u;
                        const bool wrong = any && ((now.vm[p][g] & 0x7C000000u) == 0x7C000000u || (now.vm[p][g] & 0x7C00u) == 0x7C00u);
                        now.vm[p][g] = any && !wrong ? now.vm[p][g] : 0;
#pragma unroll
                        for (int r = 0; r < 4; r++) acc_min[g][r] = wrong && (sees >> (4 * p + r) & 1) ? NAN : acc_min[g][r];
                    }
#pragma unroll
                    for (int g = 0; g < G; g++) now.km[p][g] = any && !unsound ? now.km[p][g] : 0;
                }
                uint4_t minima;
#pragma unroll
                for (int j = 0; j < 4; j++)  // (G is 2: the last four depths have zero rows, and zeros here)
                    minima[j] = G == 4 || j < 2 ? __builtin_amdgcn_perm(now.km[p][2 * j % G + 1], now.km[p][2 * j % G], 0x07060302u) : 0;
                const float4_t low = __builtin_amdgcn_mfma_f32_16x16x32_f16(q_sums, __builtin_bit_cast(half8_t, minima), float4_t{}, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    float even = 0, odd = 0;
#pragma unroll
                    for (int g = 0; g < G; g += 2) {
                        even = __builtin_fmaf(low_half(now.km[p][g]), d[g][r], even);
                        odd = __builtin_fmaf(low_half(now.km[p][g + 1]), d[g + 1][r], odd);
                    }
                    raw[p][r] = __builtin_fmaf(even, c_even, __builtin_fmaf(odd, c_odd, low[r] * (32.0f * c_low)));
                }
                if (!whole) {
                    asm volatile("");
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        raw[p][r] = unsound ? NAN : raw[p][r];
                        raw[p][r] = sees >> (4 * p + r) & 1 ? raw[p][r] : -INFINITY;
                    }
                }
#pragma unroll
                for (int r = 0; r < 4; r++) most = fmaxf(most, raw[p][r] - base[r]);
#pragma unroll
                for (int g = 0; g < G; g++) largest = max(largest, now.vm[p][g] & 0xFFFFu);
            }
            const bool grown = most > (float)(kHeadroom + kTopPower - power) || largest > power_bits;
            if (__ballot(grown)) {
                // rare after the first steps: new bases (a base is the row's largest score so far, moved by the powers)
                int bits = (int)largest;
#pragma unroll
                for (int off = 1; off < kWave; off <<= 1) bits = max(bits, __shfl_xor(bits, off, kWave));
                const float moved = (float)(power - kTopPower);
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
                    m = quad_max(m);
#pragma unroll
                    for (int off = 4 * kRows; off < kWave; off <<= 1) m = fmaxf(m, __shfl_xor(m, off, kWave));
                    const float to = fmaxf(base[r] - moved, m) + (float)(power - kTopPower);
                    keep[r] = __builtin_amdgcn_exp2f(base[r] - to);
                    base[r] = to;
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
                unsigned char *to = lds + (16 * (p * D::kPack + pack) + t16) * D::kRowBytes + row_quad * 8;
#pragma unroll
                for (int g = 0; g < G; g++) {
                    const float size = low_half(now.vm[p][g]) * sign, low = __builtin_fmaf(low_half(now.vm[p][g]), flipped, high_half(now.vm[p][g]));
                    float ws[4];
                    uint32_t hi[2], lo[2];
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        ws[r] = w[r] * size;
                        acc_min[g][r] = __builtin_fmaf(w[r], low, acc_min[g][r]);
                    }
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const half2_t h = {(_Float16)ws[2 * j], (_Float16)ws[2 * j + 1]};
                        const half2_t l = {(_Float16)__builtin_fmaf((float)h[0], minus_one, ws[2 * j]), (_Float16)__builtin_fmaf((float)h[1], minus_one, ws[2 * j + 1])};
                        hi[j] = __builtin_bit_cast(uint32_t, h);
                        lo[j] = __builtin_bit_cast(uint32_t, l);
                    }
                    *(uint2_t *)(to + g * kRows * 2) = uint2_t{hi[0], hi[1]};
                    *(uint2_t *)(to + D::kColumns * 2 + g * kRows * 2) = uint2_t{lo[0], lo[1]};
                }
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
                            unsigned char *from = lds + (16 * (2 * half + i) + 4 * quad + (lane >> 2 & 3)) * D::kRowBytes + piece * D::kColumns * 2 + e * 32 + (lane & 3) * 8;
                            two[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t *)from);
                        }
                        struct Both { short4_t x[2]; } both = {{two[0], two[1]}};
                        weights[e][piece] = __builtin_bit_cast(half8_t, both);
                    }
#pragma unroll
                for (int e = 0; e < D::kSets; e++) {
                    const uint4_t va = values.v[2 * half][e], vb = values.v[2 * half + 1][e];
#pragma unroll
                    for (int byte = 0; byte < D::kNibbles / 2; byte++) {
                        // this lane's byte `byte` of two positions' words, one per half
                        const uint32_t which = (uint32_t)(t16 % D::kLanesPerWord * (D::kNibbles / 2) + byte), select = which * 0x00010001u + 0x0C040C00u;
                        const uint32_t pairs[4] = {__builtin_amdgcn_perm(va[1], va[0], select), __builtin_amdgcn_perm(va[3], va[2], select),
                                                   __builtin_amdgcn_perm(vb[1], vb[0], select), __builtin_amdgcn_perm(vb[3], vb[2], select)};
#pragma unroll
                        for (int odd = 0; odd < 2; odd++) {
                            uint4_t codes;
#pragma unroll
                            for (int j = 0; j < 4; j++) codes[j] = ((odd ? pairs[j] : pairs[j] << 4) ^ kSecondFlipped) & kOddCodes;
                            float4_t &into = acc[e][2 * byte + odd];
                            into = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, codes), weights[e][0], into, 0, 0, 0);
                            into = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, codes), weights[e][1], into, 0, 0, 0);
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            now = next;
        }

        // ---- the sums of weights and minima over the lanes: inside each quad, then through LDS. A lane's results are column
        // (group in the set, row); of its set's groups a dim has one, and all dims of the quad the same: other lanes have none.
        const int row = t16 % kRows, in_set = t16 / kRows;
        constexpr int kQuadFloats = G * 4 + 8;  // minima [group][row], sums, bases
        float *quads = (float *)lds;
#pragma unroll
        for (int r = 0; r < 4; r++) {
            sum[r] = quad_sum(sum[r]);
#pragma unroll
            for (int g = 0; g < G; g++) acc_min[g][r] = quad_sum(acc_min[g][r]);
        }
        if (t16 == 0) {
            float4_t *to = (float4_t *)(quads + quad * kQuadFloats);
#pragma unroll
            for (int g = 0; g < G; g++) to[g] = float4_t{acc_min[g][0], acc_min[g][1], acc_min[g][2], acc_min[g][3]};
            to[G] = float4_t{sum[0], sum[1], sum[2], sum[3]};
            to[G + 1] = float4_t{base[0], base[1], base[2], base[3]};
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        float total = 0, low[D::kSets] = {};
        const float *from = quads + (row >> 2) * kQuadFloats + (row & 3);
#pragma unroll
        for (int u = 0; u < D::kPack; u++) {
            const float *one = from + u * (kRows / 4) * kQuadFloats;
            total += one[G * 4];
#pragma unroll
            for (int e = 0; e < D::kSets; e++) low[e] += one[(e * D::kSetGroups + (in_set < D::kSetGroups ? in_set : 0)) * 4];
        }
        const float own_base = from[G * 4 + 4];
        if constexpr (kAlone) __syncthreads();  // every wave is through with its weights and sums
        if (row < tile.rows_left && in_set == quad * D::kSetGroups / 4) {
            const Segments segments(a, plan, kRows);
            const int at_row = tile.first_row + row;
            const size_t query = (size_t)(tile.row0 + at_row / heads);
            const int head = kv * heads + at_row % heads;
            const size_t slot = ((size_t)kv * segments.per_head + worker + number) * kRows + row;
            if (!entire && quad * D::kSetGroups % 4 == 0 && in_set == 0) *(float2 *)(segments.bases + slot * 2) = make_float2(own_base, total);
            if (kAlone && quad * D::kSetGroups % 4 == 0 && in_set == 0) join_bases[wave][row] = make_float2(own_base, total);
#pragma unroll
            for (int e = 0; e < D::kSets; e++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int n = 4 * quad + r;  // the operand's row: word n / kLanesPerWord of the set, part n % kLanesPerWord of it
                    const int d = (e * D::kSetWords + n / D::kLanesPerWord) * 8 + n % D::kLanesPerWord * D::kNibbles;
                    float v[D::kNibbles];
#pragma unroll
                    for (int i = 0; i < D::kNibbles; i++) v[i] = __builtin_fmaf(acc[e][i][r], 1048576.0f, low[e]);
                    if constexpr (kAlone) {
                        float *to = (float *)lds_all + ((size_t)wave * kRows + row) * kDim + d;
#pragma unroll
                        for (int i = 0; i < D::kNibbles; i++) to[i] = v[i];
                    } else if (entire) {
                        uint16_t *to = a.output + query * a.output_stride + (size_t)head * kDim + d;
                        const float inv = total == 0.0f ? 0.0f : 1.0f / total;  // nothing seen: 0
#pragma unroll
                        for (int i = 0; i < D::kNibbles; i += 2) ((uint32_t *)to)[i / 2] = (uint32_t)f2h(v[i] * inv) | (uint32_t)f2h(v[i + 1] * inv) << 16;
                    } else {
                        float *to = segments.sums + slot * kDim + d;
#pragma unroll
                        for (int i = 0; i < D::kNibbles; i++) to[i] = v[i];
                    }
                }
        }
        if constexpr (kAlone) {
            __syncthreads();
            constexpr int kParts = kDim / 4;  // float4s of a row
            for (int j = threadIdx.x; j < kRows * kParts; j += kWaves * kWave) {
                const int r = j / kParts, d = j % kParts * 4;
                if (r >= tile.rows_left) break;
                float m = kEmpty, all = 0;
                float4_t o = {};
#pragma unroll
                for (int w = 0; w < kWaves; w++) m = fmaxf(m, join_bases[w][r].x);
#pragma unroll
                for (int w = 0; w < kWaves; w++) {
                    const float keep = __builtin_amdgcn_exp2f(join_bases[w][r].x - m);
                    all += join_bases[w][r].y * keep;
                    o += *(const float4_t *)((const float *)lds_all + ((size_t)w * kRows + r) * kDim + d) * keep;
                }
                const int at_row = tile.first_row + r;
                store_row(a, (size_t)(tile.row0 + at_row / heads), kv * heads + at_row % heads, d, o, all);
            }
            return;
        }
        left -= count;
        if (left <= 0) return;
        offset = 0;
        do {
            if (++number >= numbers) return;
            tile = RowTile(a, plan, number, kRows, D::kStep);
        } while (tile.steps == 0);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// Joins the segments of four rows of a row tile, or writes the zeros of rows that see nothing. kLanes lanes a row and
// segment: kDim / 4 for all dims, or 8 and a workgroup for every 32 dims, which makes enough of them even for one sequence,
// whose hundreds of segments are then read in a few round trips.
constexpr int kJoinThreads = 256;
template <int kDim, int kRows, int kLanes>
__global__ __launch_bounds__(kJoinThreads) void attention_join_kernel(const AttentionKv4Args a, const DecodePlan plan) {
    constexpr int kAtOnce = kJoinThreads / (4 * kLanes), kParts = kDim / (4 * kLanes), kJoinWaves = kJoinThreads / kWave;
    extern __shared__ float weights[];  // [4][parts]
    __shared__ float highest[4][kJoinWaves], totals[4][kJoinWaves];
    __shared__ float4_t sums[kAtOnce][4][kLanes];
    const int number = blockIdx.x, kv = blockIdx.y, first_row = blockIdx.z / kParts * 4, first_dim = blockIdx.z % kParts * 4 * kLanes;
    const Segments segments(a, plan, kRows);
    const int2 parts = segments.parts[number];
    const RowTile tile(a, plan, number, kRows, Decode<kDim, kRows>::kStep);
    if (parts.y == 1 || first_row >= tile.rows_left) return;  // stored at once; no such rows
    const size_t slot = ((size_t)kv * segments.per_head + parts.x + number) * kRows + first_row;
    const float2 *bases = (const float2 *)segments.bases + slot;
    float m[4] = {kEmpty, kEmpty, kEmpty, kEmpty}, total[4] = {};
    const int wave = threadIdx.x / kWave;
    for (int p = threadIdx.x; p < parts.y; p += kJoinThreads)
#pragma unroll
        for (int r = 0; r < 4; r++) m[r] = fmaxf(m[r], bases[(size_t)p * kRows + r].x);
#pragma unroll
    for (int r = 0; r < 4; r++) {
        m[r] = quad_max(m[r]);
        m[r] = fmaxf(m[r], __shfl_xor(m[r], 16, kWave));
        m[r] = fmaxf(m[r], __shfl_xor(m[r], 32, kWave));
        if (threadIdx.x % kWave == 0) highest[r][wave] = m[r];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
        for (int w = 0; w < kJoinWaves; w++) m[r] = fmaxf(m[r], highest[r][w]);
    for (int p = threadIdx.x; p < parts.y; p += kJoinThreads)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const float2 one = bases[(size_t)p * kRows + r];
            const float w = __builtin_amdgcn_exp2f(one.x - m[r]);
            weights[r * parts.y + p] = w;
            total[r] += one.y * w;
        }
#pragma unroll
    for (int r = 0; r < 4; r++) {
        total[r] = quad_sum(total[r]);
        total[r] += __shfl_xor(total[r], 16, kWave);
        total[r] += __shfl_xor(total[r], 32, kWave);
        if (threadIdx.x % kWave == 0) totals[r][wave] = total[r];
    }
    __syncthreads();
    const int d = threadIdx.x % kLanes, r = threadIdx.x / kLanes % 4, group = threadIdx.x / (4 * kLanes);
    const float4_t *from = (const float4_t *)(segments.sums + (slot + r) * kDim + first_dim) + d;
    float4_t o = {};
#pragma unroll 8
    for (int p = group; p < parts.y; p += kAtOnce) o += from[(size_t)p * kRows * (kDim / 4)] * weights[r * parts.y + p];
    sums[group][r][d] = o;
    __syncthreads();
    if (group || first_row + r >= tile.rows_left) return;
#pragma unroll
    for (int j = 1; j < kAtOnce; j++) o += sums[j][r][d];
    float all = 0;
#pragma unroll
    for (int w = 0; w < kJoinWaves; w++) all += totals[r][w];
    const int heads = a.n_heads / a.cache.n_kv_heads, at_row = tile.first_row + first_row + r;
    store_row(a, (size_t)(tile.row0 + at_row / heads), kv * heads + at_row % heads, first_dim + d * 4, o, all);
}

int decode_rows(const AttentionKv4Args &a) {
    const long long rows = (long long)a.max_query * (a.n_heads / a.cache.n_kv_heads);
    return rows <= 4 ? 4 : rows <= 8 ? 8 : 16;
}

DecodePlan decode_plan(const AttentionKv4Args &a) {
    const int rows = decode_rows(a), step = rows == 4 ? 64 : 32;
    const long long heads = a.n_heads / a.cache.n_kv_heads;
    DecodePlan p;
    p.tiles = (int)((a.max_query * heads + rows - 1) / rows);
    p.least = 1;
    long long reach = a.max_length;  // positions that a row tile may see, and the steps that they may touch
    if (a.window > 0 && (long long)a.window + a.max_query < reach) reach = (long long)a.window + a.max_query;
    const long long steps = (reach + step - 1) / step + 1;
    p.alone = steps <= kAloneSteps;
    const int slots = 8 * std::min(current_device_cus(), 256);  // two waves a SIMD; the join holds a weight per worker in LDS
    p.workers = p.alone ? a.batch.batch * p.tiles : (slots + a.cache.n_kv_heads - 1) / a.cache.n_kv_heads;
    return p;
}

template <int kDim, int kRows>
hipError_t launch_decode_rows(const AttentionKv4Args &a, const DecodePlan &plan, hipStream_t s) {
    const int across = plan.workers < 32768 ? plan.workers : 32768;
    const dim3 grid((unsigned)a.cache.n_kv_heads, (unsigned)across, (unsigned)((plan.workers + across - 1) / across));
    if (plan.alone) {
        attention_decode_kernel<kDim, kRows, kAloneWaves><<<grid, kAloneWaves * kWave, 0, s>>>(a, plan);
        return hipGetLastError();
    }
    attention_decode_kernel<kDim, kRows, 1><<<grid, kWave, 0, s>>>(a, plan);
    if (hipError_t e = hipGetLastError()) return e;
    const unsigned tiles = (unsigned)(a.batch.batch * plan.tiles), kv = (unsigned)a.cache.n_kv_heads;
    const size_t lds = 16 * (size_t)plan.workers;
    if ((long long)tiles * kv * (kRows / 4) < current_device_cus())
        attention_join_kernel<kDim, kRows, 8><<<dim3(tiles, kv, kRows / 4 * (kDim / 32)), kJoinThreads, lds, s>>>(a, plan);
    else
        attention_join_kernel<kDim, kRows, kDim / 4><<<dim3(tiles, kv, kRows / 4), kJoinThreads, lds, s>>>(a, plan);
    return hipGetLastError();
}

template <int kDim>
hipError_t launch_decode(const AttentionKv4Args &a, hipStream_t s) {
    const DecodePlan plan = decode_plan(a);
    switch (decode_rows(a)) {
        case 4: return launch_decode_rows<kDim, 4>(a, plan, s);
        case 8: return launch_decode_rows<kDim, 8>(a, plan, s);
        default: return launch_decode_rows<kDim, 16>(a, plan, s);
    }
}

}  // namespace

size_t attention_kv4_workspace(const AttentionKv4Args &a) {
    const DecodePlan plan = decode_plan(a);
    return plan.alone ? 0 : Segments::bytes(a, plan, decode_rows(a));
}

hipError_t launch_attention_kv4(const AttentionKv4Args &a, hipStream_t s) {
    return a.cache.head_dim == 64 ? launch_decode<64>(a, s) : launch_decode<128>(a, s);
}

}  // namespace tllm
