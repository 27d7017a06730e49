// Attention of the rows of a batch over the 4-bit paged cache: o = softmax(scale q k^T) v over the positions a row sees.
//
// A key is k[d] = m_g + s_g c[d] with one (s, m) per group g of 32 dims, so a score is
//   q . k = sum_g s_g (sum_{d in g} q[d] c[d]) + m_g (sum_{d in g} q[d]),
// and the matrix cores multiply q with the bare codes: a 4-bit field that a mask leaves in place IS an fp16 number, the
// subnormal c * 2^-24 (bits 0-3) or c * 2^-20 (bits 4-7), and v_mfma_f32_16x16x32_f16 takes subnormals as they are. 32 dims
// are the depth of one such instruction, so one instruction sums one group; s and m are applied to its fp32 result. The
// same holds for the values: sum_t p_t (m_tg + s_tg c_td) = sum_t (p_t s_tg) c_td + sum_t p_t m_tg with bare codes as one
// operand and p s as the other. p s is taken in two fp16 pieces (the second is what the first's rounding left), times a power of two
// that follows the steps, or each row's and group's products (see kStepPower): the only roundings to fewer than 32 bits are 2^-22 of p s,
// or 2^-29 of the largest of its row and group, and the result's. So up to 8 rows; more rows share keys and values that are brought to
// fp16 once (the second and third kernel).
#include <algorithm>

#include "kv4.h"
#include "kv4_rows.h"

namespace tllm {
namespace {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));
typedef uint32_t uint4_t __attribute__((ext_vector_type(4)));
typedef uint32_t uint2_t __attribute__((ext_vector_type(2)));
typedef float float16_t __attribute__((ext_vector_type(16)));

constexpr float kEmpty = -1e30f;  // below every score (|q.k| < 2^40, |scale| <= 2^40): no position yet
constexpr int kHeadroom = 4;      // powers of two that a weight may outgrow its base by before everything is rescaled
// What a weight times a step is multiplied by before it becomes fp16 (its lift) is a power of two. The steps of a group mostly lie within
// a small factor of each other; then the largest of the first positions gives the group's lift: it comes to lie between
// 2^(kStepPower - 1) and 2^kStepPower, and all steps of the piece have to lie between a 32nd of that and its double (a weight is at most
// 2^kHeadroom: the products stay in fp16, whose pieces hold them to 2^-25). A row's largest product is then 2^4 at least. But the steps of
// two positions may be any fp16 numbers apart, and one row look at the one and another row at the other (one lift for all lost 1.7 % of
// the weights of steps of 2^-14 beside one of 8000). So a wave that meets other steps begins its piece again with a lift for each row and
// group, by the products themselves: the largest so far came to lie between 2^(kTopPower - 1) and 2^kTopPower, taken anew where one
// reaches 2^kLimitPower and raised where a new base leaves the earlier weights small. (Those in every piece from the start: 50.4 us for
// 131 072 positions of one sequence, where this takes 46.7 if steps are alike; if none are, 74.)
constexpr int kStepPower = 10, kTopPower = 10, kLimitPower = 15;
constexpr int kMostLift = (127 + 32) << 23;  // 2^32 as a float's bits: the smallest step with a weight of 1 comes to 2^8, and what is lost is below 2^-57
constexpr int kInverse = 254 << 23;          // less the bits of a power of two: those of its inverse
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
__device__ __forceinline__ float as_float(int bits) { return __builtin_bit_cast(float, bits); }
// The larger of two 16-bit halves each; over the lanes of a quad, in every lane; of a word of this half of the wave (kLanes 32; 16: of this
// quad) and its partner, the even halves (quads) of the first word and the odd ones of the second.
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(ushort2_t, a), __builtin_bit_cast(ushort2_t, b)));
}
__device__ __forceinline__ uint32_t quad_larger(uint32_t v) {
    const auto turned = [](uint32_t x, auto by) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x120 + by.value, 0xF, 0xF, false); };
    v = larger(v, turned(v, std::integral_constant<int, 8>{}));
    v = larger(v, turned(v, std::integral_constant<int, 4>{}));
    v = larger(v, turned(v, std::integral_constant<int, 2>{}));
    return larger(v, turned(v, std::integral_constant<int, 1>{}));
}
template <int kLanes>
__device__ __forceinline__ uint32_t larger_of_swapped(uint32_t a, uint32_t b) {
    const uint2_t both = kLanes == 32 ? __builtin_amdgcn_permlane32_swap(a, b, false, false) : __builtin_amdgcn_permlane16_swap(a, b, false, false);
    return larger(both[0], both[1]);
}
__device__ __forceinline__ float quad_max(float v) {
    v = fmaxf(v, rotated<8>(v));
    v = fmaxf(v, rotated<4>(v));
    v = fmaxf(v, rotated<2>(v));
    return fmaxf(v, rotated<1>(v));
}

__device__ __forceinline__ int position_limit(const AttentionKv4Args &a) { return min(a.batch.width << a.cache.page_shift, a.max_length); }

// ------------------------------------------------------------------------------------------------- few rows: decode
//
// Bound: HBM, the cache's 5 bits per value; the work per position has to stay small beside it, above all the work on scores,
// of which 16 x 16 come out of every matrix instruction however few rows there are. So the row operand repeats its kRows
// rows (query rows times the heads that share a kv head: 4 or 8), and of kPack = 16 / kRows tiles of 16 positions each
// quad of lanes keeps the results of its own tile: each of the 64 lanes then has ONE position and four rows of its own (lane
// = (position t, quad)), steps and minima are one coalesced word per lane and group, and softmax runs on four registers. For
// the values, weights p s go through LDS ([position][group][row], fp16) and come back transposed (ds_read_b64_tr_b16) with
// (group, row) pairs as the 16 columns of the operand: one instruction multiplies a row tile's weights of all groups in the
// set, of which each dim uses its own group's.
//
// The positions of all sequences are one line of steps, cut into equal pieces, one per wave (each kv head its own line):
// however ragged the batch, all waves end together. A piece may end inside a sequence and begin inside another; its stretch
// of a sequence is a segment. A sequence that lies in one piece is stored at once, the segments of others are joined by a
// second launch. A wave is a workgroup of its own: nothing waits for another wave. The other form, for short contexts or
// many sequences (see plans_of): a workgroup of kAloneWaves waves has a whole row tile, the waves take its steps in turn and
// meet in LDS, and there is no second launch.
// Measured (32 query heads, 8 kv heads of 128 dims): 32 sequences of 4096 positions 33 us, a read of their 5 bits 28; the
// line, 72 000 positions of 32 ragged sequences: 29 us and 5 for the joins, a read 15; 131 072 positions of one sequence with
// 64 heads: 41 and 6, a read 28. What is left is the vector pipe (some 800 instructions a step of 64 positions, two waves a
// SIMD for the registers) and, in the line, the chain of loads before a wave's first step and behind its last.
constexpr int kAloneWaves = 8;
struct RowPlan {
    int workers;  // waves per kv head
    int tiles;    // row tiles per sequence; row tile t of sequence b is number b * tiles + t of the line
    int least;    // steps that a piece has at least
    int alone;    // every workgroup has a whole row tile (no second launch)
    int from_rows, to_rows;  // sequences with from_rows <= rows < to_rows are this launch's, rows counted with the heads
};

template <int kDim, int kRows>
struct Decode {
    static constexpr int kGroups = kDim / kKvGroup, kWords = kDim / 8;
    static constexpr int kPack = 16 / kRows;
    static constexpr int kTiles = kRows == 4 ? 4 : 2, kStep = 16 * kTiles;
    static_assert(kTiles == kPack, "a position per lane");
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
        uint32_t km[kGroups], vm[kGroups];  // step | minimum << 16 of this lane's position, keys and values
    };
    struct Values {
        uint4_t v[kTiles][kSets];
    };
};

// One row tile: its rows and the steps of positions that some row of it sees.
struct RowTile {
    int row0, rows_left, first_row, pos0, pos_low, pos_high, first_step, steps;
    __device__ RowTile(const AttentionKv4Args &a, const RowPlan &plan, int number, int rows_per_tile, int step) {
        const int seq = plan.tiles == 1 ? number : number / plan.tiles, tile = plan.tiles == 1 ? 0 : number - seq * plan.tiles;
        const int heads = a.n_heads / a.cache.n_kv_heads;
        const SequenceRows s = sequence_rows(a.batch.starts[seq], a.batch.starts[seq + 1], a.batch.lengths[seq], a.batch.n_tokens, a.max_query);
        row0 = s.row0;
        pos0 = s.pos0;
        first_row = tile * rows_per_tile;
        const TileSpan t = tile_span(s, first_row, heads, rows_per_tile, step, a.window, position_limit(a), plan.from_rows, plan.to_rows);
        rows_left = t.rows_left;
        pos_low = t.pos_low;
        pos_high = t.pos_high;
        first_step = t.first_step;
        steps = t.steps;
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
    __host__ __device__ Segments(const AttentionKv4Args &a, const RowPlan &plan, int rows, size_t at = 0) {
        const int numbers = a.batch.batch * plan.tiles;
        per_head = plan.workers + numbers;
        const size_t all = (size_t)a.cache.n_kv_heads * per_head * rows;
        sums = (float *)((char *)a.workspace + at);
        bases = sums + all * a.cache.head_dim;
        parts = (int2 *)(bases + all * 2);
    }
    __host__ __device__ static size_t bytes(const AttentionKv4Args &a, const RowPlan &plan, int rows) {
        const size_t numbers = (size_t)a.batch.batch * plan.tiles;
        return (size_t)a.cache.n_kv_heads * (plan.workers + numbers) * rows * (a.cache.head_dim + 2) * 4 + numbers * 8;
    }
};

// The worker's piece of the line: `left` steps from step `offset` of row tile `number` on; false if it has none. With
// `parts`, the wave also writes down for every row tile which workers have parts of it. All lanes take part.
__device__ __forceinline__ bool find_piece(const AttentionKv4Args &a, const RowPlan &plan, int worker, int rows, int step, bool first,
                                           int2 *parts, int *number, int *offset, int *left, RowTile *tile) {
    const int lane = threadIdx.x % kWave, numbers = a.batch.batch * plan.tiles;
    RowTile own;
    const auto running = [&](int base) {
        own.steps = 0;
        if (base + lane < numbers) own = RowTile(a, plan, base + lane, rows, step);
        return running_sum(own.steps);
    };
    int total = 0, upto = 0;
    for (int base = 0; base < numbers; base += kWave) {
        upto = running(base);
        total += __builtin_amdgcn_readlane(upto, kWave - 1);
    }
    const int per = max(plan.least, (total + plan.workers - 1) / plan.workers);
    const long long begin = (long long)worker * per;
    const int n = (int)min((long long)per, total - begin);
    if (n <= 0 && !first) return false;
    int before = 0, at = -1;
    for (int base = 0; base < numbers && (at < 0 || parts); base += kWave) {
        if (numbers > kWave) upto = running(base);
        const int from = before + upto - own.steps;
        if (parts && base + lane < numbers)
            parts[base + lane] = make_int2(from / per, own.steps ? (from + own.steps - 1) / per - from / per + 1 : 0);
        const unsigned long long here = __ballot(at < 0 && own.steps > 0 && begin >= from && begin < from + own.steps);
        if (here) {
            const int l = __builtin_amdgcn_readfirstlane(__ffsll(here) - 1);
            at = base + l;
            *offset = (int)begin - __builtin_amdgcn_readlane(from, l);
            *tile = own.of_lane(l);
        }
        before += __builtin_amdgcn_readlane(upto, kWave - 1);
    }
    *number = __builtin_amdgcn_readfirstlane(at);
    *left = __builtin_amdgcn_readfirstlane(n);
    return n > 0;  // (none at all to see: only the parts were written)
}

__device__ __forceinline__ void store_row(const AttentionKv4Args &a, size_t query, int head, int d, float4_t o, float total) {
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;  // nothing seen: 0
    const uint2_t packed = {(uint32_t)f2h(o[0] * inv) | (uint32_t)f2h(o[1] * inv) << 16, (uint32_t)f2h(o[2] * inv) | (uint32_t)f2h(o[3] * inv) << 16};
    *(uint2_t *)(a.output + query * a.output_stride + (size_t)head * a.cache.head_dim + d) = packed;
}

// Joins the sums of a workgroup's waves ([wave][row][kStride], a row's dims first) and stores the rows.
template <int kDim, int kRows, int kWaves, int kStride>
__device__ __forceinline__ void join_waves(const AttentionKv4Args &a, const RowTile &tile, int kv, int heads, const float2 (&bases)[kWaves][kRows], const float *sums) {
    constexpr int kParts = kDim / 4;  // float4s of a row
    for (int j = threadIdx.x; j < kRows * kParts; j += kWaves * kWave) {
        const int r = j / kParts, d = j % kParts * 4;
        if (r >= tile.rows_left) break;
        float m = kEmpty, all = 0;
        float4_t o = {};
#pragma unroll
        for (int w = 0; w < kWaves; w++) m = fmaxf(m, bases[w][r].x);
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            const float keep = __builtin_amdgcn_exp2f(bases[w][r].x - m);
            all += bases[w][r].y * keep;
            o += *(const float4_t *)(sums + ((size_t)w * kRows + r) * kStride + d) * keep;
        }
        const int at_row = tile.first_row + r;
        store_row(a, (size_t)(tile.row0 + at_row / heads), kv * heads + at_row % heads, d, o, all);
    }
}

template <int kDim, int kRows, int kWaves>
__global__ __launch_bounds__(kWaves *kWave, 2) void attention_decode_kernel(const AttentionKv4Args a, const RowPlan plan) {
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
        const bool scribe = kv == 0 && worker == 0;
        const Segments segments(a, plan, kRows);
        if (!find_piece(a, plan, worker, kRows, D::kStep, scribe, scribe ? segments.parts : nullptr, &number, &offset, &left, &tile)) return;
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
    // (with 4 rows a tile all lanes have the same rows: their lifts are the wave's)
    const auto of_wave = [](int x) { return kRows == 4 ? __builtin_amdgcn_readfirstlane(x) : x; };
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
                for (int g = 0; g < G; g++) {
                    x.km[g] = *(const uint32_t *)(bytes(c.k_scales, word + ((size_t)g << c.page_shift)) + scale_offset);
                    x.vm[g] = *(const uint32_t *)(bytes(c.v_scales, word + ((size_t)g << c.page_shift)) + scale_offset);
                }
            } else {
                uint32_t b = at.block[0], sl = at.slot[0];
#pragma unroll
                for (int u = 1; u < D::kPack; u++)
                    if (pack == u) b = at.block[u], sl = at.slot[u];
                const size_t word = b * scale_words + sl + t16;
#pragma unroll
                for (int g = 0; g < G; g++) {
                    x.km[g] = c.k_scales[word + ((size_t)g << c.page_shift)];
                    x.vm[g] = c.v_scales[word + ((size_t)g << c.page_shift)];
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
        // more operand: first and second fp16 piece, times a power of two that brings the largest of the row's groups to 2^13 and
        // more (small queries keep their bits beside large keys), at the depth of the quad that holds the minima of the row's tile
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
        float c_sums[4];  // of this lane's rows: what undoes the power, and the scale
        {
            float group_sum[G], largest = 0;
#pragma unroll
            for (int g = 0; g < G; g++) {
                group_sum[g] = 0;
#pragma unroll
                for (int j = 0; j < 8; j++) group_sum[g] += (float)q[g][j];
                group_sum[g] += __shfl_xor(group_sum[g], 16, kWave);
                group_sum[g] += __shfl_xor(group_sum[g], 32, kWave);
                largest = fmaxf(largest, fabsf(group_sum[g]));
            }
            const int power = (__builtin_bit_cast(int, fminf(fmaxf(largest, 1e-30f), 1e30f)) >> 23) - 13;
            const float by = as_float((254 - power) << 23);
#pragma unroll
            for (int g = 0; g < G; g++) {
                const float sum = group_sum[g] * by;
                if (quad == t16 / kRows * (kRows / 4)) {
                    q_sums[g] = (_Float16)sum;
                    q_sums[G + g] = (_Float16)(sum - (float)q_sums[g]);
                }
            }
#pragma unroll
            for (int r = 0; r < 4; r++) c_sums[r] = as_float(__shfl(power, 4 * row_quad + r, kWave) << 23) * c_low;
        }

        float4_t acc[D::kSets][D::kNibbles];
        float acc_min[G][4], sum[4], base[4];
        int column_lift[D::kSets];  // of the column that this lane's sums of values belong to; lifts are the bits of their floats
        // The piece's sums; with `each`, a lift for each row and group. False: the steps of some group are not alike.
        const auto attend = [&](auto each) {
            constexpr bool kEach = each.value;
#pragma unroll
            for (int e = 0; e < D::kSets; e++)
#pragma unroll
                for (int i = 0; i < D::kNibbles; i++) acc[e][i] = float4_t{};
#pragma unroll
            for (int r = 0; r < 4; r++) {
                sum[r] = 0;
                base[r] = kEmpty;
#pragma unroll
                for (int g = 0; g < G; g++) acc_min[g][r] = 0;
            }
            bool fresh = true, alike = true;           // (one lift a group:) no step of a value has been met; they are alike so far
            int stop = end;                            // (one way out of the loop: a second costs copies of all sums in every step)
            int group_lift[G], lift[kEach ? G : 1][4];  // of the groups; of this lane's rows (4 rows a tile: of the wave's)
#pragma unroll
            for (int g = 0; g < G; g++) {
                group_lift[g] = kMostLift;
#pragma unroll
                for (int r = 0; r < 4; r++) lift[kEach ? g : 0][r] = kMostLift;
            }
#pragma unroll
            for (int e = 0; e < D::kSets; e++) column_lift[e] = kMostLift;
            // a column's new lift, and its sums under it
            const auto change_column = [&](int e, int to) {
                const float by = as_float(to) * as_float(kInverse - column_lift[e]);
                column_lift[e] = to;
#pragma unroll
                for (int i = 0; i < D::kNibbles; i++) acc[e][i] *= by;
            };

            // this step's values, which the work on the scores covers, then the next step's keys
            while (step < stop) {
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
                float raw[4], most = -INFINITY;
                uint32_t sees = ~0u;  // a bit per row r
                bool any = true;      // some row may see this lane's position
                float4_t d[G];
#pragma unroll
                for (int pair = 0; pair < G / 2; pair++)
#pragma unroll
                    for (int u = 0; u < D::kPack; u++) {
                        const uint32_t w0 = now.k[u][2 * pair], w1 = now.k[u][2 * pair + 1];
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
                    const int t = first + 16 * pack + t16;
                    const bool there = (pages >> pack & 1) && t < limit;
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const int row = 4 * row_quad + r, pos = tile.pos0 + (tile.first_row + row) / heads;
                        const bool one = there && row < tile.rows_left && t <= pos && (a.window == 0 || t > pos - a.window);
                        sees &= ~((uint32_t)!one << r);
                    }
                    // What no row sees may be anything, and must reach neither the powers below nor, in the product of the
                    // minima, the other tiles' positions. Nor must what is not finite and only some rows see reach the others:
                    // a key's rows get their NaN in the scores below, a value's in the sum of its group's minima.
                    any = there && t <= tile.pos_high && (a.window == 0 || t > tile.pos_low - a.window);
#pragma unroll
                    for (int g = 0; g < G; g++) {
                        unsound |= any && (now.km[g] & 0x7C000000u) == 0x7C000000u;
                        const bool wrong = any && ((now.vm[g] & 0x7C000000u) == 0x7C000000u || (now.vm[g] & 0x7C00u) == 0x7C00u);
                        now.vm[g] = any && !wrong ? now.vm[g] : 0;
#pragma unroll
                        for (int r = 0; r < 4; r++) acc_min[g][r] = wrong && (sees >> r & 1) ? NAN : acc_min[g][r];
                    }
#pragma unroll
                    for (int g = 0; g < G; g++) now.km[g] = any && !unsound ? now.km[g] : 0;
                }
                uint4_t minima;
#pragma unroll
                for (int j = 0; j < 4; j++)  // (G is 2: the last four depths have zero rows, and zeros here)
                    minima[j] = G == 4 || j < 2 ? __builtin_amdgcn_perm(now.km[2 * j % G + 1], now.km[2 * j % G], 0x07060302u) : 0;
                const float4_t low = __builtin_amdgcn_mfma_f32_16x16x32_f16(q_sums, __builtin_bit_cast(half8_t, minima), float4_t{}, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    float even = 0, odd = 0;
#pragma unroll
                    for (int g = 0; g < G; g += 2) {
                        even = __builtin_fmaf(low_half(now.km[g]), d[g][r], even);
                        odd = __builtin_fmaf(low_half(now.km[g + 1]), d[g + 1][r], odd);
                    }
                    raw[r] = __builtin_fmaf(even, c_even, __builtin_fmaf(odd, c_odd, low[r] * c_sums[r]));
                }
                if (!whole) {
                    asm volatile("");
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        raw[r] = unsound ? NAN : raw[r];
                        raw[r] = sees >> r & 1 ? raw[r] : -INFINITY;
                    }
                }
#pragma unroll
                for (int r = 0; r < 4; r++) most = fmaxf(most, raw[r] - base[r]);
                float size[G];  // steps times their group's lift; odd positions' are negative (see kSecondFlipped)
                if constexpr (!kEach) {
                    if (fresh) {
                        uint32_t steps[G / 2];  // of two groups
#pragma unroll
                        for (int i = 0; i < G / 2; i++) steps[i] = __builtin_amdgcn_perm(now.vm[2 * i + 1], now.vm[2 * i], 0x05040100u);
                        uint32_t highest = larger_of_swapped<32>(steps[0], steps[G / 2 - 1]);  // halves of the wave: of these two
                        highest = quad_larger(larger_of_swapped<16>(highest, highest));
                        fresh = !__ballot(highest);
#pragma unroll
                        for (int g = 0; g < G; g++) {
                            const int one = __builtin_amdgcn_readlane(highest, g / 2 * 32) >> g % 2 * 16 & 0xFFFF;
                            group_lift[g] = one ? (127 + kStepPower + 14 - (one >> 10)) << 23 : kMostLift;
                        }
                    }
                    float most_size = 0, least_size = INFINITY;
#pragma unroll
                    for (int g = 0; g < G; g++) {
                        size[g] = low_half(now.vm[g]) * (as_float(group_lift[g]) * sign);
                        most_size = fmaxf(most_size, fabsf(size[g]));
                        least_size = fminf(least_size, fabsf(size[g]));
                    }
                    if (__ballot(any && (most_size > (float)(2 << kStepPower) || least_size < (float)(1 << kStepPower >> 5)))) stop = step, alike = false;
                } else {
#pragma unroll
                    for (int g = 0; g < G; g++) size[g] = low_half(now.vm[g]) * sign;
                }
                if (__ballot(most > (float)kHeadroom)) {
                    // rare after the first steps: new bases, whole numbers, so that what they change are powers of two
                    float keep[4];
                    int more[4];  // powers of two, as a float's bits, that the lifts are raised by
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        float m = quad_max(raw[r]);
#pragma unroll
                        for (int off = 4 * kRows; off < kWave; off <<= 1) m = fmaxf(m, __shfl_xor(m, off, kWave));
                        const float to = fmaxf(base[r], ceilf(m));
                        keep[r] = __builtin_amdgcn_exp2f(base[r] - to);
                        more[r] = of_wave((int)fminf(to - base[r], 64.0f) << 23);
                        base[r] = to;
                        sum[r] *= keep[r];
#pragma unroll
                        for (int g = 0; g < G; g++) acc_min[g][r] *= keep[r];
                    }
                    const int row = t16 % kRows;
                    float column = 0;
                    int column_more = 0;
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const float k = kRows == 4 ? keep[r] : __shfl(keep[r], (row >> 2) * 16, kWave);
                        column = (row & 3) == r ? k : column;
                        if constexpr (kEach) {
                            const int one = kRows == 4 ? more[r] : __shfl(more[r], (row >> 2) * 16, kWave);
                            column_more = (row & 3) == r ? one : column_more;
#pragma unroll
                            for (int g = 0; g < G; g++) lift[g][r] = min(lift[g][r] + more[r], kMostLift);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < D::kSets; e++) {
#pragma unroll
                        for (int i = 0; i < D::kNibbles; i++) acc[e][i] *= column;
                        if constexpr (kEach) change_column(e, min(column_lift[e] + column_more, kMostLift));
                    }
                }
                float w[4];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    w[r] = __builtin_amdgcn_exp2f(raw[r] - base[r]);
                    sum[r] += w[r];
                }
                // the weights of all groups in two pieces; the larger of the first pieces' bits (a lane's all have one sign)
                const auto put_weights = [&] {
                    unsigned char *to = lds + (16 * pack + t16) * D::kRowBytes + row_quad * 8;
                    ushort2_t high = {0, 0};
#pragma unroll
                    for (int g = 0; g < G; g++) {
                        uint32_t hi[2], lo[2];
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            float one = w[2 * j] * size[g], two = w[2 * j + 1] * size[g];
                            if constexpr (kEach) one *= as_float(lift[g][2 * j]), two *= as_float(lift[g][2 * j + 1]);
                            // (rounded to fp32 here: a product that is rounded to fp16 at once, beside one that is not, makes the second piece
                            // that of another first piece, a step off, where the fp32 product lies half-way between two fp16 numbers)
                            asm("" : "+v"(one), "+v"(two));
                            const half2_t h = {(_Float16)one, (_Float16)two};
                            const half2_t l = {(_Float16)__builtin_fmaf((float)h[0], minus_one, one), (_Float16)__builtin_fmaf((float)h[1], minus_one, two)};
                            hi[j] = __builtin_bit_cast(uint32_t, h);
                            lo[j] = __builtin_bit_cast(uint32_t, l);
                            high = __builtin_elementwise_max(high, __builtin_bit_cast(ushort2_t, h));
                        }
                        *(uint2_t *)(to + g * kRows * 2) = uint2_t{hi[0], hi[1]};
                        *(uint2_t *)(to + D::kColumns * 2 + g * kRows * 2) = uint2_t{lo[0], lo[1]};
                    }
                    return __builtin_bit_cast(uint32_t, high);
                };
                if constexpr (!kEach) {
                    put_weights();
                } else if (__ballot(((put_weights() & 0x7FFF7FFFu) + 0x00010001u * (0x8000u - ((15u + kLimitPower) << 10))) & 0x80008000u)) {
                    // (bits 15 and 31: an exponent of kLimitPower or more.) Lifts by the largest products, of which the exponents are enough: the
                    // upper halves of two rows' in a word
                    uint32_t high[2 * G];  // [2 g + j]: group g, rows 2 j and 2 j + 1
#pragma unroll
                    for (int g = 0; g < G; g++)
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            const float size = fabsf(low_half(now.vm[g]));
                            high[2 * g + j] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, w[2 * j + 1] * size), __builtin_bit_cast(uint32_t, w[2 * j] * size), 0x07060302u);
                        }
                    const auto new_lift = [](int old, uint32_t pair, bool second) {
                        const int power = (int)(pair >> (second ? 23 : 7) & 0xFF);  // (infinite or NaN, 255: the weights carry it on)
                        return (old >> 23) + power < 254 + kLimitPower ? old : (253 + kTopPower - power) << 23;
                    };
                    // swapping halves of the wave between two words and taking the larger leaves each half with one word's: [k] and [k + G]
#pragma unroll
                    for (int k = 0; k < G; k++) high[k] = larger_of_swapped<32>(high[k], high[k + G]);
                    const int row = t16 % kRows;
                    if constexpr (kRows == 4) {
                        // the same with quads: quad n has words n * G / 2 + k
#pragma unroll
                        for (int k = 0; k < G / 2; k++) high[k] = quad_larger(larger_of_swapped<16>(high[k], high[k + G / 2]));
#pragma unroll
                        for (int n = 0; n < 2 * G; n++) {
                            const uint32_t pair = __builtin_amdgcn_readlane(high[n % (G / 2)], n / (G / 2) * 16);
#pragma unroll
                            for (int i = 0; i < 2; i++) lift[n / 2][2 * (n & 1) + i] = new_lift(lift[n / 2][2 * (n & 1) + i], pair, i);
                        }
                        // this lane's column: group t16 / 4 (or none), word 2 * group + row / 2
                        const int word = 2 * (t16 / 4 % G) + (row >> 1);
                        uint32_t pair = __shfl(high[0], word / (G / 2) * 16, kWave);
                        if constexpr (G == 4) {
                            const uint32_t odd = __shfl(high[1], word / 2 * 16, kWave);
                            pair = word & 1 ? odd : pair;
                        }
                        change_column(0, new_lift(column_lift[0], pair, row & 1));
                    } else {
#pragma unroll
                        for (int k = 0; k < G; k++) {
                            high[k] = quad_larger(high[k]);
                            const uint2_t both = __builtin_amdgcn_permlane32_swap(high[k], high[k], false, false);
                            high[k] = both[0];
                            high[k + G] = both[1];
                        }
#pragma unroll
                        for (int n = 0; n < 2 * G; n++)
#pragma unroll
                            for (int i = 0; i < 2; i++) lift[n / 2][2 * (n & 1) + i] = new_lift(lift[n / 2][2 * (n & 1) + i], high[n], i);
#pragma unroll
                        for (int e = 0; e < D::kSets; e++) {
                            uint32_t pair = 0;
#pragma unroll
                            for (int n = 0; n < 2 * D::kSetGroups; n++) {
                                const uint32_t one = __shfl(high[2 * e * D::kSetGroups + n], (row >> 2) * 16, kWave);
                                pair = n == 2 * (t16 / kRows) + (row >> 1 & 1) ? one : pair;
                            }
                            change_column(e, new_lift(column_lift[e], pair, row & 1));
                        }
                    }
                    put_weights();
                }
#pragma unroll
                for (int g = 0; g < G; g++) {
                    const float low = __builtin_fmaf(low_half(now.vm[g]), flipped, high_half(now.vm[g]));
#pragma unroll
                    for (int r = 0; r < 4; r++) acc_min[g][r] = __builtin_fmaf(w[r], low, acc_min[g][r]);
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
            if constexpr (!kEach)
#pragma unroll
                for (int g = 0; g < G; g++)
                    if (g % D::kSetGroups == 0 || t16 / kRows == g % D::kSetGroups) column_lift[g / D::kSetGroups] = group_lift[g];
            return alike;
        };
        if (!attend(std::false_type{})) {
            step = tile.first_step + offset + wave;
            held_from = (tile.first_step + offset) * D::kStep >> c.page_shift;
            held = table[min(held_from + lane, a.batch.width - 1)];
            at = find(step);
            load_keys(now, at);
            attend(std::true_type{});
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
                    for (int i = 0; i < D::kNibbles; i++) v[i] = __builtin_fmaf(acc[e][i][r], 1048576.0f * as_float(kInverse - column_lift[e]), low[e]);
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
            join_waves<kDim, kRows, kWaves, kDim>(a, tile, kv, heads, join_bases, (const float *)lds_all);
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

// From 9 rows on k and v are brought to fp16, with one rounding and kept within its range, as kv4_read writes them: the code as
// 1024 + c (64 + c from bits 4-7) less the rest, exactly, then c s + m. (Halves of s and m cannot overflow, but lose the last bits
// of steps and minima below 2^-14: values of 1e-4 came out 4e-3 off.) m + 15 s may be half a step of s above fp16's largest
// number; groups that are large enough for that (or not finite) show in one look at the exponents of s and m, and what becomes of
// them then (kCut) is a piece of code of its own.
constexpr uint32_t kEvenBits = 0x64006400u, kOddBits = 0x54005400u;
// Bits 15 and 31 of what is added up with `or`: a step from 2^11 or a minimum from 2^15 on (15 * 2^11 + 2^15 < 65504), infinities and NaN.
__device__ __forceinline__ uint32_t large_bits(uint32_t scale) { return (scale & 0x7C007C00u) + 0x08001800u; }
constexpr uint32_t kLargeMask = 0x80008000u;
// The compiler does not know that the words stay the same: what was made of them is made anew, not kept in registers for a rare branch.
template <class T>
__device__ __forceinline__ void anew(T &words) {
    asm volatile("" : "+v"(words));
}
__device__ __forceinline__ bool not_finite(uint32_t scale) { return ((scale & 0x7C007C00u) + 0x04000400u) & 0x80008000u; }
// Two values of the codes in `field` (under the even or the odd mask), whose group's steps and minima are s and m in each half.
template <bool kCut>
__device__ __forceinline__ uint32_t values_of(uint32_t field, bool odd, uint32_t bits, half2_t s, half2_t m) {
    const half2_t code = __builtin_bit_cast(half2_t, (field & (odd ? kOddCodes : kEvenCodes)) | bits) - (odd ? half2_t{64, 64} : half2_t{1024, 1024});
    half2_t x = __builtin_elementwise_fma(code, s, m);
    if constexpr (kCut) {
        // (the smaller of a number and NaN is the number: the limits of a group that is not finite are NaN too)
        const half2_t none = __builtin_elementwise_fma(s, half2_t{0, 0}, m * half2_t{0, 0});
        x = __builtin_elementwise_max(__builtin_elementwise_min(x, none + half2_t{65504, 65504}), none - half2_t{65504, 65504});
    }
    return __builtin_bit_cast(uint32_t, x);
}

// ------------------------------------------------------------------------------------------------- up to 32 rows a tile
//
// Bound: the vector pipe, which brings the cache to fp16: a position's 2 kDim values cost some eight instructions a wave, whatever
// the rows, and a score tile of 32 rows three more. A wave works alone on steps of 32 positions (line or alone, as for few
// rows), and nothing goes through LDS: a lane brings to fp16 what it is to feed the matrix instructions itself. Products are
// transposed (k q^T, v^T p^T). For the first a lane has half of one position's dims, in whatever order q's operand repeats; a
// row's scores then lie in one lane and its partner 32 lanes on, and p is the second product's operand as it lies. Its other
// operand has dims as rows: a lane has one word's dims of 16 positions, and of the row tiles' order only the stores know. k, v
// and p are rounded to fp16 (see the next section).
// Measured (32 heads, 8 kv heads of 128): five drafts for 16 users in a window of 1024 18 us as whole row tiles, 36 in line;
// 16 sequences of 8192 positions with 32 rows each 74 us, with 64 rows 111, a read of the cache 28.
template <int kDim>
struct Rows32 {
    static constexpr int kGroups = kDim / kKvGroup, kWords = kDim / 8;
    static constexpr int kRows = 32, kStep = 32;
    static constexpr int kLanesPerWord = 32 / kWords, kNibbles = 8 / kLanesPerWord;  // (kNibbles == kGroups: result tiles)
    static constexpr int kJoinStride = kDim + 4;  // floats of a row in LDS: the lanes store the same dims of all rows at once
    struct Keys {
        uint4_t k[kGroups / 2];
        uint32_t scales[kGroups];
    };
};

template <int kDim, int kWaves>
__global__ __launch_bounds__(kWaves *kWave, 2) void attention_rows_kernel(const AttentionKv4Args a, const RowPlan plan) {
    using R = Rows32<kDim>;
    constexpr int G = R::kGroups, kRows = R::kRows;
    constexpr bool kAlone = kWaves > 1;
    __shared__ __align__(16) float join_sums[kAlone ? kWaves : 1][kAlone ? kRows : 1][kAlone ? R::kJoinStride : 4];
    __shared__ float2 join_bases[kAlone ? kWaves : 1][kRows];
    const Kv4Cache &c = a.cache;
    const int lane = threadIdx.x % kWave, half = lane >> 5, l32 = lane & 31;
    const int wave = kAlone ? __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) : 0;
    const int kv = blockIdx.x, worker = blockIdx.y + blockIdx.z * gridDim.y;
    if (worker >= plan.workers) return;
    const int heads = a.n_heads / c.n_kv_heads, numbers = a.batch.batch * plan.tiles;
    int number = worker, offset = 0, left = INT32_MAX;
    RowTile tile;
    if constexpr (kAlone) {
        tile = RowTile(a, plan, number, kRows, R::kStep);
        if (tile.rows_left <= 0) return;
    } else {
        const bool scribe = kv == 0 && worker == 0;
        const Segments segments(a, plan, kRows);
        if (!find_piece(a, plan, worker, kRows, R::kStep, scribe, scribe ? segments.parts : nullptr, &number, &offset, &left, &tile)) return;
    }
    const int limit = position_limit(a);
    const size_t code_words = kv4_code_words(1 << c.page_shift, kDim), scale_words = kv4_scale_words(1 << c.page_shift, kDim);
    const int v_word = l32 % R::kWords, v_part = l32 / R::kWords;
    // this lane's bytes in 16 positions of a page
    const uint32_t key_offset = (uint32_t)((l32 & 15) * R::kWords + half * 2 * G) * 4, key_scale_offset = (uint32_t)(l32 & 15) * 4;
    const uint32_t value_offset = (uint32_t)(half * R::kWords + v_word) * 16;
    const size_t value_scale_offset = (((size_t)(v_word / 4) << c.page_shift) + 4 * half) * 4;  // (the fourth group of the largest page: beyond 32 bits)
    const float to_log2 = (a.scale == 0.0f ? 1.0f : fabsf(a.scale)) * 1.44269504088896f;
    uint32_t even_bits = kEvenBits, odd_bits = kOddBits;  // (in registers: two constants make two instructions)
    asm("" : "+v"(even_bits), "+v"(odd_bits));
    const auto value2 = [&](auto cut, uint32_t field, bool odd, half2_t s, half2_t m) { return values_of<cut.value>(field, odd, odd ? odd_bits : even_bits, s, m); };

    while (true) {
        const int count = min(tile.steps - offset, left);
        const bool entire = kAlone || (offset == 0 && count == tile.steps);
        const int *table = a.batch.table + (size_t)(plan.tiles == 1 ? number : number / plan.tiles) * a.batch.width;
        int step = tile.first_step + offset + wave;
        const int end = tile.first_step + offset + count;

        // 64 entries of the page table at a time, one per lane
        int held_from = (tile.first_step + offset) * R::kStep >> c.page_shift, held = table[min(held_from + lane, a.batch.width - 1)];
        uint32_t block[2], slot[2], there = 0;  // of each 16 positions: page * n_kv_heads + head, first slot; bit i: they have a page
        auto find = [&] {
            const int at = step * R::kStep;
            if ((at + 16) >> c.page_shift >= held_from + kWave) {
                held_from = at >> c.page_shift;
                held = table[min(held_from + lane, a.batch.width - 1)];
            }
            there = 0;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int index = (at + 16 * i) >> c.page_shift, page = __builtin_amdgcn_readlane(held, index - held_from);
                const bool real = index < a.batch.width && page >= 0 && page < c.n_pages;
                there |= (uint32_t)real << i;
                block[i] = (real ? page : 0) * c.n_kv_heads + kv;
                slot[i] = (at + 16 * i) & ((1 << c.page_shift) - 1);
            }
        };
        const auto bytes = [](const void *at, size_t words) { return (const unsigned char *)at + words * 4; };
        auto load_keys = [&](typename R::Keys &x) {
            const bool second = l32 >= 16;
            const unsigned char *codes[2], *scales[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                codes[i] = bytes(c.k_codes, block[i] * code_words + (size_t)slot[i] * R::kWords);
                scales[i] = bytes(c.k_scales, block[i] * scale_words + slot[i]);
            }
            const unsigned char *from = (second ? codes[1] : codes[0]) + key_offset, *scale = (second ? scales[1] : scales[0]) + key_scale_offset;
#pragma unroll
            for (int i = 0; i < G / 2; i++) x.k[i] = ((const uint4_t *)from)[i];
#pragma unroll
            for (int g = 0; g < G; g++) x.scales[g] = *(const uint32_t *)(scale + ((size_t)g << (c.page_shift + 2)));
        };

        // this lane's row, and its operand: depth (word pair, odd or even, quad) of a key's order
        const int at_row = tile.first_row + l32;
        const bool real = l32 < tile.rows_left;
        const size_t query = (size_t)(tile.row0 + (real ? at_row / heads : 0));
        const int head = kv * heads + (real ? at_row % heads : 0), pos = real ? tile.pos0 + at_row / heads : -1;
        half8_t q[2 * G];
#pragma unroll
        for (int k = 0; k < 2 * G; k++) {
            q[k] = real ? *(const half8_t *)(a.q + query * a.q_stride + (size_t)head * kDim + (k >> 1) * 32 + (2 * half + (k & 1)) * 8) : half8_t{};
            if (a.scale < 0) q[k] = -q[k];
            if (a.scale == 0) q[k] = half8_t{};
        }
        typename R::Keys now;
        if (step < end) {
            find();
            load_keys(now);
        }
        float16_t acc[G] = {};
        float sum = 0, base = kEmpty;
        while (step < end) {
            // this step's values, which the work on the scores covers, then the next step's keys
            uint4_t v[4], v_scales[4];  // [8 positions]: four of them, of this lane's word; their steps and minima
#pragma unroll
            for (int i = 0; i < 4; i++) {
                v[i] = *(const uint4_t *)(bytes(c.v_codes, block[i >> 1] * code_words + (size_t)slot[i >> 1] * R::kWords + (i & 1) * 8 * R::kWords) + value_offset);
                v_scales[i] = *(const uint4_t *)(bytes(c.v_scales, block[i >> 1] * scale_words + slot[i >> 1] + (i & 1) * 8) + value_scale_offset);
            }
            const uint32_t pages = there;
            const int first = step * R::kStep;
            typename R::Keys next;
            step += kWaves;
            if (step < end) {
                find();
                load_keys(next);
            }
            const bool whole = pages == 3 && first + R::kStep - 1 <= tile.pos_low && first + R::kStep <= limit && (a.window == 0 || first > tile.pos_high - a.window);
            float16_t x;
            const auto scores = [&](auto cut) {
                x = float16_t{};
#pragma unroll
                for (int quad = 0; quad < 2; quad++)
#pragma unroll
                    for (int pair = 0; pair < G / 2; pair++) {
                        const int word = quad * G + 2 * pair;
                        const uint32_t w0 = now.k[word >> 2][word & 3], w1 = now.k[word >> 2][(word & 3) + 1];
#pragma unroll
                        for (int odd = 0; odd < 2; odd++) {
                            const half2_t both = __builtin_bit_cast(half2_t, now.scales[2 * pair + odd]), s = {both[0], both[0]}, m = {both[1], both[1]};
                            const uint4_t key = {value2(cut, w0, odd, s, m), value2(cut, w0 >> 8, odd, s, m), value2(cut, w1, odd, s, m), value2(cut, w1 >> 8, odd, s, m)};
                            x = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, key), q[(2 * pair + odd) * 2 + quad], x, 0, 0, 0);
                        }
                    }
            };
            scores(std::false_type{});
            uint32_t large = 0;
#pragma unroll
            for (int g = 0; g < G; g++) large |= large_bits(now.scales[g]);
            if (__ballot(large & kLargeMask)) {
#pragma unroll
                for (int i = 0; i < G / 2; i++) anew(now.k[i]);
                scores(std::true_type{});  // (again, with what is beyond fp16's range cut)
            }
            if (!whole) {
                asm volatile("");  // (a branch: not worked out and chosen from in every step)
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    const int t = first + 8 * (j >> 2) + 4 * half + (j & 3);
                    const bool sees = t <= pos && t < limit && (a.window == 0 || t > pos - a.window) && (pages >> (j >> 3) & 1);
                    x[j] = sees ? x[j] : -INFINITY;
                }
            }
            float most = -INFINITY;
#pragma unroll
            for (int j = 0; j < 16; j++) most = fmaxf(most, x[j]);
            most = fmaxf(most, __shfl_xor(most, 32, kWave)) * to_log2;
            if (__ballot(most - base > 14.0f)) {
                const float to = fmaxf(base, most - 6.0f), keep = __builtin_amdgcn_exp2f(base - to);
                base = to;
                sum *= keep;
#pragma unroll
                for (int g = 0; g < G; g++) acc[g] *= keep;
            }
            half8_t weights[2];
#pragma unroll
            for (int j = 0; j < 16; j++) weights[j >> 3][j & 7] = (_Float16)__builtin_amdgcn_exp2f(__builtin_fmaf(x[j], to_log2, -base));
#pragma unroll
            for (int j = 0; j < 16; j += 2)  // (of the rounded weights, which is what the values are multiplied with)
                sum = __builtin_amdgcn_fdot2(half2_t{weights[j >> 3][j & 7], weights[j >> 3][(j & 7) + 1]}, half2_t{1, 1}, sum, false);

            const auto weigh_values = [&](auto cut, const uint4_t (&scales)[4]) {
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    uint4_t values[R::kNibbles];
#pragma unroll
                    for (int b = 0; b < 2; b++) {
                        const uint4_t words = v[2 * k + b], pairs = scales[2 * k + b];
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            const half2_t s = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(pairs[2 * j + 1], pairs[2 * j], 0x05040100u));
                            const half2_t m = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(pairs[2 * j + 1], pairs[2 * j], 0x07060302u));
#pragma unroll
                            for (int byte = 0; byte < R::kNibbles / 2; byte++) {
                                // this lane's byte `byte` of two positions' words, one per half
                                const uint32_t which = (uint32_t)(v_part * (R::kNibbles / 2) + byte), select = which * 0x00010001u + 0x0C040C00u;
                                const uint32_t field = __builtin_amdgcn_perm(words[2 * j + 1], words[2 * j], select);
                                values[2 * byte][2 * b + j] = value2(cut, field, false, s, m);
                                values[2 * byte + 1][2 * b + j] = value2(cut, field, true, s, m);
                            }
                        }
                    }
#pragma unroll
                    for (int n = 0; n < R::kNibbles; n++) acc[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, values[n]), weights[k], acc[n], 0, 0, 0);
                }
            };
            // what no row sees may be anything: its values are zeros (its weights are). So are groups that are not finite, and
            // the rows that see them get a NaN
            large = 0;
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) large |= large_bits(v_scales[i][j]);
            const bool any_large = __ballot(large & kLargeMask);
            if (!whole || any_large) {
                uint4_t cut[4] = {};  // steps and minima of the groups that are large: a product of their own
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int t = first + 8 * i + j;  // (of the lower half of the lanes)
                        const int own = t + 4 * half;
                        const bool seen = (pages >> (i >> 1) & 1) && own <= tile.pos_high && own < limit && (a.window == 0 || own > tile.pos_low - a.window);
                        const bool bad = seen && not_finite(v_scales[i][j]);
                        v_scales[i][j] = seen && !bad ? v_scales[i][j] : 0;
                        cut[i][j] = large_bits(v_scales[i][j]) & kLargeMask ? v_scales[i][j] : 0;
                        v_scales[i][j] ^= cut[i][j];
                        const unsigned long long all_bad = __ballot(bad);
                        if (all_bad) {
                            for (int h = 0; h < 2; h++) {
                                const int its = t + 4 * h;
                                const bool sees = its <= pos && (a.window == 0 || its > pos - a.window);
#pragma unroll
                                for (int e = 0; e < 16; e++) {
                                    const int group = (2 * (e >> 2) + half) % G;  // of this lane's results e
                                    if (sees && (all_bad >> (32 * h + 4 * group) & 1)) {
#pragma unroll
                                        for (int g = 0; g < G; g++) acc[g][e] = NAN;
                                    }
                                }
                            }
                        }
                    }
                if (any_large) {
#pragma unroll
                    for (int i = 0; i < 4; i++) anew(v[i]);
                    weigh_values(std::true_type{}, cut);
                }
            }
            weigh_values(std::false_type{}, v_scales);
            now = next;
        }

        sum += __shfl_xor(sum, 32, kWave);
        if (kAlone && half == 0) join_bases[wave][l32] = make_float2(base, sum);
        const Segments segments(a, plan, kRows);
        const size_t place = ((size_t)kv * segments.per_head + worker + number) * kRows + l32;
        if (!entire && real && half == 0) *(float2 *)(segments.bases + place * 2) = make_float2(base, sum);
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // nothing seen: 0
        if (kAlone || real) {
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int at = 8 * (e >> 2) + 4 * half + (e & 3), d = at % R::kWords * 8 + at / R::kWords * R::kNibbles;  // first of kNibbles dims
                float *to = kAlone ? &join_sums[wave][kAlone ? l32 : 0][kAlone ? d : 0] : segments.sums + place * kDim + d;
                uint16_t *out = a.output + query * a.output_stride + (size_t)head * kDim + d;
#pragma unroll
                for (int n = 0; n < R::kNibbles; n += 2) {
                    if (!kAlone && entire) *(uint32_t *)(out + n) = (uint32_t)f2h(acc[n][e] * inv) | (uint32_t)f2h(acc[n + 1][e] * inv) << 16;
                    else *(float2 *)(to + n) = make_float2(acc[n][e], acc[n + 1][e]);
                }
            }
        }
        if constexpr (kAlone) {
            __syncthreads();
            join_waves<kDim, kRows, kWaves, R::kJoinStride>(a, tile, kv, heads, join_bases, (const float *)join_sums);
            return;
        }
        left -= count;
        if (left <= 0) return;
        offset = 0;
        do {
            if (++number >= numbers) return;
            tile = RowTile(a, plan, number, kRows, R::kStep);
        } while (tile.steps == 0);
    }
}

// Joins the segments of four rows of a row tile, or writes the zeros of rows that see nothing. kLanes lanes a row and
// segment: kDim / 4 for all dims, or 8 and a workgroup for every 32 dims, which makes enough of them even for one sequence,
// whose hundreds of segments are then read in a few round trips.
constexpr int kJoinThreads = 256;
template <int kDim, int kRows, int kStep, int kLanes>
__global__ __launch_bounds__(kJoinThreads) void attention_join_kernel(const AttentionKv4Args a, const RowPlan plan, size_t segments_at) {
    constexpr int kAtOnce = kJoinThreads / (4 * kLanes), kParts = kDim / (4 * kLanes), kJoinWaves = kJoinThreads / kWave;
    extern __shared__ float weights[];  // [4][parts]
    __shared__ float highest[4][kJoinWaves], totals[4][kJoinWaves];
    __shared__ float4_t sums[kAtOnce][4][kLanes];
    const int number = blockIdx.x, kv = blockIdx.y, first_row = blockIdx.z / kParts * 4, first_dim = blockIdx.z % kParts * 4 * kLanes;
    const Segments segments(a, plan, kRows, segments_at);
    const int2 parts = segments.parts[number];
    const RowTile tile(a, plan, number, kRows, kStep);
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

// ------------------------------------------------------------------------------------------------- many rows: prompts
//
// Bound: the matrix cores, 4 * kDim flops per row, head and seen position, with the vector pipe close behind (a score costs
// some eight instructions, and a position's 10 kDim bits become 32 kDim). A workgroup has 256 rows (query rows times the
// heads that share a kv head), 32 per wave; tiles of kTile positions are brought to fp16 once for all of them, into LDS,
// while the tile before is worked on. 128 rows a workgroup took 211 us for a prompt of 4096 (32 heads, 8 kv heads of 128),
// 256 take 171, 804 TFLOP/s of the seen half; a library's product of 8192^3 runs at 1177 on the card.
// k and v are rounded to fp16 there, and p for the second product: three roundings of 2^-12 (root mean square) next to the
// result's own; exact codes and two pieces of p, as for few rows, would cost as much again as all the rest.
// v's rows of positions are stored with their 16-byte pieces exchanged by the row's eight (an exclusive or): the writes of a wave,
// eight rows apart, would otherwise meet in two banks.
// Transposed products (k q^T, v^T p^T) put a row's scores into one lane and its partner 32 lanes on, and p is then the next
// product's operand as it lies, if v's positions are ordered like the result rows of the first product (8 b + 4 h + r).
template <int kDim, int kWaves_>
struct Prompt {
    static constexpr int kGroups = kDim / kKvGroup, kWords = kDim / 8;
    static constexpr int kWaves = kWaves_, kThreads = kWaves * kWave, kRows = kWaves * 32;
    static constexpr int kTile = 32 * kThreads / kDim;  // 32 values of k and of v per thread
    static constexpr int kKeyBytes = kDim * 2 + 16, kValueBytes = kTile * 2 + 16;  // rows in LDS, off the banks' period
    static constexpr int kKeyTile = kTile * kKeyBytes, kStage = kKeyTile + kDim * kValueBytes;
    static constexpr int kChunk = 64, kSub = kChunk / 32, kDepths = kDim / 16;  // positions that a wave has scores of at once
};
template <int kDim, int kWaves>
__global__ __launch_bounds__(kWaves *kWave, 2) void attention_prompt_kernel(const AttentionKv4Args a, const RowPlan plan, size_t segments_at) {
    using P = Prompt<kDim, kWaves>;
    constexpr int G = P::kGroups;
    __shared__ __align__(16) unsigned char stage[2][P::kStage];
    __shared__ uint32_t unsound[2][P::kTile + 1];  // groups of each position's value that are not finite; and whether any is
    const Kv4Cache &c = a.cache;
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), half = lane >> 5, l32 = lane & 31;
    const int kv = blockIdx.x, worker = blockIdx.y + blockIdx.z * gridDim.y;
    if (worker >= plan.workers) return;
    const int heads = a.n_heads / c.n_kv_heads, numbers = a.batch.batch * plan.tiles;
    int number, offset = 0, left = INT32_MAX;
    RowTile tile;
    if (plan.alone) {
        // last tiles first: they see the most
        number = worker % a.batch.batch * plan.tiles + plan.tiles - 1 - worker / a.batch.batch;
        tile = RowTile(a, plan, number, P::kRows, P::kTile);
        if (tile.rows_left <= 0) return;
    } else {
        const bool scribe = kv == 0 && worker == 0 && wave == 0;
        const Segments segments(a, plan, P::kRows, segments_at);
        if (!find_piece(a, plan, worker, P::kRows, P::kTile, kv == 0 && worker == 0, scribe ? segments.parts : nullptr, &number, &offset, &left, &tile)) return;
    }
    const int limit = position_limit(a);
    const size_t code_words = kv4_code_words(1 << c.page_shift, kDim), scale_words = kv4_scale_words(1 << c.page_shift, kDim);
    // (the sign is the row operand's; a scale of 0 makes that 0, so that what is left out can stay at minus infinity)
    const float to_log2 = (a.scale == 0.0f ? 1.0f : fabsf(a.scale)) * 1.44269504088896f;

    while (true) {
        const int count = min(tile.steps - offset, left);
        const bool entire = plan.alone || (offset == 0 && count == tile.steps);
        const int *table = a.batch.table + (size_t)(plan.tiles == 1 ? number : number / plan.tiles) * a.batch.width;
        const int first = tile.first_step + offset, end = first + count;

        // this lane's row, and its operand
        const int in_tile = wave * 32 + l32, at_row = tile.first_row + in_tile;
        const bool real = in_tile < tile.rows_left;
        const size_t query = (size_t)(tile.row0 + (real ? at_row / heads : 0));
        const int head = kv * heads + (real ? at_row % heads : 0), pos = real ? tile.pos0 + at_row / heads : -1;
        half8_t q[P::kDepths];
#pragma unroll
        for (int k = 0; k < P::kDepths; k++) {
            q[k] = real ? *(const half8_t *)(a.q + query * a.q_stride + (size_t)head * kDim + k * 16 + half * 8) : half8_t{};
            if (a.scale < 0) q[k] = -q[k];
            if (a.scale == 0) q[k] = half8_t{};
        }
        const int wave_rows = min(32, tile.rows_left - wave * 32);  // (none: the wave only helps with the tiles)
        const int wave_low = max(tile.pos0 + (tile.first_row + wave * 32) / heads, -1), wave_high = tile.pos0 + (tile.first_row + wave * 32 + max(wave_rows, 1) - 1) / heads;

        int held_from = first * P::kTile >> c.page_shift, held = table[min(held_from + lane, a.batch.width - 1)];
        struct Raw {
            uint4_t k, v, v_scales;
            uint32_t k_scales[4];
            uint32_t there;  // bit i: positions 16 i .. 16 i + 15 have a page
        };
        static_assert(P::kTile / 16 == kWaves * (4 / G) && P::kTile <= 512, "a wave takes 16 positions (kDim 64: two times 16); a bit each");
        // A wave takes 16 whole positions of the tile, so that their page is the same for all its lanes: of the keys, a lane has
        // one depth quad of every group of a position, of the values a word of four positions (kDim 64: half the lanes each 16).
        constexpr int kBlocks = 4 / G;
        const int k_quad = lane & 3, k_pos = lane >> 2;
        const int v_block = lane & 3, v_word = G == 4 ? lane >> 2 : lane >> 2 & 7, v_part = G == 4 ? 0 : lane >> 5;
        const uint32_t k_offset = (uint32_t)(k_pos * P::kWords + k_quad * G) * 4, ks_offset = (uint32_t)k_pos * 4;
        const uint32_t v_offset = (uint32_t)(v_block * 4 * P::kWords + v_word * 4) * 4;
        const size_t vs_offset = (((size_t)(v_word / 4) << c.page_shift) + v_block * 4) * 4;  // (the fourth group of the largest page: beyond 32 bits)
        const int slots = (1 << c.page_shift) - 1;
        auto load = [&](int step) {
            Raw x;
            const int at = step * P::kTile, last = (at + P::kTile - 16) >> c.page_shift;
            if (last >= held_from + kWave) {
                held_from = at >> c.page_shift;
                held = table[min(held_from + lane, a.batch.width - 1)];
            }
            const int index = (at + 16 * lane) >> c.page_shift, its = __shfl(held, min(index - held_from, kWave - 1), kWave);
            x.there = (uint32_t)__ballot(lane < P::kTile / 16 && index < a.batch.width && its >= 0 && its < c.n_pages);
            const unsigned char *v_at[2], *vs_at[2];
#pragma unroll
            for (int i = 0; i < kBlocks; i++) {
                const int part = wave + kWaves * i, from = at + 16 * part;
                const int page = x.there >> part & 1 ? __builtin_amdgcn_readlane(held, (from >> c.page_shift) - held_from) : 0;
                const size_t block = (size_t)(page * c.n_kv_heads + kv), slot = from & slots;
                const unsigned char *k_at = (const unsigned char *)(c.k_codes + block * code_words + slot * P::kWords) + k_offset;
                const unsigned char *ks_at = (const unsigned char *)(c.k_scales + block * scale_words + slot) + ks_offset;
                v_at[i] = (const unsigned char *)(c.v_codes + block * code_words + slot * P::kWords) + v_offset;
                vs_at[i] = (const unsigned char *)(c.v_scales + block * scale_words + slot) + vs_offset;
                if constexpr (G == 4) {
                    x.k = *(const uint4_t *)k_at;
                } else {
                    const uint2_t two = *(const uint2_t *)k_at;
                    x.k[2 * i] = two[0];
                    x.k[2 * i + 1] = two[1];
                }
#pragma unroll
                for (int g = 0; g < G; g++) x.k_scales[G * i + g] = *(const uint32_t *)(ks_at + ((size_t)g << (c.page_shift + 2)));
            }
            x.v = *(const uint4_t *)(kBlocks == 2 && v_part ? v_at[1] : v_at[0]);
            x.v_scales = *(const uint4_t *)(kBlocks == 2 && v_part ? vs_at[1] : vs_at[0]);
            return x;
        };
        uint32_t even_bits = kEvenBits, odd_bits = kOddBits;  // (in registers: two constants make two instructions)
        asm("" : "+v"(even_bits), "+v"(odd_bits));
        const auto value2 = [&](auto cut, uint32_t field, bool odd, half2_t s, half2_t m) { return values_of<cut.value>(field, odd, odd ? odd_bits : even_bits, s, m); };
        auto store = [&](const Raw &x, int step, int into) {
            const int at = step * P::kTile;
            unsigned char *keys = stage[into], *values = stage[into] + P::kKeyTile;
            const auto put_keys = [&](auto cut, const uint4_t &words) {
#pragma unroll
                for (int pair = 0; pair < 2; pair++) {
                    const uint32_t w0 = words[2 * pair], w1 = words[2 * pair + 1];
                    const int to = 16 * (wave + (G == 4 ? 0 : kWaves * pair)) + k_pos, group = G == 4 ? 2 * pair : 0;
#pragma unroll
                    for (int odd = 0; odd < 2; odd++) {
                        const half2_t both = __builtin_bit_cast(half2_t, x.k_scales[2 * pair + odd]), s = {both[0], both[0]}, m = {both[1], both[1]};
                        const uint4_t out = {value2(cut, w0, odd, s, m), value2(cut, w0 >> 8, odd, s, m), value2(cut, w1, odd, s, m), value2(cut, w1 >> 8, odd, s, m)};
                        *(uint4_t *)(keys + to * P::kKeyBytes + ((group + odd) * 32 + k_quad * 8) * 2) = out;
                    }
                }
            };
            uint32_t large_key = 0, large = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) large_key |= large_bits(x.k_scales[i]);
            put_keys(std::false_type{}, x.k);
            if (__ballot(large_key & kLargeMask)) {
                uint4_t words = x.k;
                anew(words);
                put_keys(std::true_type{}, words);  // (again, with what is beyond fp16's range cut)
            }
            // what no row sees may be anything: its values are zeros (its scores are left out); so are the groups that are not
            // finite, which the rows that see them get from `unsound`
            const int part = wave + kWaves * v_part, from = at + 16 * part + v_block * 4;
            uint32_t scales[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                scales[j] = x.v_scales[j];
                large |= large_bits(scales[j]);
            }
            // (positions of this step that all lie where some row sees them: all but the ends)
            const bool inside = x.there == (uint32_t)((1ull << (P::kTile / 16)) - 1) && at + P::kTile - 1 <= min(tile.pos_high, limit - 1) && (a.window == 0 || at > tile.pos_low - a.window);
            const bool any_large = __ballot(large & kLargeMask);
            if (!inside || any_large) {
                asm volatile("");
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int t = from + j;
                    const bool seen = (x.there >> part & 1) && t <= tile.pos_high && t < limit && (a.window == 0 || t > tile.pos_low - a.window);
                    const uint32_t w = scales[j];
                    const bool bad = not_finite(w);
                    if (seen && bad) {
                        atomicOr(&unsound[into][t - at], 1u << (v_word / 4));
                        unsound[into][P::kTile] = 1;
                    }
                    scales[j] = seen && !bad ? w : 0;
                }
            }
            half2_t s[2], m[2];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                s[j] = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(scales[2 * j + 1], scales[2 * j], 0x05040100u));
                m[j] = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(scales[2 * j + 1], scales[2 * j], 0x07060302u));
            }
            unsigned char *to = values + v_word * 8 * P::kValueBytes + ((part * 32 + (v_block & 1) * 16) ^ (v_word & 15) << 4) + (v_block >> 1) * 8;
            const auto put_values = [&](auto cut, const uint4_t &words) {
#pragma unroll
                for (int piece = 0; piece < 2; piece++) {
                    const uint32_t select = piece ? 0x07060302u : 0x05040100u;
                    const uint32_t p0 = __builtin_amdgcn_perm(words[1], words[0], select), p1 = __builtin_amdgcn_perm(words[3], words[2], select);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint2_t out = {value2(cut, i & 2 ? p0 >> 8 : p0, i & 1, s[0], m[0]), value2(cut, i & 2 ? p1 >> 8 : p1, i & 1, s[1], m[1])};
                        *(uint2_t *)(to + (piece * 4 + i) * P::kValueBytes) = out;
                    }
                }
            };
            put_values(std::false_type{}, x.v);
            if (any_large) {
                uint4_t words = x.v;
                anew(words);
                put_values(std::true_type{}, words);
            }
        };

        float16_t acc[G] = {};  // 32 dims each: transposed, this lane's row
        float sum = 0, base = kEmpty;
        uint32_t there = 0;
        for (int t = threadIdx.x; t <= P::kTile; t += P::kThreads) unsound[0][t] = unsound[1][t] = 0;
        __syncthreads();
        Raw next;
        if (first < end) {
            next = load(first);
            there = next.there;
            store(next, first, 0);
            if (first + 1 < end) next = load(first + 1);
        }
        __syncthreads();
        for (int step = first; step < end; step++) {
            const int now = (step - first) & 1, at = step * P::kTile;
            const bool any_unsound = unsound[now][P::kTile];
            uint32_t then = 0;
            auto prepare = [&] {
                if (step + 1 >= end) return;
                then = next.there;
                store(next, step + 1, now ^ 1);
                if (step + 2 < end) next = load(step + 2);
            };
            // (the two waves of a SIMD begin a tile with different work: one uses the vector pipe while the other multiplies)
            if (wave >= kWaves / 2) prepare();
#pragma unroll 1
            for (int chunk = 0; chunk < P::kTile; chunk += P::kChunk) {
                const int from = at + chunk;
                // (a wave none of whose rows sees any of the positions leaves them out)
                if (wave_rows <= 0 || from > wave_high || (a.window > 0 && from + P::kChunk - 1 <= wave_low - a.window)) continue;
                const unsigned char *keys = stage[now] + (chunk + l32) * P::kKeyBytes + half * 16;
                const unsigned char *values = stage[now] + P::kKeyTile + l32 * P::kValueBytes;
                const uint32_t pages = there >> (chunk / 16) & ((1u << (P::kChunk / 16)) - 1);
                const bool whole = pages == (1u << (P::kChunk / 16)) - 1 && from + P::kChunk - 1 <= wave_low && from + P::kChunk <= limit && (a.window == 0 || from > wave_high - a.window);
                float16_t x[P::kSub];
                float most = -INFINITY;
                // (the order written here is kept: a read of LDS 4 matrix instructions ahead of its use. Left to itself the compiler
                // puts each read right before its use, and both waves of a SIMD wait for LDS half the time: a prompt of 4096 takes 180 us, 170 so)
                constexpr int kReads = P::kSub * P::kDepths, kAhead = 4;
                const auto key = [&](int at) { return *(const half8_t *)(keys + 32 * (at / P::kDepths) * P::kKeyBytes + at % P::kDepths * 32); };
                half8_t ahead[kAhead];
#pragma unroll
                for (int j = 0; j < kAhead; j++) ahead[j] = key(j);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < P::kSub; i++) x[i] = float16_t{};
#pragma unroll
                for (int j = 0; j < kReads; j++) {
                    x[j / P::kDepths] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ahead[j % kAhead], q[j % P::kDepths], x[j / P::kDepths], 0, 0, 0);
                    if (j + kAhead < kReads) ahead[j % kAhead] = key(j + kAhead);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (!whole) {
                    asm volatile("");
#pragma unroll
                    for (int i = 0; i < P::kSub; i++)
#pragma unroll
                        for (int j = 0; j < 16; j++) {
                            const int t = from + 32 * i + 8 * (j >> 2) + 4 * half + (j & 3);
                            const bool sees = t <= pos && t < limit && (a.window == 0 || t > pos - a.window) && (pages >> (2 * i + (j >> 3)) & 1);
                            x[i][j] = sees ? x[i][j] : -INFINITY;
                        }
                }
#pragma unroll
                for (int i = 0; i < P::kSub; i++)
#pragma unroll
                    for (int j = 0; j < 16; j++) most = fmaxf(most, x[i][j]);
                most = fmaxf(most, __shfl_xor(most, 32, kWave)) * to_log2;
                if (__ballot(most - base > 14.0f)) {
                    const float to = fmaxf(base, most - 6.0f), keep = __builtin_amdgcn_exp2f(base - to);
                    base = to;
                    sum *= keep;
#pragma unroll
                    for (int g = 0; g < G; g++) acc[g] *= keep;
                }
                // the second 32 positions' weights are worked out between the first's matrix instructions
                constexpr int kProducts = 2 * G, kPiece = 16 / kProducts;
                const auto read = [&](int i, int j) {
                    const int k = j / G, g = j % G;
                    return *(const half8_t *)(values + 32 * g * P::kValueBytes + ((chunk * 2 + (32 * i + 16 * k) * 2 + half * 16) ^ ((4 * g + (l32 >> 3)) & 15) << 4));
                };
                half8_t value[kProducts], weights[P::kSub][2];
                const auto weigh = [&](int i, int from_j, int n) {
#pragma unroll
                    for (int j = from_j; j < from_j + n; j++) weights[i][j >> 3][j & 7] = (_Float16)__builtin_amdgcn_exp2f(__builtin_fmaf(x[i][j], to_log2, -base));
#pragma unroll
                    for (int j = from_j; j < from_j + n; j += 2)  // (of the rounded weights, which is what the values are multiplied with)
                        sum = __builtin_amdgcn_fdot2(half2_t{weights[i][j >> 3][j & 7], weights[i][j >> 3][(j & 7) + 1]}, half2_t{1, 1}, sum, false);
                };
#pragma unroll
                for (int j = 0; j < kProducts; j++) value[j] = read(0, j);
                weigh(0, 0, 16);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < P::kSub; i++)
#pragma unroll
                    for (int j = 0; j < kProducts; j++) {
                        acc[j % G] = __builtin_amdgcn_mfma_f32_32x32x16_f16(value[j], weights[i][j / G], acc[j % G], 0, 0, 0);
                        if (i + 1 < P::kSub) {
                            value[j] = read(i + 1, j);
                            weigh(i + 1, j * kPiece, kPiece);
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    }
                if (any_unsound) {
                    for (int t = chunk; t < chunk + P::kChunk; t++) {
                        const uint32_t groups = unsound[now][t];
                        const bool sees = at + t <= pos && (a.window == 0 || at + t > pos - a.window);
#pragma unroll
                        for (int g = 0; g < G; g++)
                            if (groups >> g & 1) acc[g] = sees ? float16_t{} + NAN : acc[g];
                    }
                }
            }
            if (wave < kWaves / 2) prepare();
            there = then;
            __syncthreads();
            if (any_unsound) {
                for (int t = threadIdx.x; t <= P::kTile; t += P::kThreads) unsound[now][t] = 0;
                __syncthreads();
            }
        }

        sum += __shfl_xor(sum, 32, kWave);
        if (real) {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // nothing seen: 0
            const Segments segments(a, plan, P::kRows, segments_at);
            const size_t slot = ((size_t)kv * segments.per_head + worker + number) * P::kRows + in_tile;
            if (!entire && half == 0) *(float2 *)(segments.bases + slot * 2) = make_float2(base, sum);
#pragma unroll
            for (int g = 0; g < G; g++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int d = 32 * g + 8 * j + 4 * half;
                    if (entire) {
                        const uint2_t packed = {(uint32_t)f2h(acc[g][4 * j] * inv) | (uint32_t)f2h(acc[g][4 * j + 1] * inv) << 16,
                                                (uint32_t)f2h(acc[g][4 * j + 2] * inv) | (uint32_t)f2h(acc[g][4 * j + 3] * inv) << 16};
                        *(uint2_t *)(a.output + query * a.output_stride + (size_t)head * kDim + d) = packed;
                    } else {
                        *(float4_t *)(segments.sums + slot * kDim + d) =
                            float4_t{acc[g][4 * j], acc[g][4 * j + 1], acc[g][4 * j + 2], acc[g][4 * j + 3]};
                    }
                }
        }
        left -= count;
        if (plan.alone || left <= 0) return;
        offset = 0;
        do {
            if (++number >= numbers) return;
            tile = RowTile(a, plan, number, P::kRows, P::kTile);
        } while (tile.steps == 0);
    }
}

// ------------------------------------------------------------------------------------------------- launches

// Rows (query rows times heads of a kv head) up to which a sequence goes the way of few rows. 16 sequences of 8192 positions,
// 64 rows each: 111 us, 138 as a prompt; 128 rows: 181 and 140. (One sequence of 8192 positions, 64 rows: 35 and 20.)
constexpr int kFewRows = 64;

// Rows of a tile: 4 and 8 take bare codes, 32 values brought to fp16. 8 rows, 131 072 positions: 47 us with 8, 56 with 32; 4
// rows, 72 000 positions: 34 with 4, 42 with 32. (Bare codes with 16 rows a tile took as long as 32 rows take now: 60 us for
// 16 rows of 16 sequences of 8192, and 99 for 32.)
int decode_rows(long long rows) { return rows <= 4 ? 4 : rows <= 8 ? 8 : 32; }

// What a call launches: for sequences of few rows, for sequences of many, or both.
struct Plans {
    bool few, many;
    RowPlan few_plan, many_plan;
    int few_rows;  // per tile
    int many_waves;
    size_t few_bytes, many_bytes;
};

// Positions that a row tile may see, as far as the host knows.
long long reach(const AttentionKv4Args &a) {
    return a.window > 0 ? std::min((long long)a.window + a.max_query, (long long)a.max_length) : a.max_length;
}

constexpr int kPromptWaves = 8;
template <int kDim>
Plans plans_of(const AttentionKv4Args &a) {
    const int kv = a.cache.n_kv_heads, cus = std::min(current_device_cus(), 256), heads = a.n_heads / kv;
    const long long rows = (long long)a.max_query * heads;
    Plans p{};
    // One sequence, or as many rows as all sequences can have: no sequence is expected to be shorter than the others
    const bool alike = a.batch.batch == 1 || (long long)a.batch.batch * a.max_query <= a.batch.n_tokens;
    p.many = rows > kFewRows;
    p.few = !p.many || !alike;
    if (p.few) {
        const long long most = std::min<long long>(rows, kFewRows);
        p.few_rows = decode_rows(most);
        // (32 rows' sums are 16 KB a segment: fewer, of four steps at least. One sequence of 8192 positions and 16 rows: 18 us,
        // with one step at least 24, with eight 23)
        p.few_plan = RowPlan{0, (int)((most + p.few_rows - 1) / p.few_rows), p.few_rows == 32 ? 4 : 1, 0, 0, p.many ? kFewRows + 1 : INT32_MAX};
        // A row tile a workgroup takes the time of its positions on one CU, 8 us and some 5 per 1024; the line takes 11 us and
        // what all positions cost on all CUs. 4 rows, 1 sequence: 512 positions 10 us alone and 11 in line, 1024 12 and 12,
        // 2048 18 and 12; 8 sequences (64 workgroups): 1024 13 and 14, 2048 18 and 17, 4096 30 and 22; 32 (256): 4096 32 and
        // 39. Only a bound of the lengths is known here: a single long sequence among many short ones costs more alone (8192
        // among 200 to 8192: 51 us, in line 34), so that 4096 positions are the most.
        const long long groups = (long long)a.batch.batch * p.few_plan.tiles * kv;
        p.few_plan.alone = reach(a) <= std::min(512 + 16 * groups, 4096ll);
        // two waves a SIMD
        p.few_plan.workers = p.few_plan.alone ? a.batch.batch * p.few_plan.tiles : (8 * cus + kv - 1) / kv;
        p.few_bytes = p.few_plan.alone ? 0 : (Segments::bytes(a, p.few_plan, p.few_rows) + 15) / 16 * 16;
    }
    if (p.many) {
        p.many_waves = kPromptWaves;
        const int tile_rows = p.many_waves * 32, step = 2048 * p.many_waves / kDim;
        p.many_plan = RowPlan{0, (int)((rows + tile_rows - 1) / tile_rows), 1, 0, p.few ? kFewRows + 1 : 0, INT32_MAX};
        const long long tiles = (long long)a.batch.batch * p.many_plan.tiles;
        const int slots = 8 / p.many_waves * cus;  // two waves a SIMD
        // A row tile alone takes some 4.5 us per step of the longest; in line all steps are shared out evenly, and what a tile of 256
        // rows leaves behind and its join cost some 32 us. (32 heads, 8 kv heads of 128, rows behind positions: 512 of 512 28 us
        // alone and 43 in line, 1024 of 1024 43 and 63, 2048 of 2048 75 and 115; twice 512 of 2048 73 and 75; 512 of 2048 73 and
        // 56, 100 of 2000 71 and 31.)
        const long long steps = (reach(a) + step - 1) / step;
        p.many_plan.alone = steps * (slots - tiles * kv) <= 7ll * slots;
        p.many_plan.workers = p.many_plan.alone ? (int)tiles : (slots + kv - 1) / kv;
        p.many_plan.least = 2;
        p.many_bytes = p.many_plan.alone ? 0 : Segments::bytes(a, p.many_plan, tile_rows);
    }
    return p;
}

// The kernels count row tiles, and in line the steps of positions of all of them, in 32 bits (as many as the sizes allow, whatever
// the arrays hold), and the counts are rounded up to whole grids and pieces.
template <int kDim>
bool counts_fit(const AttentionKv4Args &a) {
    const Plans p = plans_of<kDim>(a);
    const auto fits = [&](const RowPlan &plan, int step) {
        const long long numbers = (long long)a.batch.batch * plan.tiles, steps = (a.max_length - 1) / step + 1;
        return (plan.alone ? numbers : numbers * steps) < INT32_MAX - (1 << 16);
    };
    return (!p.few || fits(p.few_plan, p.few_rows == 4 ? Decode<kDim, 4>::kStep : Decode<kDim, 8>::kStep)) &&
           (!p.many || fits(p.many_plan, Prompt<kDim, kPromptWaves>::kTile));
}

dim3 worker_grid(const AttentionKv4Args &a, const RowPlan &plan) {
    const int across = std::min(plan.workers, 32768);
    return dim3((unsigned)a.cache.n_kv_heads, (unsigned)across, (unsigned)((plan.workers + across - 1) / across));
}

template <int kDim, int kRows, int kStep>
hipError_t launch_join(const AttentionKv4Args &a, const RowPlan &plan, size_t segments_at, hipStream_t s) {
    const unsigned tiles = (unsigned)(a.batch.batch * plan.tiles), kv = (unsigned)a.cache.n_kv_heads;
    const size_t lds = 16 * (size_t)plan.workers;  // a weight per row and part, of which there are at most `workers`
    // 8 lanes a row and segment for few rows always, for more where the workgroups of kDim / 4 lanes would not give every CU one:
    // 131 072 positions of one sequence 47.5 us with 8 and 52.1 with 32, 32 ragged users 33.4 and 34.0; 512 rows behind 9000
    // positions, three times, 320 and 279, 64 rows behind 8192, 16 times, 116 and 108.
    if (kRows <= 8 || (long long)tiles * kv * (kRows / 4) < current_device_cus()) {
        attention_join_kernel<kDim, kRows, kStep, 8><<<dim3(tiles, kv, kRows / 4 * (kDim / 32)), kJoinThreads, lds, s>>>(a, plan, segments_at);
        return hipGetLastError();
    }
    if constexpr (kRows > 8) attention_join_kernel<kDim, kRows, kStep, kDim / 4><<<dim3(tiles, kv, kRows / 4), kJoinThreads, lds, s>>>(a, plan, segments_at);
    return hipGetLastError();
}

template <int kDim>
hipError_t launch_rows32(const AttentionKv4Args &a, const RowPlan &plan, hipStream_t s) {
    if (plan.alone) {
        attention_rows_kernel<kDim, kAloneWaves><<<worker_grid(a, plan), kAloneWaves * kWave, 0, s>>>(a, plan);
        return hipGetLastError();
    }
    attention_rows_kernel<kDim, 1><<<worker_grid(a, plan), kWave, 0, s>>>(a, plan);
    if (hipError_t e = hipGetLastError()) return e;
    return launch_join<kDim, 32, Rows32<kDim>::kStep>(a, plan, 0, s);
}

template <int kDim, int kRows>
hipError_t launch_few(const AttentionKv4Args &a, const RowPlan &plan, hipStream_t s) {
    if (plan.alone) {
        attention_decode_kernel<kDim, kRows, kAloneWaves><<<worker_grid(a, plan), kAloneWaves * kWave, 0, s>>>(a, plan);
        return hipGetLastError();
    }
    attention_decode_kernel<kDim, kRows, 1><<<worker_grid(a, plan), kWave, 0, s>>>(a, plan);
    if (hipError_t e = hipGetLastError()) return e;
    return launch_join<kDim, kRows, Decode<kDim, kRows>::kStep>(a, plan, 0, s);
}

template <int kDim, int kWaves>
hipError_t launch_many(const AttentionKv4Args &a, const RowPlan &plan, size_t segments_at, hipStream_t s) {
    using P = Prompt<kDim, kWaves>;
    attention_prompt_kernel<kDim, kWaves><<<worker_grid(a, plan), P::kThreads, 0, s>>>(a, plan, segments_at);
    if (hipError_t e = hipGetLastError()) return e;
    return plan.alone ? hipSuccess : launch_join<kDim, P::kRows, P::kTile>(a, plan, segments_at, s);
}

template <int kDim>
hipError_t launch(const AttentionKv4Args &a, hipStream_t s) {
    const Plans p = plans_of<kDim>(a);
    if (p.many)
        if (hipError_t e = launch_many<kDim, kPromptWaves>(a, p.many_plan, p.few_bytes, s)) return e;
    if (!p.few) return hipSuccess;
    switch (p.few_rows) {
        case 4: return launch_few<kDim, 4>(a, p.few_plan, s);
        case 8: return launch_few<kDim, 8>(a, p.few_plan, s);
        default: return launch_rows32<kDim>(a, p.few_plan, s);
    }
}

}  // namespace

bool attention_kv4_fits(const AttentionKv4Args &a) { return a.cache.head_dim == 64 ? counts_fit<64>(a) : counts_fit<128>(a); }

size_t attention_kv4_workspace(const AttentionKv4Args &a) {
    const Plans p = a.cache.head_dim == 64 ? plans_of<64>(a) : plans_of<128>(a);
    return p.few_bytes + p.many_bytes;
}

hipError_t launch_attention_kv4(const AttentionKv4Args &a, hipStream_t s) {
    return a.cache.head_dim == 64 ? launch<64>(a, s) : launch<128>(a, s);
}

}  // namespace tllm
