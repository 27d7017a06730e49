// Writing rows into the 4-bit paged key/value cache and reading them back.
//
// A group of 32 dims of a row x is held as m = min x and s = fp16((max x - m) / 15), both fp16, and a code per value,
// c = rint((x - m) / s) of the exact quotient, kept in 0..15 (0 where s is 0); it stands for m + s c. A group with an
// element that is not finite is held as s = m = NaN.
//
// Bound: HBM, once the places are known. A row's place hangs on a chain of loads (starts, length, table), so a wave that has it
// takes two heads of k and v with it, all their loads in flight: reading 71 000 rows of 8 heads back takes 83 us so (a copy of
// as many bytes 76), 122 with one head a wave (the chain), 91 with all eight in turn (the last waves run alone); writing and
// reading 49 000 takes 116 (106), 143 and 121. Where that would give a CU fewer than sixteen waves, a wave takes one head, and
// where it still would, only k or v (48 rows of 8 heads: 6.6 us for both calls, 7.6 with k and v in one wave).
// A row of one head is read in 16-byte pieces by head_dim / 8 neighbouring lanes (8 dims each, so four lanes share a group), and
// the next lanes take the next rows of the SAME head: the cache keeps four tokens' words of v next to each other (see
// tllm_kv4_cache), so the stores of a wave fill whole 256-byte stretches where the rows are consecutive tokens. Lanes by
// token and head in the order of the input would store 4 bytes of every 16.
#include "kv4.h"

namespace tllm {
namespace {

constexpr int kThreads = 256;

// The value of the lane next to this one, next but one, next but three (DPP: no trip through LDS as a shuffle makes).
template <int kControl>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, kControl, 0xF, 0xF, false);
}
__device__ __forceinline__ uint32_t lane_xor1(uint32_t x) { return dpp<0xB1>(x); }         // quad_perm 1 0 3 2
__device__ __forceinline__ uint32_t lane_xor2(uint32_t x) { return dpp<0x4E>(x); }         // quad_perm 2 3 0 1
__device__ __forceinline__ uint32_t lane_xor4(uint32_t x) { return dpp<0x1B>(dpp<0x141>(x)); }  // mirrored in eight, then in four

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ half2_t as_half2(uint32_t x) { return __builtin_bit_cast(half2_t, x); }
__device__ __forceinline__ uint32_t as_word(half2_t x) { return __builtin_bit_cast(uint32_t, x); }

// Codes of this lane's eight values (one per entry), and the step and minimum of their group (four lanes).
__device__ __forceinline__ uint32_t quantise8(const uint4 &in, uint32_t (&code)[8]) {
    const uint32_t words[4] = {in.x, in.y, in.z, in.w};
    half2_t low = as_half2(in.x), high = low;
    uint32_t odd_one = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        low = __builtin_elementwise_min(low, as_half2(words[j]));
        high = __builtin_elementwise_max(high, as_half2(words[j]));
        // an exponent of ones carries into its half's top bit (the minimum and the maximum drop a NaN)
        odd_one |= (words[j] & 0x7C007C00u) + 0x04000400u;
    }
    low = __builtin_elementwise_min(low, as_half2(lane_xor1(as_word(low))));
    high = __builtin_elementwise_max(high, as_half2(lane_xor1(as_word(high))));
    odd_one |= lane_xor1(odd_one);
    low = __builtin_elementwise_min(low, as_half2(lane_xor2(as_word(low))));
    high = __builtin_elementwise_max(high, as_half2(lane_xor2(as_word(high))));
    odd_one |= lane_xor2(odd_one);
    if (odd_one & 0x80008000u) {
#pragma unroll
        for (int j = 0; j < 8; j++) code[j] = 0;
        return 0x7E007E00u;
    }
    const float lo = fminf((float)low[0], (float)low[1]), hi = fmaxf((float)high[0], (float)high[1]);
    // The difference of two fp16 values is exact in 64 bits and nearly always in 32. Where it is, its quotient by 15 rounds to
    // fp16 as the exact one does: 15 t has 16 bits for a tie t of fp16, so a range of 24 bits that is not 15 t is a unit of its
    // last place away from it, a fifteenth of which is more than half a unit of the quotient's. (The quotient: a product with
    // the rounded 1 / 15, then its residue, which the fused product gives exactly: rounded correctly.)
    const float range = hi - lo, back = range - hi, first = range * (1.0f / 15.0f);
    uint16_t step = f2h(__builtin_fmaf(__builtin_fmaf(first, -15.0f, range), 1.0f / 15.0f, first));
    if ((hi - (range - back)) + (-lo - back) != 0.0f) step = f2h((float)(((double)hi - (double)lo) / 15.0));
    const float s = h2f(step), inv = step ? __builtin_amdgcn_rcpf(s) : 0.0f;
    float off = 0.0f;  // how far from their codes the quotients are
#pragma unroll
    for (int j = 0; j < 8; j++) {
        // |q - exact quotient| < 16 * 4 * 2^-24 (two roundings and a reciprocal within a unit; the quotient is below 16 wherever
        // the code is not cut to 15 anyway): only within that of a half are the quotients taken in 64 bits, where halves of
        // fp16 data show exactly
        const float q = ((float)as_half2(words[j / 2])[j & 1] - lo) * inv, c = rintf(q);
        off = fmaxf(off, fabsf(q - c));
        code[j] = (uint32_t)fminf(c, 15.0f);
    }
    if (off > 0.5f - 5e-6f && step) {
        for (int j = 0; j < 8; j++)
            code[j] = (uint32_t)fmin(rint(((double)(float)as_half2(words[j / 2])[j & 1] - (double)lo) / (double)s), 15.0);
    }
    return (uint32_t)step | (uint32_t)f2h(lo) << 16;
}

// Where the row of this lane goes. kDim / 8 lanes per row.
struct Place {
    int row, slot;
    long long page;  // -1: no place
};
template <int kDim>
__device__ __forceinline__ Place find_place(const Kv4Cache &c, const Kv4Batch &b) {
    constexpr int kLanes = kDim / 8, kRows = kThreads / kLanes, kWaveRows = kWave / kLanes;
    const int wave = threadIdx.x / kWave, in_wave = (threadIdx.x & (kWave - 1)) / kLanes;
    const int first = blockIdx.x * kRows + wave * kWaveRows;
    Place p;
    p.row = first + in_wave;
    p.page = -1;
    p.slot = 0;
    int seq = kv4_find_sequence(b.starts, b.batch, first);
    if (p.row >= b.n_tokens) {
        p.row = -1;
        return p;
    }
    while (seq < b.batch && b.starts[seq + 1] <= p.row) seq++;
    if (seq >= b.batch || b.starts[seq] > p.row) {  // behind the last sequence, or before the first: left as it is
        p.row = -1;
        return p;
    }
    const int pos = kv4_position(b, seq, p.row, b.width << c.page_shift);
    if (pos < 0) return p;
    const int page = b.table[(size_t)seq * b.width + (pos >> c.page_shift)];
    if (page < 0 || page >= c.n_pages) return p;
    p.page = page;
    p.slot = pos & ((1 << c.page_shift) - 1);
    return p;
}

// This lane's word of a row in its (page, head) block, k's and v's.
template <int kDim>
__device__ __forceinline__ size_t key_word(int slot, int lane) {
    return (size_t)slot * (kDim / 8) + (lane & 3) * (kDim / 32) + 2 * (lane >> 3);
}
template <int kDim>
__device__ __forceinline__ size_t value_word(int slot, int lane) {
    return (size_t)(slot >> 2) * (kDim / 2) + lane * 4 + (slot & 3);
}

template <int kDim, bool kBoth>
__global__ __launch_bounds__(kThreads) void kv4_append_kernel(const Kv4Cache c, const Kv4Batch b, const uint16_t *__restrict__ k,
                                                              const uint16_t *__restrict__ v, int64_t k_stride, int64_t v_stride, int heads) {
    constexpr int kWords = kDim / 8;
    const int lane = threadIdx.x % kWords, h = blockIdx.y * heads;
    const bool two = heads == 2 && h + 1 < c.n_kv_heads;
    const bool keys = kBoth || blockIdx.z == 0, vals = kBoth || blockIdx.z == 1;
    const Place p = find_place<kDim>(c, b);
    // (lanes without a place work on zeros: their neighbours need them in the exchanges)
    const bool here = p.row >= 0 && p.page >= 0;
    const int page_size = 1 << c.page_shift;
    const size_t code_words = kv4_code_words(page_size, kDim), scale_words = kv4_scale_words(page_size, kDim);
    const size_t row = here ? p.row : 0, page = here ? p.page : 0;
    const uint16_t *k_row = k + row * k_stride + lane * 8, *v_row = v + row * v_stride + lane * 8;
    const bool odd = lane & 4, scribe = here && (lane & 3) == 0;
    auto put_key = [&](const uint4 &in, size_t block) {
        uint32_t code[8];
        const uint32_t pair = quantise8(in, code);
        // two groups share a word: the even nibbles are the even group's. A lane holds 8 dims of its group, half of them for each
        // of two words; the even group's lane stores the first word, the odd group's the second.
        uint32_t half[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; j++) half[j >> 2] |= code[j] << (4 * (4 * (j & 1) + (j & 2)));
        const uint32_t other = lane_xor4(odd ? half[0] : half[1]);
        if (here) c.k_codes[block * code_words + key_word<kDim>(p.slot, lane) + (odd ? 1 : 0)] = odd ? (half[1] << 4 | other) : (half[0] | other << 4);
        if (scribe) c.k_scales[block * scale_words + (size_t)(lane >> 2) * page_size + p.slot] = pair;
    };
    auto put_value = [&](const uint4 &in, size_t block) {
        uint32_t code[8], word = 0;
        const uint32_t pair = quantise8(in, code);
#pragma unroll
        for (int j = 0; j < 8; j++) word |= code[j] << (4 * j);
        if (here) c.v_codes[block * code_words + value_word<kDim>(p.slot, lane)] = word;
        if (scribe) c.v_scales[block * scale_words + (size_t)(lane >> 2) * page_size + p.slot] = pair;
    };
    uint4 in[4];
    in[0] = in[1] = in[2] = in[3] = make_uint4(0, 0, 0, 0);
    if (here && keys) {
        in[0] = *(const uint4 *)(k_row + h * kDim);
        in[1] = *(const uint4 *)(k_row + (h + two) * kDim);
    }
    if (here && vals) {
        in[2] = *(const uint4 *)(v_row + h * kDim);
        in[3] = *(const uint4 *)(v_row + (h + two) * kDim);
    }
    const size_t block = page * c.n_kv_heads + h;
    if (keys) {
        put_key(in[0], block);
        if (two) put_key(in[1], block + 1);
    }
    if (vals) {
        put_value(in[2], block);
        if (two) put_value(in[3], block + 1);
    }
}

template <int kDim, bool kBoth>
__global__ __launch_bounds__(kThreads) void kv4_read_kernel(const Kv4Cache c, const Kv4Batch b, uint16_t *__restrict__ k,
                                                            uint16_t *__restrict__ v, int64_t k_stride, int64_t v_stride, int heads) {
    constexpr int kWords = kDim / 8;
    const int lane = threadIdx.x % kWords, h = blockIdx.y * heads;
    const bool two = heads == 2 && h + 1 < c.n_kv_heads;
    const bool keys = kBoth || blockIdx.z == 0, vals = kBoth || blockIdx.z == 1;
    const Place p = find_place<kDim>(c, b);
    if (p.row < 0) return;
    const int page_size = 1 << c.page_shift;
    uint16_t *k_row = k + (size_t)p.row * k_stride + lane * 8, *v_row = v + (size_t)p.row * v_stride + lane * 8;
    if (p.page < 0) {
        for (int i = h; i <= h + two; i++) {
            if (keys) *(uint4 *)(k_row + i * kDim) = make_uint4(0, 0, 0, 0);
            if (vals) *(uint4 *)(v_row + i * kDim) = make_uint4(0, 0, 0, 0);
        }
        return;
    }
    const size_t code_words = kv4_code_words(page_size, kDim), scale_words = kv4_scale_words(page_size, kDim);
    // value = minimum + code * step for the codes of two dims at bits 0 and 16 of `codes`, in fp16 with one rounding (the code as
    // 1024 + code, less 1024: exact). It may be half a step above the largest fp16 value: what would round beyond stays that.
    auto pair_of = [&](uint32_t codes, uint32_t pair) {
        const half2_t code = as_half2((codes & 0x000F000Fu) | 0x64006400u) - (half2_t){(_Float16)1024, (_Float16)1024};
        const half2_t sm = as_half2(pair);
        return as_word(__builtin_elementwise_fma(code, (half2_t){sm[0], sm[0]}, (half2_t){sm[1], sm[1]}));
    };
    auto finite = [&](uint4 o, uint32_t pair) {
        const float s = h2f((uint16_t)pair), m = h2f((uint16_t)(pair >> 16));
        if (fabsf(__builtin_fmaf(15.0f, s, m)) > 65504.0f) {
            asm volatile("");  // (a branch that is hardly ever taken, not eight selects)
            uint32_t *word = &o.x;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if ((word[j] & 0x00007FFFu) == 0x00007C00u) word[j] -= 1;
                if ((word[j] & 0x7FFF0000u) == 0x7C000000u) word[j] -= 1u << 16;
            }
        }
        return o;
    };
    const size_t block = (size_t)p.page * c.n_kv_heads + h, scale = (size_t)(lane >> 2) * page_size + p.slot;
    const uint32_t *kc = c.k_codes + block * code_words + key_word<kDim>(p.slot, lane), *ks = c.k_scales + block * scale_words + scale;
    const uint32_t *vc = c.v_codes + block * code_words + value_word<kDim>(p.slot, lane), *vs = c.v_scales + block * scale_words + scale;
    uint2 k0 = make_uint2(0, 0), k1 = k0;
    uint32_t v0 = 0, v1 = 0, ks0 = 0, ks1 = 0, vs0 = 0, vs1 = 0;
    if (keys) {
        k0 = *(const uint2 *)kc, k1 = *(const uint2 *)(kc + two * code_words), ks0 = *ks, ks1 = ks[two * scale_words];
    }
    if (vals) {
        v0 = *vc, v1 = vc[two * code_words], vs0 = *vs, vs1 = vs[two * scale_words];
    }
    auto put_key = [&](int head, const uint2 &in, uint32_t pair) {
        const uint32_t w0 = in.x >> (lane & 4), w1 = in.y >> (lane & 4);  // (the odd group's nibbles are 4 bits up)
        *(uint4 *)(k_row + head * kDim) =
            finite(make_uint4(pair_of(w0, pair), pair_of(w0 >> 8, pair), pair_of(w1, pair), pair_of(w1 >> 8, pair)), pair);
    };
    auto put_value = [&](int head, uint32_t in, uint32_t pair) {
        const uint32_t o04 = pair_of(in, pair), o15 = pair_of(in >> 4, pair), o26 = pair_of(in >> 8, pair), o37 = pair_of(in >> 12, pair);
        auto lows = [](uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); };
        auto highs = [](uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); };
        *(uint4 *)(v_row + head * kDim) = finite(make_uint4(lows(o04, o15), lows(o26, o37), highs(o04, o15), highs(o26, o37)), pair);
    };
    if (keys) {
        put_key(h, k0, ks0);
        if (two) put_key(h + 1, k1, ks1);
    }
    if (vals) {
        put_value(h, v0, vs0);
        if (two) put_value(h + 1, v1, vs1);
    }
}

// Heads a wave takes, and the grid (rows, heads, k and v apart or not): see the top.
dim3 grid_of(const Kv4Cache &c, const Kv4Batch &b, int *heads) {
    const unsigned rows = kThreads / (c.head_dim / 8), groups = ((unsigned)b.n_tokens + rows - 1) / rows;
    const size_t full = 4 * (size_t)current_device_cus();  // workgroups of four waves
    const unsigned pairs = (unsigned)(c.n_kv_heads + 1) / 2;
    *heads = (size_t)groups * pairs >= full ? 2 : 1;
    const unsigned parts = *heads == 2 ? pairs : (unsigned)c.n_kv_heads;
    return dim3(groups, parts, (size_t)groups * parts >= full ? 1 : 2);
}

}  // namespace

hipError_t launch_kv4_append(const Kv4Cache &c, const Kv4Batch &b, const uint16_t *k, const uint16_t *v, int64_t k_stride,
                             int64_t v_stride, hipStream_t s) {
    int heads;
    const dim3 grid = grid_of(c, b, &heads);
    const auto kernel = c.head_dim == 64 ? (grid.z == 1 ? kv4_append_kernel<64, true> : kv4_append_kernel<64, false>)
                                         : (grid.z == 1 ? kv4_append_kernel<128, true> : kv4_append_kernel<128, false>);
    kernel<<<grid, kThreads, 0, s>>>(c, b, k, v, k_stride, v_stride, heads);
    return hipGetLastError();
}

hipError_t launch_kv4_read(const Kv4Cache &c, const Kv4Batch &b, uint16_t *k, uint16_t *v, int64_t k_stride, int64_t v_stride,
                           hipStream_t s) {
    int heads;
    const dim3 grid = grid_of(c, b, &heads);
    const auto kernel = c.head_dim == 64 ? (grid.z == 1 ? kv4_read_kernel<64, true> : kv4_read_kernel<64, false>)
                                         : (grid.z == 1 ? kv4_read_kernel<128, true> : kv4_read_kernel<128, false>);
    kernel<<<grid, kThreads, 0, s>>>(c, b, k, v, k_stride, v_stride, heads);
    return hipGetLastError();
}

}  // namespace tllm
