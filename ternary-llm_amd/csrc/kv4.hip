// Writing rows into the 4-bit paged key/value cache and reading them back.
//
// A group of 32 dims of a row x is held as m = min x and s = fp16((max x - m) / 15), both fp16, and a code per value,
// c = rint((x - m) / s) of the exact quotient, kept in 0..15 (0 where s is 0); it stands for m + s c. A group with an
// element that is not finite is held as s = m = NaN.
//
// Bound: HBM, once the places are known: a row's place hangs on four loads in a row (starts, length, table, then the data),
// so a wave finds it once and goes through `heads` heads of k and v with it, two heads at a time in flight. (One head per wave
// took 190 us for reading 71 000 rows of 8 heads back, a chain of loads per 16 bytes a lane, and 222 us for writing and reading
// 34 000.) A row of one head is read in 16-byte pieces by head_dim / 8 neighbouring lanes (8 dims each, so four lanes share a group), and
// the next lanes take the next rows of the SAME head: the cache keeps four tokens' words of v next to each other (see
// tllm_kv4_cache), so the stores of a wave fill whole 256-byte stretches where the rows are consecutive tokens. Lanes by
// token and head in the order of the input would store 4 bytes of every 16.
#include "kv4.h"

namespace tllm {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ void unpack8(const uint4 &w, float (&x)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 4; j++) {
        x[2 * j] = h2f((uint16_t)u[j]);
        x[2 * j + 1] = h2f((uint16_t)(u[j] >> 16));
    }
}

// Codes of this lane's eight values (one per entry), and the step and minimum of their group (four lanes).
__device__ __forceinline__ uint32_t quantise8(const uint4 &in, uint32_t (&code)[8]) {
    float x[8];
    unpack8(in, x);
    float lo = x[0], hi = x[0];
#pragma unroll
    for (int j = 1; j < 8; j++) {
        lo = fminf(lo, x[j]);
        hi = fmaxf(hi, x[j]);
    }
    // an exponent of ones carries into its half's top bit (fmin and fmax drop a NaN)
    uint32_t odd_one = 0;
    const uint32_t words[4] = {in.x, in.y, in.z, in.w};
#pragma unroll
    for (int j = 0; j < 4; j++) odd_one |= (words[j] & 0x7C007C00u) + 0x04000400u;
#pragma unroll
    for (int off = 1; off <= 2; off <<= 1) {
        lo = fminf(lo, __shfl_xor(lo, off, kWave));
        hi = fmaxf(hi, __shfl_xor(hi, off, kWave));
        odd_one |= (uint32_t)__shfl_xor((int)odd_one, off, kWave);
    }
    if (odd_one & 0x80008000u) {
#pragma unroll
        for (int j = 0; j < 8; j++) code[j] = 0;
        return 0x7E007E00u;
    }
    // The difference of two fp16 values is exact in 64 bits and nearly always in 32. Where it is, its quotient by 15 rounds to
    // fp16 as the exact one does: 15 t has 16 bits for a tie t of fp16, so a range of 24 bits that is not 15 t is a unit of its
    // last place away from it, a fifteenth of which is more than half a unit of the quotient's.
    const float range = hi - lo, back = range - hi;
    uint16_t step = f2h(range / 15.0f);
    if ((hi - (range - back)) + (-lo - back) != 0.0f) step = f2h((float)(((double)hi - (double)lo) / 15.0));
    const float s = h2f(step), inv = step ? 1.0f / s : 0.0f;
    float nearest = 1.0f;  // how far from a half the quotients stay
#pragma unroll
    for (int j = 0; j < 8; j++) {
        // |q - exact quotient| < 16 * 3 * 2^-24 (three roundings, a quotient below 16 wherever the code is not cut to 15
        // anyway): only within that of a half are the quotients taken in 64 bits, where halves of fp16 data show exactly
        const float q = (x[j] - lo) * inv, c = rintf(q);
        nearest = fminf(nearest, 0.5f - fabsf(q - c));
        code[j] = (uint32_t)fminf(c, 15.0f);
    }
    if (nearest < 4e-6f && step) {
        for (int j = 0; j < 8; j++) code[j] = (uint32_t)fmin(rint(((double)x[j] - (double)lo) / (double)s), 15.0);
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

template <int kDim>
__global__ __launch_bounds__(kThreads) void kv4_append_kernel(const Kv4Cache c, const Kv4Batch b, const uint16_t *__restrict__ k,
                                                              const uint16_t *__restrict__ v, int64_t k_stride, int64_t v_stride, int heads) {
    constexpr int kWords = kDim / 8;
    const int lane = threadIdx.x % kWords, first = blockIdx.y * heads, end = min(first + heads, c.n_kv_heads);
    const bool keys = gridDim.z == 1 || blockIdx.z == 0, vals = gridDim.z == 1 || blockIdx.z == 1;
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
        const uint32_t other = __shfl_xor(odd ? half[0] : half[1], 4, kWave);
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
    for (int h = first; h < end; h += 2) {
        const int h1 = min(h + 1, end - 1);
        uint4 in[4];
        in[0] = in[1] = in[2] = in[3] = make_uint4(0, 0, 0, 0);
        if (here && keys) {
            in[0] = *(const uint4 *)(k_row + h * kDim);
            in[1] = *(const uint4 *)(k_row + h1 * kDim);
        }
        if (here && vals) {
            in[2] = *(const uint4 *)(v_row + h * kDim);
            in[3] = *(const uint4 *)(v_row + h1 * kDim);
        }
        const size_t block = page * c.n_kv_heads + h;
        if (keys) put_key(in[0], block);
        if (vals) put_value(in[2], block);
        if (h + 1 < end) {
            if (keys) put_key(in[1], block + 1);
            if (vals) put_value(in[3], block + 1);
        }
    }
}

template <int kDim>
__global__ __launch_bounds__(kThreads) void kv4_read_kernel(const Kv4Cache c, const Kv4Batch b, uint16_t *__restrict__ k,
                                                            uint16_t *__restrict__ v, int64_t k_stride, int64_t v_stride, int heads) {
    constexpr int kWords = kDim / 8;
    const int lane = threadIdx.x % kWords, first = blockIdx.y * heads, end = min(first + heads, c.n_kv_heads);
    const bool keys = gridDim.z == 1 || blockIdx.z == 0, vals = gridDim.z == 1 || blockIdx.z == 1;
    const Place p = find_place<kDim>(c, b);
    if (p.row < 0) return;
    const int page_size = 1 << c.page_shift;
    uint16_t *k_row = k + (size_t)p.row * k_stride + lane * 8, *v_row = v + (size_t)p.row * v_stride + lane * 8;
    if (p.page < 0) {
        for (int h = first; h < end; h++) {
            if (keys) *(uint4 *)(k_row + h * kDim) = make_uint4(0, 0, 0, 0);
            if (vals) *(uint4 *)(v_row + h * kDim) = make_uint4(0, 0, 0, 0);
        }
        return;
    }
    const size_t code_words = kv4_code_words(page_size, kDim), scale_words = kv4_scale_words(page_size, kDim);
    auto values = [&](auto nibble, uint32_t pair) {
        const float s = h2f((uint16_t)pair), m = h2f((uint16_t)(pair >> 16));
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            // m + 15 s may be half a step of s above the largest value: what would round beyond fp16 stays its largest
            float x = __builtin_fmaf((float)nibble(j), s, m);
            x = x != x ? x : fminf(fmaxf(x, -65504.0f), 65504.0f);
            if (j & 1) o[j / 2] |= (uint32_t)f2h(x) << 16;
            else o[j / 2] = f2h(x);
        }
        return make_uint4(o[0], o[1], o[2], o[3]);
    };
    const size_t block = (size_t)p.page * c.n_kv_heads, scale = (size_t)(lane >> 2) * page_size + p.slot;
    const uint32_t *kc = c.k_codes + block * code_words + key_word<kDim>(p.slot, lane), *ks = c.k_scales + block * scale_words + scale;
    const uint32_t *vc = c.v_codes + block * code_words + value_word<kDim>(p.slot, lane), *vs = c.v_scales + block * scale_words + scale;
    for (int h = first; h < end; h += 2) {
        const int h1 = min(h + 1, end - 1);
        uint2 k0 = make_uint2(0, 0), k1 = k0;
        uint32_t v0 = 0, v1 = 0, ks0 = 0, ks1 = 0, vs0 = 0, vs1 = 0;
        if (keys) {
            k0 = *(const uint2 *)(kc + h * code_words), k1 = *(const uint2 *)(kc + h1 * code_words);
            ks0 = ks[h * scale_words], ks1 = ks[h1 * scale_words];
        }
        if (vals) {
            v0 = vc[h * code_words], v1 = vc[h1 * code_words];
            vs0 = vs[h * scale_words], vs1 = vs[h1 * scale_words];
        }
        auto put = [&](int head, const uint2 &kw, uint32_t kp, uint32_t vw, uint32_t vp) {
            const uint32_t w[2] = {kw.x >> (lane & 4), kw.y >> (lane & 4)};  // (lane & 4: the odd group's nibbles are 4 bits up)
            if (keys) *(uint4 *)(k_row + head * kDim) = values([&](int j) { return w[j >> 2] >> (4 * (4 * (j & 1) + (j & 2))) & 15; }, kp);
            if (vals) *(uint4 *)(v_row + head * kDim) = values([&](int j) { return vw >> (4 * j) & 15; }, vp);
        };
        put(h, k0, ks0, v0, vs0);
        if (h + 1 < end) put(h + 1, k1, ks1, v1, vs1);
    }
}

// Heads per wave: all of them, or as few as it takes to give every CU sixteen waves; with a head a wave and still no more than
// that, k and v go to different workgroups. PLACEHOLDER
int heads_per_wave(const Kv4Cache &c, const Kv4Batch &b) {
    const unsigned rows = kThreads / (c.head_dim / 8), row_groups = ((unsigned)b.n_tokens + rows - 1) / rows;
    const unsigned want = 4 * (unsigned)current_device_cus();  // workgroups of four waves
    unsigned parts = (want + row_groups - 1) / row_groups;
    if (parts > (unsigned)c.n_kv_heads) parts = (unsigned)c.n_kv_heads;
    return (int)((c.n_kv_heads + parts - 1) / parts);
}

dim3 grid_of(const Kv4Cache &c, const Kv4Batch &b, int heads) {
    const unsigned rows = kThreads / (c.head_dim / 8), groups = ((unsigned)b.n_tokens + rows - 1) / rows;
    const unsigned parts = (unsigned)((c.n_kv_heads + heads - 1) / heads);
    return dim3(groups, parts, heads == 1 && (size_t)groups * parts * 2 <= 4 * (size_t)current_device_cus() ? 2 : 1);
}

}  // namespace

hipError_t launch_kv4_append(const Kv4Cache &c, const Kv4Batch &b, const uint16_t *k, const uint16_t *v, int64_t k_stride,
                             int64_t v_stride, hipStream_t s) {
    const int heads = heads_per_wave(c, b);
    const dim3 grid = grid_of(c, b, heads);
    if (c.head_dim == 64) kv4_append_kernel<64><<<grid, kThreads, 0, s>>>(c, b, k, v, k_stride, v_stride, heads);
    else kv4_append_kernel<128><<<grid, kThreads, 0, s>>>(c, b, k, v, k_stride, v_stride, heads);
    return hipGetLastError();
}

hipError_t launch_kv4_read(const Kv4Cache &c, const Kv4Batch &b, uint16_t *k, uint16_t *v, int64_t k_stride, int64_t v_stride,
                           hipStream_t s) {
    const int heads = heads_per_wave(c, b);
    const dim3 grid = grid_of(c, b, heads);
    if (c.head_dim == 64) kv4_read_kernel<64><<<grid, kThreads, 0, s>>>(c, b, k, v, k_stride, v_stride, heads);
    else kv4_read_kernel<128><<<grid, kThreads, 0, s>>>(c, b, k, v, k_stride, v_stride, heads);
    return hipGetLastError();
}

}  // namespace tllm
