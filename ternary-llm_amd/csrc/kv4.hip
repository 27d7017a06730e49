// Writing rows into the 4-bit paged key/value cache and reading them back.
//
// A group of 32 dims of a row x is held as m = min x and s = fp16((max x - m) / 15), both fp16, and a code per value,
// c = rint((x - m) / s) of the exact quotient, kept in 0..15 (0 where s is 0); it stands for m + s c. A group with an
// element that is not finite is held as s = m = NaN.
//
// Bound: HBM. A row of one head is read in 16-byte pieces by head_dim / 8 neighbouring lanes (8 dims each, so four lanes
// share a group), and the next lanes take the next rows of the SAME head: the cache keeps four tokens' words of v next to
// each other (see tllm_kv4_cache), so the stores of a wave fill whole 256-byte stretches where the rows are consecutive
// tokens. Lanes by token and head in the order of the input would store 4 bytes of every 16.
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
    bool bad = false;  // (fmin and fmax drop a NaN)
#pragma unroll
    for (int j = 0; j < 8; j++) {
        lo = fminf(lo, x[j]);
        hi = fmaxf(hi, x[j]);
        bad |= !(fabsf(x[j]) <= 65504.0f);
    }
#pragma unroll
    for (int off = 1; off <= 2; off <<= 1) {
        lo = fminf(lo, __shfl_xor(lo, off, kWave));
        hi = fmaxf(hi, __shfl_xor(hi, off, kWave));
        bad |= (bool)__shfl_xor((int)bad, off, kWave);
    }
    if (bad) {
#pragma unroll
        for (int j = 0; j < 8; j++) code[j] = 0;
        return 0x7E007E00u;
    }
    // in 64 bits: the difference of two fp16 values is exact there and need not be in 32
    const uint16_t step = f2h((float)(((double)hi - (double)lo) / 15.0));
    const float s = h2f(step), inv = step ? 1.0f / s : 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        // |q - exact quotient| < 16 * 3 * 2^-24 (three roundings, a quotient below 16 wherever the code is not cut to 15
        // anyway): only within that of a half is the quotient taken in 64 bits, where halves of fp16 data show exactly
        const float q = (x[j] - lo) * inv;
        float c = rintf(q);
        if (fabsf(q - c) > 0.5f - 4e-6f && step) c = (float)rint(((double)x[j] - (double)lo) / (double)s);
        code[j] = (uint32_t)fminf(c, 15.0f);
    }
    return (uint32_t)step | (uint32_t)f2h(lo) << 16;
}

// Where the rows of this lane go: row index, its sequence's position, its page's first words. kDim / 8 lanes per row.
template <int kDim>
struct Place {
    int row, slot;
    long long block;  // page * n_kv_heads + head, or -1: no place
};
template <int kDim>
__device__ __forceinline__ Place<kDim> find_place(const Kv4Cache &c, const Kv4Batch &b, int head) {
    constexpr int kLanes = kDim / 8, kRows = kThreads / kLanes, kWaveRows = kWave / kLanes;
    const int wave = threadIdx.x / kWave, in_wave = (threadIdx.x & (kWave - 1)) / kLanes;
    const int first = blockIdx.x * kRows + wave * kWaveRows;
    Place<kDim> p;
    p.row = first + in_wave;
    p.block = -1;
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
    p.block = (long long)page * c.n_kv_heads + head;
    p.slot = pos & ((1 << c.page_shift) - 1);
    return p;
}

template <int kDim>
__global__ __launch_bounds__(kThreads) void kv4_append_kernel(const Kv4Cache c, const Kv4Batch b, const uint16_t *__restrict__ k,
                                                              const uint16_t *__restrict__ v, int64_t k_stride, int64_t v_stride) {
    constexpr int kWords = kDim / 8;
    const int head = blockIdx.y, lane = threadIdx.x % kWords;
    const Place<kDim> p = find_place<kDim>(c, b, head);
    // (lanes without a place work on zeros: their neighbours need them in the exchange below)
    const bool here = p.row >= 0 && p.block >= 0;
    const int page_size = 1 << c.page_shift;
    const bool is_v = blockIdx.z;
    uint4 in = make_uint4(0, 0, 0, 0);
    if (here) in = *(const uint4 *)((is_v ? v + (size_t)p.row * v_stride : k + (size_t)p.row * k_stride) + head * kDim + lane * 8);
    uint32_t code[8];
    const uint32_t pair = quantise8(in, code);
    uint32_t word;
    size_t at;
    if (is_v) {
        word = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) word |= code[j] << (4 * j);
        at = (size_t)(p.slot >> 2) * (kWords * 4) + lane * 4 + (p.slot & 3);
    } else {
        // two groups share a word: the even nibbles are the even group's. A lane holds 8 dims of its group, half of them
        // for each of two words; the even group's lane stores the first word, the odd group's the second.
        uint32_t half[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; j++) half[j >> 2] |= code[j] << (4 * (4 * (j & 1) + (j & 2)));
        const bool odd = lane & 4;
        const uint32_t other = __shfl_xor(odd ? half[0] : half[1], 4, kWave);
        word = odd ? (half[1] << 4 | other) : (half[0] | other << 4);
        at = (size_t)p.slot * kWords + (lane & 3) * (kDim / 32) + 2 * (lane >> 3) + (odd ? 1 : 0);
    }
    if (!here) return;
    (is_v ? c.v_codes : c.k_codes)[p.block * kv4_code_words(page_size, kDim) + at] = word;
    if ((lane & 3) == 0)
        (is_v ? c.v_scales : c.k_scales)[p.block * kv4_scale_words(page_size, kDim) + (size_t)(lane >> 2) * page_size + p.slot] = pair;
}

template <int kDim>
__global__ __launch_bounds__(kThreads) void kv4_read_kernel(const Kv4Cache c, const Kv4Batch b, uint16_t *__restrict__ k,
                                                            uint16_t *__restrict__ v, int64_t k_stride, int64_t v_stride) {
    constexpr int kWords = kDim / 8;
    const int head = blockIdx.y, lane = threadIdx.x % kWords;
    const Place<kDim> p = find_place<kDim>(c, b, head);
    if (p.row < 0) return;
    const int page_size = 1 << c.page_shift;
    const bool is_v = blockIdx.z;
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (p.block >= 0) {
        const uint32_t pair = (is_v ? c.v_scales : c.k_scales)[p.block * kv4_scale_words(page_size, kDim) + (size_t)(lane >> 2) * page_size + p.slot];
        const float s = h2f((uint16_t)pair), m = h2f((uint16_t)(pair >> 16));
        if (is_v) {
            const uint32_t w = c.v_codes[p.block * kv4_code_words(page_size, kDim) + (size_t)(p.slot >> 2) * (kWords * 4) + lane * 4 + (p.slot & 3)];
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = __builtin_fmaf((float)(w >> (4 * j) & 15), s, m);
        } else {
            const uint32_t *at = c.k_codes + p.block * kv4_code_words(page_size, kDim) + (size_t)p.slot * kWords + (lane & 3) * (kDim / 32) + 2 * (lane >> 3);
            const uint2 two = *(const uint2 *)at;
            const uint32_t w[2] = {two.x >> (lane & 4), two.y >> (lane & 4)};  // (lane & 4: the odd group's nibbles are 4 bits up)
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = __builtin_fmaf((float)(w[j >> 2] >> (4 * (4 * (j & 1) + (j & 2))) & 15), s, m);
        }
    }
    // m + 15 s may be half a step of s above the largest value: what would round beyond fp16 stays its largest
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = x[j] != x[j] ? x[j] : fminf(fmaxf(x[j], -65504.0f), 65504.0f);
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; j++) o[j] = (uint32_t)f2h(x[2 * j]) | (uint32_t)f2h(x[2 * j + 1]) << 16;
    *(uint4 *)((is_v ? v + (size_t)p.row * v_stride : k + (size_t)p.row * k_stride) + head * kDim + lane * 8) = make_uint4(o[0], o[1], o[2], o[3]);
}

dim3 row_grid(const Kv4Cache &c, const Kv4Batch &b) {
    const int rows = kThreads / (c.head_dim / 8);
    return dim3((unsigned)((b.n_tokens + rows - 1) / rows), (unsigned)c.n_kv_heads, 2);
}

}  // namespace

hipError_t launch_kv4_append(const Kv4Cache &c, const Kv4Batch &b, const uint16_t *k, const uint16_t *v, int64_t k_stride,
                             int64_t v_stride, hipStream_t s) {
    if (c.head_dim == 64) kv4_append_kernel<64><<<row_grid(c, b), kThreads, 0, s>>>(c, b, k, v, k_stride, v_stride);
    else kv4_append_kernel<128><<<row_grid(c, b), kThreads, 0, s>>>(c, b, k, v, k_stride, v_stride);
    return hipGetLastError();
}

hipError_t launch_kv4_read(const Kv4Cache &c, const Kv4Batch &b, uint16_t *k, uint16_t *v, int64_t k_stride, int64_t v_stride,
                           hipStream_t s) {
    if (c.head_dim == 64) kv4_read_kernel<64><<<row_grid(c, b), kThreads, 0, s>>>(c, b, k, v, k_stride, v_stride);
    else kv4_read_kernel<128><<<row_grid(c, b), kThreads, 0, s>>>(c, b, k, v, k_stride, v_stride);
    return hipGetLastError();
}

}  // namespace tllm
