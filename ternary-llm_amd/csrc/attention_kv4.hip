// Attention of the rows of a batch over the 4-bit paged cache: o = softmax(scale q k^T) v over the positions a row sees.
#include "kv4.h"

namespace tllm {
namespace {

// Simple form: one wave per (row, head). 64 positions at a time, a lane each for the scores, two dims (one) of the output
// per lane for the values; running maximum and sum in fp32.
template <int kDim>
__global__ __launch_bounds__(64) void attention_rows_kernel(const AttentionKv4Args a) {
    constexpr int kWords = kDim / 8, kPer = kDim / 64;
    __shared__ float q[kDim], p[64];
    __shared__ int blocks[64];
    const Kv4Cache &c = a.cache;
    const Kv4Batch &b = a.batch;
    const int lane = threadIdx.x, row = blockIdx.x, head = blockIdx.y, kv = head / (a.n_heads / c.n_kv_heads);
    const int seq = kv4_find_sequence(b.starts, b.batch, row);
    if (seq >= b.batch || b.starts[seq] > row) return;
    const int page_size = 1 << c.page_shift;
    const int capacity = min(b.width << c.page_shift, a.max_length);
    const int pos = kv4_position(b, seq, row, INT32_MAX);
    const int end = min(pos + 1, capacity);
    const int begin = a.window > 0 ? max(0, pos + 1 - a.window) : 0;
    for (int d = lane; d < kDim; d += 64) q[d] = h2f(a.q[(size_t)row * a.q_stride + head * kDim + d]);
    __syncthreads();
    float sums[kDim / 32];
    for (int g = 0; g < kDim / 32; g++) {
        sums[g] = 0;
        for (int d = 0; d < 32; d++) sums[g] += q[g * 32 + d];
    }
    float top = -INFINITY, total = 0, o[kPer] = {};
    for (int t0 = begin & ~63; t0 < end; t0 += 64) {
        const int t = t0 + lane;
        float score = -INFINITY;
        int block = -1;
        const int slot = t & (page_size - 1);
        if (t >= begin && t < end) {
            const int page = b.table[(size_t)seq * b.width + (t >> c.page_shift)];
            if (page >= 0 && page < c.n_pages) block = page * c.n_kv_heads + kv;
        }
        if (block >= 0) {
            const uint32_t *kc = c.k_codes + (size_t)block * kv4_code_words(page_size, kDim) + (size_t)slot * kWords;
            const uint32_t *ks = c.k_scales + (size_t)block * kv4_scale_words(page_size, kDim) + slot;
            float acc[kDim / 32] = {};
            for (int w = 0; w < kWords; w++) {
                const int quad = w / (kDim / 32), g = w % (kDim / 32) & ~1, half = w & 1;
                for (int j = 0; j < 4; j++) {
                    const int shift = 4 * (4 * (j & 1) + (j & 2)), d = quad * 8 + half * 4 + j;
                    acc[g] += (float)(kc[w] >> shift & 15) * q[g * 32 + d];
                    acc[g + 1] += (float)(kc[w] >> (shift + 4) & 15) * q[g * 32 + 32 + d];
                }
            }
            score = 0;
            for (int g = 0; g < kDim / 32; g++) {
                const uint32_t pair = ks[(size_t)g * page_size];
                score += h2f((uint16_t)pair) * acc[g] + h2f((uint16_t)(pair >> 16)) * sums[g];
            }
            score *= a.scale;
        }
        float most = score;
        for (int off = 32; off; off >>= 1) most = fmaxf(most, __shfl_xor(most, off, 64));
        const float now = fmaxf(top, most);
        const float base = now == -INFINITY ? 0.0f : now, keep = expf(top - base);
        const float e = expf(score - base);
        top = now;
        total = total * keep + wave_sum(e);
        p[lane] = e;
        blocks[lane] = block;
        __syncthreads();
        for (int i = 0; i < kPer; i++) o[i] *= keep;
        for (int j = 0; j < 64; j++) {
            if (blocks[j] < 0) continue;
            const int at = (t0 + j) & (page_size - 1);
            for (int i = 0; i < kPer; i++) {
                const int d = lane + 64 * i;
                const uint32_t w = c.v_codes[(size_t)blocks[j] * kv4_code_words(page_size, kDim) + (size_t)(at >> 2) * (kWords * 4) + (d >> 3) * 4 + (at & 3)];
                const uint32_t pair = c.v_scales[(size_t)blocks[j] * kv4_scale_words(page_size, kDim) + (size_t)(d >> 5) * page_size + at];
                o[i] += p[j] * ((float)(w >> (4 * (d & 7)) & 15) * h2f((uint16_t)pair) + h2f((uint16_t)(pair >> 16)));
            }
        }
        __syncthreads();
    }
    for (int i = 0; i < kPer; i++)
        a.output[(size_t)row * a.output_stride + head * kDim + lane + 64 * i] = f2h(total > 0 || total != total ? o[i] / total : 0.0f);
}

}  // namespace

size_t attention_kv4_workspace(const AttentionKv4Args &a) {
    (void)a;
    return 0;
}

hipError_t launch_attention_kv4(const AttentionKv4Args &a, hipStream_t s) {
    const dim3 grid((unsigned)a.batch.n_tokens, (unsigned)a.n_heads);
    if (a.cache.head_dim == 64) attention_rows_kernel<64><<<grid, 64, 0, s>>>(a);
    else attention_rows_kernel<128><<<grid, 64, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace tllm
