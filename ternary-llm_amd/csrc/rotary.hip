// Rotary position embedding with a position per token, both pair layouts, part of the head and scaled rates.
//
// Pair i of a head (i < rotary_dim / 2) of the token at position p turns by the angle p * w_i and is multiplied by
// `magnitude`: (x0, x1) -> (x0 c - x1 s, x0 s + x1 c), c = magnitude cos(p w_i), s = magnitude sin(p w_i).
// w_i = theta^(-2i / rotary_dim), changed by the scaling (RotaryArgs below).
//
// Bound: HBM, 4 bytes per element of q and k. The angles are a matter of latency only: a workgroup works out the
// cosines and sines of its tokens once (one lane per pair, fp64 up to the fraction of a turn, which is where far
// positions would lose their digits, fp32 from there) and uses them for every head through LDS.
#include "common.h"

namespace tllm {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ double pair_rate(const RotaryArgs &a, int i) {
    const double rate = exp2(-a.log2_theta * (2.0 * i) / (double)a.rotary_dim);
    double blend;  // share of the kept rate; the rest is divided by the factor
    switch (a.scaling) {
        case TLLM_ROTARY_LINEAR: return rate * a.inv_factor;
        case TLLM_ROTARY_BANDED: blend = (a.turns_per_rate * rate - a.low) * a.inv_width; break;
        case TLLM_ROTARY_YARN: blend = 1.0 - (i - a.low) * a.inv_width; break;
        default: return rate;  // none, and NTK (whose theta the host has changed)
    }
    blend = fmin(fmax(blend, 0.0), 1.0);
    return rate * (a.inv_factor + (1.0 - a.inv_factor) * blend);
}

__device__ __forceinline__ void turn(uint32_t &w0, uint32_t &w1, const float2 (&cs)[2]) {
    // (w0, w1) hold the first and the second members of two pairs, low and high half
    const float a0 = h2f((uint16_t)w0), b0 = h2f((uint16_t)w1), a1 = h2f((uint16_t)(w0 >> 16)), b1 = h2f((uint16_t)(w1 >> 16));
    w0 = (uint32_t)f2h(a0 * cs[0].x - b0 * cs[0].y) | (uint32_t)f2h(a1 * cs[1].x - b1 * cs[1].y) << 16;
    w1 = (uint32_t)f2h(a0 * cs[0].y + b0 * cs[0].x) | (uint32_t)f2h(a1 * cs[1].y + b1 * cs[1].x) << 16;
}

// A unit of work: one head of one token, one piece of it. Vector form: pieces of 16 bytes (interleaved, and the part of
// the head behind rotary_dim) or of two times 16 bytes half a rotary_dim apart (half layout). Scalar form (sizes, strides
// or pointers that 16-byte pieces do not fit): one pair, or one element behind rotary_dim.
template <bool kVec>
__global__ __launch_bounds__(kThreads) void rotary_kernel(const RotaryArgs a, int tokens_per_wg, int units_per_head, int turned_units) {
    extern __shared__ float2 cs[];  // [tokens_per_wg][pairs]
    const int pairs = a.rotary_dim / 2;
    const int first = blockIdx.x * tokens_per_wg;
    const int tokens = min(tokens_per_wg, a.n_tokens - first);
    for (int j = threadIdx.x; j < tokens * pairs; j += kThreads) {
        const int t = j / pairs, i = j - t * pairs;
        const double turns = (double)a.positions[first + t] * (pair_rate(a, i) * 0.15915494309189533577);  // 1 / (2 pi)
        float s, c;
        sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
        cs[j] = make_float2(c * a.magnitude, s * a.magnitude);
    }
    __syncthreads();
    const int units = (a.n_heads + a.n_kv_heads) * units_per_head;  // of one token
    for (int j = blockIdx.y * kThreads + threadIdx.x; j < tokens * units; j += kThreads * gridDim.y) {
        const int t = j / units, rest = j - t * units;
        int head = rest / units_per_head;
        const int u = rest - head * units_per_head;
        const uint16_t *x;
        uint16_t *y;
        const size_t token = (size_t)(first + t);
        if (head < a.n_heads) {
            x = a.q + token * a.q_stride + (size_t)head * a.head_dim;
            y = a.q_out + token * a.q_out_stride + (size_t)head * a.head_dim;
        } else {
            head -= a.n_heads;
            x = a.k + token * a.k_stride + (size_t)head * a.head_dim;
            y = a.k_out + token * a.k_out_stride + (size_t)head * a.head_dim;
        }
        const float2 *w = cs + t * pairs;
        if constexpr (kVec) {
            if (u >= turned_units) {  // behind rotary_dim: as it is
                const int at = a.rotary_dim + (u - turned_units) * 8;
                if (x != y) *(uint4 *)(y + at) = *(const uint4 *)(x + at);
            } else if (a.half_layout) {
                const uint4 p = *(const uint4 *)(x + u * 8), q = *(const uint4 *)(x + pairs + u * 8);
                uint32_t pw[4] = {p.x, p.y, p.z, p.w}, qw[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float2 two[2] = {w[u * 8 + 2 * e], w[u * 8 + 2 * e + 1]};
                    turn(pw[e], qw[e], two);
                }
                *(uint4 *)(y + u * 8) = make_uint4(pw[0], pw[1], pw[2], pw[3]);
                *(uint4 *)(y + pairs + u * 8) = make_uint4(qw[0], qw[1], qw[2], qw[3]);
            } else {
                const uint4 p = *(const uint4 *)(x + u * 8);
                uint32_t pw[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    // two neighbouring words hold two pairs side by side: sorted into first and second members and back
                    uint32_t f = (pw[e] & 0xFFFFu) | pw[e + 1] << 16, s = pw[e] >> 16 | (pw[e + 1] & 0xFFFF0000u);
                    const float2 two[2] = {w[u * 4 + e], w[u * 4 + e + 1]};
                    turn(f, s, two);
                    pw[e] = (f & 0xFFFFu) | s << 16;
                    pw[e + 1] = f >> 16 | (s & 0xFFFF0000u);
                }
                *(uint4 *)(y + u * 8) = make_uint4(pw[0], pw[1], pw[2], pw[3]);
            }
        } else {
            if (u >= turned_units) {
                const int at = a.rotary_dim + (u - turned_units);
                y[at] = x[at];
            } else {
                const int i0 = a.half_layout ? u : 2 * u, i1 = a.half_layout ? u + pairs : 2 * u + 1;
                const float x0 = h2f(x[i0]), x1 = h2f(x[i1]), c = w[u].x, s = w[u].y;
                y[i0] = f2h(x0 * c - x1 * s);
                y[i1] = f2h(x0 * s + x1 * c);
            }
        }
    }
}

}  // namespace

hipError_t launch_rotary(const RotaryArgs &a, hipStream_t s) {
    const int pairs = a.rotary_dim / 2;
    uintptr_t all = (uintptr_t)a.q | (uintptr_t)a.q_out | (uintptr_t)((a.q_stride | a.q_out_stride) * 2);
    if (a.n_kv_heads) all |= (uintptr_t)a.k | (uintptr_t)a.k_out | (uintptr_t)((a.k_stride | a.k_out_stride) * 2);
    const bool vec = (all & 15) == 0 && a.head_dim % 8 == 0 && a.rotary_dim % (a.half_layout ? 16 : 8) == 0;
    const int turned = vec ? a.rotary_dim / (a.half_layout ? 16 : 8) : pairs;
    const int per_head = turned + (a.head_dim - a.rotary_dim) / (vec ? 8 : 1);
    // One lane per cosine in the first phase: as many tokens as fill a workgroup. When that leaves CUs without work, one
    // token per workgroup, its heads dealt to several.
    int per_wg = kThreads / pairs;
    if (per_wg < 1) per_wg = 1;
    int split = 1;
    const int cus = current_device_cus();
    if ((a.n_tokens + per_wg - 1) / per_wg < 2 * cus) {
        per_wg = 1;
        const long long units = (long long)(a.n_heads + a.n_kv_heads) * per_head;
        const long long want = (units + kThreads - 1) / kThreads, room = (4 * cus + a.n_tokens - 1) / a.n_tokens;
        split = (int)(want < room ? want : room);
    }
    const dim3 grid((unsigned)((a.n_tokens + per_wg - 1) / per_wg), (unsigned)split);
    const size_t lds = (size_t)per_wg * pairs * sizeof(float2);
    if (vec) rotary_kernel<true><<<grid, kThreads, lds, s>>>(a, per_wg, per_head, turned);
    else rotary_kernel<false><<<grid, kThreads, lds, s>>>(a, per_wg, per_head, turned);
    return hipGetLastError();
}

}  // namespace tllm
