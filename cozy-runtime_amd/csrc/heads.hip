// Queries and keys between the QKV projection and attention: each head's RMS norm and its rotation
// to the token's position, one read and one write of every element.
//
//   y = x · rsqrt(mean(x²) + eps) · gain,   (y_a, y_b) -> (y_a·cos − y_b·sin, y_b·cos + y_a·sin)
//
// over the first `rotated` elements of a head, paired as halves (i, i + rotated/2) or as neighbours
// (2i, 2i + 1), with cos and sin of the token's position from a float32 table. Everything between the
// 16-bit load and the one rounding at the store is float32.
#include <hip/hip_runtime.h>

#include "common.h"
#include "kernels.h"
#include "sixteen.h"

namespace cozyq {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ void load8f(const float* p, float* v) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const f32x4 raw = *reinterpret_cast<const f32x4*>(p + 4 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * i + j] = raw[j];
    }
}

// A head is width/16 units of 16 elements, one a lane, on `lanes` lanes (a power of two). A unit of
// the rotated part holds both elements of eight pairs, so that a rotation needs no other lane: for
// halves the chunks u and u + rotated/16 of eight elements, otherwise the neighbours 2u and 2u + 1.
// Bound by memory over a prompt: 8191 tokens of 32 + 8 heads of 128 in 34.8 us, 172 MB at 4.9 TB/s, where a
// large copy runs at 5.6; the vector unit is busy 82% of that time, which is why the 16-bit type is a template
// parameter (chosen at run time both types' conversions were worked out). 4173 tokens of 20 + 20 heads of 64, 44 MB,
// take 12.1 us: the vector unit, busy 71%, beside memory at 3.6 TB/s, and the launch's beginning and end. 24 tokens take
// 3.7 us: a launch and one trip to memory, and one for the tables.
template <bool kHalf>
__global__ __launch_bounds__(kThreads) void norm_rope_kernel(HeadRows r) {
    const int64_t head_slot = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / r.lanes;
    const int u = threadIdx.x & (r.lanes - 1);
    const int heads = r.q_heads + r.k_heads;
    const int64_t token = head_slot / heads;
    const int head = static_cast<int>(head_slot - token * heads);
    const int units = r.width / 16, turning = r.rotated / 16;
    const bool live = token < r.tokens && u < units;
    float a[8], b[8];
    int at_a = 0, at_b = 0;
    uint16_t* out = nullptr;
    const void* gain = nullptr;
    if (live) {
        const bool is_q = head < r.q_heads;
        const int h = is_q ? head : head - r.q_heads;
        const uint16_t* x = is_q ? r.q + token * r.q_token + h * r.q_head : r.k + token * r.k_token + h * r.k_head;
        out = is_q ? r.q_out + (token * r.q_heads + h) * r.width : r.k_out + (token * r.k_heads + h) * r.width;
        gain = is_q ? r.q_gain : r.k_gain;
        at_a = 16 * u;
        at_b = 16 * u + 8;
        if (!r.interleaved && u < turning) {
            at_a = 8 * u;
            at_b = 8 * u + r.rotated / 2;
        }
        load8<kHalf>(x + at_a, a);
        load8<kHalf>(x + at_b, b);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = b[i] = 0.0f;
    }
    if (r.norm) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = __builtin_fmaf(a[i], a[i], __builtin_fmaf(b[i], b[i], sum));
        for (int step = 1; step < r.lanes; step *= 2) sum += __shfl_xor(sum, step);
        const float inv = __builtin_amdgcn_rsqf(sum / static_cast<float>(r.width) + r.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            a[i] *= inv;
            b[i] *= inv;
        }
        if (live && gain) {
            float ga[8], gb[8];
            if (r.gain_wide) {
                load8f(static_cast<const float*>(gain) + at_a, ga);
                load8f(static_cast<const float*>(gain) + at_b, gb);
            } else {
                load8<kHalf>(static_cast<const uint16_t*>(gain) + at_a, ga);
                load8<kHalf>(static_cast<const uint16_t*>(gain) + at_b, gb);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                a[i] *= ga[i];
                b[i] *= gb[i];
            }
        }
    }
    if (!live) return;
    if (u < turning) {
        int64_t row = r.positions ? r.positions[token] : token;
        row = row < 0 ? 0 : (row < r.table_rows ? row : r.table_rows - 1);
        const int64_t base = row * (r.rotated / 2) + 8 * u;
        float c[8], s[8];
        load8f(r.cos + base, c);
        load8f(r.sin + base, s);
        if (r.interleaved) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float a0 = a[2 * i], a1 = a[2 * i + 1], b0 = b[2 * i], b1 = b[2 * i + 1];
                a[2 * i] = a0 * c[i] - a1 * s[i];
                a[2 * i + 1] = a1 * c[i] + a0 * s[i];
                b[2 * i] = b0 * c[4 + i] - b1 * s[4 + i];
                b[2 * i + 1] = b1 * c[4 + i] + b0 * s[4 + i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x0 = a[i], x1 = b[i];
                a[i] = x0 * c[i] - x1 * s[i];
                b[i] = x1 * c[i] + x0 * s[i];
            }
        }
    }
    store8<kHalf>(out + at_a, a);
    store8<kHalf>(out + at_b, b);
}

}  // namespace

hipError_t head_norm_rope(HeadRows rows, hipStream_t s) {
    rows.lanes = 1;
    while (rows.lanes * 16 < rows.width) rows.lanes *= 2;
    const int64_t threads = static_cast<int64_t>(rows.tokens) * (rows.q_heads + rows.k_heads) * rows.lanes;
    if (threads == 0) return hipSuccess;
    const unsigned groups = static_cast<unsigned>((threads + kThreads - 1) / kThreads);
    if (rows.half) norm_rope_kernel<true><<<groups, kThreads, 0, s>>>(rows);
    else norm_rope_kernel<false><<<groups, kThreads, 0, s>>>(rows);
    return hipGetLastError();
}

}  // namespace cozyq
