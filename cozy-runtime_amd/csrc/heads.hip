// Queries and keys between the QKV projection and attention: each head's RMS norm and its rotation
// to the token's position, one read and one write of every element.
//
//   y = x · rsqrt(mean(x²) + eps) · gain,   (y_a, y_b) -> (y_a·cos − y_b·sin, y_b·cos + y_a·sin)
//
// over the first `rotated` elements of a head, paired as halves (i, i + rotated/2) or as neighbours
// (2i, 2i + 1), with cos and sin of the token's position from a float32 table. A token may have a position on each
// of several axes (time, height, width): every pair then belongs to one of them. Everything between the
// 16-bit load and the one rounding at the store is float32.
#include <hip/hip_runtime.h>

#include "common.h"
#include "kernels.h"
#include "sixteen.h"

namespace cozyq {
namespace {

constexpr int kThreads = 256;
// From so many waves of one run each on, a wave takes several, one after another, of one token: its cosines and sines are
// then read fewer times, but with fewer waves there is less to hide a wave's waiting behind. On one axis, one run and up
// to three a wave, us (bf16, cold): 8500 waves (1700 tokens of 32 + 8 heads of 128) 12.8 / 12.6, 12500 15.6 / 15.8, 16500
// 19.8 / 18.5, 40955 40.1 / 37.5; 9900 of 12 + 12 13.7 / 13.4, 24573 27.3 / 24.2; 12519 of 20 + 20 of 64 14.2 / 15.1,
// 24573 23.6 / 22.8. On three axes, whose tables are three times as much, one and up to four: 6000 waves of 32 + 8 10.9 /
// 11.9, 8500 14.4 / 13.9, 40955 48.5 / 40.5; 7500 of 12 + 12 13.7 / 12.8, 24573 31.3 / 26.5; 7500 of 20 + 20 of 64 11.3 /
// 12.2, 12519 16.0 / 16.4, 18000 21.8 / 20.0.
constexpr int kManyWaves = 16384, kMostRuns = 3, kManyAxesWaves = 7168, kMostAxesRuns = 4;

// The tables' row of a position, the nearest one where there is none.
__device__ __forceinline__ int64_t table_row(const HeadRows& r, int position) {
    return position < 0 ? 0 : (position < r.table_rows ? position : r.table_rows - 1);
}

// The cosines and sines of eight pairs from 8 * u on, of a token. On several axes a lane reads every axis' rows and keeps,
// of each pair, its own axis': whole lines that the token's other lanes share, rather than a gather a pair.
template <bool kAxes>
__device__ __forceinline__ void turns_of(const HeadRows& r, int token, int u, float* c, float* s) {
    const int64_t row = table_row(r, r.positions ? r.positions[token] : token) * (r.rotated / 2) + 8 * u;
    load8f(r.cos + row, c);
    load8f(r.sin + row, s);
    if constexpr (!kAxes) return;
    const uint32_t axis = r.axis_of[u];
    for (int a = 1; a < r.axes; ++a) {
        const int64_t other = table_row(r, r.positions[static_cast<int64_t>(a) * r.tokens + token]) * (r.rotated / 2) + 8 * u;
        float ca[8], sa[8];
        load8f(r.cos + other, ca);
        load8f(r.sin + other, sa);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const bool mine = ((axis >> (2 * i)) & 3) == static_cast<uint32_t>(a);
            c[i] = mine ? ca[i] : c[i];
            s[i] = mine ? sa[i] : s[i];
        }
    }
}

// A head is width/16 units of 16 elements, one a lane, on `lanes` lanes (a power of two). A unit of
// the rotated part holds both elements of eight pairs, so that a rotation needs no other lane: for
// halves the chunks u and u + rotated/16 of eight elements, otherwise the neighbours 2u and 2u + 1.
// A wave takes the next 64 / lanes heads, of whatever tokens; or (kRuns) 64 / lanes heads of one token at a time, `runs`
// times: a lane's cosines and sines are then the same for all of them and are read once.
// Bound by memory over a prompt on one axis: 8191 tokens of 32 + 8 heads of 128 in 31.5 us, 172 MB at 5.5 TB/s, where a
// large copy runs at 5.6 (VALU 78% busy); by memory and the vector unit on three: 35.1 us, 4.9 TB/s, VALU 75%. 4173 tokens of
// 20 + 20 heads of 64, 44 MB, take 13.6 us and 14.8 on three axes: waves that wait (66% and 71% of their life) and the
// launch's beginning and end. 24 tokens take 3.9 and 4.7 us: a launch and two trips to memory. What is a template parameter
// saves the other's instructions (both types' conversions) or registers (72 with several axes, 55 with one).
template <bool kHalf, bool kAxes, bool kRuns>
__global__ __launch_bounds__(kThreads) void norm_rope_kernel(HeadRows r, int parts) {
    const int lane = threadIdx.x & 63, u = lane & (r.lanes - 1), slots = 64 / r.lanes;
    const int64_t wave = static_cast<int64_t>(blockIdx.x) * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int heads = r.q_heads + r.k_heads;
    int token, head;
    if constexpr (kRuns) {
        token = static_cast<int>(wave / parts);
        head = static_cast<int>(wave - static_cast<int64_t>(token) * parts) * r.runs * slots + lane / r.lanes;
    } else {
        const int64_t slot = wave * slots + lane / r.lanes;
        token = static_cast<int>(slot / heads);
        head = static_cast<int>(slot - static_cast<int64_t>(token) * heads);
    }
    if (token >= r.tokens) return;  // with all of its head's lanes
    const int units = r.width / 16, turning = r.rotated / 16;
    int at_a = 16 * u, at_b = 16 * u + 8;
    if (!r.interleaved && u < turning) {
        at_a = 8 * u;
        at_b = 8 * u + r.rotated / 2;
    }
    float c[8], s[8];
    if (kRuns && u < turning) turns_of<kAxes>(r, token, u, c, s);
    for (int run = 0; run < (kRuns ? r.runs : 1); ++run, head += slots) {
        const bool live = head < heads && u < units;
        float a[8], b[8];
        uint16_t* out = nullptr;
        const void* gain = nullptr;
        if (live) {
            const bool is_q = head < r.q_heads;
            const int h = is_q ? head : head - r.q_heads;
            const uint16_t* x = is_q ? r.q + token * r.q_token + h * r.q_head : r.k + token * r.k_token + h * r.k_head;
            out = is_q ? r.q_out + (static_cast<int64_t>(token) * r.q_heads + h) * r.width
                       : r.k_out + (static_cast<int64_t>(token) * r.k_heads + h) * r.width;
            gain = is_q ? r.q_gain : r.k_gain;
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
        if (!live) continue;
        if (u < turning) {
            if (!kRuns) turns_of<kAxes>(r, token, u, c, s);
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
}

template <bool kHalf, bool kAxes>
void launch(const HeadRows& rows, int most, hipStream_t s) {
    const int heads = rows.q_heads + rows.k_heads, slots = 64 / rows.lanes, parts = (most + rows.runs - 1) / rows.runs;
    const int64_t waves = rows.runs > 1 ? static_cast<int64_t>(rows.tokens) * parts : (static_cast<int64_t>(rows.tokens) * heads + slots - 1) / slots;
    const unsigned groups = static_cast<unsigned>((waves + kThreads / 64 - 1) / (kThreads / 64));
    if (rows.runs > 1) norm_rope_kernel<kHalf, kAxes, true><<<groups, kThreads, 0, s>>>(rows, parts);
    else norm_rope_kernel<kHalf, kAxes, false><<<groups, kThreads, 0, s>>>(rows, 1);
}

}  // namespace

hipError_t head_norm_rope(HeadRows rows, hipStream_t s) {
    rows.lanes = 1;
    while (rows.lanes * 16 < rows.width) rows.lanes *= 2;
    const int slots = 64 / rows.lanes, heads = rows.q_heads + rows.k_heads, most = (heads + slots - 1) / slots;
    if (rows.tokens == 0 || heads == 0) return hipSuccess;
    const bool axes = rows.axes > 1;
    // The same number of runs for every wave of a token, but for the last one's.
    const int up_to = axes ? kMostAxesRuns : kMostRuns, parts = (most + up_to - 1) / up_to;
    rows.runs = static_cast<int64_t>(rows.tokens) * most >= (axes ? kManyAxesWaves : kManyWaves) ? (most + parts - 1) / parts : 1;
    if (rows.half) axes ? launch<true, true>(rows, most, s) : launch<true, false>(rows, most, s);
    else axes ? launch<false, true>(rows, most, s) : launch<false, false>(rows, most, s);
    return hipGetLastError();
}

}  // namespace cozyq
