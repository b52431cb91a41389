// The residual's addition, the RMS norm of the sum and its quantization, one read and one write of every element:
//
//   t = round16(x + r),   n = t · rsqrt(mean(t²) + eps) · gain
//   E4M3: s = max(amax(n) / 448, 1e-12), code = e4m3(n / s)
//   int8: u = H256 n / 16 over blocks of 256, s = max(amax(u) / 127, 1e-12), code = rne(u / s)
//
// t is rounded to the rows' type before its norm: the norm is that of the stream as it is stored, which every later
// reader sees. From there to the code everything is float32. H256 = H4⊗H4⊗H4⊗H4 is the int8 linears' rotation.
#include <hip/hip_runtime.h>

#include "common.h"
#include "kernels.h"
#include "rotate.h"
#include "sixteen.h"

namespace cozyq {
namespace {

// H4 of four values, (a + b + c − d, a + b − c + d, a − b + c + d, b + c + d − a): each is the four's sum with one of
// them, in reverse order, taken away twice. Seven operations where the written order takes twelve.
__device__ __forceinline__ void h4_sum(float& a, float& b, float& c, float& d) {
    const float sum = (a + b) + (c + d);
    const float o0 = __builtin_fmaf(-2.0f, d, sum), o1 = __builtin_fmaf(-2.0f, c, sum);
    const float o2 = __builtin_fmaf(-2.0f, b, sum), o3 = __builtin_fmaf(-2.0f, a, sum);
    a = o0;
    b = o1;
    c = o2;
    d = o3;
}

// 16 · H256 over the 256 values of 16 neighbouring lanes, 16 contiguous ones a lane: the inner two stages in the lane's
// registers, the outer two over a quad of lanes and over the quads of a row of 16, by DPP.
__device__ __forceinline__ void rotate256(float* v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) h4_sum(v[i], v[4 + i], v[8 + i], v[12 + i]);
#pragma unroll
    for (int i = 0; i < 4; ++i) h4_sum(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float pair = v[i] + dpp_move<0xB1>(v[i]);                    // quad_perm 1,0,3,2
        const float sum = pair + dpp_move<0x4E>(pair);                     // quad_perm 2,3,0,1
        v[i] = __builtin_fmaf(-2.0f, dpp_move<0x1B>(v[i]), sum);           // quad_perm 3,2,1,0
        const float two = v[i] + dpp_move<0x128>(v[i]);                    // row_ror:8
        const float all = two + dpp_move<0x124>(two);                      // row_ror:4
        const float across = dpp_move<0x1B>(dpp_move<0x140>(v[i]));        // row_mirror, the quad's order kept
        v[i] = __builtin_fmaf(-2.0f, across, all);
    }
}

// The workgroup's sum, the same for every thread, through `waves` places of their own.
__device__ __forceinline__ float block_total(float v, float* places) {
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) places[threadIdx.x >> 6] = v;
    __syncthreads();
    v = places[0];
    for (int w = 1; w < static_cast<int>(blockDim.x >> 6); ++w) v += places[w];
    return v;
}

// One workgroup a row, 16 contiguous elements a thread and run (a second run past 16384), held in registers from the load
// to the code, so that a row is read once however its norm and its scale depend on all of it. A thread's 16 elements are a
// sixteenth of a rotation's block: two of its four stages stay in the lane, the others move by DPP, and nothing but the
// two reductions passes through LDS.
// Bound by the vector unit and memory alike where there is a rotation (6001 rows of 4096: 172 MB in 32.6 us, 5.3 TB/s of a
// large copy's 5.6; VALU 94% busy), by memory without (1531 rows of 12288 to E4M3: 132 MB in 25.3 us, 5.2 TB/s); few rows by
// the launch and one row's chain of reductions (one row 3.6 us, 48 of 5120 4.4).
template <bool kHalf, bool kFp8, int kRuns>
__global__ __launch_bounds__(1024) void add_rms_kernel(AddRms p) {
    __shared__ float sums[2][16], tops[16];
    const int64_t row = static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x;
    if (row >= p.rows) return;
    const int thread = threadIdx.x, waves = blockDim.x >> 6;
    const uint16_t* x = p.x + row * p.width;
    const uint16_t* r = p.residual ? p.residual + row * p.width : nullptr;
    float v[kRuns][16];
    float squares = 0.0f;
#pragma unroll
    for (int k = 0; k < kRuns; ++k) {
        const int e = 16 * (thread + k * blockDim.x);
#pragma unroll
        for (int i = 0; i < 16; ++i) v[k][i] = 0.0f;
        if (e < p.width) {
            load8<kHalf>(x + e, v[k]);
            load8<kHalf>(x + e + 8, v[k] + 8);
            if (r) {
                float w[16];
                load8<kHalf>(r + e, w);
                load8<kHalf>(r + e + 8, w + 8);
                i32x4 packed[2];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    packed[i / 4][i % 4] = static_cast<int32_t>(narrow2<kHalf>(v[k][2 * i] + w[2 * i], v[k][2 * i + 1] + w[2 * i + 1]));
                i32x4* out = reinterpret_cast<i32x4*>(p.total + row * p.width + e);
                out[0] = packed[0];
                out[1] = packed[1];
                widen8<kHalf>(packed[0], v[k]);
                widen8<kHalf>(packed[1], v[k] + 8);
            }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) squares = __builtin_fmaf(v[k][i], v[k][i], squares);
    }
    float sum = block_total(squares, sums[0]), eps = p.eps;
    if (sum >= __builtin_huge_valf()) {  // the same for every thread
        // Squares past float32's range: the row, and with it the root, is taken 2^-80 times as large, where eps is nothing.
        squares = eps = 0.0f;
#pragma unroll
        for (int k = 0; k < kRuns; ++k) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                v[k][i] *= 0x1p-80f;
                squares = __builtin_fmaf(v[k][i], v[k][i], squares);
            }
        }
        sum = block_total(squares, sums[1]);
    }
    // An infinity in the row makes all of it NaN (sum - sum), not zeros beside one NaN.
    const float inv = rsqrtf((sum + (sum - sum)) / static_cast<float>(p.width) + eps);
    float top = 0.0f;
#pragma unroll
    for (int k = 0; k < kRuns; ++k) {
        const int e = 16 * (thread + k * blockDim.x);
        if (e < p.width) {
#pragma unroll
            for (int i = 0; i < 16; ++i) v[k][i] *= inv;
            if (p.gain) {
                float g[16];
                if (p.gain_wide) {
                    load8f(static_cast<const float*>(p.gain) + e, g);
                    load8f(static_cast<const float*>(p.gain) + e + 8, g + 8);
                } else {
                    load8<kHalf>(static_cast<const uint16_t*>(p.gain) + e, g);
                    load8<kHalf>(static_cast<const uint16_t*>(p.gain) + e + 8, g + 8);
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) v[k][i] *= g[i];
            }
        }
        if constexpr (!kFp8) rotate256(v[k]);
#pragma unroll
        for (int i = 0; i < 16; ++i) top = nan_max(top, __builtin_fabsf(v[k][i]));
    }
    top = wave_max_nan(top);
    if ((thread & 63) == 0) tops[thread >> 6] = top;
    __syncthreads();
    top = tops[0];
    for (int w = 1; w < waves; ++w) top = nan_max(top, tops[w]);
    // The rotation's 1/16 is a power of two: it scales the maximum and leaves the quotients as they are.
    constexpr float kUnit = kFp8 ? 1.0f : 16.0f;
    const float scale = nan_max(top / (kUnit * (kFp8 ? kE4m3Max : 127.0f)), kScaleFloor);
    if (thread == 0) p.scales[row] = scale;
    const float unit = kUnit * scale, back = 1.0f / unit;
#pragma unroll
    for (int k = 0; k < kRuns; ++k) {
        const int e = 16 * (thread + k * blockDim.x);
        if (e >= p.width) continue;
        i32x4 word;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (kFp8) {
                float c[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) c[i] = fminf(fmaxf(div_rn(v[k][4 * j + i], unit, back), -kE4m3Max), kE4m3Max);
                word[j] = static_cast<int32_t>(e4m3x4(c[0], c[1], c[2], c[3]));
            } else {
                word[j] = static_cast<int32_t>(q8x4<true>(v[k] + 4 * j, unit, back));
            }
        }
        *reinterpret_cast<i32x4*>(p.codes + row * p.width + e) = word;
    }
}

template <bool kHalf, bool kFp8>
hipError_t launch(const AddRms& p, hipStream_t s) {
    const int lanes = (p.width / 16 + 63) / 64 * 64;
    // A dimension of a grid has fewer than 2^32 threads: lines of 2^21 rows, of up to 1024 threads each.
    constexpr int kLine = 1 << 21;
    const dim3 grid(p.rows < kLine ? p.rows : kLine, (p.rows + kLine - 1) / kLine);
    if (lanes <= 1024) add_rms_kernel<kHalf, kFp8, 1><<<grid, lanes, 0, s>>>(p);
    else add_rms_kernel<kHalf, kFp8, 2><<<grid, (lanes / 2 + 63) / 64 * 64, 0, s>>>(p);
    return hipGetLastError();
}

}  // namespace

hipError_t add_rms(const AddRms& p, bool fp8, hipStream_t s) {
    if (p.rows == 0) return hipSuccess;
    if (p.half) return fp8 ? launch<true, true>(p, s) : launch<true, false>(p, s);
    return fp8 ? launch<false, true>(p, s) : launch<false, false>(p, s);
}

}  // namespace cozyq
