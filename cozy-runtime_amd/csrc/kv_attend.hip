// Attention of a step's queries over the paged 8-bit cache (kv_cache.hip's layout):
//
//   out_i = Σ_t softmax_t(scale · q_i · k_t) v_t,   k_t = kc_t · ks,  v_t = vc_t · vs
//
// over the tokens t that row i sees: up to its own position where causal, the last `window` of them
// where there is a window. ks and vs are the scales of t's page and head. One pass over the pages
// with the running maximum and sum of the softmax.
//
// The products run on the f16 matrix unit. A code, int8 or E4M3, is exact in f16, so the cache is
// multiplied as it is stored and its scales stay outside: ks multiplies a score, and vs goes into the
// weight's exponent, p = 2^(s·log2(e) + log2(vs) − m), so that m bounds what a token adds to the
// output rather than its probability, and the denominator takes p/vs. A query row is brought near
// 2^12 by a power of two and is then exact in f16, but for what lies below 2^-26 of its largest
// element. Weights are
// rounded to f16 (11 bits, three more than bf16) for the second product alone; maxima, sums and both
// products' accumulators are float32.
#include <hip/hip_runtime.h>

#include "common.h"
#include "kernels.h"

namespace cozyq {
namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.44269504f;
// Below any finite score: an all-masked row's maximum, so that 2^(−inf − m) is 0 and not NaN.
constexpr float kNoScore = -1e30f;
// Weights are taken 2^10 above the true ones (the denominator alike), which keeps those down to
// 2^-24 of the largest normal in f16.
constexpr float kLift = 10.0f;

// Four codes of a dword as f16, exactly.
template <bool kFp8>
__device__ __forceinline__ void codes4(uint32_t c, f16x2& lo, f16x2& hi) {
    if constexpr (kFp8) {
        lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, 1.0f, false);
        hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, 1.0f, true);
    } else {
        // u = code + 128 in the significand of 1024 + u, then 1152 less.
        const uint32_t u = c ^ 0x80808080u;
        const f16x2 off = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
        lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + off;
        hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + off;
    }
}

template <bool kFp8>
__device__ __forceinline__ f16x8 codes8(uint32_t a, uint32_t b) {
    f16x2 v[4];
    codes4<kFp8>(a, v[0], v[1]);
    codes4<kFp8>(b, v[2], v[3]);
    return __builtin_bit_cast(f16x8, v);
}

// A finite scale, NaN for an infinite one: whoever sees its page gets NaN, not a score of either sign.
__device__ __forceinline__ float or_nan(float scale) { return scale + (scale - scale); }

// Where request r's rows begin, never past the step's.
__device__ __forceinline__ int row_start(const CacheAttend& p, int r) { return min(max(p.starts[r], 0), p.tokens); }

// The request and row tile (of kRows rows) that the tile number `item` names, over all requests in
// order; false past the last. Called by a whole wave.
template <int kRows>
__device__ bool locate(const CacheAttend& p, int item, int& request, int& tile) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < p.requests; base += 64) {
        const int r = base + lane;
        int tiles = 0;
        if (r < p.requests) tiles = ((row_start(p, r + 1) - row_start(p, r)) * p.group + kRows - 1) / kRows;
        int sum = tiles;
        for (int step = 1; step < 64; step *= 2) {
            const int below = __shfl_up(sum, step);
            if (lane >= step) sum += below;
        }
        const int all = __shfl(sum, 63);
        if (item < before + all) {
            const uint64_t past = __ballot(before + sum > item);
            const int first = __ffsll(static_cast<unsigned long long>(past)) - 1;
            request = base + first;
            tile = item - before - (__shfl(sum, first) - __shfl(tiles, first));
            return true;
        }
        before += all;
    }
    return false;
}

// One wave a tile of 16 query rows of one key head (the heads that share it, token by token) and all
// the tokens they see, 64 at a time. Both products are taken transposed, Sᵀ = K·Qᵀ and Oᵀ = Vᵀ·Pᵀ, on
// v_mfma_f32_16x16x32_f16, so that a query row is a column of both results: lane l holds column l%16.
// Score tile j's row m is token 16·(m/4) + 4j + m%4 of the step, which leaves lane group g = l/16 with
// the scores of tokens 16g .. 16g+15 in order: all of one page (pages are multiples of 16 tokens), one
// scale each, and exactly the 16 bytes of a channel's values that the group loads for the second
// product. No operand passes through LDS.
template <int kWidth, bool kFp8>
__global__ __launch_bounds__(64) void attend_kernel(CacheAttend p) {
    constexpr int kBlocks = kWidth / 64, kOut = kWidth / 16;
    const int lane = threadIdx.x, col = lane & 15, g = lane >> 4;
    const int kv = blockIdx.y;
    int request, tile;
    if (!locate<16>(p, blockIdx.x, request, tile)) return;
    const int first = row_start(p, request), fresh = row_start(p, request + 1) - first, length = p.lengths[request];
    const int row = 16 * tile + col;
    const bool live = row < fresh * p.group;
    const int token = live ? row / p.group : 0;
    const int head = kv * p.group + (live ? row % p.group : 0);
    const int position = length - fresh + token;
    // Tokens [low, high) of this row; of the tile's rows together.
    const int high = live ? (p.causal ? position + 1 : length) : 0;
    const int low = live ? (p.window > 0 ? max(0, position + 1 - p.window) : 0) : 0x7fffffff;
    int begin = low, end = high;
    for (int step = 1; step < 16; step *= 2) {
        begin = min(begin, __shfl_xor(begin, step));
        end = max(end, __shfl_xor(end, step));
    }

    // The row, brought to a largest magnitude of about 2^12; a lane holds elements 64b + 16g .. + 15 of
    // each block of 64, as two operands.
    f16x8 q[kBlocks][2];
    float unit;
    {
        const uint16_t* x = p.q + (first + token) * p.q_token + head * p.q_head;
        float v[kBlocks][16];
        uint32_t most = 0;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const i32x4 raw = *reinterpret_cast<const i32x4*>(x + 64 * b + 16 * g + 8 * c);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint16_t h = static_cast<uint16_t>(static_cast<uint32_t>(raw[i / 2]) >> (16 * (i & 1)));
                    const float f = p.half ? widen<true>(h) : widen<false>(h);
                    v[b][8 * c + i] = f;
                    most = max(most, bits_of(f) & 0x7fffffffu);
                }
            }
        }
        most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 16)));
        most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 32)));
        // 2^(exponent − 12) and its inverse, both normal numbers.
        const int e = min(max(static_cast<int>(most >> 23) - 12, 10), 240);
        unit = float_of(static_cast<uint32_t>(e) << 23);
        const float down = float_of(static_cast<uint32_t>(254 - e) << 23);
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
            for (int i = 0; i < 16; ++i) q[b][i / 8][i % 8] = static_cast<_Float16>(v[b][i] * down);
        }
    }
    const float sharp = unit * p.scale * kLog2e;

    f32x4 acc[kOut];
#pragma unroll
    for (int i = 0; i < kOut; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float top = kNoScore, total = 0.0f;
    const int* pages = p.table + static_cast<int64_t>(request) * p.width;
    const int last_page = min((length - 1) >> p.shift, p.width - 1);
    const int64_t head_bytes = static_cast<int64_t>(p.page) * kWidth;
    const int within = p.page - 1;

    for (int t0 = begin & ~63; t0 < end; t0 += 64) {
        // The pages of the 16 tokens whose keys this lane loads and of those whose scores it holds;
        // one that the table lacks is read as page 0 and masked.
        const int tk = t0 + 16 * (col >> 2), tv = t0 + 16 * g;
        int page_k = pages[min(tk >> p.shift, last_page)], page_v = pages[min(tv >> p.shift, last_page)];
        const bool there = page_v >= 0 && page_v < p.pages && (tv >> p.shift) <= last_page;
        page_k = page_k >= 0 && page_k < p.pages ? page_k : 0;
        page_v = there ? page_v : 0;
        const uint8_t* k = p.k_codes + (static_cast<int64_t>(page_k) * p.heads + kv) * head_bytes +
                           static_cast<int64_t>((tk & within) + (col & 3)) * kWidth + 16 * g;
        const uint8_t* v = p.v_codes + (static_cast<int64_t>(page_v) * p.heads + kv) * head_bytes +
                           static_cast<int64_t>(col) * p.page + (tv & within);
        const int64_t at_scale = static_cast<int64_t>(page_v) * p.heads + kv;
        const float ks = there ? or_nan(p.k_scale[at_scale]) : 1.0f;
        const float vs = there ? nan_max(or_nan(p.v_scale[at_scale]), 1e-30f) : 1.0f;

        f32x4 s[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            s[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                const i32x4 c = *reinterpret_cast<const i32x4*>(k + 4 * j * kWidth + 64 * b);
                s[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8<kFp8>(c[0], c[1]), q[b][0], s[j], 0, 0, 0);
                s[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8<kFp8>(c[2], c[3]), q[b][1], s[j], 0, 0, 0);
            }
        }
        const float mul = sharp * ks, add = __builtin_amdgcn_logf(vs);
        float x[16], most = kNoScore;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            x[i] = __builtin_fmaf(s[i / 4][i % 4], mul, add);
            if (!there || tv + i < low || tv + i >= high) x[i] = -__builtin_inff();
            most = fmaxf(most, x[i]);
        }
        most = fmaxf(most, __shfl_xor(most, 16));
        most = fmaxf(most, __shfl_xor(most, 32));
        most = fmaxf(most - kLift, top);
        const float shrink = __builtin_amdgcn_exp2f(top - most);
        top = most;
        float sum = 0.0f;
        f16x8 w[2];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float e = __builtin_amdgcn_exp2f(x[i] - top);
            sum += e;
            w[i / 8][i % 8] = static_cast<_Float16>(e);
        }
        // A group whose tokens the row does not see adds nothing, whatever its page's scale is.
        total = total * shrink + (sum == 0.0f ? 0.0f : sum / vs);
        // Bytes past the request's tokens may hold anything, a NaN of the format too.
        const int left = length - tv;
        uint32_t kept[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int n = there ? left - 4 * i : 0;
            kept[i] = n >= 4 ? 0xffffffffu : n <= 0 ? 0u : (1u << (8 * n)) - 1u;
        }
#pragma unroll
        for (int o = 0; o < kOut; ++o) {
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[o][i] *= shrink;
            const i32x4 c = *reinterpret_cast<const i32x4*>(v + static_cast<int64_t>(16 * o) * p.page);
            acc[o] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8<kFp8>(c[0] & kept[0], c[1] & kept[1]), w[0], acc[o], 0, 0, 0);
            acc[o] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8<kFp8>(c[2] & kept[2], c[3] & kept[3]), w[1], acc[o], 0, 0, 0);
        }
    }
    total += __shfl_xor(total, 16);
    total += __shfl_xor(total, 32);
    if (!live) return;
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    uint16_t* out = p.out + (static_cast<int64_t>(first + token) * p.q_heads + head) * kWidth + 4 * g;
#pragma unroll
    for (int o = 0; o < kOut; ++o) {
        uint16_t h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float f = acc[o][i] * inv;
            h[i] = p.half ? narrow<true>(f) : narrow<false>(f);
        }
        i32x2 two = {static_cast<int32_t>(h[0] | (static_cast<uint32_t>(h[1]) << 16)),
                     static_cast<int32_t>(h[2] | (static_cast<uint32_t>(h[3]) << 16))};
        *reinterpret_cast<i32x2*>(out + 16 * o) = two;
    }
}

// Rows of the step that no request has (past the last one's tokens) are zeros.
__global__ __launch_bounds__(256) void rest_kernel(CacheAttend p) {
    const int first = row_start(p, p.requests);
    const int64_t row = static_cast<int64_t>(p.q_heads) * p.head_width / 8;
    const int64_t all = (p.tokens - first) * row;
    i32x4* out = reinterpret_cast<i32x4*>(p.out) + first * row;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < all; i += 256 * gridDim.x) out[i] = i32x4{0, 0, 0, 0};
}

template <bool kFp8>
hipError_t attend(const CacheAttend& p, hipStream_t s) {
    const int tiles = (static_cast<int64_t>(p.tokens) * p.group + 15) / 16 + p.requests;
    const dim3 grid(static_cast<unsigned>(tiles), static_cast<unsigned>(p.heads));
    if (p.head_width == 64) attend_kernel<64, kFp8><<<grid, 64, 0, s>>>(p);
    else if (p.head_width == 128) attend_kernel<128, kFp8><<<grid, 64, 0, s>>>(p);
    else attend_kernel<256, kFp8><<<grid, 64, 0, s>>>(p);
    return hipGetLastError();
}

}  // namespace

hipError_t cache_attend(const CacheAttend& p, bool fp8, hipStream_t s) {
    rest_kernel<<<64, 256, 0, s>>>(p);
    const hipError_t error = hipGetLastError();
    if (error != hipSuccess) return error;
    return fp8 ? attend<true>(p, s) : attend<false>(p, s);
}

}  // namespace cozyq
