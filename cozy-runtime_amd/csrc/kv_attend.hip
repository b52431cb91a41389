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
// A row's weights are taken up to 2^6 at first (the denominator alike), so that f16 holds those down to
// 2^-30 of the largest; no more, because of scores so large that float32 steps by 16: six less then
// rounds to no change, ten less would round to 2^16, which f16 has not.
constexpr float kLift = 6.0f;

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

// Four elements from d on of a row's result: the sums over its denominator, 0 for a row that sees nothing.
__device__ __forceinline__ void store_row(const CacheAttend& p, int token, int head, int width, int d, f32x4 v, float total) {
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    uint16_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float f = v[i] * inv;
        h[i] = p.half ? narrow<true>(f) : narrow<false>(f);
    }
    const i32x2 two = {static_cast<int32_t>(h[0] | (static_cast<uint32_t>(h[1]) << 16)),
                       static_cast<int32_t>(h[2] | (static_cast<uint32_t>(h[3]) << 16))};
    *reinterpret_cast<i32x2*>(p.out + (static_cast<int64_t>(token) * p.q_heads + head) * width + d) = two;
}

// Where request r's rows begin, never past the step's.
__device__ __forceinline__ int row_start(const CacheAttend& p, int r) { return min(max(p.starts[r], 0), p.tokens); }

// x from the lane that DPP control kCtrl names, 0 where it names none or the row is masked out.
template <int kCtrl, int kRowMask, typename T>
__device__ __forceinline__ T dpp_or_zero(T x) {
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), kCtrl, kRowMask, 0xF, false));
}

// Inclusive prefix sums over a wave: within rows of 16 lanes, then a row's last sum into the next rows.
template <typename T>
__device__ __forceinline__ T wave_prefix(T x) {
    x += dpp_or_zero<0x111, 0xF>(x);  // row_shr:1
    x += dpp_or_zero<0x112, 0xF>(x);  // row_shr:2
    x += dpp_or_zero<0x114, 0xF>(x);  // row_shr:4
    x += dpp_or_zero<0x118, 0xF>(x);  // row_shr:8
    x += dpp_or_zero<0x142, 0xA>(x);  // row_bcast:15 into rows 1 and 3
    x += dpp_or_zero<0x143, 0xC>(x);  // row_bcast:31 into rows 2 and 3
    return x;
}

// ------------------------------------------------------------------- few rows a request

constexpr int kStep = 64;       // tokens a wave takes at a time
constexpr int kMinSteps = 16;   // steps a workgroup takes at the least

// A request's part of the work: row tiles, and the 64-token steps that any of its rows sees.
struct Extent {
    int tiles, steps;
};

template <int kRows>
__device__ __forceinline__ Extent extent(const CacheAttend& p, int r) {
    const int fresh = row_start(p, r + 1) - row_start(p, r), length = p.lengths[r];
    const int low = p.window > 0 ? max(0, length - fresh + 1 - p.window) : 0;
    const int steps = (max(length, 0) + kStep - 1) / kStep - low / kStep;
    return {(fresh * p.group + kRows - 1) / kRows, max(steps, 0)};
}

// Tile `tile` of request `request`, its steps split in `splits` workgroups, this one number `split`,
// whose partial results stand `split` places after place `first`.
struct Share {
    int request, tile, split, splits, first;
};

// All the row tiles' steps are shared out evenly: with N steps in all (a head), a workgroup takes
// c = max(kMinSteps, ⌈N / shares⌉) of one row tile's, so that there are at most shares + tiles
// workgroups, whatever the requests' lengths are, and the host can size the launch without knowing
// them. Finds workgroup `id`'s share (kById), or row tile `id`'s first; false past the last. Every wave
// scans all requests, 64 at a time.
template <int kRows, bool kById>
__device__ bool find_share(const CacheAttend& p, int id, Share& out) {
    const int lane = threadIdx.x & 63;
    float work = 0.0f;  // in float32, which no number of steps overflows; the margin is over its rounding
    for (int base = 0; base < p.requests; base += 64) {
        Extent e = {0, 0};
        if (base + lane < p.requests) e = extent<kRows>(p, base + lane);
        const float sum = wave_prefix(static_cast<float>(e.tiles) * static_cast<float>(e.steps));
        work += __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, sum), 63));
    }
    const int c = max(kMinSteps, static_cast<int>(work * 1.001f / static_cast<float>(p.shares)) + 1);
    int groups_before = 0, tiles_before = 0;
    for (int base = 0; base < p.requests; base += 64) {
        Extent e = {0, 0};
        if (base + lane < p.requests) e = extent<kRows>(p, base + lane);
        const int splits = max(1, (e.steps + c - 1) / c);
        const int groups = wave_prefix(e.tiles * splits), tiles = wave_prefix(e.tiles);
        const int mine = kById ? groups_before + groups : tiles_before + tiles;
        const uint64_t past = __ballot(mine > id);
        if (past) {
            const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
            const int n = __builtin_amdgcn_readlane(splits, at), t = __builtin_amdgcn_readlane(e.tiles, at);
            const int g0 = groups_before + __builtin_amdgcn_readlane(groups, at) - t * n;
            const int t0 = tiles_before + __builtin_amdgcn_readlane(tiles, at) - t;
            const int tile = kById ? (id - g0) / n : id - t0;
            out = {base + at, tile, kById ? (id - g0) % n : 0, n, g0 + tile * n};
            return true;
        }
        groups_before += __builtin_amdgcn_readlane(groups, 63);
        tiles_before += __builtin_amdgcn_readlane(tiles, 63);
    }
    return false;
}

// What a workgroup keeps of a page of its tokens: its number (-1: none of the cache's), the keys'
// scale, log2 and inverse of the values'.
struct PageScales {
    int page;
    float keys, values_log, values_inv;
};

// Four waves take a row tile of 16 rows (kTiles of them) of one key head, the heads that share it token
// by token, over the workgroup's share of its tokens: each wave every fourth step of 64. Both products
// are taken transposed, Sᵀ = K·Qᵀ and Oᵀ = Vᵀ·Pᵀ, on v_mfma_f32_16x16x32_f16, so that a query row is a
// column of both results: lane l holds column l%16. Score tile j's row m is token 16·(m/4) + 4j + m%4
// of the step, which leaves lane group g = l/16 with the scores of tokens 16g .. 16g+15 in order: all
// of one page (pages are multiples of 16 tokens), one scale each, and exactly the 16 bytes of a channel's
// values that the group loads for the second product. Codes go from memory to registers to the matrix
// unit; nothing of the cache passes through LDS but its pages' numbers and scales, read once a share.
// A step's keys are loaded over the previous step's second product and its values over its first.
template <int kWidth, int kTiles, bool kFp8>
__global__ __launch_bounds__(256, kWidth == 256 ? 1 : 2) void few_kernel(CacheAttend p) {
    constexpr int kWaves = 4, kBlocks = kWidth / 64, kOut = kWidth / 16, kRows = 16 * kTiles;
    constexpr int kStage = 128, kEntries = kStage * kStep / 16 + 1;
    __shared__ PageScales entries[kEntries];
    __shared__ float merged[kWaves][16][kWidth + 4];
    __shared__ float tops[kWaves][16], totals[kWaves][16];
    const int thread = threadIdx.x, lane = thread & 63, wave = thread >> 6, col = lane & 15, g = lane >> 4;
    const int kv = blockIdx.x % p.heads, id = blockIdx.x / p.heads;
    Share share;
    if (!find_share<kRows, true>(p, id, share)) return;
    const int first = row_start(p, share.request), fresh = row_start(p, share.request + 1) - first;
    const int length = p.lengths[share.request], rows = fresh * p.group;

    // Tokens [low, high) of each of the lane's rows, of which the tile's steps span [begin, end).
    int low[kTiles], high[kTiles], token[kTiles], head[kTiles];
    bool live[kTiles];
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
        const int row = kRows * share.tile + 16 * n + col;
        live[n] = row < rows;
        token[n] = live[n] ? row / p.group : 0;
        head[n] = kv * p.group + (live[n] ? row - token[n] * p.group : 0);
        const int position = length - fresh + token[n];
        high[n] = live[n] ? (p.causal ? position + 1 : length) : 0;
        low[n] = live[n] ? (p.window > 0 ? max(0, position + 1 - p.window) : 0) : 0x7fffffff;
    }
    const int t_first = kRows * share.tile / p.group, t_last = min(rows, kRows * (share.tile + 1)) - 1;
    const int low_least = p.window > 0 ? max(0, length - fresh + t_first + 1 - p.window) : 0;
    const int low_most = p.window > 0 ? max(0, length - fresh + t_last / p.group + 1 - p.window) : 0;
    const int high_least = p.causal ? length - fresh + t_first + 1 : length;
    const int high_most = p.causal ? length - fresh + t_last / p.group + 1 : length;
    const int steps_from = low_least / kStep, steps = max(0, (high_most + kStep - 1) / kStep - steps_from);
    const int begin = steps_from + static_cast<int>(static_cast<int64_t>(steps) * share.split / share.splits);
    const int end = steps_from + static_cast<int>(static_cast<int64_t>(steps) * (share.split + 1) / share.splits);

    // Each row brought to a largest magnitude of about 2^12; a lane holds elements 64b + 16g .. + 15 of
    // each block of 64, as two operands.
    f16x8 q[kTiles][kBlocks][2];
    float sharp[kTiles];
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
        const uint16_t* x = p.q + (first + token[n]) * p.q_token + head[n] * p.q_head;
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
        sharp[n] = float_of(static_cast<uint32_t>(e) << 23) * p.scale * kLog2e;
        const float down = float_of(static_cast<uint32_t>(254 - e) << 23);
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
            for (int i = 0; i < 16; ++i) q[n][b][i / 8][i % 8] = static_cast<_Float16>(v[b][i] * down);
        }
    }

    // `ref` is subtracted from every exponent. It follows the row's largest, set 2^kLift below it when a
    // row sees its first token and moved up only when a weight would pass 2^15: most steps need neither
    // the maximum over the lane groups nor the accumulators' scaling. `bound` is −inf until it is set.
    f32x4 acc[kTiles][kOut];
    float ref[kTiles], bound[kTiles], total[kTiles];
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
#pragma unroll
        for (int i = 0; i < kOut; ++i) acc[n][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        ref[n] = total[n] = 0.0f;
        bound[n] = -__builtin_inff();
    }
    const int* table = p.table + static_cast<int64_t>(share.request) * p.width;
    const int within = p.page - 1;
    const uint8_t* k_lane = p.k_codes + static_cast<int64_t>(kv) * p.page * kWidth + (col & 3) * kWidth + 16 * g;
    const uint8_t* v_lane = p.v_codes + static_cast<int64_t>(kv) * p.page * kWidth + col * p.page;
    const int64_t page_bytes = static_cast<int64_t>(p.heads) * p.page * kWidth;

    i32x4 kc[4][kBlocks], vc[kOut];
    for (int stage = begin; stage < end; stage += kStage) {
        const int stage_end = min(end, stage + kStage);
        const int page_first = stage * kStep >> p.shift;
        const int pages = ((stage_end * kStep - 1) >> p.shift) - page_first + 1;
        if (stage != begin) __syncthreads();
        for (int i = thread; i < pages; i += 256) {
            const int index = page_first + i;
            const int page = index < p.width && (index << p.shift) < length ? table[index] : -1;
            PageScales e = {-1, 0.0f, 0.0f, 0.0f};
            if (page >= 0 && page < p.pages) {
                const int64_t at = static_cast<int64_t>(page) * p.heads + kv;
                const float values = nan_max(or_nan(p.v_scale[at]), 1e-30f);
                e = {page, or_nan(p.k_scale[at]), __builtin_amdgcn_logf(values), 1.0f / values};
            }
            entries[i] = e;
        }
        __syncthreads();

        const auto load_keys = [&](int step) {
            const int t = step * kStep + 16 * (col >> 2);
            const int page = max(entries[(t >> p.shift) - page_first].page, 0);
            const uint8_t* k = k_lane + page * page_bytes + static_cast<int64_t>(t & within) * kWidth;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) kc[j][b] = *reinterpret_cast<const i32x4*>(k + 4 * j * kWidth + 64 * b);
            }
        };
        const auto load_values = [&](int step) {
            const int t = step * kStep + 16 * g;
            const int page = max(entries[(t >> p.shift) - page_first].page, 0);
            const uint8_t* v = v_lane + page * page_bytes + (t & within);
#pragma unroll
            for (int o = 0; o < kOut; ++o) vc[o] = *reinterpret_cast<const i32x4*>(v + 16 * o * p.page);
        };
        int step = stage + wave;
        if (step < stage_end) {
            load_keys(step);
            load_values(step);
        }
        for (; step < stage_end; step += kWaves) {
            const int t0 = step * kStep, mine = t0 + 16 * g;
            const PageScales page = entries[(mine >> p.shift) - page_first];
            const bool whole = t0 >= low_most && t0 + kStep <= high_least && __all(page.page >= 0);
            f32x4 s[kTiles][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
#pragma unroll
                for (int n = 0; n < kTiles; ++n) s[n][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) {
                    const f16x8 k0 = codes8<kFp8>(kc[j][b][0], kc[j][b][1]), k1 = codes8<kFp8>(kc[j][b][2], kc[j][b][3]);
#pragma unroll
                    for (int n = 0; n < kTiles; ++n) {
                        s[n][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, q[n][b][0], s[n][j], 0, 0, 0);
                        s[n][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, q[n][b][1], s[n][j], 0, 0, 0);
                    }
                }
            }
            if (step + kWaves < stage_end) load_keys(step + kWaves);

            f16x8 w[kTiles][2];
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
                const float mul = sharp[n] * page.keys, add = page.values_log - ref[n];
                float x[16], most = -__builtin_inff();
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    x[i] = __builtin_fmaf(s[n][i / 4][i % 4], mul, add);
                    if (!whole && (page.page < 0 || mine + i < low[n] || mine + i >= high[n])) x[i] = -__builtin_inff();
                    most = fmaxf(most, x[i]);
                }
                if (__any(most > bound[n])) {
                    most = fmaxf(most, __shfl_xor(most, 16));
                    most = fmaxf(most, __shfl_xor(most, 32));
                    const float up = most > bound[n] ? most - kLift : 0.0f;
                    // Nothing is there to scale before the row's first token, and 0 · 2^-up may be 0 · inf.
                    const float shrink = bound[n] > 0.0f ? __builtin_amdgcn_exp2f(-up) : 0.0f;
                    if (most > bound[n]) bound[n] = 15.0f;
                    ref[n] += up;
                    total[n] *= shrink;
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[i] -= up;
#pragma unroll
                    for (int o = 0; o < kOut; ++o) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[n][o][i] *= shrink;
                    }
                }
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float e = __builtin_amdgcn_exp2f(x[i]);
                    sum += e;
                    w[n][i / 8][i % 8] = static_cast<_Float16>(e);
                }
                // A group whose tokens the row does not see adds nothing, whatever its page's scale is.
                total[n] += sum == 0.0f ? 0.0f : sum * page.values_inv;
            }
            if (!whole) {
                // Bytes past the request's tokens may hold anything, a NaN of the format too.
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int n = page.page >= 0 ? length - mine - 4 * i : 0;
                    const int kept = n >= 4 ? -1 : n <= 0 ? 0 : (1 << (8 * n)) - 1;
#pragma unroll
                    for (int o = 0; o < kOut; ++o) vc[o][i] &= kept;
                }
            }
#pragma unroll
            for (int o = 0; o < kOut; ++o) {
                const f16x8 v0 = codes8<kFp8>(vc[o][0], vc[o][1]), v1 = codes8<kFp8>(vc[o][2], vc[o][3]);
#pragma unroll
                for (int n = 0; n < kTiles; ++n) {
                    acc[n][o] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, w[n][0], acc[n][o], 0, 0, 0);
                    acc[n][o] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, w[n][1], acc[n][o], 0, 0, 0);
                }
            }
            if (step + kWaves < stage_end) load_values(step + kWaves);
        }
    }

    // The four waves' sums, brought to one reference; then the rows, or their part of them.
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
        total[n] += __shfl_xor(total[n], 16);
        total[n] += __shfl_xor(total[n], 32);
        const float top = bound[n] > 0.0f ? ref[n] : kNoScore;
        if (n) __syncthreads();
        if (g == 0) {
            tops[wave][col] = top;
            totals[wave][col] = total[n];
        }
        __syncthreads();
        float most = kNoScore;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) most = nan_max(most, tops[w][col]);
        const float factor = __builtin_amdgcn_exp2f(top - most);
#pragma unroll
        for (int o = 0; o < kOut; ++o) {
            f32x4 v = acc[n][o];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] *= factor;
            *reinterpret_cast<f32x4*>(&merged[wave][col][16 * o + 4 * g]) = v;
        }
        __syncthreads();
        const int row0 = kRows * share.tile + 16 * n, count = min(16, rows - row0);
        for (int i = thread; i < count * (kWidth / 4); i += 256) {
            const int r = i / (kWidth / 4), d = 4 * (i - r * (kWidth / 4));
            float best = kNoScore, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) best = nan_max(best, tops[w][r]);
            f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                v += *reinterpret_cast<const f32x4*>(&merged[w][r][d]);
                sum += totals[w][r] * __builtin_amdgcn_exp2f(tops[w][r] - best);
            }
            if (share.splits == 1) {
                const int t = (row0 + r) / p.group, h = kv * p.group + (row0 + r) - t * p.group;
                store_row(p, first + t, h, kWidth, d, v, sum);
            } else {
                const int64_t at = (static_cast<int64_t>(share.first + share.split) * p.heads + kv) * kRows + 16 * n + r;
                *reinterpret_cast<f32x4*>(p.work + at * (kWidth + 4) + d) = v;
                if (d == 0) {
                    p.work[at * (kWidth + 4) + kWidth] = best;
                    p.work[at * (kWidth + 4) + kWidth + 1] = sum;
                }
            }
        }
    }
}

// Joins the parts of the row tiles that several workgroups took: one workgroup a row tile and head,
// every part brought to the largest reference, in the order of their tokens.
template <int kWidth, int kTiles>
__global__ __launch_bounds__(256) void join_kernel(CacheAttend p) {
    constexpr int kRows = 16 * kTiles;
    const int kv = blockIdx.y;
    Share share;
    if (!find_share<kRows, false>(p, blockIdx.x, share) || share.splits == 1) return;
    const int first = row_start(p, share.request), rows = (row_start(p, share.request + 1) - first) * p.group;
    const int row0 = kRows * share.tile, count = min(kRows, rows - row0);
    for (int i = threadIdx.x; i < count * (kWidth / 4); i += 256) {
        const int r = i / (kWidth / 4), d = 4 * (i - r * (kWidth / 4));
        const float* part = p.work + ((static_cast<int64_t>(share.first) * p.heads + kv) * kRows + r) * (kWidth + 4);
        const int64_t next = static_cast<int64_t>(p.heads) * kRows * (kWidth + 4);
        float best = kNoScore, sum = 0.0f;
        for (int s = 0; s < share.splits; ++s) best = nan_max(best, part[s * next + kWidth]);
        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int s = 0; s < share.splits; ++s) {
            const float factor = __builtin_amdgcn_exp2f(part[s * next + kWidth] - best);
            const f32x4 one = *reinterpret_cast<const f32x4*>(part + s * next + d);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = __builtin_fmaf(one[j], factor, v[j]);
            sum = __builtin_fmaf(part[s * next + kWidth + 1], factor, sum);
        }
        const int t = (row0 + r) / p.group, h = kv * p.group + (row0 + r) - t * p.group;
        store_row(p, first + t, h, kWidth, d, v, sum);
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

struct AttendShape {
    int tiles, shares;
    int64_t row_tiles;
    bool splits;
};

int64_t few_tiles(const CacheAttend& p, int rows) {
    return (static_cast<int64_t>(p.tokens) * p.group + rows - 1) / rows + p.requests;
}

template <int kWidth, int kTiles, bool kFp8>
hipError_t few(const CacheAttend& p, hipStream_t s) {
    const int64_t tiles = few_tiles(p, 16 * kTiles);
    few_kernel<kWidth, kTiles, kFp8><<<static_cast<unsigned>((p.shares + tiles) * p.heads), 256, 0, s>>>(p);
    const hipError_t error = hipGetLastError();
    if (error != hipSuccess || !p.work) return error;
    join_kernel<kWidth, kTiles><<<dim3(static_cast<unsigned>(tiles), static_cast<unsigned>(p.heads)), 256, 0, s>>>(p);
    return hipGetLastError();
}

template <bool kFp8>
hipError_t attend(const CacheAttend& p, hipStream_t s) {
    const bool one = p.tiles == 1;
    if (p.head_width == 64) return one ? few<64, 1, kFp8>(p, s) : few<64, 2, kFp8>(p, s);
    if (p.head_width == 128) return one ? few<128, 1, kFp8>(p, s) : few<128, 2, kFp8>(p, s);
    return one ? few<256, 1, kFp8>(p, s) : few<256, 2, kFp8>(p, s);
}

// The launch's shape, which the workspace goes by too.
AttendShape shape_of(int64_t tokens, int group, int requests, int heads, int columns, int page, int64_t most) {
    AttendShape a;
    a.tiles = most > 0 && most * group <= 16 ? 1 : 2;
    a.row_tiles = (tokens * group + 16 * a.tiles - 1) / (16 * a.tiles) + requests;
    // Two workgroups a CU at a time, and twice as many for the requests' different lengths.
    a.shares = max(1, 2 * 512 / heads);
    a.splits = static_cast<int64_t>(columns) * page > kMinSteps * kStep;
    return a;
}

}  // namespace

int64_t cache_attend_work(int64_t tokens, int group, int requests, int heads, int columns, int page, int width, int64_t most) {
    const AttendShape a = shape_of(tokens, group, requests, heads, columns, page, most);
    return a.splits ? (a.shares + a.row_tiles) * heads * 16 * a.tiles * (width + 4) * 4 : 0;
}

hipError_t cache_attend(CacheAttend p, int64_t most, bool fp8, hipStream_t s) {
    const AttendShape a = shape_of(p.tokens, p.group, p.requests, p.heads, p.width, p.page, most);
    p.tiles = a.tiles;
    p.shares = a.shares;
    if (!a.splits) p.work = nullptr;
    rest_kernel<<<64, 256, 0, s>>>(p);
    const hipError_t error = hipGetLastError();
    if (error != hipSuccess) return error;
    return fp8 ? attend<true>(p, s) : attend<false>(p, s);
}

}  // namespace cozyq
