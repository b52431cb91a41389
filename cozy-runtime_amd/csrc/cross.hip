// Attention of a decoder's rows to an encoder's states of another length, keys and values dense in 16 bits:
//
//   out_i = Σ_t softmax_t(scale · q_i · k_t) v_t
//
// over the states t of row i's request: those below its length that its mask has, all of them seen by every row. One
// pass over the states with the running maximum and sum of the softmax.
//
// Both products run on the matrix unit in the inputs' type, transposed (Sᵀ = K·Qᵀ, Oᵀ = Vᵀ·Pᵀ), so that a row is a
// column of both results and a lane holds 16 scores of one row for every 32 states. Weights are rounded to the inputs'
// type for the second product alone: float32 runs at a sixteenth of the rate there. Scores, maxima, sums and
// accumulators are float32. States that are not seen are zeros by the time they are in LDS, whatever memory holds.
#include <hip/hip_runtime.h>

#include "common.h"
#include "kernels.h"
#include "sixteen.h"

namespace cozyq {
namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 LdsFour;

constexpr float kLog2e = 1.44269504f;
// A row's weights are taken up to 2^6 at first and up to 2^15 before their reference moves, so that f16 holds those
// down to 2^-30 of the largest.
constexpr float kLift = 6.0f, kBound = 15.0f;
// Below any reference: that of a row without a finite score.
constexpr float kNoScore = -1e30f;
constexpr int kStage = 256;  // steps whose seen states are staged at a time
// States taken at a time: 64, or 32 of wide heads, whose accumulators leave fewer registers.
constexpr int step_of(int width) { return width == 256 ? 32 : 64; }

template <bool kHalf>
__device__ __forceinline__ f32x16 mfma32(const i32x4& a, const i32x4& b, f32x16 c) {
    if constexpr (kHalf)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Two float32 values in the inputs' type, rounded to nearest even.
template <bool kHalf>
__device__ __forceinline__ int32_t pack2(float a, float b) {
    if constexpr (kHalf) {
        const f16x2 two = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
        return __builtin_bit_cast(int32_t, two);
    } else {
        return static_cast<int32_t>(narrow2<false>(a, b));
    }
}

// Keeps a branch a branch: without it the compiler works out both sides and selects.
__device__ __forceinline__ void rarely() { asm volatile(""); }

// Request b's rows of the call, in order and never past its last: [first, first + count), and how many states it has.
struct Rows {
    int first, count, length;
};

__device__ __forceinline__ Rows rows_of(const CrossAttend& p, int b) {
    Rows r;
    if (p.starts) {
        r.first = min(max(p.starts[b], 0), p.tokens);
        r.count = min(max(p.starts[b + 1], r.first), p.tokens) - r.first;
    } else {
        r.first = b * p.each;
        r.count = p.each;
    }
    r.length = p.lengths ? min(max(p.lengths[b], 0), p.states) : p.states;
    return r;
}

// The tile number `id` of all requests' row tiles of kRows rows, one request after another; false past the last.
template <int kRows>
__device__ bool find_tile(const CrossAttend& p, int id, int& request, int& tile, int& count) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < p.requests; base += 64) {
        int tiles = 0;
        if (base + lane < p.requests)
            tiles = static_cast<int>((static_cast<int64_t>(rows_of(p, base + lane).count) * p.group + kRows - 1) / kRows);
        int sum = tiles;
#pragma unroll
        for (int step = 1; step < 64; step *= 2) {
            const int other = __shfl_up(sum, step);
            if (lane >= step) sum += other;
        }
        const uint64_t past = __ballot(before + sum > id);
        if (past) {
            const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
            request = base + at;
            tile = id - before - (__builtin_amdgcn_readlane(sum, at) - __builtin_amdgcn_readlane(tiles, at));
            return true;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    count = before;
    return false;
}

// Rows of the call that no request has are zeros: the workgroups without a tile write them, those from number `busy` on.
__device__ void clear_rest(const CrossAttend& p, int busy) {
    const int64_t row = static_cast<int64_t>(p.q_heads) * p.width / 8;
    const int64_t from = rows_of(p, 0).first * row;
    const Rows last = rows_of(p, p.requests - 1);
    const int64_t after = static_cast<int64_t>(last.first + last.count) * row, count = from + p.tokens * row - after;
    const int64_t stride = static_cast<int64_t>(gridDim.x - busy) * blockDim.x;
    for (int64_t i = static_cast<int64_t>(blockIdx.x - busy) * blockDim.x + threadIdx.x; i < count; i += stride)
        reinterpret_cast<i32x4*>(p.out)[i < from ? i : i - from + after] = i32x4{0, 0, 0, 0};
}

// Four elements of a row's result from d on, of the sums v with the denominator `total`: the result, or this split's
// part of it with its reference `ref`. `some`: whether a state was seen; nothing seen is 0, nothing but scores of minus
// infinity the quotient 0 / 0.
template <int kWidth, bool kHalf>
__device__ __forceinline__ void store_row(const CrossAttend& p, int split, int64_t at, int d, f32x4 v, float ref, float total, bool some) {
    if (p.splits == 1) {
        if (d >= p.width) return;
        const float inv = some ? 1.0f / total : 0.0f;
        *reinterpret_cast<i32x2*>(p.out + at * p.width + d) = i32x2{pack2<kHalf>(v[0] * inv, v[1] * inv), pack2<kHalf>(v[2] * inv, v[3] * inv)};
    } else {
        const int64_t places = static_cast<int64_t>(p.tokens) * p.q_heads;
        *reinterpret_cast<f32x4*>(p.work + (split * places + at) * kWidth + d) = v;
        if (d == 0) {
            float* parts = p.work + p.splits * places * kWidth + 2 * (split * places + at);
            parts[0] = some ? ref : -__builtin_inff();
            parts[1] = total;
        }
    }
}

// A view of `left` rows (none below 1) of `width` 16-bit elements, `stride` apart, from `base` on: what lies past them
// reads as zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t states_view(const uint16_t* base, int left, int64_t stride, int width) {
    const int bytes = left < 1 ? 0 : static_cast<int>(2 * ((left - 1) * stride + width));
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(base), 0, bytes, 0x00020000);
}
// An offset past every view.
constexpr uint32_t kNowhere = 0x7fffffffu;

// Eight elements of a query row from d on, zeros of a row that is not there (whose address is that of one that is) and
// past the row's width.
__device__ __forceinline__ i32x4 query8(const uint16_t* row, bool live, int d, int width) {
    const bool there = d < width;
    const i32x4 raw = *reinterpret_cast<const i32x4*>(row + (there ? d : 0));
    return live && there ? raw : i32x4{0, 0, 0, 0};
}

// Where the 16-byte chunks of a tile's row stand: exclusive-or'ed so that the 16 lanes that one cycle of a read serves
// find different banks (64 of 4 bytes). Keys are read a chunk of 16 neighbouring rows at a time, values 64 bytes of
// four neighbouring rows.
template <int kWidth>
__device__ __forceinline__ int key_place(int row, int chunk) {
    return chunk ^ (kWidth == 64 ? (row >> 1) & 7 : row & 15);
}
template <int kWidth>
__device__ __forceinline__ int value_place(int row, int chunk) {
    return chunk ^ (kWidth == 64 ? 4 * ((row >> 1) & 1) : 4 * (row & 3));
}

// kWaves waves take a tile of 32 rows each of one key head over its states a step at a time, which all of them share in
// LDS. A step's keys and values are in registers by the step before it, when they are written to LDS, and asked for a
// step before that.
template <int kWidth, int kWaves, bool kHalf>
__global__ __launch_bounds__(64 * kWaves, kWidth == 256 ? 1 : 2) void cross_kernel(CrossAttend p) {
    constexpr int kRows = 32 * kWaves, kOut = kWidth / 32, kDepth = kWidth / 16;
    constexpr int kStep = step_of(kWidth), kScores = kStep / 2, kBytes = kStep * kWidth * 2;
    constexpr int kChunks = kWidth / 8, kPerLoad = 64 / kChunks, kLoads = kBytes / 1024 / kWaves;
    constexpr uint64_t kAll = kStep == 64 ? ~0ull : 0xffffffffull;
    __shared__ __attribute__((aligned(1024))) uint8_t tiles[2][2][kBytes];
    __shared__ uint64_t seen_of[kStage];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, h = lane >> 5;
    const int kv = blockIdx.x % p.kv_heads, id = blockIdx.x / p.kv_heads;
    int request, tile, found;
    if (!find_tile<kRows>(p, id / p.splits, request, tile, found)) {
        if (p.splits == 1) clear_rest(p, found * p.kv_heads);
        return;
    }
    const int split = id % p.splits;
    const Rows of = rows_of(p, request);
    const int rows = of.count * p.group, mine = kRows * tile + 32 * wave, row = mine + col;
    const bool busy = mine < rows, live = row < rows;
    const int token = of.first + (live ? row / p.group : 0), head = kv * p.group + (live ? row % p.group : 0);
    const int steps = (of.length + kStep - 1) / kStep;
    const int begin = static_cast<int>(static_cast<int64_t>(steps) * split / p.splits);
    const int end = static_cast<int>(static_cast<int64_t>(steps) * (split + 1) / p.splits);

    i32x4 q[kDepth];
#pragma unroll
    for (int b = 0; b < kDepth; ++b) q[b] = query8(p.q + token * p.q_token + head * p.q_head, live, 16 * b + 8 * h, p.width);
    const float sharp = p.scale * kLog2e;

    // This wave's shares of a step's keys and values: 1 KiB each, whole rows.
    const uint16_t* k_base = p.k + request * p.k_request + kv * p.k_head;
    const uint16_t* v_base = p.v + request * p.v_request + kv * p.v_head;
    const uint8_t* mask = p.mask ? p.mask + request * p.mask_request : nullptr;
    uint32_t k_from[kLoads], v_from[kLoads], row_of[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int r = (wave * kLoads + i) * kPerLoad + lane / kChunks;
        const int kc = key_place<kWidth>(r, lane % kChunks), vc = value_place<kWidth>(r, lane % kChunks);
        row_of[i] = r;
        k_from[i] = 8 * kc < p.width ? 2u * (r * static_cast<uint32_t>(p.k_state) + 8 * kc) : kNowhere;
        v_from[i] = 8 * vc < p.width ? 2u * (r * static_cast<uint32_t>(p.v_state) + 8 * vc) : kNowhere;
    }
    const auto seen_at = [&](int i) {
        const uint64_t word = seen_of[i];
        return static_cast<uint64_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(word >> 32))) << 32 |
               static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(word)));
    };
    i32x4 k_raw[kLoads], v_raw[kLoads];
    const auto load = [&](int step) {
        const int64_t t0 = static_cast<int64_t>(step) * kStep;
        const int left = static_cast<int>(min(of.length - t0, static_cast<int64_t>(kStep)));
        const __amdgpu_buffer_rsrc_t kr = states_view(k_base + t0 * p.k_state, left, p.k_state, p.width);
        const __amdgpu_buffer_rsrc_t vr = states_view(v_base + t0 * p.v_state, left, p.v_state, p.width);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            k_raw[i] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(kr, k_from[i], 0, 0));
            v_raw[i] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(vr, v_from[i], 0, 0));
        }
    };
    // Values of states that are not seen become zeros here; their scores are made minus infinity whatever they are.
    const auto put = [&](int slot, uint64_t seen) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int to = 1024 * (wave * kLoads + i) + 16 * lane;
            *reinterpret_cast<i32x4*>(&tiles[slot][0][to]) = k_raw[i];
            if (seen != kAll) {
                rarely();
                if (!((seen >> row_of[i]) & 1)) v_raw[i] = i32x4{0, 0, 0, 0};
            }
            *reinterpret_cast<i32x4*>(&tiles[slot][1][to]) = v_raw[i];
        }
    };

    f32x16 acc[kOut];
#pragma unroll
    for (int o = 0; o < kOut; ++o) {
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[o][i] = 0.0f;
    }
    float ref = 0.0f, bound = -__builtin_inff(), total = 0.0f;
    bool any = false;

    // The matrix unit's operands in a tile: row col of a half's 32 keys, elements 16b + 8h ..; and, transposed by the
    // read, channel 32o + col of the states that the lane's weights are of, 4h .. and 8 + 4h .. of each 16.
    int k_at[kDepth], v_at[kOut];
    const int v_row = 4 * h + (lane & 15) / 4, v_piece = 2 * ((lane >> 4) & 1) + (lane & 3) / 2;
#pragma unroll
    for (int b = 0; b < kDepth; ++b) k_at[b] = col * 2 * kWidth + 16 * key_place<kWidth>(col, 2 * b + h);
#pragma unroll
    for (int o = 0; o < kOut; ++o) v_at[o] = v_row * 2 * kWidth + 16 * value_place<kWidth>(v_row, 4 * o + v_piece) + 8 * (lane & 1);

    const auto compute = [&](int slot, uint64_t seen) {
        const uint8_t* keys = tiles[slot][0];
        const uint8_t* values = tiles[slot][1];
        f32x16 s[kStep / 32];
#pragma unroll
        for (int i = 0; i < kScores; ++i) s[i / 16][i % 16] = 0.0f;
#pragma unroll
        for (int b = 0; b < kDepth; ++b) {
#pragma unroll
            for (int j = 0; j < kStep / 32; ++j)
                s[j] = mfma32<kHalf>(*reinterpret_cast<const i32x4*>(keys + k_at[b] + 64 * kWidth * j), q[b], s[j]);
        }
        float most = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < kScores; ++i) s[i / 16][i % 16] = __builtin_fmaf(s[i / 16][i % 16], sharp, -ref);
        if (seen != kAll) {
            rarely();
            const uint64_t own = seen >> (4 * h);
#pragma unroll
            for (int i = 0; i < kScores; ++i)
                if (!((own >> (8 * (i / 4) + i % 4)) & 1)) s[i / 16][i % 16] = -__builtin_inff();
        }
#pragma unroll
        for (int i = 0; i < kScores; ++i) most = fmaxf(most, s[i / 16][i % 16]);
        if (__any(most > bound)) {
            most = fmaxf(most, __shfl_xor(most, 32));
            const float up = most > bound ? most - kLift : 0.0f;
            const float shrink = bound > 0.0f ? __builtin_amdgcn_exp2f(-up) : 0.0f;
            if (most > bound) bound = kBound;
            ref += up;
            total *= shrink;
#pragma unroll
            for (int i = 0; i < kScores; ++i) s[i / 16][i % 16] -= up;
#pragma unroll
            for (int o = 0; o < kOut; ++o) {
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[o][i] *= shrink;
            }
        }
        i32x4 w[kStep / 16];
#pragma unroll
        for (int i = 0; i < kScores; i += 2) {
            const float x = __builtin_amdgcn_exp2f(s[i / 16][i % 16]), y = __builtin_amdgcn_exp2f(s[i / 16][i % 16 + 1]);
            total += x + y;
            w[i / 8][i % 8 / 2] = pack2<kHalf>(x, y);
        }
#pragma unroll
        for (int a = 0; a < kStep / 16; ++a) {
#pragma unroll
            for (int o = 0; o < kOut; ++o) {
                const uint8_t* at = values + v_at[o] + 32 * kWidth * a;
                const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsFour*)(at));
                const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsFour*)(at + 16 * kWidth));
                const i32x2 l2 = __builtin_bit_cast(i32x2, lo), h2 = __builtin_bit_cast(i32x2, hi);
                acc[o] = mfma32<kHalf>(i32x4{l2[0], l2[1], h2[0], h2[1]}, w[a], acc[o]);
            }
        }
    };

    for (int stage = begin; stage < end; stage += kStage) {
        const int stage_end = min(end, stage + kStage);
        if (stage != begin) __syncthreads();
        for (int i = wave; i < stage_end - stage; i += kWaves) {
            const int t = (stage + i) * kStep + lane;
            const uint64_t word = __ballot(lane < kStep && t < of.length && (!mask || mask[t]));
            if (lane == 0) seen_of[i] = word;
        }
        __syncthreads();
        load(stage);
        put(stage & 1, seen_at(0));
        load(stage + 1);
        for (int step = stage; step < stage_end; ++step) {
            __syncthreads();
            if (step + 1 < stage_end) put((step + 1) & 1, seen_at(step + 1 - stage));
            load(step + 2);
            const uint64_t seen = seen_at(step - stage);
            any |= seen != 0;
            if (busy) compute(step & 1, seen);
        }
    }

    if (!live) return;
    total += __shfl_xor(total, 32);
    const int64_t at = static_cast<int64_t>(token) * p.q_heads + head;
#pragma unroll
    for (int o = 0; o < kOut; ++o) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            store_row<kWidth, kHalf>(p, split, at, 32 * o + 8 * i + 4 * h, f32x4{acc[o][4 * i], acc[o][4 * i + 1], acc[o][4 * i + 2], acc[o][4 * i + 3]},
                                     bound > 0.0f ? ref : kNoScore, total, any);
    }
}

// ------------------------------------------------------------------------------ few rows a request

template <bool kHalf>
__device__ __forceinline__ f32x4 mfma16(const i32x4& a, const i32x4& b, f32x4 c) {
    if constexpr (kHalf)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// LDS accesses of the wave's own lanes, before and after: done, and in that order.
__device__ __forceinline__ void wave_sync() {
    fence();
    wait_lgkmcnt0();
    __builtin_amdgcn_wave_barrier();
    fence();
}

// Waves of a workgroup: as many as leave each the registers that it needs.
constexpr int few_waves(int width, int tiles) { return width * tiles > 128 ? 4 : 8; }

// kWaves waves take the rows of one request and key head, 16 · kTiles at a time, over a share of its states: each wave
// every kWaves-th step of 32, by itself. Keys go from memory into registers as the matrix unit wants them, values
// through a tile of the wave's own in LDS, whose transposed read makes them the second product's operand. The waves'
// sums are joined in LDS.
template <int kWidth, int kTiles, bool kHalf>
__global__ __launch_bounds__(64 * few_waves(kWidth, kTiles), few_waves(kWidth, kTiles) / 4) void cross_few_kernel(CrossAttend p) {
    constexpr int kWaves = few_waves(kWidth, kTiles), kStep = 32, kDepth = kWidth / 32, kOut = kWidth / 16, kRows = 16 * kTiles;
    constexpr int kChunks = kWidth / 8, kPerLoad = 64 / kChunks, kLoads = kStep / kPerLoad;
    constexpr int kPad = kWidth + 4;
    __shared__ __attribute__((aligned(1024))) float merged[kWaves][16 * kPad];
    __shared__ float tops[kWaves][16], totals[kWaves][16];
    static_assert(16 * kPad * 4 >= kStep * kWidth * 2, "a tile of values fits the place of a wave's sums");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int kv = blockIdx.x % p.kv_heads, id = blockIdx.x / p.kv_heads, request = id / p.splits, split = id % p.splits;
    const Rows of = rows_of(p, request);
    const int rows = of.count * p.group, length = of.length;
    const int steps = (length + kStep - 1) / kStep;
    const int begin = static_cast<int>(static_cast<int64_t>(steps) * split / p.splits);
    const int end = static_cast<int>(static_cast<int64_t>(steps) * (split + 1) / p.splits);
    const uint16_t* k_base = p.k + request * p.k_request + kv * p.k_head;
    const uint16_t* v_base = p.v + request * p.v_request + kv * p.v_head;
    const __amdgpu_buffer_rsrc_t mask = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(p.mask ? p.mask + request * p.mask_request : nullptr), 0, p.mask ? length : 0, 0x00020000);
    const float sharp = p.scale * kLog2e;
    uint8_t* const values = reinterpret_cast<uint8_t*>(merged[wave]);

    uint32_t k_from[kDepth];
#pragma unroll
    for (int b = 0; b < kDepth; ++b)
        k_from[b] = 32 * b + 8 * g < p.width ? 2u * (col * static_cast<uint32_t>(p.k_state) + 32 * b + 8 * g) : kNowhere;
    const int v_row = 4 * g + col / 4, v_piece = (col & 3) / 2;
    int v_at[kOut];
#pragma unroll
    for (int o = 0; o < kOut; ++o) v_at[o] = v_row * 2 * kWidth + 16 * value_place<kWidth>(v_row, 2 * o + v_piece) + 8 * (col & 1);

    for (int row0 = 0; row0 < rows; row0 += kRows) {
        i32x4 q[kTiles][kDepth];
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
            const int row = row0 + 16 * n + col;
            const bool live = row < rows;
            const uint16_t* x = p.q + (of.first + (live ? row / p.group : 0)) * p.q_token + (kv * p.group + (live ? row % p.group : 0)) * p.q_head;
#pragma unroll
            for (int b = 0; b < kDepth; ++b) q[n][b] = query8(x, live, 32 * b + 8 * g, p.width);
        }
        f32x4 acc[kTiles][kOut];
        float ref[kTiles], bound[kTiles], total[kTiles];
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
            ref[n] = total[n] = 0.0f;
            bound[n] = -__builtin_inff();
#pragma unroll
            for (int o = 0; o < kOut; ++o) acc[n][o] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        bool any = false;

        i32x4 k_raw[2][kDepth], v_raw[kLoads];
        uint8_t shown = 0;
        const auto load_keys = [&](int step) {
            const int64_t t0 = static_cast<int64_t>(step) * kStep;
            const __amdgpu_buffer_rsrc_t kr =
                states_view(k_base + t0 * p.k_state, static_cast<int>(min(length - t0, static_cast<int64_t>(kStep))), p.k_state, p.width);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int b = 0; b < kDepth; ++b)
                    k_raw[j][b] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(
                        kr, k_from[b] + j * 32u * static_cast<uint32_t>(p.k_state), 0, 0));
            }
        };
        const auto load_values = [&](int step) {
            const int64_t t0 = static_cast<int64_t>(step) * kStep;
            const __amdgpu_buffer_rsrc_t vr =
                states_view(v_base + t0 * p.v_state, static_cast<int>(min(length - t0, static_cast<int64_t>(kStep))), p.v_state, p.width);
            shown = __builtin_amdgcn_raw_buffer_load_b8(mask, static_cast<int>(min(t0, static_cast<int64_t>(length))) + lane, 0, 0);
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int r = i * kPerLoad + lane / kChunks, c = value_place<kWidth>(r, lane % kChunks);
                v_raw[i] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(
                    vr, 8 * c < p.width ? 2u * (r * static_cast<uint32_t>(p.v_state) + 8 * c) : kNowhere, 0, 0));
            }
        };
        if (begin + wave < end) {
            load_keys(begin + wave);
            load_values(begin + wave);
        }
        for (int step = begin + wave; step < end; step += kWaves) {
            const uint32_t seen = static_cast<uint32_t>(__ballot(step * kStep + lane < length && (!p.mask || shown)));
            any |= seen != 0;
            f32x4 s[kTiles][2];
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    s[n][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int b = 0; b < kDepth; ++b) s[n][j] = mfma16<kHalf>(k_raw[j][b], q[n][b], s[n][j]);
                }
            }
            load_keys(step + kWaves);
            wave_sync();  // the last step's reads
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                i32x4 raw = v_raw[i];
                if (seen != 0xffffffffu) {
                    rarely();
                    if (!((seen >> (i * kPerLoad + lane / kChunks)) & 1)) raw = i32x4{0, 0, 0, 0};
                }
                *reinterpret_cast<i32x4*>(values + 1024 * i + 16 * lane) = raw;
            }
            load_values(step + kWaves);
            i32x4 w[kTiles];
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
                float x[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = __builtin_fmaf(s[n][i / 4][i % 4], sharp, -ref[n]);
                if (seen != 0xffffffffu) {
                    rarely();
                    const uint32_t own = seen >> (4 * g);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (!((own >> (16 * (i / 4) + i % 4)) & 1)) x[i] = -__builtin_inff();
                }
                float most = x[0];
#pragma unroll
                for (int i = 1; i < 8; ++i) most = fmaxf(most, x[i]);
                if (__any(most > bound[n])) {
                    most = fmaxf(most, __shfl_xor(most, 16));
                    most = fmaxf(most, __shfl_xor(most, 32));
                    const float up = most > bound[n] ? most - kLift : 0.0f;
                    const float shrink = bound[n] > 0.0f ? __builtin_amdgcn_exp2f(-up) : 0.0f;
                    if (most > bound[n]) bound[n] = kBound;
                    ref[n] += up;
                    total[n] *= shrink;
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] -= up;
#pragma unroll
                    for (int o = 0; o < kOut; ++o) acc[n][o] *= shrink;
                }
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const float a = __builtin_amdgcn_exp2f(x[i]), b = __builtin_amdgcn_exp2f(x[i + 1]);
                    total[n] += a + b;
                    w[n][i / 2] = pack2<kHalf>(a, b);
                }
            }
            wave_sync();
#pragma unroll
            for (int o = 0; o < kOut; ++o) {
                const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsFour*)(values + v_at[o]));
                const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsFour*)(values + v_at[o] + 32 * kWidth));
                const i32x2 l2 = __builtin_bit_cast(i32x2, lo), h2 = __builtin_bit_cast(i32x2, hi);
#pragma unroll
                for (int n = 0; n < kTiles; ++n) acc[n][o] = mfma16<kHalf>(i32x4{l2[0], l2[1], h2[0], h2[1]}, w[n], acc[n][o]);
            }
        }

        // The waves' sums, brought to one reference; then the rows, or their part of them.
        const bool some = __syncthreads_or(any);
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
            if (n) __syncthreads();
            total[n] += __shfl_xor(total[n], 16);
            total[n] += __shfl_xor(total[n], 32);
            const float top = bound[n] > 0.0f ? ref[n] : kNoScore;
            if (g == 0) {
                tops[wave][col] = top;
                totals[wave][col] = total[n];
            }
#pragma unroll
            for (int o = 0; o < kOut; ++o) *reinterpret_cast<f32x4*>(&merged[wave][col * kPad + 16 * o + 4 * g]) = acc[n][o];
            __syncthreads();
            const int first = row0 + 16 * n, count = min(16, rows - first);
            for (int i = threadIdx.x; i < count * (kWidth / 4); i += 64 * kWaves) {
                const int r = i / (kWidth / 4), d = 4 * (i % (kWidth / 4));
                float most = kNoScore, sum = 0.0f;
#pragma unroll
                for (int w = 0; w < kWaves; ++w) most = nan_max(most, tops[w][r]);
                f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int w = 0; w < kWaves; ++w) {
                    const float factor = __builtin_amdgcn_exp2f(tops[w][r] - most);
                    v += *reinterpret_cast<const f32x4*>(&merged[w][r * kPad + d]) * factor;
                    sum += totals[w][r] * factor;
                }
                const int64_t at = static_cast<int64_t>(of.first + (first + r) / p.group) * p.q_heads + kv * p.group + (first + r) % p.group;
                store_row<kWidth, kHalf>(p, split, at, d, v, most, sum, some);
            }
        }
        if (row0 + kRows < rows) __syncthreads();
    }
    if (p.starts && p.splits == 1) clear_rest(p, 0);
}

// Joins a row's parts, kWidth / 4 threads a row: Σ sums · 2^(ref − most) over Σ totals · 2^(ref − most).
template <int kWidth>
__global__ __launch_bounds__(256) void cross_join_kernel(CrossAttend p) {
    constexpr int kEach = kWidth / 4;
    const int64_t places = static_cast<int64_t>(p.tokens) * p.q_heads;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * (256 / kEach) + threadIdx.x / kEach;
    const int d = 4 * (threadIdx.x % kEach);
    if (at >= places || d >= p.width) return;
    const int token = static_cast<int>(at / p.q_heads);
    const Rows last = rows_of(p, p.requests - 1);
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (token >= rows_of(p, 0).first && token < last.first + last.count) {
        const float* parts = p.work + p.splits * places * kWidth;
        float most = -__builtin_inff();
        for (int i = 0; i < p.splits; ++i) most = nan_max(most, parts[2 * (i * places + at)]);
        if (most != -__builtin_inff()) {
            float total = 0.0f;
            for (int i = 0; i < p.splits; ++i) {
                const float factor = __builtin_amdgcn_exp2f(parts[2 * (i * places + at)] - most);
                total += parts[2 * (i * places + at) + 1] * factor;
                v += *reinterpret_cast<const f32x4*>(p.work + (i * places + at) * kWidth + d) * factor;
            }
            v *= 1.0f / total;
        }
    }
    *reinterpret_cast<i32x2*>(p.out + at * p.width + d) =
        i32x2{static_cast<int32_t>(narrow2(v[0], v[1], p.half)), static_cast<int32_t>(narrow2(v[2], v[3], p.half))};
}

constexpr int padded(int width) { return width <= 64 ? 64 : width <= 128 ? 128 : 256; }
constexpr int waves_of(int width) { return width == 256 ? 4 : 8; }

// Requests of up to so many rows a key head are cross_few_kernel's: two tiles of 16, whose accumulators fit the registers
// up to 128 wide.
constexpr int64_t few_rows(int width) { return width > 128 ? 16 : 32; }

// The shape of a call, which its workspace goes by too: the kernel, its rows a tile, and how many workgroups a tile's
// states are split over.
struct Shape {
    bool few;
    int rows, splits;
};

Shape shape_of(int64_t tokens, int group, int requests, int kv_heads, int states, int width, int64_t most) {
    const int64_t rows = (most > 0 && most < tokens ? most : tokens) * group;
    Shape a = {rows <= few_rows(width), 0, 1};
    int64_t groups, step, wanted, least;
    if (a.few) {
        a.rows = rows > 16 ? 32 : 16;
        groups = static_cast<int64_t>(requests) * kv_heads;
        step = 32 * 8;
        wanted = 512 / groups;
        least = 4;
    } else {
        a.rows = 32 * waves_of(padded(width));
        groups = ((tokens * group + a.rows - 1) / a.rows + requests - 1) * kv_heads;
        step = step_of(padded(width));
        wanted = 256 / groups;
        least = 4;
    }
    const int64_t fit = (states + step - 1) / step / least;
    const int64_t splits = wanted < fit ? wanted : fit;
    a.splits = static_cast<int>(splits < 1 ? 1 : splits > 64 ? 64 : splits);
    return a;
}

template <int kWidth, bool kHalf>
hipError_t attend(const CrossAttend& p, const Shape& a, hipStream_t s) {
    if (a.few) {
        const unsigned groups = static_cast<unsigned>(p.requests) * p.kv_heads * p.splits;
        constexpr int kMost = few_rows(kWidth) / 16;
        if (a.rows == 16) cross_few_kernel<kWidth, 1, kHalf><<<groups, 64 * few_waves(kWidth, 1), 0, s>>>(p);
        else cross_few_kernel<kWidth, kMost, kHalf><<<groups, 64 * few_waves(kWidth, kMost), 0, s>>>(p);
    } else {
        constexpr int kWaves = waves_of(kWidth), kRows = 32 * kWaves;
        const int64_t tiles = (static_cast<int64_t>(p.tokens) * p.group + kRows - 1) / kRows + p.requests;
        const unsigned groups = static_cast<unsigned>(tiles * p.kv_heads * p.splits);
        cross_kernel<kWidth, kWaves, kHalf><<<groups, 64 * kWaves, 0, s>>>(p);
    }
    if (p.splits > 1) {
        const int64_t rows = static_cast<int64_t>(p.tokens) * p.q_heads;
        constexpr int kEach = 256 / (kWidth / 4);
        cross_join_kernel<kWidth><<<static_cast<unsigned>((rows + kEach - 1) / kEach), 256, 0, s>>>(p);
    }
    return hipGetLastError();
}

template <int kWidth>
hipError_t attend(const CrossAttend& p, const Shape& a, hipStream_t s) {
    return p.half ? attend<kWidth, true>(p, a, s) : attend<kWidth, false>(p, a, s);
}

}  // namespace

int64_t cross_attend_work(int64_t tokens, int group, int requests, int kv_heads, int states, int width, int64_t most) {
    const int64_t splits = shape_of(tokens, group, requests, kv_heads, states, width, most).splits;
    return splits == 1 ? 0 : 4 * splits * tokens * group * kv_heads * (padded(width) + 2);
}

hipError_t cross_attend(CrossAttend p, int64_t most, hipStream_t s) {
    const Shape a = shape_of(p.tokens, p.group, p.requests, p.kv_heads, p.states, p.width, most);
    p.splits = a.splits;
    const int width = padded(p.width);
    if (width == 64) return attend<64>(p, a, s);
    if (width == 128) return attend<128>(p, a, s);
    return attend<256>(p, a, s);
}

}  // namespace cozyq
