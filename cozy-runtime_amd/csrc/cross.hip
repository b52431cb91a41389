// Attention of a decoder's rows to an encoder's states of another length, keys and values dense in 16 bits:
//
//   out_i = Σ_t softmax_t(scale · q_i · k_t) v_t
//
// over the states t of row i's request: those below its length that its mask has, all of them seen by every row. One
// pass over the states with the running maximum and sum of the softmax.
//
// Both products run on the matrix unit in the inputs' type, transposed (Sᵀ = K·Qᵀ, Oᵀ = Vᵀ·Pᵀ), so that a row is a
// column of both results and a lane holds 16 scores of one row for every 32 states. Weights are rounded to the inputs'
// type for the second product alone: float32 runs at a sixteenth of the rate there. (Against 64 bits the result is off
// by 0.0021 of its size in bf16 and 0.00024 in fp16 over 30000 states, where weights of 32 bits leave 0.0017 and 0.00021,
// the output's rounding.) Scores, maxima, sums and accumulators are float32. States that are not seen are zeros by the
// time they are in LDS, whatever memory holds.
#include <hip/hip_runtime.h>

#include "common.h"
#include "kernels.h"
#include "sixteen.h"

namespace cozyq {
namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 LdsFour;

constexpr float kLog2e = 1.44269504f;
// A row's weights are taken up to 2^kLift at first and 2^kSlack times that, 2^kMost at the most, before their reference
// moves. f16: up to 2^6 and 2^15, so that it holds those down to 2^-30 of the largest. bf16, whose values have float32's
// range: up to 2^-14 and 2^-6, between its two ends. Before they are divided, sums of 2^14 values of up to 2^128 stay finite
// at weights alike (of 2^6 values where most weights have crept up to the bound); and a sum of values down to 2^-126, in
// steps of 2^-149, is off by half of one a matrix instruction, each 2^-136 of the mean at the most. (A bound of 2^-8 costs
// 1.8% of 2311 masked rows' time in more moves.)
template <bool kHalf>
constexpr float kLift = kHalf ? 6.0f : -14.0f;
template <bool kHalf>
constexpr float kSlack = kHalf ? 9.0f : 8.0f;
constexpr float kMost = 15.0f;
// Below any reference, as the lowest finite number: that of a row without a finite score.
constexpr float kNoScore = -3.40282347e38f;
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

// Moves a row's reference for exponents of up to `most`, if they pass `bound` (minus infinity: there is no reference yet):
// `up` is how far, and the result what sums so far are to be taken times. Where scores are so large that float32 has no
// kLift more or less of them, the bound is of the weight that comes of it.
template <bool kHalf>
__device__ __forceinline__ float move(float most, float& ref, float& bound, float& up) {
    const bool over = most > bound;
    up = over ? most - kLift<kHalf> : 0.0f;
    const float shrink = bound > -__builtin_inff() ? __builtin_amdgcn_exp2f(-up) : 0.0f;
    if (over) bound = fminf(most - up + kSlack<kHalf>, kMost);
    ref += up;
    return shrink;
}

// Request b's rows of the call, in order and never past its last: [first, first + count), and how many states it has.
struct Rows {
    int first, count, length;
};

__host__ __device__ __forceinline__ Rows rows_of(const CrossAttend& p, int b) {
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

// Tiles and steps of a call are fewer than kMany, and sums end there, so that no `starts`, in order or not, carries an
// index past its request.
constexpr int kMany = 1 << 30;

// Two numbers of up to kMany, added up.
__host__ __device__ __forceinline__ int add_up(int a, int b) {
    const uint32_t sum = static_cast<uint32_t>(a) + static_cast<uint32_t>(b);
    return sum < kMany ? static_cast<int>(sum) : kMany;
}

// x from the lane that DPP control kCtrl names, 0 where it names none or the row is masked out.
template <int kCtrl, int kRowMask>
__device__ __forceinline__ int dpp_or_zero(int x) {
    return __builtin_amdgcn_update_dpp(0, x, kCtrl, kRowMask, 0xF, false);
}

// Inclusive sums over a wave of numbers of up to kMany: within rows of 16 lanes, then a row's last sum into the next.
__device__ __forceinline__ int wave_prefix(int n) {
    n = add_up(n, dpp_or_zero<0x111, 0xF>(n));  // row_shr:1
    n = add_up(n, dpp_or_zero<0x112, 0xF>(n));  // row_shr:2
    n = add_up(n, dpp_or_zero<0x114, 0xF>(n));  // row_shr:4
    n = add_up(n, dpp_or_zero<0x118, 0xF>(n));  // row_shr:8
    n = add_up(n, dpp_or_zero<0x142, 0xA>(n));  // row_bcast:15 into rows 1 and 3
    return add_up(n, dpp_or_zero<0x143, 0xC>(n));  // row_bcast:31 into rows 2 and 3
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
        const int sum = wave_prefix(tiles);
        const uint64_t past = __ballot(before - id > -sum);
        if (past) {
            const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
            request = base + at;
            tile = id - before - (__builtin_amdgcn_readlane(sum, at) - __builtin_amdgcn_readlane(tiles, at));
            return true;
        }
        before = add_up(before, __builtin_amdgcn_readlane(sum, 63));
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

// The inputs' type's largest number, and a finite result within it: a mean is no larger than its values, but where weights
// were rounded up and their sum was not, the quotient may be.
template <bool kHalf>
constexpr float kLargest = kHalf ? 65504.0f : 0x1.fep127f;
template <bool kHalf>
__device__ __forceinline__ float within(float x) {
    const float bounded = fminf(fmaxf(x, -kLargest<kHalf>), kLargest<kHalf>);
    return __builtin_fabsf(x) < __builtin_inff() ? bounded : x;
}

// Four elements of a row's result from d on, of the sums v with the denominator `total`. `some`: whether a state was
// seen; nothing seen is 0, nothing but scores of minus infinity the quotient 0 / 0.
template <bool kHalf>
__device__ __forceinline__ void store_row(const CrossAttend& p, int64_t at, int d, f32x4 v, float total, bool some) {
    if (d >= p.width) return;
    const float inv = some ? 1.0f / total : 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = within<kHalf>(v[i] * inv);
    *reinterpret_cast<i32x2*>(p.out + at * p.width + d) = i32x2{pack2<kHalf>(v[0], v[1]), pack2<kHalf>(v[2], v[3])};
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

// LDS accesses of the wave's own lanes, before and after: done, and in that order.
__device__ __forceinline__ void wave_sync() {
    fence();
    wait_lgkmcnt0();
    __builtin_amdgcn_wave_barrier();
    fence();
}

// A workgroup's part of a tile of kRows rows: their sums, as the lanes hold them, then their references and denominators.
template <int kWidth, int kRows>
__device__ __forceinline__ float* place_of(const CrossAttend& p, int64_t group) {
    return p.work + group * (kRows * (kWidth + 2));
}

// kWaves waves take a tile of 32 rows each of one key head over its states a step at a time, which all of them share in
// LDS. A step's keys and values are in registers by the step before it, when they are written to LDS, and asked for a
// step before that; one barrier a step. Queries and results cross LDS too, so that memory sees whole lines: read and
// written 8 and 16 bytes a row at a time they took 18000 rows of 24 heads of 128 over 512 states from 131 to 152 us.
// Where tiles are fewer than CUs a tile's states are split (301 rows of 28 heads over 30000 states: six ways, 154 us, and
// 746 in one), and cross_join_kernel adds the parts.
// Bound by no unit alone (matrix unit 28 to 39% of the cycles, vector unit 35 to 45%, a wave waits 33 to 39% of its life):
// of a step's 2.0 us (256 rows, 64 states, 128 wide) the products alone take 0.95. Left out one at a time, the scores
// are 0.5 of it, their exponentials and the second product 0.75, waiting for states 0.25, writing them to LDS and the
// barrier 0.15; the other 0.35 is no single part's. Two waves a SIMD are all that its registers hold. Tried and not faster: the
// next step's scores over this one's exponentials; half of the waves half a step late; 4 waves of 64 rows (copies
// between register files, +50%); 4 waves of 32, two workgroups a CU (states read twice as often, +12%); equal runs of
// steps as few rows have them (+5%: their parts' traffic, and requests' states no longer shared in L2).
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
    const int kv = blockIdx.x % p.kv_heads;
    const float sharp = p.scale * kLog2e;

    // This wave's shares of a step's keys and values: 1 KiB each, whole rows.
    uint32_t k_from[kLoads], v_from[kLoads], row_of[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int r = (wave * kLoads + i) * kPerLoad + lane / kChunks;
        const int kc = key_place<kWidth>(r, lane % kChunks), vc = value_place<kWidth>(r, lane % kChunks);
        row_of[i] = r;
        k_from[i] = 8 * kc < p.width ? 2u * (r * static_cast<uint32_t>(p.k_state) + 8 * kc) : kNowhere;
        v_from[i] = 8 * vc < p.width ? 2u * (r * static_cast<uint32_t>(p.v_state) + 8 * vc) : kNowhere;
    }
    // The matrix unit's operands in a tile: row col of a half's 32 keys, elements 16b + 8h ..; and, transposed by the
    // read, channel 32o + col of the states that the lane's weights are of, 4h .. and 8 + 4h .. of each 16.
    // Chunks' places are exclusive-or's, so that of 2b or 4o chunks further on is this one's with 32b or 64o.
    const int k_at = col * 2 * kWidth + 16 * key_place<kWidth>(col, h);
    const int v_row = 4 * h + (lane & 15) / 4, v_piece = 2 * ((lane >> 4) & 1) + (lane & 3) / 2;
    const int v_at = v_row * 2 * kWidth + 16 * value_place<kWidth>(v_row, v_piece) + 8 * (lane & 1);

    uint8_t* const own = &tiles[0][0][0] + wave * 64 * kWidth;
    static_assert(sizeof(tiles) >= kWaves * 64 * kWidth, "32 rows a wave");
    const int turn_tokens = kPerLoad / p.group, turn_heads = kPerLoad % p.group;
    const int id = blockIdx.x / p.kv_heads;
    int request, tile, found;
    if (!find_tile<kRows>(p, id / p.splits, request, tile, found)) {
        if (p.splits == 1) clear_rest(p, found * p.kv_heads);
        return;
    }
    const int split = id % p.splits;
    const Rows of = rows_of(p, request);
    const int rows = of.count * p.group, mine = kRows * tile + 32 * wave;
    const bool busy = mine < rows;
    const int steps = (of.length + kStep - 1) / kStep;
    const int begin = static_cast<int>(static_cast<int64_t>(steps) * split / p.splits);
    const int end = static_cast<int>(static_cast<int64_t>(steps) * (split + 1) / p.splits);
    const uint16_t* k_base = p.k + request * p.k_request + kv * p.k_head;
    const uint16_t* v_base = p.v + request * p.v_request + kv * p.v_head;
    const uint8_t* mask = p.mask ? p.mask + request * p.mask_request : nullptr;
    // Queries and results go through the wave's share of LDS, in whole lines to and from memory: piece i is rows
    // kPerLoad * i + lane / kChunks of the wave, and each(i, its token, its head, its chunk) is called for those
    // that are there.
    const auto each_line = [&](auto&& each) {
        int r0 = mine + lane / kChunks;
        asm volatile("" : "+v"(r0));  // worked out anew at each call, rather than kept in registers over the steps
        int token = of.first + r0 / p.group, head = r0 % p.group;
#pragma unroll
        for (int i = 0; i < 32 / kPerLoad; ++i) {
            const int r = i * kPerLoad + lane / kChunks, chunk = key_place<kWidth>(r, lane % kChunks);
            if (mine + r < rows && 8 * chunk < p.width) each(i, token, kv * p.group + head, 8 * chunk);
            token += turn_tokens;
            head += turn_heads;
            if (head >= p.group) {
                head -= p.group;
                ++token;
            }
        }
    };
    i32x4 q[kDepth];
    {
        i32x4 raw[32 / kPerLoad];
#pragma unroll
        for (int i = 0; i < 32 / kPerLoad; ++i) raw[i] = i32x4{0, 0, 0, 0};
        each_line([&](int i, int token, int head, int d) { raw[i] = *reinterpret_cast<const i32x4*>(p.q + token * p.q_token + head * p.q_head + d); });
#pragma unroll
        for (int i = 0; i < 32 / kPerLoad; ++i) *reinterpret_cast<i32x4*>(own + 1024 * i + 16 * lane) = raw[i];
        wave_sync();
#pragma unroll
        for (int b = 0; b < kDepth; ++b) q[b] = *reinterpret_cast<const i32x4*>(own + (k_at ^ 32 * b));
        wave_sync();
    }

    const auto same = [](uint64_t word) {
        return static_cast<uint64_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(word >> 32))) << 32 |
               static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(word)));
    };
    i32x4 k_raw[kLoads], v_raw[kLoads];
    const uint16_t* k_next = k_base + static_cast<int64_t>(begin) * kStep * p.k_state;
    const uint16_t* v_next = v_base + static_cast<int64_t>(begin) * kStep * p.v_state;
    int left = of.length - begin * kStep;
    // The next step's share.
    const auto load = [&] {
        const __amdgpu_buffer_rsrc_t kr = states_view(k_next, min(left, kStep), p.k_state, p.width);
        const __amdgpu_buffer_rsrc_t vr = states_view(v_next, min(left, kStep), p.v_state, p.width);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            k_raw[i] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(kr, k_from[i], 0, 0));
            v_raw[i] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(vr, v_from[i], 0, 0));
        }
        k_next += kStep * p.k_state;
        v_next += kStep * p.v_state;
        left -= kStep;
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

    f32x16 s[kStep / 32];
    const auto score = [&](int slot) {
        const int at = slot * 2 * kBytes + k_at;
        const uint8_t* keys = &tiles[0][0][0];
#pragma unroll
        for (int i = 0; i < kScores; ++i) s[i / 16][i % 16] = 0.0f;
#pragma unroll
        for (int b = 0; b < kDepth; ++b) {
#pragma unroll
            for (int j = 0; j < kStep / 32; ++j)
                s[j] = mfma32<kHalf>(*reinterpret_cast<const i32x4*>(keys + (at ^ 32 * b) + 64 * kWidth * j), q[b], s[j]);
        }
        // Eight operands read ahead: the compiler by itself reads two, and waits for LDS at each pair of products.
        constexpr int kProducts = kDepth * (kStep / 32), kAhead = 8;
        __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
        for (int i = 0; i < kProducts; i += 2) {
            __builtin_amdgcn_sched_group_barrier(0x8, 2, 0);
            if (i + kAhead < kProducts) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
    };
    const auto add = [&](int slot, uint64_t seen) {
        const int from = slot * 2 * kBytes + kBytes + v_at;
        const uint8_t* values = &tiles[0][0][0];
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
            float up;
            const float shrink = move<kHalf>(most, ref, bound, up);
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
                const uint8_t* at = values + (from ^ 64 * o) + 32 * kWidth * a;
                const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsFour*)(at));
                const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsFour*)(at + 16 * kWidth));
                const i32x2 l2 = __builtin_bit_cast(i32x2, lo), h2 = __builtin_bit_cast(i32x2, hi);
                acc[o] = mfma32<kHalf>(i32x4{l2[0], l2[1], h2[0], h2[1]}, w[a], acc[o]);
            }
        }
    };

    for (int stage = begin; stage < end; stage += kStage) {
        const int stage_end = min(end, stage + kStage);
        __syncthreads();  // the last stage's reads
        for (int i = wave; i < stage_end - stage; i += kWaves) {
            const int t = (stage + i) * kStep + lane;
            const uint64_t word = __ballot(lane < kStep && t < of.length && (!mask || mask[t]));
            if (lane == 0) seen_of[i] = word;
        }
        __syncthreads();
        if (stage == begin) load();
        uint64_t seen = same(seen_of[0]);
        put(stage & 1, seen);
        load();
        for (int step = stage; step < stage_end; ++step) {
            __syncthreads();
            const uint64_t word = step + 1 < stage_end ? seen_of[step + 1 - stage] : 0;
            if (busy) score(step & 1);
            const uint64_t next = same(word);
            if (step + 1 < stage_end) {
                put((step + 1) & 1, next);
                load();
            }
            any |= seen != 0;
            if (busy) add(step & 1, seen);
            seen = next;
        }
    }

    total += __shfl_xor(total, 32);
    if (p.splits == 1) {
        __syncthreads();
        const float inv = any ? 1.0f / total : 0.0f;
        float largest = 0.0f;
        const auto leave = [&](auto&& number) {
#pragma unroll
            for (int o = 0; o < kOut; ++o) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float x[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[j] = number(acc[o][4 * i + j]);
                    *reinterpret_cast<i32x2*>(own + col * 2 * kWidth + 16 * key_place<kWidth>(col, 4 * o + i) + 8 * h) =
                        i32x2{pack2<kHalf>(x[0], x[1]), pack2<kHalf>(x[2], x[3])};
                }
            }
        };
        leave([&](float sum) {
            const float x = sum * inv;
            largest = fmaxf(largest, __builtin_fabsf(x));
            return x;
        });
        if (__any(largest > kLargest<kHalf>)) {
            rarely();
            leave([&](float sum) { return within<kHalf>(sum * inv); });
        }
        wave_sync();
        each_line([&](int i, int token, int head, int d) {
            *reinterpret_cast<i32x4*>(p.out + (static_cast<int64_t>(token) * p.q_heads + head) * p.width + d) =
                *reinterpret_cast<const i32x4*>(own + 1024 * i + 16 * lane);
        });
        return;
    }
    if (!busy) return;
    float* const to = place_of<kWidth, kRows>(p, blockIdx.x);
#pragma unroll
    for (int o = 0; o < kOut; ++o) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            reinterpret_cast<f32x4*>(to)[(4 * kOut * wave + 4 * o + i) * 64 + lane] =
                f32x4{acc[o][4 * i], acc[o][4 * i + 1], acc[o][4 * i + 2], acc[o][4 * i + 3]};
    }
    if (h == 0)
        reinterpret_cast<f32x2*>(to + kRows * kWidth)[32 * wave + col] =
            f32x2{any ? (bound > -__builtin_inff() ? ref : kNoScore) : -__builtin_inff(), total};
}

// Joins a tile's parts, one a split: a workgroup the 32 rows of one wave, in the order in which it left them.
template <int kWidth, int kWaves>
__global__ __launch_bounds__(256) void cross_join_kernel(CrossAttend p) {
    constexpr int kRows = 32 * kWaves, kOut = kWidth / 32;
    const int lane = threadIdx.x & 63, side = threadIdx.x >> 6, wave = blockIdx.x % kWaves;
    const int id = blockIdx.x / kWaves, kv = id % p.kv_heads, col = lane & 31, h = lane >> 5;
    int request, tile, found;
    if (!find_tile<kRows>(p, id / p.kv_heads, request, tile, found)) {
        clear_rest(p, found * p.kv_heads * kWaves);
        return;
    }
    const Rows of = rows_of(p, request);
    const int row = kRows * tile + 32 * wave + col;
    if (row >= of.count * p.group) return;
    float most = -__builtin_inff(), total = 0.0f;
    f32x4 v[kOut];
#pragma unroll
    for (int o = 0; o < kOut; ++o) v[o] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 2
    for (int split = 0; split < p.splits; ++split) {
        const float* from = place_of<kWidth, kRows>(p, (id / p.kv_heads * p.splits + split) * p.kv_heads + kv);
        const f32x2 rest = reinterpret_cast<const f32x2*>(from + kRows * kWidth)[32 * wave + col];
        f32x4 one[kOut];
#pragma unroll
        for (int o = 0; o < kOut; ++o) one[o] = reinterpret_cast<const f32x4*>(from)[(4 * kOut * wave + kOut * side + o) * 64 + lane];
        const float up = nan_max(most, rest[0]);
        // Nothing seen so far, and here: minus infinity less itself is no reference.
        const float old = most == up ? 1.0f : __builtin_amdgcn_exp2f(most - up), factor = rest[0] == up ? 1.0f : __builtin_amdgcn_exp2f(rest[0] - up);
        total = total * old + rest[1] * factor;
#pragma unroll
        for (int o = 0; o < kOut; ++o) v[o] = v[o] * old + one[o] * factor;
        most = up;
    }
    const int64_t at = static_cast<int64_t>(of.first + row / p.group) * p.q_heads + kv * p.group + row % p.group;
    const bool some = most != -__builtin_inff();
#pragma unroll
    for (int o = 0; o < kOut; ++o) {
        const int chunk = kOut * side + o, d = 32 * (chunk / 4) + 8 * (chunk % 4) + 4 * h;
        if (p.half) store_row<true>(p, at, d, v[o], total, some);
        else store_row<false>(p, at, d, v[o], total, some);
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

// The eight XCDs take workgroups in turn: one share's heads begin further on than the last one's, so that each XCD reads
// rows of all key heads at a time. One head's rows alone, which are the heads' number times their bytes apart, may all
// lie in one of the 16 channels of an XCD's L2.
__device__ __forceinline__ int turn(int share, int kv_heads) { return (kv_heads >= 8 ? share : share / (8 / kv_heads)) % kv_heads; }

// Few rows' work is the steps of 32 states of all row tiles, one tile after another, the same for every key head: cut
// into `shares` equal runs, one a workgroup and head, wherever the cuts fall, so that requests of any lengths keep
// every CU at its share of the reading (one CU alone draws some 30 GB/s). A workgroup takes the end of one tile,
// whole tiles and the beginning of another, and leaves sums to be joined for the first and the last alone: two places
// each.
constexpr int kFewStep = 32;
// The loads' mark of what is read once.
constexpr int kOnce = 2;
// Steps of a tile that are not cut, and those of a run at the least.
constexpr int kWholeSteps = 24, kLeastSteps = 8;

// A request's row tiles, and a tile's steps: at the least one, so that a tile that sees nothing is written too.
struct Extent {
    int tiles, steps;
    Rows of;
};

template <int kRows>
__host__ __device__ __forceinline__ Extent extent_of(const CrossAttend& p, int b) {
    if (b >= p.requests) return {0, 0, {0, 0, 0}};
    const Rows r = rows_of(p, b);
    const int steps = max(1, (r.length + kFewStep - 1) / kFewStep);
    return {min((r.count * p.group + kRows - 1) / kRows, kMany / steps), steps, r};
}

// How the steps are cut: runs of `run`, at the least p.cut. Where runs of p.cut are few enough even if none of them holds
// two tiles' steps (`apart`), none does: the second tile would only wait for the first. Without cuts a run is a tile.
struct Cuts {
    Extent first;  // of the lane's request among the first 64
    int run;
    bool apart;
};

template <int kRows>
__device__ __forceinline__ Extent extent_at(const CrossAttend& p, const Cuts& c, int base) {
    return base == 0 ? c.first : extent_of<kRows>(p, base + static_cast<int>(threadIdx.x & 63));
}

// A request's runs of p.cut steps, if none holds two tiles' steps.
__host__ __device__ __forceinline__ int runs_of(const CrossAttend& p, const Extent& e) { return e.tiles * ((e.steps + p.cut - 1) / p.cut); }

// Cuts `total` steps in all (kMany: or more), of `runs` such runs; `longer`: whether a tile has more than kWholeSteps.
// run * shares > total, so that every step is of one of the runs.
__host__ __device__ __forceinline__ void cut(const CrossAttend& p, int total, int runs, bool longer, Cuts& c) {
    c.apart = runs <= p.shares;
    c.run = c.apart ? (longer ? p.cut : kWholeSteps) : max(p.cut, total / p.shares + 1);
}

// A tile's steps as they are counted.
__host__ __device__ __forceinline__ int counted(const Extent& e, const Cuts& c) {
    return c.apart ? (e.steps + c.run - 1) / c.run * c.run : e.steps;
}

// The first step of tile `tile` of a request's `tiles` of `one` steps each, the last of which ends at `end`.
__host__ __device__ __forceinline__ int first_step(int end, int tiles, int tile, int one) { return end - (tiles - tile) * one; }

// The runs that a tile's steps are in, from the first to the last.
struct Runs {
    int first, last;
};

__host__ __device__ __forceinline__ Runs runs_of(int start, int steps, int run) { return {start / run, (start + steps - 1) / run}; }

template <int kRows>
__device__ Cuts cuts_of(const CrossAttend& p) {
    Cuts c = {extent_of<kRows>(p, threadIdx.x & 63), 1, !p.cut};
    if (!p.cut) {
        c.run = kMany;
        return c;
    }
    int total = 0, runs = 0;
    bool longer = false;
    for (int base = 0; base < p.requests; base += 64) {
        const Extent e = extent_at<kRows>(p, c, base);
        longer |= __any(e.steps > kWholeSteps);
        total = add_up(total, __builtin_amdgcn_readlane(wave_prefix(e.tiles * e.steps), 63));
        runs = add_up(runs, __builtin_amdgcn_readlane(wave_prefix(runs_of(p, e)), 63));
    }
    cut(p, total, runs, longer, c);
    return c;
}

// A row tile: its request, its number there, its first step among all, its steps.
struct Item {
    int request, tile, start, steps;
    Rows of;
};

// The tile that step `id` is of (kByStep), or tile number `id`; false past the last.
template <int kRows, bool kByStep>
__device__ bool find_item(const CrossAttend& p, const Cuts& c, int id, Item& out) {
    int ids_before = 0, steps_before = 0;
    for (int base = 0; base < p.requests; base += 64) {
        const Extent e = extent_at<kRows>(p, c, base);
        const int one = p.cut ? counted(e, c) : 0;
        const int steps = wave_prefix(e.tiles * one), tiles = wave_prefix(e.tiles);
        const int ids = kByStep ? steps : tiles;
        const uint64_t past = __ballot(ids_before - id > -ids);
        if (past) {
            const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
            const int n = __builtin_amdgcn_readlane(one, at), t = __builtin_amdgcn_readlane(e.tiles, at);
            const int from = id - ids_before - __builtin_amdgcn_readlane(ids, at) + (kByStep ? t * n : t);
            const int tile = kByStep ? from / n : from;
            out = {base + at, tile, first_step(steps_before + __builtin_amdgcn_readlane(steps, at), t, tile, n), __builtin_amdgcn_readlane(e.steps, at),
                   {__builtin_amdgcn_readlane(e.of.first, at), __builtin_amdgcn_readlane(e.of.count, at), __builtin_amdgcn_readlane(e.of.length, at)}};
            return true;
        }
        ids_before = add_up(ids_before, __builtin_amdgcn_readlane(ids, 63));
        steps_before = add_up(steps_before, __builtin_amdgcn_readlane(steps, 63));
    }
    return false;
}

// The place of a part of kRows rows: their sums, then their references and denominators.
template <int kWidth, int kRows>
__device__ __forceinline__ float* place_of(const CrossAttend& p, int place, int kv) {
    return p.work + (static_cast<int64_t>(place) * p.kv_heads + kv) * (kRows * (kWidth + 2));
}

// kWaves waves take a run of steps of one key head, a row tile of 16 · kTiles rows at a time: each wave
// every kWaves-th step by itself. Keys and values go in whole lines through registers and then, one after the other,
// through a tile of the wave's own in LDS, from which they are read as the matrix unit wants them, values by a transposed
// read. (Keys loaded as the first product's operand, 64 bytes of 16 rows at a time: 35.4 us for 32.9, 24 requests over 1600
// states each.) The waves' sums are joined in LDS.
// Bound by memory: those 157 MB at 4.8 TB/s, where reads alone of the same rows, 256 bytes at a stride of 4 KiB, reach
// 5.1 to 5.5; before the first of them 4 us of launch and search.
template <int kWidth, int kTiles, bool kHalf>
__global__ __launch_bounds__(256, kWidth * kTiles > 128 ? 1 : kWidth * kTiles == 64 ? 4 : 2) void cross_few_kernel(CrossAttend p) {
    constexpr int kWaves = 4, kStep = kFewStep, kDepth = kWidth / 32, kOut = kWidth / 16, kRows = 16 * kTiles;
    constexpr int kChunks = kWidth / 8, kPerLoad = 64 / kChunks, kLoads = kStep / kPerLoad;
    constexpr int kPad = kWidth + 4;
    __shared__ __attribute__((aligned(1024))) float merged[kWaves][16 * kPad];
    __shared__ float tops[kWaves][16], totals[kWaves][16];
    static_assert(16 * kPad * 4 >= kStep * kWidth * 2, "a tile of values fits the place of a wave's sums");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    const float sharp = p.scale * kLog2e;
    uint8_t* const tile = reinterpret_cast<uint8_t*>(merged[wave]);
    const int share = blockIdx.x / p.kv_heads, kv = (blockIdx.x % p.kv_heads + turn(share, p.kv_heads)) % p.kv_heads;

    int k_at[kDepth];
#pragma unroll
    for (int b = 0; b < kDepth; ++b) k_at[b] = col * 2 * kWidth + 16 * key_place<kWidth>(col, 4 * b + g);
    const int v_row = 4 * g + col / 4, v_piece = (col & 3) / 2;
    int v_at[kOut];
#pragma unroll
    for (int o = 0; o < kOut; ++o) v_at[o] = v_row * 2 * kWidth + 16 * value_place<kWidth>(v_row, 2 * o + v_piece) + 8 * (col & 1);

    const Cuts cuts = cuts_of<kRows>(p);
    const int run_from = static_cast<int>(min(static_cast<int64_t>(share) * cuts.run, static_cast<int64_t>(kMany)));
    int at = p.cut ? run_from : 0, run_to = p.cut ? run_from + cuts.run : 1;
    Item item;
    while (at < run_to) {
        if (p.cut ? !find_item<kRows, true>(p, cuts, at, item) : !find_item<kRows, false>(p, cuts, share, item)) break;
        if (!p.cut) run_to = item.steps;
        const int request = item.request, begin = at - item.start, last = min(item.steps, run_to - item.start);
        const bool whole = begin == 0 && last == item.steps;
        const int part = 2 * share + (begin == 0 && at != run_from ? 1 : 0);
        at = cuts.apart ? run_to : item.start + last;
        const Rows of = item.of;
        const int length = of.length, row0 = kRows * item.tile, rows = min(of.count * p.group, row0 + kRows);
        const int end = min(last, (length + kStep - 1) / kStep);
        const uint16_t* k_base = p.k + request * p.k_request + kv * p.k_head;
        const uint16_t* v_base = p.v + request * p.v_request + kv * p.v_head;
        const __amdgpu_buffer_rsrc_t mask = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint8_t*>(p.mask ? p.mask + request * p.mask_request : nullptr), 0, p.mask ? length : 0, 0x00020000);
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

        i32x4 k_raw[kLoads], v_raw[kLoads];
        uint8_t shown = 0;
        const auto load_keys = [&](int step) {
            const int64_t t0 = static_cast<int64_t>(step) * kStep;
            const __amdgpu_buffer_rsrc_t kr = states_view(k_base + t0 * p.k_state, static_cast<int>(step < end ? min(length - t0, static_cast<int64_t>(kStep)) : 0), p.k_state, p.width);
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int r = i * kPerLoad + lane / kChunks, c = key_place<kWidth>(r, lane % kChunks);
                k_raw[i] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(
                    kr, 8 * c < p.width ? 2u * (r * static_cast<uint32_t>(p.k_state) + 8 * c) : kNowhere, 0, kOnce));
            }
        };
        const auto load_values = [&](int step) {
            const int64_t t0 = static_cast<int64_t>(step) * kStep;
            const __amdgpu_buffer_rsrc_t vr =
                states_view(v_base + t0 * p.v_state, static_cast<int>(step < end ? min(length - t0, static_cast<int64_t>(kStep)) : 0), p.v_state, p.width);
            shown = __builtin_amdgcn_raw_buffer_load_b8(mask, static_cast<int>(min(t0, static_cast<int64_t>(length))) + lane, 0, 0);
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int r = i * kPerLoad + lane / kChunks, c = value_place<kWidth>(r, lane % kChunks);
                v_raw[i] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(
                    vr, 8 * c < p.width ? 2u * (r * static_cast<uint32_t>(p.v_state) + 8 * c) : kNowhere, 0, kOnce));
            }
        };
        load_keys(begin + wave);
        load_values(begin + wave);
        for (int step = begin + wave; step < end; step += kWaves) {
            const uint32_t seen = static_cast<uint32_t>(__ballot(step * kStep + lane < length && (!p.mask || shown)));
            any |= seen != 0;
            wave_sync();  // the last step's reads
#pragma unroll
            for (int i = 0; i < kLoads; ++i) *reinterpret_cast<i32x4*>(tile + 1024 * i + 16 * lane) = k_raw[i];
            load_keys(step + kWaves);
            wave_sync();
            f32x4 s[kTiles][2];
#pragma unroll
            for (int n = 0; n < kTiles; ++n) s[n][0] = s[n][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int b = 0; b < kDepth; ++b) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const i32x4 k = *reinterpret_cast<const i32x4*>(tile + k_at[b] + 32 * kWidth * j);
#pragma unroll
                    for (int n = 0; n < kTiles; ++n) s[n][j] = mfma16<kHalf>(k, q[n][b], s[n][j]);
                }
            }
            wave_sync();  // the keys' reads
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                i32x4 raw = v_raw[i];
                if (seen != 0xffffffffu) {
                    rarely();
                    if (!((seen >> (i * kPerLoad + lane / kChunks)) & 1)) raw = i32x4{0, 0, 0, 0};
                }
                *reinterpret_cast<i32x4*>(tile + 1024 * i + 16 * lane) = raw;
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
                    float up;
                    const float shrink = move<kHalf>(most, ref[n], bound[n], up);
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
                const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsFour*)(tile + v_at[o]));
                const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsFour*)(tile + v_at[o] + 32 * kWidth));
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
            if (g == 0) {
                tops[wave][col] = bound[n] > -__builtin_inff() ? ref[n] : kNoScore;
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
                if (whole) {
                    const int row = first + r;
                    store_row<kHalf>(p, static_cast<int64_t>(of.first + row / p.group) * p.q_heads + kv * p.group + row % p.group, d, v, sum, some);
                } else {
                    float* to = place_of<kWidth, kRows>(p, part, kv);
                    *reinterpret_cast<f32x4*>(to + (16 * n + r) * kWidth + d) = v;
                    if (d == 0) *reinterpret_cast<f32x2*>(to + kRows * kWidth + 2 * (16 * n + r)) = f32x2{some ? most : -__builtin_inff(), sum};
                }
            }
        }
        __syncthreads();
    }
    if (p.starts) clear_rest(p, 0);
}

// Joins the parts of few rows' tiles that runs cut: a workgroup a tile and key head.
template <int kWidth, int kRows>
__global__ __launch_bounds__(256) void cross_few_join_kernel(CrossAttend p) {
    constexpr int kEach = kWidth / 4;
    const int kv = blockIdx.x % p.kv_heads;
    const Cuts cuts = cuts_of<kRows>(p);
    const int run = cuts.run;
    Item item;
    if (!find_item<kRows, false>(p, cuts, blockIdx.x / p.kv_heads, item)) return;
    const Runs parts = runs_of(item.start, item.steps, run);
    const int first = parts.first, last = parts.last;
    if (first == last) return;  // whole
    const Rows of = item.of;
    const int row0 = kRows * item.tile, count = min(kRows, of.count * p.group - row0);
    // Each wave takes every fourth part of a row, 64 / kEach rows at a time; then the waves' sums are joined in LDS.
    constexpr int kSide = kEach < 64 ? 64 / kEach : 1;
    __shared__ f32x4 sums[4][64];
    __shared__ f32x2 rests[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int r0 = 0; r0 < count; r0 += kSide) {
        const int r = min(r0 + lane / kEach, count - 1), d = 4 * (lane % kEach);
        const auto part = [&](int share) { return place_of<kWidth, kRows>(p, 2 * share + (share == first && item.start % run ? 1 : 0), kv); };
        float most = -__builtin_inff(), total = 0.0f;
        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
        for (int share = first + wave; share <= last; share += 4) {
            const float* from = part(share);
            const f32x2 rest = *reinterpret_cast<const f32x2*>(from + kRows * kWidth + 2 * r);
            const f32x4 one = *reinterpret_cast<const f32x4*>(from + r * kWidth + d);
            const float up = nan_max(most, rest[0]);
            // Nothing seen so far, and here: minus infinity less itself is no reference.
            const float old = most == up ? 1.0f : __builtin_amdgcn_exp2f(most - up), factor = rest[0] == up ? 1.0f : __builtin_amdgcn_exp2f(rest[0] - up);
            total = total * old + rest[1] * factor;
            v = v * old + one * factor;
            most = up;
        }
        sums[wave][lane] = v;
        rests[wave][lane] = f32x2{most, total};
        __syncthreads();
        if (wave == 0 && r0 + lane / kEach < count) {
#pragma unroll
            for (int w = 1; w < 4; ++w) {
                const f32x2 rest = rests[w][lane];
                const float up = nan_max(most, rest[0]);
                const float old = most == up ? 1.0f : __builtin_amdgcn_exp2f(most - up), factor = rest[0] == up ? 1.0f : __builtin_amdgcn_exp2f(rest[0] - up);
                total = total * old + rest[1] * factor;
                v = v * old + sums[w][lane] * factor;
                most = up;
            }
            const int row = row0 + r;
            const int64_t at = static_cast<int64_t>(of.first + row / p.group) * p.q_heads + kv * p.group + row % p.group;
            const bool some = most != -__builtin_inff();
            if (p.half) store_row<true>(p, at, d, v, total, some);
            else store_row<false>(p, at, d, v, total, some);
        }
        __syncthreads();
    }
}

constexpr int padded(int width) { return width <= 64 ? 64 : width <= 128 ? 128 : 256; }
constexpr int waves_of(int width) { return width == 256 ? 4 : 8; }

// Requests of up to so many rows a key head are cross_few_kernel's: two tiles of 16, whose accumulators fit the registers
// up to 128 wide. By that alone; cross_few_kernel / cross_kernel, us, requests of so many rows each: 24 requests over 1600
// states, 8 key heads of 128, 16 rows 34.4 / 37.7, 20 rows 35.7 / 37.4, 32 rows 35.1 / 38.0, 20 key heads of 64 40.8 /
// 56.5, 41.4 / 56.8, 40.3 / 55.1; but 4 requests, whose steps are cut, 16 rows 24.9 / 17.8, 20 rows 29.7 / 18.0, 32 rows
// 38.9 / 18.7, of 64 20.7 / 19.9, 26.2 / 20.1, 31.5 / 20.9.
constexpr int64_t few_rows(int width) { return width > 128 ? 16 : 32; }

// Whether few rows' steps are cut into equal runs, which costs a second launch and a workgroup's search for its tiles,
// some 8 us, or every tile is one workgroup's, which then draws 30 to 40 GB/s alone. Cut / whole, us, one row a request
// and 32 heads over 8 of 128: 24 requests over 400 to 1601 states 29.4 / 27.2, over 1600 each 40.7 / 32.9; 6 over 1601 16.3 /
// 25.3; 8 over 6400 41 / 90; 1 over 6400 17 / 80; 20 heads of 64 over 1500 11.0 / 16.8. Past 128 steps always: the
// lengths, which are on the GPU, may be of very different sizes.
bool few_cut(int64_t pairs, int64_t steps, int width) {
    return steps > kWholeSteps && (steps > 128 || (256 - pairs) * steps * width > 4096 * 128);
}

// The shape of a call, which its workspace goes by too: the kernel, its rows a tile, and how its states are shared out.
struct Shape {
    bool few;
    int rows;
    int64_t tiles;  // at the most, of a key head
    int splits;     // many rows: workgroups of a tile
    int cut, shares;  // few rows: a run's steps at the least (0: runs are tiles), runs at the most
    int64_t floats;
    int64_t threads;  // of the larger launch
};

Shape shape_of(int64_t tokens, int group, int requests, int kv_heads, int states, int width, int64_t most) {
    const int64_t rows = (most > 0 && most < tokens ? most : tokens) * group;
    Shape a = {rows <= few_rows(width), 0, 0, 1, 0, 0, 0, 0};
    if (a.few) {
        a.rows = rows > 16 ? 32 : 16;
        a.tiles = tokens * group / a.rows + requests;
        const int64_t steps = (states + kFewStep - 1) / kFewStep;
        a.few = a.tiles * (steps + 1) < (1 << 30);
        if (few_cut(static_cast<int64_t>(requests) * kv_heads, steps, padded(width))) {
            const int64_t runs = a.tiles * ((steps + kLeastSteps - 1) / kLeastSteps), shares = max((padded(width) == 64 ? 1024 : 512) / kv_heads, 1);
            a.cut = kLeastSteps;
            a.shares = static_cast<int>(min(runs, shares));
            a.floats = 2ll * a.shares * kv_heads * a.rows * (padded(width) + 2);
        }
        a.threads = 256 * kv_heads * (a.shares > a.tiles ? a.shares : a.tiles);
    }
    if (!a.few) {
        const int waves = waves_of(padded(width));
        a = {false, 32 * waves, 0, 1, 0, 0, 0, 0};
        a.tiles = (tokens * group + a.rows - 1) / a.rows + requests;
        const int64_t step = step_of(padded(width)), steps = (states + step - 1) / step;
        const int64_t splits = min(256 / (a.tiles * kv_heads), steps / 4);
        a.splits = static_cast<int>(splits < 1 ? 1 : splits > 64 ? 64 : splits);
        if (a.splits > 1) a.floats = a.tiles * a.splits * kv_heads * a.rows * (padded(width) + 2);
        a.threads = a.tiles * kv_heads * waves * (a.splits > 4 ? 64 * a.splits : a.splits > 1 ? 256 : 64);
    }
    return a;
}

template <int kWidth, int kTiles, bool kHalf>
void attend_few(const CrossAttend& p, const Shape& a, hipStream_t s) {
    const unsigned groups = static_cast<unsigned>((a.cut ? a.shares : a.tiles) * p.kv_heads);
    cross_few_kernel<kWidth, kTiles, kHalf><<<groups, 256, 0, s>>>(p);
    if (a.cut) cross_few_join_kernel<kWidth, 16 * kTiles><<<static_cast<unsigned>(a.tiles * p.kv_heads), 256, 0, s>>>(p);
}

template <int kWidth, bool kHalf>
hipError_t attend(const CrossAttend& p, const Shape& a, hipStream_t s) {
    if (a.few) {
        if (a.rows == 16) attend_few<kWidth, 1, kHalf>(p, a, s);
        else attend_few<kWidth, few_rows(kWidth) / 16, kHalf>(p, a, s);
        return hipGetLastError();
    }
    constexpr int kWaves = waves_of(kWidth);
    const unsigned groups = static_cast<unsigned>(a.tiles * p.kv_heads * p.splits);
    cross_kernel<kWidth, kWaves, kHalf><<<groups, 64 * kWaves, 0, s>>>(p);
    if (p.splits > 1) cross_join_kernel<kWidth, kWaves><<<static_cast<unsigned>(a.tiles * p.kv_heads * kWaves), 256, 0, s>>>(p);
    return hipGetLastError();
}

template <int kWidth>
hipError_t attend(const CrossAttend& p, const Shape& a, hipStream_t s) {
    return p.half ? attend<kWidth, true>(p, a, s) : attend<kWidth, false>(p, a, s);
}

}  // namespace

int64_t cross_attend_work(int64_t tokens, int group, int requests, int kv_heads, int states, int width, int64_t most) {
    const Shape a = shape_of(tokens, group, requests, kv_heads, states, width, most);
    return a.threads < (1ll << 32) ? 4 * a.floats : -1;
}

// What cuts_of and find_item come to, 64 requests after another: the same sums and rules.
template <int kRows>
static void host_runs(const CrossAttend& p, int tiles, int* out) {
    Cuts c = {extent_of<kRows>(p, 0), 1, false};
    int total = 0, runs = 0;
    bool longer = false;
    for (int base = 0; base < p.requests; base += 64) {
        int all = 0, cut_up = 0;
        for (int b = base; b < base + 64; ++b) {
            const Extent e = extent_of<kRows>(p, b);
            longer |= e.steps > kWholeSteps;
            all = add_up(all, e.tiles * e.steps);
            cut_up = add_up(cut_up, runs_of(p, e));
        }
        total = add_up(total, all);
        runs = add_up(runs, cut_up);
    }
    cut(p, total, runs, longer, c);
    int least = 0, most = 0, steps_before = 0;
    for (int base = 0, id = 0; base < p.requests; base += 64) {
        int steps = 0;
        for (int b = base; b < base + 64; ++b) {
            const Extent e = extent_of<kRows>(p, b);
            const int one = counted(e, c);
            steps = add_up(steps, e.tiles * one);
            for (int tile = 0; tile < e.tiles && id < tiles; ++tile, ++id) {
                const Runs of = runs_of(first_step(steps_before + steps, e.tiles, tile, one), e.steps, c.run);
                least = min(least, of.first);
                most = max(most, of.last);
            }
        }
        steps_before = add_up(steps_before, steps);
    }
    out[0] = total;
    out[1] = c.run;
    out[2] = p.shares;
    out[3] = least;
    out[4] = most;
}

bool cross_runs(CrossAttend p, int64_t most, int* out) {
    const Shape a = shape_of(p.tokens, p.group, p.requests, p.kv_heads, p.states, p.width, most);
    if (!a.cut) return false;
    p.cut = a.cut;
    p.shares = a.shares;
    if (a.rows == 16) host_runs<16>(p, static_cast<int>(a.tiles), out);
    else host_runs<32>(p, static_cast<int>(a.tiles), out);
    return true;
}

hipError_t cross_attend(CrossAttend p, int64_t most, hipStream_t s) {
    const Shape a = shape_of(p.tokens, p.group, p.requests, p.kv_heads, p.states, p.width, most);
    p.splits = a.splits;
    p.cut = a.cut;
    p.shares = a.shares;
    const int width = padded(p.width);
    if (width == 64) return attend<64>(p, a, s);
    if (width == 128) return attend<128>(p, a, s);
    return attend<256>(p, a, s);
}

}  // namespace cozyq
