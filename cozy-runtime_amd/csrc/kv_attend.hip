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
// element. Weights are rounded to f16 (11 bits, three more than bf16) for the second product alone: float32 runs
// at a sixteenth of the rate there, and two f16 numbers a weight would double the product. Nothing shows of it in
// bf16; in fp16 an output's error grows from 2.1e-4 to 2.7e-4 of its norm. Maxima, sums and both products'
// accumulators are float32.
// A denominator takes p/vs where p is above 2^-126 of the reference: where a request's pages have value scales
// more than 2^110 apart, the tokens of the smallest may be missing from it.
#include <hip/hip_runtime.h>

#include "common.h"
#include "kernels.h"
#include "sixteen.h"

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

// 16 bytes of codes, marked as read once or not.
template <bool kOnce>
__device__ __forceinline__ i32x4 codes16(const uint8_t* at) {
    const i32x4* p = reinterpret_cast<const i32x4*>(at);
    if constexpr (kOnce) return __builtin_nontemporal_load(p);
    else return *p;
}

// A finite scale, NaN for an infinite one: whoever sees its page gets NaN, not a score of either sign.
__device__ __forceinline__ float or_nan(float scale) { return scale + (scale - scale); }

// Keeps a branch a branch: without it the compiler works out both sides and selects.
__device__ __forceinline__ void rarely() { asm volatile(""); }

// Four elements from d on of a row's result: the sums over its denominator, 0 for a row that sees nothing.
__device__ __forceinline__ void store_row(const CacheAttend& p, int token, int head, int width, int d, f32x4 v, float total) {
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    const i32x2 two = {static_cast<int32_t>(narrow2(v[0] * inv, v[1] * inv, p.half)),
                       static_cast<int32_t>(narrow2(v[2] * inv, v[3] * inv, p.half))};
    *reinterpret_cast<i32x2*>(p.out + (static_cast<int64_t>(token) * p.q_heads + head) * width + d) = two;
}

// Where request r's rows begin, never past the step's.
__device__ __forceinline__ int row_start(const CacheAttend& p, int r) { return min(max(p.starts[r], 0), p.tokens); }

// Request r in the step: its first row, how many of its rows the step has, the tokens before the first of them, and
// its tokens in all. A step that ends before a request's rows do cuts the last ones off: those before stay where
// they are.
struct Rows {
    int first, fresh, before, length;
};

__device__ __forceinline__ Rows rows_of(const CacheAttend& p, int r) {
    const int first = row_start(p, r), end = max(p.starts[r + 1], first), length = max(p.lengths[r], 0);
    return {first, min(end, p.tokens) - first, length - (end - first), length};
}

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

// The largest of a wave's numbers, none of them negative, in its last lane.
__device__ __forceinline__ int wave_top(int x) {
    x = max(x, dpp_or_zero<0x111, 0xF>(x));
    x = max(x, dpp_or_zero<0x112, 0xF>(x));
    x = max(x, dpp_or_zero<0x114, 0xF>(x));
    x = max(x, dpp_or_zero<0x118, 0xF>(x));
    x = max(x, dpp_or_zero<0x142, 0xA>(x));
    return max(x, dpp_or_zero<0x143, 0xC>(x));
}

// The first token that a row at `position` sees, whatever numbers the two are.
__device__ __forceinline__ int low_of(const CacheAttend& p, int position) {
    return p.window > 0 && position >= p.window ? position + 1 - p.window : 0;
}

// --------------------------------------------------------------------- sharing the work out

constexpr int kStep = 64;       // tokens taken at a time

// Which requests a launch takes: those of more than `over` and up to `upto` rows, in row tiles shared
// out over `shares` workgroups a head.
struct Part {
    int over, upto, shares;
    int least;    // steps a workgroup takes at the least
    int shift;    // a row tile is 1 << shift rows
    float* work;  // places of a row tile's rows · (width + 4) floats: a row's sums, reference, denominator; or none
    int cuts;     // how many of kCuts a long tile's steps may be cut by
};

// A request's part of the work: row tiles, and the 64-token steps that any of its rows sees.
struct Extent {
    int tiles, steps;
};

__device__ __forceinline__ Extent extent(const CacheAttend& p, const Part& part, int r) {
    const Rows own = rows_of(p, r);
    const int rows = own.fresh * p.group;
    if (rows <= part.over || rows > part.upto) return {0, 0};
    const int low = low_of(p, own.before);
    const int held = min(own.length, p.width << p.shift);  // what the table's row has pages for
    const int steps = (held + kStep - 1) / kStep - low / kStep;
    return {(rows + (1 << part.shift) - 1) >> part.shift, max(steps, 0)};
}

// Tile `tile` of request `request`, its steps split over `splits` workgroups, of which this is number
// `split`; with more than one they leave their sums in that many places from `place` on.
struct Share {
    int request, tile, split, splits, place;
};

// A workgroup's steps are N / shares over one of these, N the steps in all (a head).
constexpr float kCuts[] = {1.0f, 4.0f / 3.0f, 2.0f};
constexpr int kCutCount = 3, kMostCut = 2;

// All the row tiles' steps are shared out evenly: a workgroup takes c = max(least, N / (shares · cut)) of one
// row tile's, so that there are at most shares · cut workgroups more than tiles and at most 2 · shares · cut
// places (a tile of more than c steps splits into less than 2 · steps / c), whatever the requests' lengths
// are: the host sizes the launch and the workspace without knowing them.
// Where tiles are split and a CU holds one workgroup, the cut is the one of least cost: the rounds of `shares`
// workgroups, each as long as the longest share and kStartSteps, and a part's way through memory, 1/kPartsAStep
// of a step. (Chunks of 574 tokens among 11 requests, 64 heads over 8: at cut 1, 4/3 and 2 189, 162 and
// 176 us; 500 among 8 137, 114 and 112; but 500 among 4 of 20000 tokens 203, 255 and 219. The choice costs 3 us, so
// that it is not made over shares of less than 3/2 · least steps, where 54 became 57.)
constexpr float kStartSteps = 4.0f, kPartsAStep = 48.0f;

__device__ int steps_a_share(const CacheAttend& p, const Part& part, Extent& e0) {
    const int lane = threadIdx.x & 63;
    float work = 0.0f;  // in float32, which no number of steps overflows; the margin is over its rounding
    int longest = 0;
    e0 = {0, 0};
    for (int base = 0; base < p.requests; base += 64) {
        Extent e = {0, 0};
        if (base + lane < p.requests) e = extent(p, part, base + lane);
        const float sum = wave_prefix(static_cast<float>(e.tiles) * static_cast<float>(e.steps));
        work += __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, sum), 63));
        longest = max(longest, e.steps);
        if (base == 0) e0 = e;
    }
    const float shares = static_cast<float>(part.shares), one = work * 1.001f / shares;
    const int most = max(part.least, static_cast<int>(one) + 1);
    if (!__any(longest > most)) return 0x7fffffff;  // nothing is split
    if (part.cuts == 1 || 2 * most < 3 * part.least) return most;
    int count[kCutCount] = {}, places[kCutCount] = {}, top[kCutCount] = {};
    for (int base = 0; base < p.requests; base += 64) {
        Extent e = e0;
        if (base) e = base + lane < p.requests ? extent(p, part, base + lane) : Extent{0, 0};
#pragma unroll
        for (int k = 0; k < kCutCount; ++k) {
            const int c = max(part.least, static_cast<int>(one / kCuts[k]) + 1);
            const int splits = max(1, (e.steps + c - 1) / c);
            count[k] += __builtin_amdgcn_readlane(wave_prefix(e.tiles * splits), 63);
            places[k] += __builtin_amdgcn_readlane(wave_prefix(splits > 1 ? e.tiles * splits : 0), 63);
            top[k] = max(top[k], __builtin_amdgcn_readlane(wave_top((e.steps + splits - 1) / splits), 63));
        }
    }
    int best = most;
    float least_cost = __builtin_inff();
#pragma unroll
    for (int k = 0; k < kCutCount; ++k) {
        const float rounds = ceilf(static_cast<float>(count[k]) / shares);
        const float cost = rounds * (static_cast<float>(top[k]) + kStartSteps) + static_cast<float>(places[k]) * p.heads / kPartsAStep;
        if (cost < least_cost) {
            least_cost = cost;
            best = max(part.least, static_cast<int>(one / kCuts[k]) + 1);
        }
    }
    return __builtin_amdgcn_readfirstlane(best);
}

// Finds workgroup `id`'s share (kById), or the first of split row tile number `id`; false past the last, with
// `count` how many there are. A request's last tile comes first: where causal it has the most to do. Every wave scans all requests, 64 at
// a time.
template <bool kById>
__device__ bool find_share(const CacheAttend& p, const Part& part, int id, Share& out, int& count) {
    const int lane = threadIdx.x & 63;
    Extent e0;
    const int c = steps_a_share(p, part, e0);
    count = 0;
    if (!kById && c == 0x7fffffff) return false;  // nothing to join
    int ids_before = 0, places_before = 0;
    for (int base = 0; base < p.requests; base += 64) {
        Extent e = e0;
        if (base) e = base + lane < p.requests ? extent(p, part, base + lane) : Extent{0, 0};
        const int splits = e.steps > c ? (e.steps + c - 1) / c : 1;
        const int places = wave_prefix(splits > 1 ? e.tiles * splits : 0);
        const int ids = wave_prefix(kById ? e.tiles * splits : splits > 1 ? e.tiles : 0);
        const uint64_t past = __ballot(ids_before + ids > id);
        if (past) {
            const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
            const int n = __builtin_amdgcn_readlane(splits, at), t = __builtin_amdgcn_readlane(e.tiles, at);
            const int from = id - ids_before - __builtin_amdgcn_readlane(ids, at) + (kById ? t * n : t);
            const int tile = kById ? from / n : from;
            const int first = places_before + __builtin_amdgcn_readlane(places, at) - (n > 1 ? t * n : 0);
            out = {base + at, t - 1 - tile, kById ? from % n : 0, n, first + tile * n};
            return true;
        }
        ids_before += __builtin_amdgcn_readlane(ids, 63);
        places_before += __builtin_amdgcn_readlane(places, 63);
    }
    count = ids_before;
    return false;
}

// The few rows' work, shared out to the step: the steps of all row tiles, one tile after another, are cut
// into equal runs of c = max(least, N / shares), one a workgroup, wherever the cuts fall. A workgroup
// then takes the end of one tile, whole tiles and the beginning of another, and leaves sums to be joined for
// the first and the last alone: two places each. Where runs of `least` steps are enough workgroups even if
// none of them holds two tiles' steps (`aligned`), none does: the second tile would only wait for the first.
// Positions count units of 1 << shift steps, one but for N past 2^29.
struct Survey {
    Extent first;  // of the lane's request among the first 64
    int c, shift, total;
    bool aligned;
};

__device__ __forceinline__ Extent extent_at(const CacheAttend& p, const Part& part, const Survey& sv, int base) {
    if (base == 0) return sv.first;
    const int r = base + (threadIdx.x & 63);
    return r < p.requests ? extent(p, part, r) : Extent{0, 0};
}

// A row tile's units: at the least one, so that a tile that sees nothing is written too; whole runs where
// they are aligned.
__device__ __forceinline__ int units_of(const Extent& e, const Survey& sv) {
    const int units = max(1, (e.steps + (1 << sv.shift) - 1) >> sv.shift);
    return sv.aligned ? (units + sv.c - 1) / sv.c * sv.c : units;
}

__device__ Survey survey(const CacheAttend& p, const Part& part) {
    const int lane = threadIdx.x & 63;
    Survey sv = {lane < p.requests ? extent(p, part, lane) : Extent{0, 0}, 0, 0, 0, false};
    float work = 0.0f;
    for (int base = 0; base < p.requests; base += 64) {
        const Extent e = extent_at(p, part, sv, base);
        const float sum = wave_prefix(static_cast<float>(e.tiles) * static_cast<float>(max(e.steps, 1)));
        work += __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, sum), 63));
    }
    sv.shift = max(0, static_cast<int>(bits_of(work) >> 23) - 127 - 28);
    sv.c = max(part.least >> sv.shift, 1);
    int runs = 0;
    for (int base = 0; base < p.requests; base += 64) {
        const Extent e = extent_at(p, part, sv, base);
        const int units = units_of(e, sv);
        sv.total += __builtin_amdgcn_readlane(wave_prefix(e.tiles * units), 63);
        runs += __builtin_amdgcn_readlane(wave_prefix(e.tiles * ((units + sv.c - 1) / sv.c)), 63);
    }
    // Without places for parts (no tile can be cut) runs hold whole tiles, however many rows `starts` speaks of.
    sv.aligned = !part.work || runs <= part.shares;
    if (sv.aligned) sv.total = runs * sv.c;
    else sv.c = max(sv.c, (sv.total + part.shares - 1) / part.shares);
    return sv;
}

// A row tile, its units [start, start + units) of all.
struct Item {
    int request, tile, start, units;
};

// The tile that unit `id` is of (kByUnit), or tile number `id`; false past the last.
template <bool kByUnit>
__device__ bool find_item(const CacheAttend& p, const Part& part, const Survey& sv, int id, Item& out) {
    int ids_before = 0, units_before = 0;
    for (int base = 0; base < p.requests; base += 64) {
        const Extent e = extent_at(p, part, sv, base);
        const int one = units_of(e, sv);
        const int units = wave_prefix(e.tiles * one), tiles = wave_prefix(e.tiles);
        const int ids = kByUnit ? units : tiles;
        const uint64_t past = __ballot(ids_before + ids > id);
        if (past) {
            const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
            const int u = __builtin_amdgcn_readlane(one, at), t = __builtin_amdgcn_readlane(e.tiles, at);
            const int from = id - ids_before - __builtin_amdgcn_readlane(ids, at) + (kByUnit ? t * u : t);
            const int tile = kByUnit ? from / u : from;
            out = {base + at, tile, units_before + __builtin_amdgcn_readlane(units, at) - (t - tile) * u, u};
            return true;
        }
        ids_before += __builtin_amdgcn_readlane(ids, 63);
        units_before += __builtin_amdgcn_readlane(units, 63);
    }
    return false;
}

// Rows of the step that no request has (before the first one's and past the last one's) are zeros: the
// workgroups without a share write them, those from number `busy` on. There are `heads` at the least: a launch
// has that many more than it can have shares. They run beside the others: 24 to 216 such rows of 32 heads of 128
// added nothing to 82 us of 40 requests, 984 (8 MB) 3 us, and 4095 beside one request over 131071 tokens 36 us.
__device__ void clear_rest(const CacheAttend& p, int width, int busy) {
    const int64_t row = static_cast<int64_t>(p.q_heads) * width / 8;
    const int64_t before = row_start(p, 0) * row, after = row_start(p, p.requests) * row, count = before + p.tokens * row - after;
    const int64_t stride = static_cast<int64_t>(gridDim.x - busy) * blockDim.x;
    for (int64_t i = static_cast<int64_t>(blockIdx.x - busy) * blockDim.x + threadIdx.x; i < count; i += stride)
        reinterpret_cast<i32x4*>(p.out)[i < before ? i : i - before + after] = i32x4{0, 0, 0, 0};
}

// Where a row tile's tokens lie: steps [begin, end) of the share; rows see tokens from low_least on and
// before high_most, and all of them those in [low_most, high_least).
struct Span {
    int begin, end, low_least, low_most, high_least, high_most;
};

__device__ __forceinline__ Span span_of(const CacheAttend& p, int row0, int rows, const Rows& own, int split = 0, int splits = 1) {
    const int before = own.before, length = own.length, t0 = row0 / p.group, t1 = (rows - 1) / p.group;
    Span s;
    s.low_least = low_of(p, before + t0);
    s.low_most = low_of(p, before + t1);
    s.high_least = p.causal ? before + t0 + 1 : length;
    // Past what the table's row has pages for there is nothing to see, whatever the length says.
    s.high_most = min(p.causal ? before + t1 + 1 : length, p.width << p.shift);
    const int from = s.low_least / kStep, steps = max(0, (s.high_most + kStep - 1) / kStep - from);
    s.begin = from + static_cast<int>(static_cast<int64_t>(steps) * split / splits);
    s.end = from + static_cast<int>(static_cast<int64_t>(steps) * (split + 1) / splits);
    return s;
}

// What a workgroup keeps of a page of its tokens: its number (-1: none of the cache's), the keys'
// scale, log2 and inverse of the values'.
struct PageScales {
    int page;
    float keys, values_log, values_inv;
};

constexpr int kStage = 128;  // steps whose pages a workgroup stages at a time
constexpr int kEntries = kStage * kStep / 16 + 1;

// Stages the pages of steps [from, to) of a request, the first of them number `page_first`.
__device__ __forceinline__ void stage_pages(const CacheAttend& p, PageScales* entries, const int* table, int length, int kv,
                                            int page_first, int to) {
    const int pages = ((to * kStep - 1) >> p.shift) - page_first + 1;
    for (int i = threadIdx.x; i < pages; i += blockDim.x) {
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
}

// The largest magnitude's bits of a query row -> the exponents of the power of two that brings it to
// about 2^12 and of its inverse, both of normal numbers.
__device__ __forceinline__ void row_unit(uint32_t most, float& unit, float& down) {
    const int e = min(max(static_cast<int>(most >> 23) - 12, 10), 240);
    unit = float_of(static_cast<uint32_t>(e) << 23);
    down = float_of(static_cast<uint32_t>(254 - e) << 23);
}

// Eight elements of a query row as float32, and their largest magnitude's bits.
__device__ __forceinline__ void query8(const CacheAttend& p, const uint16_t* x, float* v, uint32_t& most) {
    widen8(*reinterpret_cast<const i32x4*>(x), p.half, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, bits_of(v[i]) & 0x7fffffffu);
}

// ------------------------------------------------------------------------ few rows a request

// Four waves take row tiles of 16 rows (kTiles of them) of one key head, the heads that share it token
// by token, over the workgroup's run of their tokens: each wave every fourth step of 64. Both products
// are taken transposed, Sᵀ = K·Qᵀ and Oᵀ = Vᵀ·Pᵀ, on v_mfma_f32_16x16x32_f16, so that a query row is a
// column of both results: lane l holds column l%16. Score tile j's row m is token 16·(m/4) + 4j + m%4
// of the step, which leaves lane group g = l/16 with the scores of tokens 16g .. 16g+15 in order: all
// of one page (pages are multiples of 16 tokens), one scale each, and exactly the 16 bytes of a channel's
// values that the group loads for the second product. Codes go from memory to registers to the matrix
// unit; nothing of the cache passes through LDS but its pages' numbers and scales, read once a tile.
// A step's keys are loaded over the previous step's second product and its values over its first.
// kOnce: lines of codes are marked as read once, which leaves the caches to what is read again. The rule is the
// page's size alone. Up to 64 tokens a row tile reads every line by one load: one token for each of 40 requests
// 86 -> 75 us, and 0.93 of the time without the mark over requests of up to 32 rows. Of more, each row tile reads
// the lines again, which the mark does not keep: 1.06 of the time without, 89 us for 74 at the worst (8 tokens of 64
// heads over 8 and 100000). The values of a larger page's channel fill a line that two steps share: with the mark
// 53 us became 57 at 131071 tokens.
// Bound by the codes' way from memory: those 40 requests' up to 12001 tokens, 8 heads of 128, are 437 MB in 75 us,
// 5.8 TB/s of the 7.2 that a large read reaches; 131071 tokens of one request, 268 MB, 53 us, 5.1 TB/s, with
// some 5 us before the first codes arrive (the requests' survey, the pages' numbers and scales) and after the
// last. 700 tokens of one request are 10.9 us on 8 workgroups of 11 steps: that chain alone.
template <int kWidth, int kTiles, bool kFp8, bool kOnce>
__global__ __launch_bounds__(256, kWidth == 256 ? 1 : 2) void few_kernel(CacheAttend p, Part part, bool clears) {
    constexpr int kWaves = 4, kBlocks = kWidth / 64, kOut = kWidth / 16, kRows = 16 * kTiles;
    __shared__ PageScales entries[kEntries];
    __shared__ float merged[kWaves][16][kWidth + 4];
    __shared__ float tops[kWaves][16], totals[kWaves][16];
    const int thread = threadIdx.x, lane = thread & 63, wave = __builtin_amdgcn_readfirstlane(thread >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int kv = blockIdx.x % p.heads, id = blockIdx.x / p.heads;
    const Survey sv = survey(p, part);
    const int64_t run_begin = static_cast<int64_t>(id) * sv.c;
    if (run_begin >= sv.total) {
        if (clears) clear_rest(p, kWidth, (sv.total + sv.c - 1) / sv.c * p.heads);
        return;
    }
    const int run_from = static_cast<int>(run_begin), run_to = static_cast<int>(min(run_begin + sv.c, static_cast<int64_t>(sv.total)));
    const int within = p.page - 1;
    const uint8_t* k_lane = p.k_codes + static_cast<int64_t>(kv) * p.page * kWidth + (col & 3) * kWidth + 16 * g;
    const uint8_t* v_lane = p.v_codes + static_cast<int64_t>(kv) * p.page * kWidth + col * p.page;
    const int64_t page_bytes = static_cast<int64_t>(p.heads) * p.page * kWidth;

    Item item;
    for (int at = run_from; at < run_to && find_item<true>(p, part, sv, at, item);) {
        const Rows own = rows_of(p, item.request);
        const int first = own.first, length = own.length, rows = own.fresh * p.group;
        const int stop = min(item.start + item.units, run_to);
        const bool split = item.start < run_from || item.start + item.units > run_to;
        const int place = 2 * id + (at != run_from);

        // Tokens [low, high) of each of the lane's rows, none of a row that is not there.
        int low[kTiles], high[kTiles], token[kTiles], head[kTiles];
        i32x4 raw[kTiles][kBlocks][2];
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
            const int row = kRows * item.tile + 16 * n + col;
            const bool live = row < rows;
            token[n] = live ? row / p.group : 0;
            head[n] = kv * p.group + (live ? row - token[n] * p.group : 0);
            const int position = own.before + token[n];
            high[n] = live ? max(p.causal ? position + 1 : length, 0) : 0;
            low[n] = live ? low_of(p, position) : 0;
        }
        // The rows, read before the pages are looked up where there is one tile of them.
        const auto read_rows = [&]() {
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
                const uint16_t* x = p.q + (first + token[n]) * p.q_token + head[n] * p.q_head + 16 * g;
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) {
                    raw[n][b][0] = *reinterpret_cast<const i32x4*>(x + 64 * b);
                    raw[n][b][1] = *reinterpret_cast<const i32x4*>(x + 64 * b + 8);
                }
            }
        };
        if constexpr (kTiles == 1) read_rows();
        const Span span = span_of(p, kRows * item.tile, min(rows, kRows * (item.tile + 1)), own);
        const int base = low_of(p, own.before) / kStep;
        const int begin = max(span.begin, base + ((at - item.start) << sv.shift));
        const int end = stop == item.start + item.units ? span.end : min(span.end, base + ((stop - item.start) << sv.shift));
        const int* table = p.table + static_cast<int64_t>(item.request) * p.width;
        at = stop;

        // Each row brought to a largest magnitude of about 2^12; a lane holds elements 64b + 16g .. + 15 of
        // each block of 64, as two operands.
        f16x8 q[kTiles][kBlocks][2];
        float sharp[kTiles];
        const auto bring_rows = [&]() {
            if constexpr (kTiles > 1) read_rows();
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
                float v[kBlocks][16], unit, down;
                uint32_t most = 0;
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) {
                    widen8(raw[n][b][0], p.half, v[b]);
                    widen8(raw[n][b][1], p.half, v[b] + 8);
#pragma unroll
                    for (int i = 0; i < 16; ++i) most = max(most, bits_of(v[b][i]) & 0x7fffffffu);
                }
                most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 16)));
                most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 32)));
                row_unit(most, unit, down);
                sharp[n] = unit * p.scale * kLog2e;
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) q[n][b][i / 8][i % 8] = static_cast<_Float16>(v[b][i] * down);
                }
            }
        };

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

        i32x4 kc[4][kBlocks], vc[kOut];
        for (int stage = begin; stage < end; stage += kStage) {
            const int stage_end = min(end, stage + kStage);
            const int page_first = stage * kStep >> p.shift;
            if (stage != begin) __syncthreads();
            stage_pages(p, entries, table, length, kv, page_first, stage_end);
            if (stage == begin) bring_rows();
            __syncthreads();
            const auto load_keys = [&](int step) {
                const int t = step * kStep + 16 * (col >> 2);
                const int page = max(entries[(t >> p.shift) - page_first].page, 0);
                const uint8_t* k = k_lane + page * page_bytes + static_cast<int64_t>(t & within) * kWidth;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
#pragma unroll
                    for (int b = 0; b < kBlocks; ++b) kc[j][b] = codes16<kOnce>(k + 4 * j * kWidth + 64 * b);
                }
            };
            const auto load_values = [&](int step) {
                const int t = step * kStep + 16 * g;
                const int page = max(entries[(t >> p.shift) - page_first].page, 0);
                const uint8_t* v = v_lane + page * page_bytes + (t & within);
#pragma unroll
                for (int o = 0; o < kOut; ++o) vc[o] = codes16<kOnce>(v + 16 * o * p.page);
            };
            int step = stage + wave;
            if (step < stage_end) {
                load_keys(step);
                load_values(step);
            }
            for (; step < stage_end; step += kWaves) {
                const int t0 = step * kStep, mine = t0 + 16 * g;
                const PageScales page = entries[(mine >> p.shift) - page_first];
                const bool whole = t0 >= span.low_most && t0 + kStep <= span.high_least && __all(page.page >= 0);
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
                    }
                    if (!whole) {
                        rarely();
                        const uint32_t seen = page.page < 0 ? 0 : high[n] - low[n];
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            if (static_cast<uint32_t>(mine + i - low[n]) >= seen) x[i] = -__builtin_inff();
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) most = fmaxf(most, x[i]);
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
                    rarely();
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
            const int row0 = kRows * item.tile + 16 * n, count = min(16, rows - row0);
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
                if (!split) {
                    const int t = (row0 + r) / p.group, h = kv * p.group + (row0 + r) - t * p.group;
                    store_row(p, first + t, h, kWidth, d, v, sum);
                } else {
                    float* to = part.work + ((static_cast<int64_t>(place) * p.heads + kv) * kRows + 16 * n + r) * (kWidth + 4);
                    *reinterpret_cast<f32x4*>(to + d) = v;
                    if (d == 0) {
                        to[kWidth] = best;
                        to[kWidth + 1] = sum;
                    }
                }
            }
        }
        if (at < run_to) __syncthreads();
    }
}

// ----------------------------------------------------------------------- many rows a request

// A step's keys and values as f16 in LDS, in 16-byte chunks whose place in a row is exclusive-or'ed with
// the row's number, so that the eight rows that a read of 128 bytes takes lie in different banks.
// Row m of a half's 32 keys holds token π(m), m with bits 2 and 3 exchanged.
__device__ __forceinline__ int exchanged(int m) { return (m & ~12) | ((m & 4) << 1) | ((m & 8) >> 1); }

// kWaves waves take a tile of 32 rows each of one key head, and the workgroup's share of its tokens 64 at
// a time: codes become f16 once for all of them, on their way through registers into LDS, a step ahead of
// their use. Products as in few_kernel, on v_mfma_f32_32x32x16_f16: lane l holds row l%32, and with row m of
// the keys at token π(m), score register 8a + e of half h = l/32 is that of token 16a + 8h + e, in the order
// that the second product reads its weights in. Bytes past the request's tokens and pages that the cache has
// not become zeros on the way to LDS.
// Bound by no unit alone: 14003 tokens of two requests, 32 heads of 128 over 8, are 857 GFLOP in 0.93 to 1.05 ms
// as the clock allows, 0.82 to 0.92 PFLOP/s where a large f16 product reaches 1.51; of a SIMD's cycles the
// matrix unit is busy in 42%, the vector unit in 54% (a fifth in both at once), of a CU's the LDS in 43%.
// Without the exponentials it was 6% faster, without the conversions 9%, without loads 3%. At width 64 (2311
// tokens of 12 requests, 16 heads over 4, a window of 4096: 30 GFLOP in 74 us) a score costs the vector unit
// as much for half the products: VALU 47%, matrix unit 20%.
template <int kWidth, int kWaves, bool kFp8>
__global__ __launch_bounds__(64 * kWaves, kWidth == 256 ? 1 : 2) void many_kernel(CacheAttend p, Part part, bool clears) {
    constexpr int kRows = 32 * kWaves, kThreads = 64 * kWaves, kOut = kWidth / 32, kDepth = kWidth / 16;
    constexpr int kBytes = kStep * kWidth * 2, kChunks = kStep * kWidth / 16 / kThreads, kSwizzle = kWidth == 64 ? 7 : 15;
    constexpr bool kLate = kWaves == 8;
    __shared__ PageScales entries[kEntries];
    __shared__ __attribute__((aligned(16))) uint8_t keys[2][kBytes], values[kLate ? 3 : 2][kBytes];
    const int thread = threadIdx.x, lane = thread & 63, wave = __builtin_amdgcn_readfirstlane(thread >> 6);
    const int col = lane & 31, h = lane >> 5;
    const int kv = blockIdx.x % p.heads, id = blockIdx.x / p.heads;
    Share share;
    int shares;
    if (!find_share<true>(p, part, id, share, shares)) {
        if (clears) clear_rest(p, kWidth, shares * p.heads);
        return;
    }
    const Rows of = rows_of(p, share.request);
    const int first = of.first, length = of.length, rows = of.fresh * p.group;
    const int row0 = kRows * share.tile, mine0 = row0 + 32 * wave, row = mine0 + col;
    const Span span = span_of(p, row0, min(rows, row0 + kRows), of, share.split, share.splits);
    // The wave's own rows; one without rows only helps to load.
    const bool busy = mine0 < rows;
    const Span own = span_of(p, busy ? mine0 : 0, min(rows, mine0 + 32), of);
    const bool live = row < rows;
    const int token = live ? row / p.group : 0, head = kv * p.group + (live ? row - token * p.group : 0);
    const int position = of.before + token;
    const int high = live ? max(p.causal ? position + 1 : length, 0) : 0;
    const int low = live ? low_of(p, position) : 0;

    f16x8 q[kDepth];
    float sharp;
    {
        const uint16_t* x = p.q + (first + token) * p.q_token + head * p.q_head + 8 * h;
        float unit, down;
        uint32_t most = 0;
        float v[kDepth][8];
#pragma unroll
        for (int b = 0; b < kDepth; ++b) query8(p, x + 16 * b, v[b], most);
        most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 32)));
        row_unit(most, unit, down);
        sharp = unit * p.scale * kLog2e;
#pragma unroll
        for (int b = 0; b < kDepth; ++b) {
#pragma unroll
            for (int i = 0; i < 8; ++i) q[b][i] = static_cast<_Float16>(v[b][i] * down);
        }
    }

    f32x16 acc[kOut];
#pragma unroll
    for (int o = 0; o < kOut; ++o) {
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[o][i] = 0.0f;
    }
    float ref = 0.0f, bound = -__builtin_inff(), total = 0.0f;
    const int* table = p.table + static_cast<int64_t>(share.request) * p.width;
    const int within = p.page - 1;
    const int64_t page_bytes = static_cast<int64_t>(p.heads) * p.page * kWidth;
    const uint8_t* k_head = p.k_codes + static_cast<int64_t>(kv) * p.page * kWidth;
    const uint8_t* v_head = p.v_codes + static_cast<int64_t>(kv) * p.page * kWidth;

    // Chunk c of a step's codes: 16 channels of token c / (width/16); 16 tokens of channel c / 4.
    i32x4 kc[kChunks], vc[kChunks];
    int page_first = 0, kept[kChunks];
    uint32_t k_to[kChunks][2], v_to[kChunks][2];
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
        const int c = thread + i * kThreads, t = c / (kWidth / 16), x = c % (kWidth / 16), d = c / 4;
        const int m = (t & 32) | exchanged(t & 31);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            k_to[i][j] = m * (2 * kWidth) + 16 * ((2 * x + j) ^ (m & kSwizzle));
            v_to[i][j] = d * (2 * kStep) + 16 * ((2 * (c & 3) + j) ^ (d & 7));
        }
    }
    const auto load_keys = [&](int step) {
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const int c = thread + i * kThreads, t = step * kStep + c / (kWidth / 16);
            const int page = max(entries[(t >> p.shift) - page_first].page, 0);
            kc[i] = *reinterpret_cast<const i32x4*>(k_head + page * page_bytes + (t & within) * kWidth + 16 * (c % (kWidth / 16)));
        }
    };
    const auto load_values = [&](int step) {
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const int c = thread + i * kThreads, t = step * kStep + 16 * (c & 3);
            const int page = entries[(t >> p.shift) - page_first].page;
            kept[i] = page < 0 ? 0 : length - t;
            vc[i] = *reinterpret_cast<const i32x4*>(v_head + max(page, 0) * page_bytes + (c / 4) * p.page + (t & within));
        }
    };
    // The tiles of values that the step before, this one and the next have.
    int v_before = kLate ? 2 * kBytes : kBytes, v_now = 0, v_next = kBytes;
    uint8_t* const values_at = &values[0][0];
    // Chunk i of a step's codes, as f16, to its places in LDS.
    const auto put_keys = [&](int step, int i) {
        *reinterpret_cast<f16x8*>(&keys[step & 1][k_to[i][0]]) = codes8<kFp8>(kc[i][0], kc[i][1]);
        *reinterpret_cast<f16x8*>(&keys[step & 1][k_to[i][1]]) = codes8<kFp8>(kc[i][2], kc[i][3]);
    };
    const auto put_values = [&](int tile, int i) {
        *reinterpret_cast<f16x8*>(values_at + tile + v_to[i][0]) = codes8<kFp8>(vc[i][0], vc[i][1]);
        *reinterpret_cast<f16x8*>(values_at + tile + v_to[i][1]) = codes8<kFp8>(vc[i][2], vc[i][3]);
    };
    // Where a step's values hold tokens past the request's or of pages that the cache has not, zeros in their
    // place, over what was put there.
    const auto cut_values = [&](int tile) {
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            if (__any(kept[i] < 16)) {
                rarely();
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int n = kept[i] - 4 * j;
                    vc[i][j] &= n >= 4 ? -1 : n <= 0 ? 0 : (1 << (8 * n)) - 1;
                }
                put_values(tile, i);
            }
        }
    };
    // The matrix unit's operands in LDS: elements 16b + 8h .. of the keys of a half's row, tokens 16a + 8h ..
    // of the values of 32 channels.
    const auto key_chunk = [&](int step, int b, int half) {
        return *reinterpret_cast<const f16x8*>(&keys[step & 1][(32 * half + col) * (2 * kWidth) + 16 * ((2 * b + h) ^ (col & kSwizzle))]);
    };
    const auto value_chunk = [&](int tile, int a, int o) {
        return *reinterpret_cast<const f16x8*>(values_at + tile + ((32 * o + col) * (2 * kStep) + 16 * ((2 * a + h) ^ (col & 7))));
    };
    // The scores of a step whose keys are in LDS, as they leave the matrix unit.
    f32x16 s[2];
    constexpr int kScores = 2 * kDepth, kSums = 4 * kOut, kAhead = 4;

    f16x8 w[4];
    // A step's weights times its values, `beside` done with the last products, a chunk each.
    const auto add_values = [&](int tile, auto beside) {
        f16x8 ring[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) ring[j] = value_chunk(tile, j / kOut, j % kOut);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < kSums; ++j) {
            acc[j % kOut] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ring[j % kAhead], w[j / kOut], acc[j % kOut], 0, 0, 0);
            if (j + kAhead < kSums) ring[j % kAhead] = value_chunk(tile, (j + kAhead) / kOut, (j + kAhead) % kOut);
            if (j >= kSums - kChunks) beside(j - (kSums - kChunks));
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // Half of the waves, one on each SIMD, are half a step behind: they multiply a step's values after the
    // barrier, while the others are at the exponentials, so that the two waves of a SIMD want the matrix
    // unit and the vector unit in turn.
    const bool late = kLate && wave >= kWaves / 2;

    for (int stage = span.begin; stage < span.end; stage += kStage) {
        const int stage_end = min(span.end, stage + kStage);
        page_first = stage * kStep >> p.shift;
        if (stage != span.begin) __syncthreads();
        stage_pages(p, entries, table, length, kv, page_first, stage_end);
        __syncthreads();
        load_keys(stage);
        load_values(stage);
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            put_keys(stage, i);
            put_values(v_now, i);
        }
        cut_values(v_now);
        if (stage + 1 < stage_end) {
            load_keys(stage + 1);
#pragma unroll
            for (int i = 0; i < kChunks; ++i) put_keys(stage + 1, i);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 16; ++i) s[0][i] = s[1][i] = 0.0f;
#pragma unroll
        for (int j = 0; j < kScores; ++j)
            s[j % 2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(key_chunk(stage, j / 2, j % 2), q[j / 2], s[j % 2], 0, 0, 0);
        for (int step = stage; step < stage_end; ++step) {
            if (step + 2 < stage_end) load_keys(step + 2);
            if (step + 1 < stage_end) load_values(step + 1);
            if (busy) {
                if (late && step > stage) add_values(v_before, [](int) {});
                const int t0 = step * kStep;
                PageScales page[4];
#pragma unroll
                for (int a = 0; a < 4; ++a) page[a] = entries[((t0 + 16 * a) >> p.shift) - page_first];
                const bool whole = t0 >= own.low_most && t0 + kStep <= own.high_least && page[0].page >= 0 &&
                                   page[1].page >= 0 && page[2].page >= 0 && page[3].page >= 0;
                float most = -__builtin_inff();
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                    const float mul = sharp * page[a].keys, add = page[a].values_log - ref;
#pragma unroll
                    for (int e = 0; e < 8; ++e) s[a / 2][8 * (a & 1) + e] = __builtin_fmaf(s[a / 2][8 * (a & 1) + e], mul, add);
                }
                if (!whole) {
                    rarely();
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const uint32_t seen = page[i / 8].page < 0 ? 0 : high - low;
                        if (static_cast<uint32_t>(t0 + 16 * (i / 8) + 8 * h + i % 8 - low) >= seen) s[i / 16][i % 16] = -__builtin_inff();
                    }
                }
#pragma unroll
                for (int i = 0; i < 32; ++i) most = fmaxf(most, s[i / 16][i % 16]);
                if (__any(most > bound)) {
                    most = fmaxf(most, __shfl_xor(most, 32));
                    const float up = most > bound ? most - kLift : 0.0f;
                    const float shrink = bound > 0.0f ? __builtin_amdgcn_exp2f(-up) : 0.0f;
                    if (most > bound) bound = 15.0f;
                    ref += up;
                    total *= shrink;
#pragma unroll
                    for (int i = 0; i < 32; ++i) s[i / 16][i % 16] -= up;
#pragma unroll
                    for (int o = 0; o < kOut; ++o) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) acc[o][i] *= shrink;
                    }
                }
                // The next step's scores on the matrix unit over this one's exponentials. Each operand is read
                // from LDS kAhead products before its own, and the order written here is kept. Past the stage's
                // last step the scores are of whatever the tile holds, and not used.
                f16x8 ring[kAhead];
                f32x16 next[2];
                const auto key_operand = [&](int j) { return key_chunk(step + 1, j / 2, j % 2); };
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i) next[0][i] = next[1][i] = 0.0f;
#pragma unroll
                for (int j = 0; j < kAhead; ++j) ring[j] = key_operand(j);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int j = 0; j < kScores; ++j) {
                    next[j % 2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ring[j % kAhead], q[j / 2], next[j % 2], 0, 0, 0);
                    if (j + kAhead < kScores) ring[j % kAhead] = key_operand(j + kAhead);
#pragma unroll
                    for (int i = 32 / kScores * j; i < 32 / kScores * (j + 1); ++i) {
                        const float x = __builtin_amdgcn_exp2f(s[i / 16][i % 16]);
                        sum = i % 8 ? sum + x : x;
                        w[i / 8][i % 8] = static_cast<_Float16>(x);
                        // A group whose tokens the row does not see adds nothing, whatever its page's scale is.
                        if (i % 8 == 7) total += sum == 0.0f ? 0.0f : sum * page[i / 8].values_inv;
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (!late) {
                    add_values(v_now, [&](int i) {
                        put_keys(step + 2, i);
                        put_values(v_next, i);
                    });
                }
                s[0] = next[0];
                s[1] = next[1];
            }
            if (!busy || late) {
#pragma unroll
                for (int i = 0; i < kChunks; ++i) {
                    put_keys(step + 2, i);
                    put_values(v_next, i);
                }
            }
            cut_values(v_next);
            __syncthreads();
            const int freed = kLate ? v_before : v_now;
            v_before = v_now;
            v_now = v_next;
            v_next = freed;
        }
        if (busy && late) add_values(v_before, [](int) {});
    }

    if (!live) return;
    total += __shfl_xor(total, 32);
    float* to = share.splits == 1 ? nullptr : part.work + ((static_cast<int64_t>(share.place + share.split) * p.heads + kv) * kRows + 32 * wave + col) * (kWidth + 4);
#pragma unroll
    for (int o = 0; o < kOut; ++o) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4 v = {acc[o][4 * i], acc[o][4 * i + 1], acc[o][4 * i + 2], acc[o][4 * i + 3]};
            const int d = 32 * o + 8 * i + 4 * h;
            if (to) *reinterpret_cast<f32x4*>(to + d) = v;
            else store_row(p, first + token, head, kWidth, d, v, total);
        }
    }
    if (to && h == 0) {
        to[kWidth] = bound > 0.0f ? ref : kNoScore;
        to[kWidth + 1] = total;
    }
}

// ------------------------------------------------------------------------------------- join

// Where a row's parts stand: the first, and the others `next` apart.
struct Parts {
    const float *first, *others;
    int64_t next;
    int count;
    __device__ const float* operator[](int s) const { return s == 0 ? first : others + s * next; }
};

// A row's parts from `slice` on, every `slices`-th, brought to `best` and added up: four elements.
__device__ __forceinline__ void add_parts(const Parts& parts, int slice, int slices, int width, int quad, float best, f32x4& v, float& sum) {
    v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    sum = 0.0f;
#pragma unroll 8
    for (int s = slice; s < parts.count; s += slices) {
        const float* one = parts[s];
        const f32x4 x = *reinterpret_cast<const f32x4*>(one + 4 * quad);
        const float factor = __builtin_amdgcn_exp2f(one[width] - best);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = __builtin_fmaf(x[j], factor, v[j]);
        sum = __builtin_fmaf(one[width + 1], factor, sum);
    }
}

// The same of all of a row's parts, four of them read at a time, their references with them.
__device__ __forceinline__ void add_all(const Parts& parts, int width, int quad, f32x4& v, float& sum) {
    v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    sum = 0.0f;
    float best = kNoScore;
    for (int from = 0; from < parts.count; from += 4) {
        f32x4 x[4];
        float top[4], one[4], most = best;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float* part = parts[min(from + i, parts.count - 1)];
            x[i] = *reinterpret_cast<const f32x4*>(part + 4 * quad);
            top[i] = part[width];
            one[i] = part[width + 1];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) most = nan_max(most, top[i]);
        const float shrink = __builtin_amdgcn_exp2f(best - most);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] *= shrink;
        sum *= shrink;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float factor = from + i < parts.count ? __builtin_amdgcn_exp2f(top[i] - most) : 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = __builtin_fmaf(x[i][j], factor, v[j]);
            sum = __builtin_fmaf(one[i], factor, sum);
        }
        best = most;
    }
}

// Joins the parts of the row tiles that several workgroups took, all of a row's parts brought to their
// largest reference; blockIdx.y says of which launch. few_kernel's rows are few and their parts many: a
// workgroup a row, kWidth/4 threads a part. many_kernel's rows are many and their parts few: kWidth/4
// threads a row, its parts one after another. Which thread sums which parts is fixed: a call's result does
// not vary. Bound by latency, of the survey and two trips to memory: one row of 32 heads for each of 40 requests
// 6.5 us (1.9 MB), 64 rows of 64 parts 7.7 us, the parts of 2311 tokens at width 64 10.2 us (22 MB).
template <int kWidth>
__global__ __launch_bounds__(256) void join_kernel(CacheAttend p, Part few, Part many, int few_rows, int many_rows, int few_items, int many_items) {
    constexpr int kQuads = kWidth / 4, kParts = 256 / kQuads;
    __shared__ f32x4 sums[kParts][kQuads];
    __shared__ float totals[kParts];
    const int thread = threadIdx.x, slice = thread / kQuads, quad = thread % kQuads;
    const bool wide = blockIdx.y != 0;
    const Part part = wide ? many : few;
    const int rows_all = 1 << part.shift, groups = wide ? many_rows : few_rows;
    const int items = wide ? many_items : few_items;
    const int64_t row_floats = kWidth + 4, place_floats = static_cast<int64_t>(p.heads) * rows_all * row_floats;
    if (blockIdx.x >= items) return;
    Survey sv;
    if (!wide) {
        sv = survey(p, part);
        if (sv.total <= sv.c) return;  // one run takes it all
    }
    for (int number = blockIdx.x; number < items; number += gridDim.x) {
        const int kv = number % p.heads, group = number / p.heads % groups, id = number / (p.heads * groups);
        int request, tile;
        Parts parts;
        if (wide) {
            Share share;
            int count;
            if (!find_share<false>(p, part, id, share, count)) return;
            request = share.request;
            tile = share.tile;
            parts = {part.work + share.place * place_floats, part.work + share.place * place_floats, place_floats, share.splits};
        } else {
            Item item;
            if (!find_item<false>(p, part, sv, id, item)) return;
            request = item.request;
            tile = item.tile;
            const int run = item.start / sv.c, last = (item.start + item.units - 1) / sv.c;
            parts = {part.work + (2 * run + (item.start != run * sv.c)) * place_floats, part.work + 2 * run * place_floats,
                     2 * place_floats, last - run + 1};
        }
        if (parts.count == 1) continue;
        const Rows own = rows_of(p, request);
        const int first = own.first, rows = own.fresh * p.group;
        const int row0 = tile << part.shift, count = min(rows_all, rows - row0);
        for (int r = wide ? group * kParts + slice : group; r < count; r += wide ? groups * kParts : groups) {
            const int64_t at = (static_cast<int64_t>(kv) * rows_all + r) * row_floats;
            const Parts row = {parts.first + at, parts.others + at, parts.next, parts.count};
            float best = kNoScore, sum;
            f32x4 v;
            if (wide) {
                add_all(row, kWidth, quad, v, sum);
            } else {
                for (int s = thread & 63; s < row.count; s += 64) best = nan_max(best, row[s][kWidth]);
                best = wave_max_nan(best);
                add_parts(row, slice, kParts, kWidth, quad, best, v, sum);
                __syncthreads();
                sums[slice][quad] = v;
                if (quad == 0) totals[slice] = sum;
                __syncthreads();
                if (slice == 0) {
#pragma unroll
                    for (int s = 1; s < kParts; ++s) {
                        v += sums[s][quad];
                        sum += totals[s];
                    }
                }
            }
            if (wide || slice == 0) {
                const int t = (row0 + r) / p.group, h = kv * p.group + (row0 + r) - t * p.group;
                store_row(p, first + t, h, kWidth, 4 * quad, v, sum);
            }
        }
    }
}

// ----------------------------------------------------------------------------------- launch

// One of a call's launches: its row tiles' rows, their number at the most, and where its places begin.
struct Launch {
    bool on;
    int rows, over, upto, shares, least, row_groups, cuts;
    int64_t tiles, offset;
};

// Workgroups that a launch's steps are cut into, at the most.
int most_shares(const Launch& l) { return l.cuts == 1 ? l.shares : kMostCut * l.shares; }

// Eight waves share a step's tiles; at width 64 those are too small for so many, at 256 a wave takes 512
// registers.
constexpr int many_waves(int width) { return width == 128 ? 8 : 4; }

struct AttendShape {
    Launch few, many;
    bool splits;
    int64_t floats;
};

constexpr int kFewShares = 512;   // few_kernel's workgroups over all heads: two a CU
constexpr int kFewSteps = 8;      // of which each takes so many steps at the least,
constexpr int kWholeSteps = 16;   // but a whole tile where none can have more than these: no join then
constexpr int kManySteps = 16;    // many_kernel's, whose parts are larger
constexpr int kCutSteps = 64;     // with more, and a CU to a workgroup, many_kernel chooses among kCuts
constexpr int64_t kJoinGroups = 1024;  // join_kernel's workgroups for each of the two launches
constexpr int kFewRows = 64;      // up to here a request's rows are few_kernel's alone,
constexpr int kFewWork = 24000;   // and so are all, up to so much work (`few_work`): one launch less
constexpr int kBesideRows = 16;   // up to here they are few_kernel's beside requests of more,
constexpr int kManyRows = 1024;   // unless so many a request on average leave few such requests

// What the few rows' kernel has to do, in rows of a key head: twice as much at width 256, where a CU holds one
// workgroup and not two; where tiles are split, times the root of a row's steps (at the most kLongSteps, as a
// table may be much wider than the requests are long), since the many rows' kernel then costs its join and parts first
// and codes made f16 once for 256 rows later. Timed over 755 steps of 125 to 12000 rows, up to 20000 tokens held, 1
// to 30 requests and six head layouts (int8, bf16, pages of 64), it takes 1.012 of the faster side's time (geometric
// mean; a limit of 1024 rows for all 1.112) and more than 1.25 of it in ten, seven of them at width 256, where the
// mean is 1.031: at the worst 76 us for 43, 1024 rows of 12 requests over 2500, and 117 for 69, 400 of one over
// 20000. Few / many rows' kernel, us, 32 heads over 8 of width 128: 100 tokens over 300
// 14 / 23, over 2500 41 / 43, over 7000 55 / 50, over 20000 101 / 68; 256 over 7000 86 / 60; 500 over 300 24 / 35, over
// 7000 159 / 92; 1750 tokens of 8 requests over 200 54 / 31; 16 heads over 2 of 256: 128 over 2500 68 / 59, over 300 28 / 34.
constexpr int64_t kLongSteps = 128;
float few_work(int64_t all_rows, int heads, int width, int64_t steps) {
    const float rows = static_cast<float>(all_rows) * static_cast<float>(heads) * (width == 256 ? 2.0f : 1.0f);
    return steps > kWholeSteps ? rows * sqrtf(static_cast<float>(min(steps, kLongSteps))) : rows;
}

// The shape of a call, which its workspace goes by too. Where a request may have more than kFewRows
// rows, those of more than kBesideRows go to many_kernel and the others, if there are others, to few_kernel.
// (With kManyRows at 256 the chunks of 2311 tokens among 12 requests took 99 us for 87, as their single tokens then
// run a wave a workgroup.)
AttendShape shape_of(int64_t tokens, int group, int requests, int heads, int columns, int page, int width, int64_t most, int window) {
    const int64_t rows = (most > 0 && most < tokens ? most : tokens) * group;
    const int all = 0x7fffffff;
    AttendShape a = {};
    const int64_t all_rows = tokens * group;
    const int64_t steps = (static_cast<int64_t>(columns) * page + kStep - 1) / kStep;  // of a tile, at the most
    const int64_t seen = window > 0 ? min(steps, static_cast<int64_t>(window) / kStep + 2) : steps;  // by a row, about
    a.many.on = rows > kFewRows && few_work(all_rows, heads, width, seen) > kFewWork;
    a.few.on = !a.many.on || (requests > 1 && all_rows < kManyRows * requests);
    a.few.rows = rows > 16 && !a.many.on ? 32 : 16;
    a.few.upto = a.many.on ? kBesideRows : all;
    a.few.tiles = a.many.on ? requests : (tokens * group + a.few.rows - 1) / a.few.rows + requests - 1;
    if (steps <= kWholeSteps) {
        a.few.least = kWholeSteps;
        a.few.shares = static_cast<int>(a.few.tiles);
    } else {  // no more workgroups than the runs that there can be
        const int64_t runs = min(a.few.tiles, requests * ((rows + a.few.rows - 1) / a.few.rows)) * ((steps + kFewSteps - 1) / kFewSteps);
        a.few.least = kFewSteps;
        a.few.shares = static_cast<int>(min(runs, static_cast<int64_t>(max(1, kFewShares / heads))));
    }
    a.few.row_groups = static_cast<int>(rows < a.few.rows ? rows : a.few.rows);
    a.many.rows = 32 * many_waves(width);
    a.many.over = a.few.on ? kBesideRows : 0;
    a.many.upto = all;
    a.many.least = kManySteps;
    a.many.shares = max(1, (width == 64 ? 512 : 256) / heads);
    a.many.cuts = width > 64 && steps > kCutSteps ? kCutCount : 1;
    a.many.tiles = (tokens * group + a.many.rows - 1) / a.many.rows + requests - 1;
    a.splits = steps > kWholeSteps;
    if (a.splits) {
        if (a.few.on) a.floats += 2ll * a.few.shares * heads * a.few.rows * (width + 4);
        a.many.offset = a.floats;
        if (a.many.on) a.floats += 2ll * most_shares(a.many) * heads * a.many.rows * (width + 4);
    }
    return a;
}

int log2_of(int n) { return n > 1 ? 1 + log2_of(n / 2) : 0; }

Part part_of(const CacheAttend& p, const AttendShape& a, const Launch& l) {
    return {l.over, l.upto, l.shares, l.least, log2_of(l.rows), a.splits ? p.work + l.offset : nullptr, l.cuts};
}

template <int kWidth, bool kFp8>
hipError_t attend(const CacheAttend& p, const AttendShape& a, hipStream_t s) {
    const Part few = part_of(p, a, a.few), many = part_of(p, a, a.many);
    if (a.many.on) {
        constexpr int kWaves = many_waves(kWidth);
        const unsigned groups = static_cast<unsigned>((most_shares(a.many) + a.many.tiles + 1) * p.heads);
        many_kernel<kWidth, kWaves, kFp8><<<groups, 64 * kWaves, 0, s>>>(p, many, true);
    }
    if (a.few.on) {
        const unsigned groups = static_cast<unsigned>((a.few.shares + 1) * p.heads);
        const bool once = p.page <= 64;
        const auto kernel = a.few.rows == 16 ? (once ? few_kernel<kWidth, 1, kFp8, true> : few_kernel<kWidth, 1, kFp8, false>)
                                             : (once ? few_kernel<kWidth, 2, kFp8, true> : few_kernel<kWidth, 2, kFp8, false>);
        kernel<<<groups, 256, 0, s>>>(p, few, !a.many.on);
    }
    if (a.splits) {
        const int64_t most = 0x7fffffff, one = 1;
        const int64_t few_items = a.few.on ? min(most, a.few.tiles * p.heads * a.few.row_groups) : 0;
        // A split tile has more steps than a share, so that there are no more of them than shares; and no more
        // groups of rows than workgroups, as each looks its tile up.
        const int64_t tiles = a.many.on ? min(a.many.tiles, static_cast<int64_t>(most_shares(a.many))) * p.heads : 0;
        const int64_t row_groups = max(one, min(kJoinGroups / max(tiles, one), static_cast<int64_t>(a.many.rows * kWidth / 1024)));
        const int64_t many_items = tiles * row_groups;
        const unsigned groups = static_cast<unsigned>(min(max(few_items, many_items), kJoinGroups));
        join_kernel<kWidth><<<dim3(groups, a.many.on ? 2 : 1), 256, 0, s>>>(
            p, few, many, a.few.row_groups, static_cast<int>(row_groups), static_cast<int>(few_items), static_cast<int>(many_items));
    }
    return hipGetLastError();
}

template <bool kFp8>
hipError_t attend(const CacheAttend& p, const AttendShape& a, hipStream_t s) {
    if (p.head_width == 64) return attend<64, kFp8>(p, a, s);
    if (p.head_width == 128) return attend<128, kFp8>(p, a, s);
    return attend<256, kFp8>(p, a, s);
}

}  // namespace

int64_t cache_attend_work(int64_t tokens, int group, int requests, int heads, int columns, int page, int width, int64_t most, int window) {
    return 4 * shape_of(tokens, group, requests, heads, columns, page, width, most, window).floats;
}

hipError_t cache_attend(const CacheAttend& p, int64_t most, bool fp8, hipStream_t s) {
    const AttendShape a = shape_of(p.tokens, p.group, p.requests, p.heads, p.width, p.page, p.head_width, most, p.window);
    return fp8 ? attend<true>(p, a, s) : attend<false>(p, a, s);
}

}  // namespace cozyq
