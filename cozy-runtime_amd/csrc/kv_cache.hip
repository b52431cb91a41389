// The paged cache of keys and values in 8 bits: the step's plan (pages, slots and positions from the
// requests' lengths), the write of new tokens into their pages, and pages read back.
//
// A page holds `page` tokens of every key head. Keys stand as [pages, heads, page, width] and values
// transposed, as [pages, heads, width, page]: each is then the operand that attention's matrix
// instructions read 16 bytes at a time, without a transpose on the way. One float32 scale a page and
// head, for keys and for values: value = code · scale.
#include <hip/hip_runtime.h>

#include "common.h"
#include "kernels.h"
#include "sixteen.h"

namespace cozyq {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

// ------------------------------------------------------------------------------------ plan

// min(a + b, top) for a, b <= top < 2^30: a sum that saturates, so that no request's count can
// carry the prefix past the step's rows.
__device__ __forceinline__ int capped(int a, int b, int top) {
    const int sum = a + b;
    return sum < top ? sum : top;
}

// In place, the exclusive prefix sums of v[0, n) in shared memory, the whole sum in v[n]; sums
// saturate at `top`. Called by the whole workgroup.
__device__ void prefix(int* v, int n, int top, int* wave_sums) {
    const int per = (n + kThreads - 1) / kThreads;
    const int begin = min(n, per * static_cast<int>(threadIdx.x)), end = min(n, begin + per);
    int mine = 0;
    for (int i = begin; i < end; ++i) mine = capped(mine, v[i], top);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int sum = mine;
    for (int step = 1; step < 64; step *= 2) {
        const int below = __shfl_up(sum, step);
        if (lane >= step) sum = capped(sum, below, top);
    }
    int before = __shfl_up(sum, 1);
    if (lane == 0) before = 0;
    if (lane == 63) wave_sums[wave] = sum;
    __syncthreads();
    for (int w = 0; w < wave; ++w) before = capped(before, wave_sums[w], top);
    for (int i = begin; i < end; ++i) {
        const int x = v[i];
        v[i] = before;
        before = capped(before, x, top);
    }
    if (threadIdx.x == kThreads - 1) v[n] = before;
    __syncthreads();
}

// The last i in [0, n) with v[i] <= x, for ascending v with v[0] = 0 <= x.
__device__ __forceinline__ int find(const int* v, int n, int x) {
    int low = 0, high = n;
    while (high - low > 1) {
        const int mid = (low + high) / 2;
        if (v[mid] <= x) low = mid;
        else high = mid;
    }
    return low;
}

struct PageOf {
    const CachePlan& p;
    const int *starts, *taken;
    int spare;

    // The page of request r's tokens index·page ..: its table's where the request held it already,
    // else popped off the end of the free list; -1 where the list or the table's row has none left.
    __device__ int operator()(int r, int held, int index) const {
        if (index >= p.width) return -1;
        const int have = min((held + p.page - 1) >> p.shift, p.width);
        if (index < have) return p.table[static_cast<int64_t>(r) * p.width + index];
        const int place = taken[r] + index - have;
        return place < spare ? p.free[spare - 1 - place] : -1;
    }
};

// Every workgroup scans all requests' lengths (a few KB from L2) and then takes its share of the
// tokens and of the runs, finding each one's request by bisection of the prefix sums: one launch,
// and nothing passes between workgroups. No entry of the table is both read and written: a page that
// was held is read, one that is new is written.
__global__ __launch_bounds__(kThreads) void plan_kernel(CachePlan p) {
    extern __shared__ int shared[];
    __shared__ int wave_sums[kWaves];
    const int R = p.requests;
    int *starts = shared, *taken = starts + R + 1, *first_run = taken + R + 1, *held_of = first_run + R + 1;
    for (int r = threadIdx.x; r < R; r += kThreads) {
        starts[r] = min(max(p.fresh[r], 0), p.tokens);
        held_of[r] = max(p.held[r], 0);
    }
    __syncthreads();
    prefix(starts, R, p.tokens, wave_sums);
    const int top = (1 << 30) - 1;
    for (int r = threadIdx.x; r < R; r += kThreads) {
        const int held = held_of[r], n = starts[r + 1] - starts[r];
        const int have = (held + p.page - 1) >> p.shift, need = (held + n + p.page - 1) >> p.shift;
        taken[r] = min(need, p.width) - min(have, p.width);
        first_run[r] = n > 0 ? ((held + n - 1) >> p.shift) - (held >> p.shift) + 1 : 0;
    }
    __syncthreads();
    prefix(taken, R, top, wave_sums);
    prefix(first_run, R, top, wave_sums);

    const int spare = min(p.spare[0], p.free_count);
    const PageOf page_of{p, starts, taken, spare};
    const int at = blockIdx.x * kThreads + threadIdx.x, stride = gridDim.x * kThreads;
    for (int t = at; t < p.tokens; t += stride) {
        int request = -1, position = 0, slot = -1;
        if (t < starts[R]) {
            request = find(starts, R + 1, t);
            const int held = held_of[request];
            position = held + t - starts[request];
            const int page = page_of(request, held, position >> p.shift);
            slot = page < 0 ? -1 : (page << p.shift) + (position & (p.page - 1));
        }
        p.requests_out[t] = request;
        p.positions[t] = position;
        p.slots[t] = slot;
    }
    for (int i = at; i < p.runs_most; i += stride) {
        i32x4 run = {0, 0, -1, 0};
        if (i < first_run[R]) {
            const int r = find(first_run, R + 1, i);
            const int held = held_of[r], n = starts[r + 1] - starts[r];
            const int index = (held >> p.shift) + i - first_run[r];
            const int begin = max(held, index << p.shift), end = min(held + n, (index + 1) << p.shift);
            const int page = page_of(r, held, index);
            run = {starts[r] + begin - held, end - begin, page, begin & (p.page - 1)};
            if (index >= (held + p.page - 1) >> p.shift && index < p.width)
                p.table[static_cast<int64_t>(r) * p.width + index] = page;
        }
        *reinterpret_cast<i32x4*>(p.runs + 4 * static_cast<int64_t>(i)) = run;
    }
    for (int r = at; r <= R; r += stride) {
        p.starts[r] = starts[r];
        if (r < R) p.lengths[r] = held_of[r] + starts[r + 1] - starts[r];
    }
    if (blockIdx.x == 0) {
        // Pages wanted and not got: those past the free list's end, and those past a row of the table.
        int past = 0;
        for (int r = threadIdx.x; r < R; r += kThreads) {
            const int held = held_of[r], n = starts[r + 1] - starts[r];
            const int have = min((held + p.page - 1) >> p.shift, p.width);
            past += ((held + n + p.page - 1) >> p.shift) - have;
        }
        for (int step = 1; step < 64; step *= 2) past += __shfl_xor(past, step);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) wave_sums[threadIdx.x >> 6] = past;
        __syncthreads();
        if (threadIdx.x == 0) {
            past = 0;
            for (int w = 0; w < kWaves; ++w) past += wave_sums[w];
            const int got = min(taken[R], max(spare, 0));
            p.spare_out[0] = spare - got;
            p.spare_out[1] = past - got;
        }
    }
}

// ---------------------------------------------------------------------------------- append

// The codes of four values (already over the scale): int8 by rint, E4M3 by the conversion, clamped to the
// format's largest. A NaN (only where the scale is not finite) becomes code 0: codes are always finite.
template <bool kFp8>
__device__ __forceinline__ uint32_t codes_of(const float* x) {
    constexpr float kMost = kFp8 ? kE4m3Max : 127.0f;
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = x[i] != x[i] ? 0.0f : fminf(fmaxf(x[i], -kMost), kMost);
    if constexpr (kFp8) {
        return e4m3x4(v[0], v[1], v[2], v[3]);
    } else {
        uint32_t c = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) c |= (static_cast<uint32_t>(static_cast<int>(__builtin_rintf(v[i]))) & 0xffu) << (8 * i);
        return c;
    }
}

// A dword of codes at a new scale: code · ratio, rounded again.
template <bool kFp8>
__device__ __forceinline__ uint32_t rescaled(uint32_t c, float ratio) {
    float v[4];
    codes4f<kFp8>(c, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] *= ratio;
    return codes_of<kFp8>(v);
}

// Bytes [from, to) of the dword whose first byte is number `at`.
__device__ __forceinline__ uint32_t byte_mask(int at, int from, int to) {
    const int a = max(from - at, 0), b = min(to - at, 4);
    if (a >= b) return 0;
    return (b == 4 ? 0xffffffffu : (1u << (8 * b)) - 1u) & ~((1u << (8 * a)) - 1u);
}

// Up to this many tokens of a page whose scale stands have their values stored byte by byte: a read of what
// the page holds would be another trip to memory for 16 bytes of which one to a few change.
constexpr int kFewTokens = 4;

// One workgroup a (run, head, keys or values): the run's new tokens of one page. The scale is
// max(the page's, largest new magnitude / largest code, 1e-12), the page's own only where it was
// begun before. Where it grows, the codes that the page holds are rounded again at the new scale
// (code · old/new); a page that the run begins is cleared past its tokens. Magnitudes compare as their bits
// do, and an infinity or NaN is above every number: what is not finite goes into the page's scale.
// Elements are read eight at a time, twice (the second time out of L1 or L2). New values are transposed in
// LDS, four tokens of a channel a dword, rows of page/4 + 1 dwords; both kinds leave 16 bytes a thread.
template <bool kFp8>
__global__ __launch_bounds__(kThreads) void append_kernel(CacheAppend p, int width_shift, int page_shift) {
    extern __shared__ uint32_t turned[];
    __shared__ uint32_t wave_most[kWaves];
    const i32x4 run = *reinterpret_cast<const i32x4*>(p.runs + 4 * static_cast<int64_t>(blockIdx.x));
    const int row = run[0], count = run[1], page = run[2], offset = run[3];
    if (count <= 0 || page < 0 || page >= p.pages || row < 0 || row + count > p.tokens || offset < 0 ||
        offset + count > p.page)
        return;
    const int head = blockIdx.y, end = offset + count, eights = width_shift - 3;
    const bool values = blockIdx.z != 0;
    const uint16_t* x = values ? p.v + row * p.v_token + head * p.v_head : p.k + row * p.k_token + head * p.k_head;
    const int64_t token_step = values ? p.v_token : p.k_token;
    const int64_t tile = static_cast<int64_t>(page) * p.heads + head;
    uint8_t* codes = (values ? p.v_codes : p.k_codes) + tile * p.page * p.width;
    float* scale_at = (values ? p.v_scale : p.k_scale) + tile;
    const float before = offset > 0 ? *scale_at : 0.0f;

    uint32_t most = 0;
    for (int i = threadIdx.x; i < count << eights; i += kThreads) {
        float v[8];
        load8(x + (i >> eights) * token_step + 8 * (i & ((1 << eights) - 1)), p.half, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) most = max(most, bits_of(v[j]) & 0x7fffffffu);
    }
    for (int step = 1; step < 64; step *= 2) most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), step)));
    if ((threadIdx.x & 63) == 0) wave_most[threadIdx.x >> 6] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) most = max(most, wave_most[w]);
    const float reach = nan_max(float_of(most) / (kFp8 ? kE4m3Max : 127.0f), kScaleFloor);
    const float scale = nan_max(before, reach);
    const float inv = 1.0f / scale;
    const float ratio = before / scale;
    const bool keep = offset > 0 && bits_of(scale) == bits_of(before);
    if (threadIdx.x == 0 && !keep) *scale_at = scale;

    if (!values) {
        // A thread: 16 channels of a token; where the scale stands, of the new tokens alone.
        const int sixteens = width_shift - 4, first = keep ? offset : 0, last = keep ? end : p.page;
        for (int i = threadIdx.x; i < (last - first) << sixteens; i += kThreads) {
            const int t = first + (i >> sixteens), d = 16 * (i & ((1 << sixteens) - 1));
            i32x4* at = reinterpret_cast<i32x4*>(codes + (static_cast<int64_t>(t) << width_shift) + d);
            i32x4 got = {0, 0, 0, 0};
            if (t >= offset && t < end) {
                float v[16];
                load8(x + (t - offset) * token_step + d, p.half, v);
                load8(x + (t - offset) * token_step + d + 8, p.half, v + 8);
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = div_rn(v[j], scale, inv);
#pragma unroll
                for (int j = 0; j < 4; ++j) got[j] = static_cast<int32_t>(codes_of<kFp8>(v + 4 * j));
            } else if (offset > 0) {
                got = *at;
#pragma unroll
                for (int j = 0; j < 4; ++j) got[j] = static_cast<int32_t>(rescaled<kFp8>(static_cast<uint32_t>(got[j]), ratio));
            }
            *at = got;
        }
        return;
    }
    if (keep && count <= kFewTokens) {
        for (int i = threadIdx.x; i < count << eights; i += kThreads) {
            const int t = i >> eights, d = 8 * (i & ((1 << eights) - 1));
            float v[8];
            load8(x + t * token_step + d, p.half, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = div_rn(v[j], scale, inv);
            const uint32_t c[2] = {codes_of<kFp8>(v), codes_of<kFp8>(v + 4)};
#pragma unroll
            for (int j = 0; j < 8; ++j) codes[((d + j) << page_shift) + offset + t] = static_cast<uint8_t>(c[j / 4] >> (8 * (j & 3)));
        }
        return;
    }
    // A thread: four tokens of the page, eight channels.
    const int pitch = (p.page >> 2) + 1, t_first = offset & ~3;
    const int fours = (end - t_first + 3) >> 2;
    for (int i = threadIdx.x; i < fours << eights; i += kThreads) {
        const int t = t_first + 4 * (i >> eights), d = 8 * (i & ((1 << eights) - 1));
        float v[4][8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (t + j >= offset && t + j < end) {
                load8(x + (t + j - offset) * token_step + d, p.half, v[j]);
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) v[j][k] = 0.0f;
            }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float four[4] = {div_rn(v[0][k], scale, inv), div_rn(v[1][k], scale, inv), div_rn(v[2][k], scale, inv),
                                   div_rn(v[3][k], scale, inv)};
            turned[(d + k) * pitch + (t >> 2)] = codes_of<kFp8>(four);
        }
    }
    __syncthreads();
    // A thread: 16 tokens of a channel; where the scale stands, of those with new tokens alone.
    const int first = keep ? offset >> 4 : 0, last = keep ? (end + 15) >> 4 : p.page >> 4;
    const int chunks = last - first;
    for (int i = threadIdx.x; i < chunks << width_shift; i += kThreads) {
        const int d = i / chunks, t = 16 * (first + i - d * chunks);
        i32x4* at = reinterpret_cast<i32x4*>(codes + (static_cast<int64_t>(d) << page_shift) + t);
        i32x4 got = {0, 0, 0, 0};
        if (offset > 0 && (t < offset || t + 16 > end)) got = *at;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t c = static_cast<uint32_t>(got[j]);
            if (!keep && offset > 0) c = rescaled<kFp8>(c, ratio);
            const uint32_t mine = byte_mask(t + 4 * j, offset, end);
            if (mine) c = (c & ~mine) | (turned[d * pitch + (t >> 2) + j] & mine);
            got[j] = static_cast<int32_t>(c);
        }
        *at = got;
    }
}

// ------------------------------------------------------------------------------------ read

// One workgroup a (listed page, head): its keys and values as 16-bit numbers, tokens by width. A thread
// takes 16 channels of a token's keys, and 16 tokens of four channels' values, which it turns in registers:
// a wave's stores of a token's values are of neighbouring channels.
template <bool kFp8>
__global__ __launch_bounds__(kThreads) void read_kernel(CacheRead p, int width_shift, int page_shift) {
    const int page = p.numbers[blockIdx.x], head = blockIdx.y;
    const int64_t to = (static_cast<int64_t>(blockIdx.x) * p.heads + head) * p.page * p.width;
    uint16_t *k_out = p.k_out + to, *v_out = p.v_out + to;
    const int elements = p.page << width_shift;
    if (page < 0 || page >= p.pages) {
        for (int i = threadIdx.x; i < elements / 8; i += kThreads) {
            reinterpret_cast<i32x4*>(k_out)[i] = i32x4{0, 0, 0, 0};
            reinterpret_cast<i32x4*>(v_out)[i] = i32x4{0, 0, 0, 0};
        }
        return;
    }
    const int64_t tile = static_cast<int64_t>(page) * p.heads + head;
    const float ks = p.k_scale[tile], vs = p.v_scale[tile];
    const uint8_t *k = p.k_codes + tile * elements, *v = p.v_codes + tile * elements;
    for (int i = threadIdx.x; i < elements / 16; i += kThreads) {
        const i32x4 c = reinterpret_cast<const i32x4*>(k)[i];
        float x[16];
#pragma unroll
        for (int j = 0; j < 4; ++j) codes4f<kFp8>(static_cast<uint32_t>(c[j]), x + 4 * j);
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] *= ks;
        store8(k_out + 16 * i, p.half, x);
        store8(k_out + 16 * i + 8, p.half, x + 8);
    }
    const int fours = width_shift - 2;
    for (int i = threadIdx.x; i < elements / 64; i += kThreads) {
        const int d = 4 * (i & ((1 << fours) - 1)), t = 16 * (i >> fours);
        i32x4 c[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) c[j] = *reinterpret_cast<const i32x4*>(v + ((d + j) << page_shift) + t);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float x[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) codes4f<kFp8>(static_cast<uint32_t>(c[j][q]), x[j]);
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const i32x2 two = {static_cast<int32_t>(narrow2(x[0][s] * vs, x[1][s] * vs, p.half)),
                                   static_cast<int32_t>(narrow2(x[2][s] * vs, x[3][s] * vs, p.half))};
                *reinterpret_cast<i32x2*>(v_out + ((t + 4 * q + s) << width_shift) + d) = two;
            }
        }
    }
}

}  // namespace

hipError_t cache_plan(const CachePlan& p, hipStream_t s) {
    const size_t shared = (4 * static_cast<size_t>(p.requests) + 3) * sizeof(int);
    const int work = p.tokens > p.requests ? p.tokens : p.requests + 1;
    int groups = (work + 4 * kThreads - 1) / (4 * kThreads);
    plan_kernel<<<groups, kThreads, shared, s>>>(p);
    return hipGetLastError();
}

static int log2_of(int n) { return n > 1 ? 1 + log2_of(n / 2) : 0; }

hipError_t cache_append(const CacheAppend& p, bool fp8, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(p.runs_most), static_cast<unsigned>(p.heads), 2);
    const size_t turned = static_cast<size_t>(p.width) * (p.page / 4 + 1) * 4;
    const int w = log2_of(p.width), t = log2_of(p.page);
    if (fp8) append_kernel<true><<<grid, kThreads, turned, s>>>(p, w, t);
    else append_kernel<false><<<grid, kThreads, turned, s>>>(p, w, t);
    return hipGetLastError();
}

hipError_t cache_read(const CacheRead& p, bool fp8, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(p.count), static_cast<unsigned>(p.heads));
    const int w = log2_of(p.width), t = log2_of(p.page);
    if (fp8) read_kernel<true><<<grid, kThreads, 0, s>>>(p, w, t);
    else read_kernel<false><<<grid, kThreads, 0, s>>>(p, w, t);
    return hipGetLastError();
}

}  // namespace cozyq
