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

// Magnitudes compare as their bits do, and an infinity or NaN is above every number: a page's
// largest magnitude carries what is not finite into the page's scale.
__device__ __forceinline__ uint32_t magnitude(uint16_t h, bool half) {
    return bits_of(half ? widen<true>(h) : widen<false>(h)) & 0x7fffffffu;
}

__device__ __forceinline__ float value16(uint16_t h, bool half) { return half ? widen<true>(h) : widen<false>(h); }

// The code of v (already over the scale): int8 by rint, E4M3 by the conversion, clamped to the
// format's largest. A NaN (only where the scale is not finite) becomes code 0, so that codes are
// always finite.
template <bool kFp8>
__device__ __forceinline__ uint32_t code_of(float v) {
    constexpr float kMost = kFp8 ? kE4m3Max : 127.0f;
    v = v != v ? 0.0f : fminf(fmaxf(v, -kMost), kMost);
    if constexpr (kFp8) return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(v, v, 0, false)) & 0xffu;
    else return static_cast<uint32_t>(static_cast<int>(__builtin_rintf(v))) & 0xffu;
}

template <bool kFp8>
__device__ __forceinline__ float code_value(uint32_t c) {
    if constexpr (kFp8) return e4m3_value(c);
    else return static_cast<float>(static_cast<int8_t>(c));
}

// One workgroup a (run, head, keys or values): the run's new tokens of one page. The scale is
// max(the page's, largest new magnitude / largest code, 1e-12), the page's own only where it was
// begun before. Where it grows, the codes that the page holds are rounded again at the new scale
// (code · old/new); a page that the run begins is cleared past its tokens.
template <bool kFp8>
__global__ __launch_bounds__(kThreads) void append_kernel(CacheAppend p) {
    __shared__ uint32_t wave_most[kWaves];
    const i32x4 run = *reinterpret_cast<const i32x4*>(p.runs + 4 * static_cast<int64_t>(blockIdx.x));
    const int row = run[0], count = run[1], page = run[2], offset = run[3];
    if (count <= 0 || page < 0 || page >= p.pages || row < 0 || row + count > p.tokens || offset < 0 ||
        offset + count > p.page)
        return;
    const int head = blockIdx.y;
    const bool values = blockIdx.z != 0;
    const uint16_t* x = values ? p.v + row * p.v_token + head * p.v_head : p.k + row * p.k_token + head * p.k_head;
    const int64_t token_step = values ? p.v_token : p.k_token;
    const int64_t tile = static_cast<int64_t>(page) * p.heads + head;
    uint8_t* codes = (values ? p.v_codes : p.k_codes) + tile * p.page * p.width;
    float* scale_at = (values ? p.v_scale : p.k_scale) + tile;

    uint32_t most = 0;
    for (int i = threadIdx.x; i < count * (p.width / 2); i += kThreads) {
        const int t = i / (p.width / 2), d = 2 * (i - t * (p.width / 2));
        const uint32_t two = *reinterpret_cast<const uint32_t*>(x + t * token_step + d);
        most = max(most, max(magnitude(static_cast<uint16_t>(two), p.half), magnitude(static_cast<uint16_t>(two >> 16), p.half)));
    }
    for (int step = 1; step < 64; step *= 2) most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), step)));
    if ((threadIdx.x & 63) == 0) wave_most[threadIdx.x >> 6] = most;
    const float before = offset > 0 ? *scale_at : 0.0f;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) most = max(most, wave_most[w]);
    const float reach = nan_max(float_of(most) / (kFp8 ? kE4m3Max : 127.0f), kScaleFloor);
    const float scale = nan_max(before, reach);
    const float inv = 1.0f / scale;
    const float ratio = before / scale;
    const bool keep = offset > 0 && bits_of(scale) == bits_of(before);
    if (threadIdx.x == 0 && !keep) *scale_at = scale;

    // 16 codes a thread and step: of one token's keys, or of one channel's values.
    const int chunks = p.page * p.width / 16;
    for (int i = threadIdx.x; i < chunks; i += kThreads) {
        // Values: neighbouring threads take neighbouring channels, whose new values are neighbours.
        const int t0 = values ? 16 * (i / p.width) : i / (p.width / 16);
        const int d0 = values ? i % p.width : 16 * (i % (p.width / 16));
        const int last = values ? t0 + 15 : t0;
        const bool any_new = last >= offset && t0 < offset + count;
        if (keep && !any_new) continue;
        i32x4* at = reinterpret_cast<i32x4*>(codes + (values ? static_cast<int64_t>(d0) * p.page + t0 : static_cast<int64_t>(t0) * p.width + d0));
        i32x4 old = {0, 0, 0, 0}, got;
        if (offset > 0) old = *at;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const int t = values ? t0 + j : t0, d = values ? d0 : d0 + j;
            uint32_t c = (static_cast<uint32_t>(old[j / 4]) >> (8 * (j & 3))) & 0xffu;
            if (t >= offset && t < offset + count)
                c = code_of<kFp8>(div_rn(value16(x[(t - offset) * token_step + d], p.half), scale, inv));
            else if (!keep && offset > 0)
                c = code_of<kFp8>(code_value<kFp8>(c) * ratio);
            got[j / 4] = j % 4 ? static_cast<int32_t>(static_cast<uint32_t>(got[j / 4]) | (c << (8 * (j & 3)))) : static_cast<int32_t>(c);
        }
        *at = got;
    }
}

// ------------------------------------------------------------------------------------ read

// One workgroup a (listed page, head): its keys and values as 16-bit numbers, tokens by width.
template <bool kFp8>
__global__ __launch_bounds__(kThreads) void read_kernel(CacheRead p) {
    const int page = p.numbers[blockIdx.x], head = blockIdx.y;
    const int64_t to = (static_cast<int64_t>(blockIdx.x) * p.heads + head) * p.page * p.width;
    const bool held = page >= 0 && page < p.pages;
    const int64_t tile = static_cast<int64_t>(held ? page : 0) * p.heads + head;
    const float ks = held ? p.k_scale[tile] : 0.0f, vs = held ? p.v_scale[tile] : 0.0f;
    const uint8_t *k = p.k_codes + tile * p.page * p.width, *v = p.v_codes + tile * p.page * p.width;
    for (int i = threadIdx.x; i < p.page * p.width; i += kThreads) {
        const int t = i / p.width, d = i - t * p.width;
        const float a = held ? code_value<kFp8>(k[i]) * ks : 0.0f;
        const float b = held ? code_value<kFp8>(v[static_cast<int64_t>(d) * p.page + t]) * vs : 0.0f;
        p.k_out[to + i] = p.half ? narrow<true>(a) : narrow<false>(a);
        p.v_out[to + i] = p.half ? narrow<true>(b) : narrow<false>(b);
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

hipError_t cache_append(const CacheAppend& p, bool fp8, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(p.runs_most), static_cast<unsigned>(p.heads), 2);
    if (fp8) append_kernel<true><<<grid, kThreads, 0, s>>>(p);
    else append_kernel<false><<<grid, kThreads, 0, s>>>(p);
    return hipGetLastError();
}

hipError_t cache_read(const CacheRead& p, bool fp8, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(p.count), static_cast<unsigned>(p.heads));
    if (fp8) read_kernel<true><<<grid, kThreads, 0, s>>>(p);
    else read_kernel<false><<<grid, kThreads, 0, s>>>(p);
    return hipGetLastError();
}

}  // namespace cozyq
