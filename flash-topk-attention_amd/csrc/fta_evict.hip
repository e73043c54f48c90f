// Eviction: of every request's K/V heads the rows that stay in the cache, by the attention that
// each received (a running sum, fta_cache_weights), and their move to the front.
//
// Of len_b rows min(len_b, budget) stay: the first `sinks`, the last `recent` and, of those
// between, the ones of largest weight; of equal weights the lower rows (NaN counts as less than
// anything).  Rows keep their order.  Two launches:
//
//  * fta_evict_select_kernel, one workgroup of 1024 threads per (b, K/V head): the weight of the
//    last row to stay is found digit by digit (11, 11 and 10 bits of the weights as ordered
//    integers, a histogram in LDS for each), then every wave counts what it keeps of its own run
//    of rows and writes their numbers behind those of the waves in front of it.  Up to 1024 rows
//    take one wave each instead, fta_evict_select_wave_kernel.
//  * fta_evict_move_kernel moves the rows.  In place, destinations never lie behind their sources
//    and both ascend, so a workgroup that reads a block of rows, waits, and then writes it may go
//    on to the next block: nothing that later blocks read has been written.  What can run side by
//    side are heads, tensors and slices of a row.  Into another cache every block of rows runs by
//    itself.
#include "fta_common.h"
#include "fta_host.h"
#include "fta_tile.h"

#include <algorithm>

namespace {

constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64;
constexpr int kMoved = 5;  // tensors at most: codes and scales of keys and values, weights

struct Moved {
    const uint8_t* src;
    uint8_t* dst;
    int64_t s_sb, s_sh, s_sn, d_sb, d_sh, d_sn;  // bytes
    int unit, units;                             // bytes of an access, accesses of a row
    int slice, slices;                           // accesses of a row that go together, such slices
};

struct EvictArgs {
    const float* w;
    int64_t w_sb, w_sh;
    const int32_t* lens;
    int32_t* new_lens;
    int32_t* kept;  // [B][Hk][budget]
    Moved t[kMoved];
    int nt, B, Hk, S, S_out, budget, recent, sinks;
    int jobs, blocks;  // slices of all tensors; out of place: blocks of rows
    bool in_place;
};

// Weights as integers in the same order: -0 as 0, NaN (1) below everything.  0 and kAlways stand for rows
// that are not there and rows that stay whatever they weigh.
constexpr uint32_t kAlways = 0xffffffffu;
__device__ __forceinline__ uint32_t ordered(float x) {
    if (x != x) return 1u;
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.f);
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}

// Sum over the workgroup of v over the threads in front of this one, and over all.
__device__ __forceinline__ int scan_threads(int v, int* sw, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o, 64);
        if (lane >= o) x += y;
    }
    if (lane == 63) sw[wave] = x;
    __syncthreads();
    int before = 0;
    total = 0;
    for (int i = 0; i < kSelWaves; ++i) {
        const int y = sw[i];
        before += i < wave ? y : 0;
        total += y;
    }
    __syncthreads();
    return before + x - v;
}

// PT > 0: a thread's weights (at most PT) stay in registers between the passes; 0: they are read again.
// What bounds it: the latency of its passes, one workgroup a CU.  8192 rows, 128 heads: 10.6 us; 16384, 512
// heads: 30; 32768, 8 heads: 23, of which two histograms are 5 and the last pass 6.
template <int PT>
__global__ __launch_bounds__(kSelThreads) void fta_evict_select_kernel(EvictArgs a) {
    __shared__ __align__(16) int hist[2048][4];  // four copies: weights crowd into few bins, whose additions wait for each other
    __shared__ int sw[kSelWaves];
    __shared__ int found[2];
    __shared__ int sgt[kSelWaves], seq[kSelWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int bhk = blockIdx.x, b = bhk / a.Hk, hk = bhk - b * a.Hk;
    const int len = min(max(a.lens[b], 0), a.S);
    int32_t* kept = a.kept + (int64_t)bhk * a.budget;
    if (hk == 0 && threadIdx.x == 0) a.new_lens[b] = min(len, a.budget);
    if (len <= a.budget) {
        for (int i = threadIdx.x; i < a.budget; i += kSelThreads) kept[i] = i < len ? i : -1;
        return;
    }
    const float* w = a.w + b * a.w_sb + hk * a.w_sh;
    const int lo = a.sinks, hi = len - a.recent;  // rows that compete
    const int m = a.budget - a.sinks - a.recent;  // how many of them stay
    // this wave's run of rows: `steps` times 64
    const int steps = PT > 0 ? PT : (len + kSelThreads - 1) / kSelThreads;
    const int64_t w0 = (int64_t)wave * steps * 64 + lane;
    // every weight is loaded, whether or not it competes: a load behind a condition waits for itself alone
    auto load = [&](int64_t j) { return w[min(j, (int64_t)len - 1)]; };
    auto value = [&](int64_t j, float x) { return j < lo || (j >= hi && j < len) ? kAlways : j < hi ? ordered(x) : 0u; };
    uint32_t held[PT > 0 ? PT : 1];
    if constexpr (PT > 0) {
#pragma unroll
        for (int i = 0; i < PT; ++i) held[i] = __builtin_bit_cast(uint32_t, load(w0 + i * 64));
#pragma unroll
        for (int i = 0; i < PT; ++i) held[i] = value(w0 + i * 64, __builtin_bit_cast(float, held[i]));
    }
    auto each = [&](auto f) __attribute__((always_inline)) {  // f(index, value) of the run's rows in order
        if constexpr (PT > 0) {
#pragma unroll
            for (int i = 0; i < PT; ++i) {
                f(i, held[i]);
                __builtin_amdgcn_sched_barrier(0);  // else every row's votes are formed first, and spill
            }
        } else {
            for (int i = 0; i < steps; ++i) f(i, value(w0 + (int64_t)i * 64, load(w0 + (int64_t)i * 64)));
        }
    };

    // the m-th largest weight, its first `done` bits in `prefix`; `need` of the rows that share them stay
    uint32_t prefix = 0;
    int need = m, done = 0;
    if (m == 0) prefix = kAlways - 1;
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
        const int bits = pass < 2 ? 11 : 10, shift = 32 - done - bits;
        for (int i = threadIdx.x; i < 2048; i += kSelThreads) *reinterpret_cast<int4*>(hist[i]) = make_int4(0, 0, 0, 0);
        __syncthreads();
        if (m > 0)
            each([&](int, uint32_t x) {
                if (x - 1u < kAlways - 1u && (done == 0 || (x >> (32 - done)) == prefix)) atomicAdd(&hist[(x >> shift) & ((1 << bits) - 1)][lane & 3], 1);
            });
        __syncthreads();
        // thread t holds bins 2 t and 2 t + 1 from the top
        const int top = 2047 - 2 * threadIdx.x;
        const int4 h1 = *reinterpret_cast<const int4*>(hist[top]), h0 = *reinterpret_cast<const int4*>(hist[top - 1]);
        const int c1 = (h1.x + h1.y) + (h1.z + h1.w), c0 = (h0.x + h0.y) + (h0.z + h0.w);
        int total;
        const int before = scan_threads(c1 + c0, sw, total);
        if (before < need && before + c1 + c0 >= need) {
            const bool first = before + c1 >= need;
            found[0] = first ? top : top - 1;
            found[1] = need - before - (first ? 0 : c1);
        }
        __syncthreads();
        if (m > 0) {
            prefix = (prefix << bits) | (uint32_t)found[0];
            need = found[1];
        }
        done += bits;
        __syncthreads();
    }

    // rows above the threshold and at it, wave by wave
    int gt = 0, eq = 0;
    each([&](int, uint32_t x) {
        gt += x > prefix;
        eq += x == prefix;
    });
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        gt += __shfl_xor(gt, o, 64);
        eq += __shfl_xor(eq, o, 64);
    }
    if (lane == 0) {
        sgt[wave] = gt;
        seq[wave] = eq;
    }
    __syncthreads();
    int eqs = 0, at = 0;  // rows at the threshold, and rows that stay, in front of this wave
    for (int i = 0; i < wave; ++i) {
        at += sgt[i] + min(max(need - eqs, 0), seq[i]);
        eqs += seq[i];
    }
    const uint64_t below = (1ull << lane) - 1;
    each([&](int i, uint32_t x) {
        const uint64_t ties = __ballot(x == prefix);
        const bool stay = x > prefix || (x == prefix && eqs + __popcll(ties & below) < need);
        const uint64_t all = __ballot(stay);
        const int p = at + __popcll(all & below);
        if (stay && p < a.budget) kept[p] = (int32_t)(w0 + (int64_t)i * 64);
        at += __popcll(all);
        eqs += __popcll(ties);
    });
}

// The same by one wave for up to 64 PT rows: the weight of the last row to stay is found bit by bit, by the
// number of rows at or above it, until that number is the budget.  No LDS and no barriers.
// What bounds it: latency, a compare, a count and an addition that wait for each other for every 64 rows.  481 rows, 512
// heads: 7.8 us, the workgroup's kernel 14; 704 rows, 404 heads: 12.3 and 15.3.  2048 rows, 8 heads, would be 17 and 10.
template <int PT>
__global__ __launch_bounds__(256) void fta_evict_select_wave_kernel(EvictArgs a) {
    const int lane = threadIdx.x & 63;
    const int bhk = fta_scalar(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (bhk >= a.B * a.Hk) return;
    const int b = fta_scalar(bhk / a.Hk), hk = bhk - b * a.Hk;
    const int len = __builtin_amdgcn_readfirstlane(min(max(a.lens[b], 0), a.S));
    int32_t* kept = a.kept + (int64_t)bhk * a.budget;
    if (hk == 0 && lane == 0) a.new_lens[b] = min(len, a.budget);
    if (len <= a.budget) {
        for (int i = lane; i < a.budget; i += 64) kept[i] = i < len ? i : -1;
        return;
    }
    const float* w = a.w + b * a.w_sb + hk * a.w_sh;
    const int hi = len - a.recent;
    float x[PT];
    uint32_t held[PT];
#pragma unroll
    for (int i = 0; i < PT; ++i) x[i] = w[min(64 * i + lane, len - 1)];
#pragma unroll
    for (int i = 0; i < PT; ++i) {
        const int j = 64 * i + lane;
        held[i] = j >= len ? 0u : (j < a.sinks || j >= hi) ? kAlways : ordered(x[i]);
    }
    auto count = [&](auto f) __attribute__((always_inline)) {
        int n = 0;
#pragma unroll
        for (int i = 0; i < PT; ++i) n += __popcll(__ballot(f(held[i])));
        return n;
    };
    uint32_t last = 0;  // more than `budget` rows are there, so it ends above 0, which stands for none
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t c = last | 1u << bit;
        const int n = count([&](uint32_t v) { return v >= c; });
        if (n >= a.budget) last = c;
        if (n == a.budget) break;
    }
    const int need = a.budget - count([&](uint32_t v) { return v > last; });
    const uint64_t below = (1ull << lane) - 1;
    int eqs = 0, at = 0;
#pragma unroll
    for (int i = 0; i < PT; ++i) {
        const uint64_t ties = __ballot(held[i] == last);
        const bool stay = held[i] > last || (held[i] == last && eqs + __popcll(ties & below) < need);
        const uint64_t all = __ballot(stay);
        const int p = at + __popcll(all & below);
        if (stay && p < a.budget) kept[p] = 64 * i + lane;
        at += __popcll(all);
        eqs += __popcll(ties);
    }
}

// ----------------------------------------------------------------------------
// The move: workgroup = (b, K/V head, slice) in place, (b, K/V head, slice, block of rows) into
// another cache.  A thread moves one access of a row, kMove rows at a time.
// What bounds it: memory, and in place for few heads the latency of its blocks, which follow each other.  16 x 8
// heads of 128 bf16, 8192 rows to 4096: 146 to 152 us in place, 118 into another cache (537 MB: 3.5 to 3.7 and 4.6
// TB/s); 64 x 8 heads of 128 in 4 bits, 16384 to 4096: 176 to 180 us (604 MB; single rows of 64 and 8 bytes out of
// 128-byte lines); 1 x 8 heads, 32768 to 8192: 34 us.  In place, of one run, 146 / 176 / 35 us, with 512 threads
// instead of 1024 152 / 184 / 42, with eight rows a thread 174 / 194 / 39.  Where few rows stay most of 1024 threads
// have none, and 256 move them: 346 rows of 64 x 8 heads bf16 45 -> 27 us, 345 rows of 101 x 4 heads in 4 bits 26 ->
// 11, 1024 rows of 128 x 8 in 4 bits 100 -> 75; but of 8 heads 1024 rows 6.8 -> 11.5, 4096 of 16 x 8 155 -> 171.
// ----------------------------------------------------------------------------
constexpr int kMove = 4;
// Bytes of a row that one workgroup moves: the fewest that memory reads at once.  32 / 64 / 128 / 256, us of
// the kernel: in place, 8192 rows to 4096, 16 x 8 heads of 128 bf16 (537 MB moved) 244 / 153 / 155 / 174,
// 32768 to 8192, 1 x 8 heads 46 / 42 / 75 / 141; into another cache, 16 x 8 heads 202 / 121 / 119 / 125.
constexpr int kSliceBytes = 64;

// The value is in its registers: a load that would still be on its way is waited for here.
__device__ __forceinline__ void arrived(uint4& x) { asm volatile("" : "+v"(x.x), "+v"(x.y), "+v"(x.z), "+v"(x.w)); }
__device__ __forceinline__ void arrived(uint2& x) { asm volatile("" : "+v"(x.x), "+v"(x.y)); }
__device__ __forceinline__ void arrived(uint32_t& x) { asm volatile("" : "+v"(x)); }
__device__ __forceinline__ void arrived(uint16_t& x) { asm volatile("" : "+v"(x)); }

// Rows [first, last) of (b, hk), this slice of them, kMove accesses of a thread in a block of rows.
// The next block's rows are asked for before this one's are written: they lie behind everything
// that this one writes.
template <typename V, bool IN_PLACE, int NT>
__device__ __forceinline__ void move_rows(const EvictArgs& a, const Moved& t, int b, int hk, int slice, int first, int last,
                                          const int32_t* kept) {
    const int u0 = slice * t.slice, un = min(t.slice, t.units - u0);  // this slice's accesses
    const int row0 = threadIdx.x / t.slice, u = threadIdx.x - row0 * t.slice;
    const int rows = NT / t.slice;  // rows of one access of the workgroup
    const bool mine = u < un && row0 < rows;
    const uint8_t* src = t.src + b * t.s_sb + hk * t.s_sh + (int64_t)(u0 + u) * sizeof(V);
    uint8_t* dst = t.dst + b * t.d_sb + hk * t.d_sh + (int64_t)(u0 + u) * sizeof(V);
    struct Block {
        V x[kMove];
        int from[kMove];
    };
    auto ask = [&](Block& k, int c) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kMove; ++i) {
            const int p = c + i * rows + row0;
            k.from[i] = mine && p < last ? kept[p] : -1;
            if (IN_PLACE && k.from[i] == p) k.from[i] = -1;  // it stays where it is
        }
#pragma unroll
        for (int i = 0; i < kMove; ++i)
            if (k.from[i] >= 0) k.x[i] = *reinterpret_cast<const V*>(src + k.from[i] * t.s_sn);
    };
    auto put = [&](Block& k, int c) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kMove; ++i) arrived(k.x[i]);
        if constexpr (IN_PLACE) __syncthreads();  // every row of the block has been read before any is written
#pragma unroll
        for (int i = 0; i < kMove; ++i)
            if (k.from[i] >= 0) *reinterpret_cast<V*>(dst + (int64_t)(c + i * rows + row0) * t.d_sn) = k.x[i];
    };
    const int step = rows * kMove;
    Block k0, k1;
    ask(k0, first);
    for (int c = first; c < last; c += 2 * step) {
        if (c + step < last) ask(k1, c + step);
        put(k0, c);
        if (c + step >= last) break;
        if (c + 2 * step < last) ask(k0, c + 2 * step);
        put(k1, c + step);
    }
}

template <bool IN_PLACE, int NT>
__global__ __launch_bounds__(NT) void fta_evict_move_kernel(EvictArgs a) {
    const int wgi = blockIdx.x;
    const int rest = wgi / a.blocks, block = wgi - rest * a.blocks;
    const int bhk = rest / a.jobs;
    int job = rest - bhk * a.jobs;
    const int b = bhk / a.Hk, hk = bhk - b * a.Hk;
    const int len = min(max(a.lens[b], 0), a.S), n = min(len, a.budget);
    int ti = 0;
    while (ti + 1 < a.nt && job >= a.t[ti].slices) job -= a.t[ti++].slices;
    const Moved& t = a.t[ti];
    const int32_t* kept = a.kept + (int64_t)bhk * a.budget;
    if (!IN_PLACE || len > a.budget) {
        const int per = IN_PLACE ? n : (n + a.blocks - 1) / a.blocks;
        const int first = min(block * per, n), last = min(n, first + per);
        if (first < last) {
            switch (t.unit) {
                case 16: move_rows<uint4, IN_PLACE, NT>(a, t, b, hk, job, first, last, kept); break;
                case 8: move_rows<uint2, IN_PLACE, NT>(a, t, b, hk, job, first, last, kept); break;
                case 4: move_rows<uint32_t, IN_PLACE, NT>(a, t, b, hk, job, first, last, kept); break;
                default: move_rows<uint16_t, IN_PLACE, NT>(a, t, b, hk, job, first, last, kept);
            }
        }
    }
    if (ti + 1 != a.nt) return;
    // weights of the rows behind those that stayed start again at zero (in place every weight has
    // been read: the last block's are waited for before it is written)
    const int end = IN_PLACE ? len : a.S_out;
    for (int j = n + block * NT + threadIdx.x; j < end; j += a.blocks * NT)
        *reinterpret_cast<float*>(t.dst + b * t.d_sb + hk * t.d_sh + j * t.d_sn) = 0.f;
}

// ---------------------------------------------------------------------- host

template <int PT>
int launch_select_wave(const EvictArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((fta_evict_select_wave_kernel<PT>), dim3((unsigned)((a.B * a.Hk + 3) / 4)), dim3(256), 0, st, a);
    return fta::check_launch("fta_evict_select_wave_kernel");
}

template <int PT>
int launch_select(const EvictArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((fta_evict_select_kernel<PT>), dim3((unsigned)(a.B * a.Hk)), dim3(kSelThreads), 0, st, a);
    return fta::check_launch("fta_evict_select_kernel");
}

}  // namespace

extern "C" {

int fta_cache_evict(int tensors, const void* const* src, const int64_t* src_strides, void* const* dst,
                    const int64_t* dst_strides, const int32_t* row_bytes, const float* weights, const int64_t* w_strides,
                    float* weights_out, const int64_t* wo_strides, int B, int Hk, int S, int S_out, int budget, int recent,
                    int num_sinks, const int32_t* cache_lens, int32_t* new_lens, int32_t* kept, void* stream) {
    FTA_TRY_BEGIN
    if (B <= 0 || Hk <= 0 || S <= 0 || S_out <= 0 || budget <= 0) return fta::arg_error("cache_evict: dims must be positive");
    if (tensors < 1 || tensors > kMoved - 1) return fta::arg_error("cache_evict: one to four tensors");
    if (recent < 0 || num_sinks < 0 || (int64_t)recent + num_sinks > budget)
        return fta::arg_error("cache_evict: recent and num_sinks must be non-negative and fit in budget");
    if (budget > S || budget > S_out) return fta::arg_error("cache_evict: budget must not pass the caches' rows");
    if (S > (1 << 29) || S_out > (1 << 29) || Hk > (1 << 20)) return fta::unsupported("cache_evict: sizes past 2^29 rows or 2^20 heads");
    if (!fta::size_fits(B, S, Hk, 256) || !fta::size_fits(B, S_out, Hk, 256)) return fta::unsupported("cache_evict: 2^60 elements and more");
    if (!fta::all_set(src, src_strides, dst, dst_strides, row_bytes, weights, w_strides, weights_out, wo_strides, cache_lens,
                      new_lens, kept))
        return fta::arg_error("cache_evict: a required pointer is null");
    EvictArgs a = {};
    a.w = weights, a.w_sb = w_strides[0], a.w_sh = w_strides[1];
    a.lens = cache_lens, a.new_lens = new_lens, a.kept = kept;
    a.nt = tensors + 1, a.B = B, a.Hk = Hk, a.S = S, a.S_out = S_out, a.budget = budget, a.recent = recent, a.sinks = num_sinks;
    a.in_place = weights == weights_out;
    for (int i = 0; i < a.nt; ++i) {
        Moved& t = a.t[i];
        const bool last = i == tensors;
        t.src = last ? (const uint8_t*)weights : (const uint8_t*)src[i];
        t.dst = last ? (uint8_t*)weights_out : (uint8_t*)dst[i];
        if (!fta::all_set(t.src, t.dst)) return fta::arg_error("cache_evict: a required pointer is null");
        if ((t.src == t.dst) != a.in_place) return fta::arg_error("cache_evict: every tensor in place, or none");
        const int64_t ss[3] = {last ? 4 * w_strides[0] : src_strides[3 * i], last ? 4 * w_strides[1] : src_strides[3 * i + 1],
                               last ? 4 : src_strides[3 * i + 2]};
        const int64_t ds[3] = {last ? 4 * wo_strides[0] : dst_strides[3 * i], last ? 4 * wo_strides[1] : dst_strides[3 * i + 1],
                               last ? 4 : dst_strides[3 * i + 2]};
        const int rb = last ? 4 : row_bytes[i];
        if (rb <= 0 || rb > 512 || rb % 2 != 0) return fta::arg_error("cache_evict: rows of 2 to 512 bytes, an even number");
        t.s_sb = ss[0], t.s_sh = ss[1], t.s_sn = ss[2], t.d_sb = ds[0], t.d_sh = ds[1], t.d_sn = ds[2];
        // the widest access that everything is a multiple of
        const uint64_t all = (uint64_t)rb | (uintptr_t)t.src | (uintptr_t)t.dst | (uint64_t)(ss[0] | ss[1] | ss[2] | ds[0] | ds[1] | ds[2]);
        t.unit = all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : 2;
        if (all % 2 != 0) return fta::arg_error("cache_evict: rows must be 2-byte aligned");
        t.units = rb / t.unit;
        t.slice = std::min(t.units, kSliceBytes / t.unit);
        t.slices = (t.units + t.slice - 1) / t.slice;
        a.jobs += t.slices;
    }
    const int64_t heads = (int64_t)B * Hk;
    a.blocks = a.in_place ? 1 : (int)std::max<int64_t>(1, std::min<int64_t>((budget + 255) / 256, (8192 + heads * a.jobs - 1) / (heads * a.jobs)));
    if (heads * a.jobs * a.blocks > (1 << 22) - 1 || heads > (1 << 22) - 1) return fta::unsupported("cache_evict: too many heads");
    hipStream_t st = (hipStream_t)stream;
    int rc = S <= 8 * 64             ? launch_select_wave<8>(a, st)
             : S <= 16 * 64          ? launch_select_wave<16>(a, st)
             : S <= 8 * kSelThreads  ? launch_select<8>(a, st)
             : S <= 16 * kSelThreads ? launch_select<16>(a, st)
             : S <= 32 * kSelThreads ? launch_select<32>(a, st)
                                     : launch_select<0>(a, st);
    if (rc != FTA_OK) return rc;
    const dim3 g((unsigned)(heads * a.jobs * a.blocks));
    if (!a.in_place)
        hipLaunchKernelGGL((fta_evict_move_kernel<false, 512>), g, dim3(512), 0, st, a);
    else if (budget <= 512 || (budget <= 1024 && heads * a.jobs >= 2048))
        hipLaunchKernelGGL((fta_evict_move_kernel<true, 256>), g, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((fta_evict_move_kernel<true, 1024>), g, dim3(1024), 0, st, a);
    return fta::check_launch("fta_evict_move_kernel");
    FTA_TRY_END
}

}  // extern "C"
