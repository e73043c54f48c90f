// Attention of new tokens over K/V caches: the last tokens of a window (and the
// sinks), or everything, of each request's own cache, and in front of it a prefix that
// all requests of the batch share.
//
// Request b holds len_b cached tokens, the T of this call included.  Its token t
// stands at p = len_b - T + t and sees own key j when
//   j <= p  and  (j >= p - left  or  j < sinks),
// and every key of the shared prefix.  Rows that see nothing give o = 0, lse = -inf.
//
// The T tokens x G query heads that share a K/V head are the rows of one tile, so
// each cached K and V row is read once for all of them.  One request's keys are cut
// into parts so that the chip is full whatever the batch; a part's workgroup gives
// every wave tiles of 32 keys of its own (private LDS stages, no barrier in the
// loop), and the waves' (O, max, sum) are merged through LDS.  The prefix is a
// different shape, all requests' rows against one K/V: its workgroups are row tiles
// that share 64-key stages.  Parts of both write fp32 (O, max, sum) and
// fta_cache_combine_kernel joins them; a call that needs one part writes o directly.
#include "fta_common.h"
#include "fta_host.h"
#include "fta_tile.h"

#include <algorithm>

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;

struct CacheArgs {
    const uint16_t *q, *k, *v, *kp, *vp;
    int64_t q_sb, q_sh, q_sn, k_sb, k_sh, k_sn, v_sb, v_sh, v_sn, kp_sh, kp_sn, vp_sh, vp_sn;
    const int32_t* lens;
    uint16_t* o;
    int64_t o_sb, o_sh, o_sn;
    float* lse;       // [B][H][T]
    float* part_o;    // [slot][row][Dk]
    float2* part_ml;  // [slot][row]: running max, sum
    int B, T, H, Hk, G, R, S, P, Dreal;  // R = T * G rows per (b, K/V head); row (b * Hk + hk) * R + t * G + g
    int left, sinks;
    float c;
    int row_tiles, ns;        // own keys: 32-row tiles of R, parts
    int pre_tiles, pre_ns;    // prefix: row tiles of B * R, parts
    int64_t rows;             // B * Hk * R
    int total, pre_total;     // workgroups of either
    bool narrow, pre_narrow;
};

// (b, t, head) of row r of (b, hk)
__device__ __forceinline__ int64_t q_offset(const CacheArgs& a, int b, int hk, int r) {
    const int t = r / a.G, g = r - t * a.G;
    return b * a.q_sb + (int64_t)(hk * a.G + g) * a.q_sh + t * a.q_sn;
}

__device__ __forceinline__ void write_row4(const CacheArgs& a, int slot, int64_t row, int Dk, int d, float4 o) {
    *reinterpret_cast<float4*>(a.part_o + ((int64_t)slot * a.rows + row) * Dk + d) = o;
}

template <int D>
struct CacheShape {
    static constexpr int NW = 4;                                           // waves
    static constexpr int STAGE_B = 2 * FtaTile<FTA_DTYPE_BF16, D>::TEN_B;  // 32 keys, each wave's own
    static constexpr int PRE_B = (D <= 128 ? 2 : 1) * STAGE_B;  // prefix: 64 (or 32) keys, shared
    static constexpr int OROW = D + 4;  // floats per row of the merge buffer
    static constexpr int OWN_B = NW * (STAGE_B > 32 * OROW * 4 ? STAGE_B : 32 * OROW * 4);  // the merge buffer reuses the stages
    static constexpr int LDS_B = OWN_B > 2 * PRE_B ? OWN_B : 2 * PRE_B;
};

// ----------------------------------------------------------------------------
// Own keys.  Workgroup = (b, K/V head, row tile, part).  A wave loads its next tile as soon
// as it has read the last one, into the same stage: the other waves of the CU (eight at
// D = 128, 128 KB of loads in all) cover its wait, and a second stage changed nothing.
// What bounds it: memory.  128 requests, 32 / 8 heads of 128, 4096 of 8192 cached tokens:
// 365 us, 5.9 TB/s (a large copy moves 5.15); one request: 7 us and 4 for the join,
// latencies.
// ----------------------------------------------------------------------------
template <int DT, int D>
__device__ void cache_own(const CacheArgs& a, int wgi, unsigned char* sStage, float2 (*sML)[32]) {
    using E = Elem<DT>;
    using T = FtaTile<DT, D>;
    using Sh = CacheShape<D>;
    constexpr int NW = Sh::NW;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rest = fta_scalar(wgi / a.ns), sp = wgi - rest * a.ns;
    const int bhk = fta_scalar(rest / a.row_tiles), rt = rest - bhk * a.row_tiles;
    const int b = fta_scalar(bhk / a.Hk), hk = bhk - b * a.Hk;
    const int r_lo = 32 * rt, r_n = min(32, a.R - r_lo);
    const int len = __builtin_amdgcn_readfirstlane(min(max(a.lens[b], 0), a.S));
    const int p0 = len - a.T + fta_scalar(r_lo / a.G), p1 = len - a.T + fta_scalar((r_lo + r_n - 1) / a.G);  // first and last position
    const int r = r_lo + (lane & 31);
    const int pos = (r < a.R) ? len - a.T + r / a.G : -1;  // this lane's row

    // 32-key tiles: the sinks', then the band's
    const int ke = max(p1 + 1, 0), kb0 = max(0, p0 - a.left);
    int ns = (min(a.sinks, ke) + 31) >> 5, c_lo = kb0 >> 5;
    const int c_hi = (ke + 31) >> 5;
    if (c_lo <= ns) c_lo = ns = 0;
    const int all = max(ns + c_hi - c_lo, 0);
    const int it0 = fta_scalar((int)((int64_t)all * sp / a.ns)), it1 = fta_scalar((int)((int64_t)all * (sp + 1) / a.ns));

    f32x16 oacc[T::DT32];
#pragma unroll
    for (int dt = 0; dt < T::DT32; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) oacc[dt][i] = 0.f;
    float m_run = -FTA_INF, l_run = 0.f;

    const uint32_t lds0 = fta_lds_addr(sStage + wave * Sh::STAGE_B);
    if (it0 + wave < it1) {  // wave-uniform
        const uint16_t* kp = a.k + b * a.k_sb + hk * a.k_sh;
        const uint16_t* vp = a.v + b * a.v_sb + hk * a.v_sh;
        fta_frag qf[T::KS];
        T::load_rows(a.q + q_offset(a, b, hk, min(r, a.R - 1)), r < a.R, a.Dreal, lane, qf);
        FtaGather<D, 1, 32> g;
        g.start(a.k_sn, a.v_sn, a.Dreal, 0, lane);
        const FtaAddr<D> ad0(lds0, lane);
        auto key = [&](int it) { return 32 * (it < ns ? it : c_lo + it - ns); };
        auto issue = [&](int it) {
            const int kb = key(it);
            if (a.narrow && kb + 32 <= ke && (kb >= kb0 || kb + 32 <= a.sinks))
                g.whole(kp + (int64_t)kb * a.k_sn, vp + (int64_t)kb * a.v_sn, lds0);
            else  // keys that no row sees are taken from one that is seen (masked)
                g.mapped(kp, vp, a.k_sn, a.v_sn, kb, a.Dreal, lds0, 0, lane,
                         [&](int t) { return t >= ke ? ke - 1 : (t < kb0 && t >= a.sinks) ? kb0 : t; });
        };
        fta_wait_vmcnt<0>();  // the Q loads: the DMAs are invisible to the compiler's wait counting
        issue(it0 + wave);
        for (int it = it0 + wave; it < it1; it += NW) {
            fta_wait_vmcnt<0>();
            asm volatile("" ::: "memory");
            const int kb = key(it);
            const FtaAddr<D> ad = ad0.here();
            f32x16 s;
            T::template qk<3>(ad, 0, qf, s);
            if (!(kb + 31 <= p0 && (kb >= p1 - a.left || kb + 31 < a.sinks)))  // (rows past R are never written)
                T::mask(fta_bits_below(pos + 1 - kb) & (~fta_bits_below(pos - a.left - kb) | fta_bits_below(a.sinks - kb)),
                        lane, s);
            T::template softmax_pv<3>(ad, T::TEN_B, s, a.c, m_run, l_run, oacc);
            if (it + NW < it1) {  // every LDS read has returned: its MFMAs were issued
                __builtin_amdgcn_sched_barrier(0);
                issue(it + NW);
            }
        }
    }

    // merge of the waves through LDS (the stages are done with)
    const float L = l_run + fta_xor32(l_run);
    __syncthreads();
    float* so = reinterpret_cast<float*>(sStage);
    if (lane < 32) sML[wave][lane] = make_float2(m_run, L);
    if ((lane & 31) < r_n) {
#pragma unroll
        for (int dt = 0; dt < T::DT32; ++dt)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<float4*>(so + (wave * 32 + (lane & 31)) * Sh::OROW + dt * 32 + c_row(i, lane)) =
                    make_float4(oacc[dt][i], oacc[dt][i + 1], oacc[dt][i + 2], oacc[dt][i + 3]);
    }
    __syncthreads();
    const bool direct = a.ns == 1 && a.pre_ns == 0;
    for (int e = threadIdx.x; e < r_n * (D / 4); e += NW * 64) {
        const int rr = e / (D / 4), d = (e - rr * (D / 4)) * 4;
        float m = -FTA_INF, l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < NW; ++w)
            if (sML[w][rr].y > 0.f) m = fmaxf(m, sML[w][rr].x);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float2 ml = sML[w][rr];
            if (!(ml.y != 0.f)) continue;  // this wave saw no key (a NaN sum goes on)
            const float f = fta_exp2((ml.x - m) * a.c);
            const float4 x = *reinterpret_cast<const float4*>(so + (w * 32 + rr) * Sh::OROW + d);
            l = fmaf(ml.y, f, l);
            o.x = fmaf(x.x, f, o.x), o.y = fmaf(x.y, f, o.y), o.z = fmaf(x.z, f, o.z), o.w = fmaf(x.w, f, o.w);
        }
        const int row_r = r_lo + rr;
        const int64_t row = (int64_t)bhk * a.R + row_r;
        if (!direct) {
            write_row4(a, a.pre_ns + sp, row, D, d, o);
            if (d == 0) a.part_ml[(int64_t)(a.pre_ns + sp) * a.rows + row] = make_float2(m, l);
            continue;
        }
        const int t = row_r / a.G, h = hk * a.G + row_r - t * a.G;
        if (d == 0) a.lse[((int64_t)b * a.H + h) * a.T + t] = l != 0.f ? fmaf(m, a.c, fta_log2(l)) * kLn2 : -FTA_INF;
        if (d >= a.Dreal) continue;
        const float f = l != 0.f ? 1.f / l : 0.f;
        *reinterpret_cast<uint2*>(a.o + b * a.o_sb + h * a.o_sh + t * a.o_sn + d) =
            make_uint2(E::pack2(o.x * f, o.y * f), E::pack2(o.z * f, o.w * f));
    }
}

// ----------------------------------------------------------------------------
// Shared prefix.  Workgroup = (K/V head, 32 NW rows of the batch's B * R, part):
// 64-key stages (32 at D = 256) shared by its waves, no mask but at the prefix's end.
// What bounds it: the forward's mix of matrix and vector work for many rows (64 requests, 32 /
// 8 heads of 128, 32768 tokens: 47 us alone, 730 TFLOP/s), the prefix's bytes for few.
// ----------------------------------------------------------------------------
template <int DT, int D>
__device__ void cache_prefix(const CacheArgs& a, int wgi, unsigned char* sStage) {
    constexpr int NH = D <= 128 ? 2 : 1, KEYS = 32 * NH, PD = D <= 128 ? 3 : 2;
    using T = FtaTile<DT, D>;
    using Sh = CacheShape<D>;
    constexpr int NW = Sh::NW;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rest = fta_scalar(wgi / a.pre_tiles), rt = wgi - rest * a.pre_tiles;
    const int hk = fta_scalar(rest / a.pre_ns), sp = rest - hk * a.pre_ns;
    const int all = (a.P + KEYS - 1) / KEYS;
    const int it0 = fta_scalar((int)((int64_t)all * sp / a.pre_ns));
    const int it1 = fta_scalar((int)((int64_t)all * (sp + 1) / a.pre_ns));
    const int64_t rows = (int64_t)a.B * a.R;
    const int64_t f0 = (int64_t)rt * 32 * NW + 32 * wave, f = f0 + (lane & 31);
    const bool ok = f < rows;
    const int b = ok ? (int)(f / a.R) : 0, r = ok ? (int)(f - (int64_t)b * a.R) : 0;

    const uint16_t* kp = a.kp + hk * a.kp_sh;
    const uint16_t* vp = a.vp + hk * a.vp_sh;
    fta_frag qf[T::KS];
    T::load_rows(a.q + q_offset(a, b, hk, r), ok, a.Dreal, lane, qf);
    f32x16 oacc[T::DT32];
#pragma unroll
    for (int dt = 0; dt < T::DT32; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) oacc[dt][i] = 0.f;
    float m_run = -FTA_INF, l_run = 0.f;
    FtaGather<D, NW, KEYS> g;
    g.start(a.kp_sn, a.vp_sn, a.Dreal, wave, lane);
    const uint32_t lds0 = fta_lds_addr(sStage), ldsw = lds0 + 1024 * wave;
    const FtaAddr<D> ad0(lds0, lane);
    auto issue = [&](int it, int st) __attribute__((always_inline)) {
        const int kb = KEYS * it;
        const uint32_t lds = ldsw + st * Sh::PRE_B;
        if (a.pre_narrow && kb + KEYS <= a.P)
            g.whole(kp + (int64_t)kb * a.kp_sn, vp + (int64_t)kb * a.vp_sn, lds);
        else
            g.mapped(kp, vp, a.kp_sn, a.vp_sn, kb, a.Dreal, lds, wave, lane, [&](int t) { return min(t, a.P - 1); });
    };
    fta_wait_vmcnt<0>();  // the Q loads: the DMAs are invisible to the compiler's wait counting
    int it = it0;
    if (it0 < it1) issue(it0, 0);
    auto tile = [&](auto st) __attribute__((always_inline)) {
        constexpr int ST = decltype(st)::value;
        fta_wait_vmcnt<0>();
        __syncthreads();  // tile `it` visible; every wave is past tile it - 1
        const int left = a.P - KEYS * it;
        if (++it < it1) issue(it, ST ^ 1);
        if (f0 >= rows) return;  // wave-uniform
#pragma unroll
        for (int sb = 0; sb < NH; ++sb) {
            const int hi = left - 32 * sb;  // keys left
            if (hi <= 0) continue;
            const FtaAddr<D> ad = ad0.here();
            f32x16 s;
            T::template qk<PD>(ad, ST * Sh::PRE_B + sb * T::TEN_B, qf, s);
            if (hi < 32) T::mask(fta_bits_below(hi), lane, s);
            T::template softmax_pv<PD>(ad, ST * Sh::PRE_B + (NH + sb) * T::TEN_B, s, a.c, m_run, l_run, oacc);
        }
    };
    while (it < it1) {
        tile(std::integral_constant<int, 0>{});
        if (it < it1) tile(std::integral_constant<int, 1>{});
    }
    const float L = l_run + fta_xor32(l_run);
    if (!ok) return;
    const int64_t row = ((int64_t)b * a.Hk + hk) * a.R + r;
    if (lane < 32) a.part_ml[(int64_t)sp * a.rows + row] = make_float2(m_run, L);
#pragma unroll
    for (int dt = 0; dt < T::DT32; ++dt)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
            write_row4(a, sp, row, D, dt * 32 + c_row(i, lane),
                       make_float4(oacc[dt][i], oacc[dt][i + 1], oacc[dt][i + 2], oacc[dt][i + 3]));
}

// One launch for both: the prefix's workgroups, bound by the matrix units for many rows, and
// the own keys', bound by memory, are spread evenly over the block ids, so that a CU holds
// some of each.  64 requests, 32 / 8 heads of 128, a prefix of 32768 and 768 own tokens on
// average: 47 + 47 us as two launches, 84 as one; prefix first or last is 3 to 5% slower.
// Each CU holds two workgroups (registers and LDS), so the mix hides less than it could.
// The own keys' workgroups go to the XCDs in turn: parts of one cache share no keys, and
// runs of requests on one XCD would leave it with the longest (128 requests of 256 to 4096
// tokens: 273 -> 212 us; of 4096 out of 8192: 370 -> 358).
template <int DT, int D>
__global__ __launch_bounds__(CacheShape<D>::NW * 64, D <= 64 ? 4 : D <= 128 ? 2 : 1) void fta_cache_attn_kernel(CacheArgs a) {
    using Sh = CacheShape<D>;
    __shared__ __align__(1024) unsigned char sStage[Sh::LDS_B];
    __shared__ float2 sML[Sh::NW][32];
    if (a.pre_total == 0) {
        cache_own<DT, D>(a, blockIdx.x, sStage, sML);
        return;
    }
    const int64_t all = a.pre_total + a.total;
    const int before = fta_scalar((int)((int64_t)blockIdx.x * a.pre_total / all));
    const bool pre = fta_scalar((int)((int64_t)(blockIdx.x + 1) * a.pre_total / all)) > before;
    if (pre)
        cache_prefix<DT, D>(a, fta_xcd_remap(before, a.pre_total), sStage);
    else
        cache_own<DT, D>(a, blockIdx.x - before, sStage, sML);
}

// Join of the parts, one workgroup per row: D / 8 column groups x 2048 / D slices of
// the parts, each slice with its own running max; the slices are joined through LDS.
template <int DT, int D>
__global__ __launch_bounds__(256) void fta_cache_combine_kernel(CacheArgs a, int slots) {
    using E = Elem<DT>;
    constexpr int DC = D / 8, NSL = 256 / DC;
    __shared__ float so[NSL][D + 4];
    __shared__ float2 sml[NSL];
    const int64_t row = blockIdx.x;
    const int dc = threadIdx.x % DC, sl = threadIdx.x / DC;
    float m = -FTA_INF, l = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int s = sl; s < slots; s += NSL) {
        const float2 ml = a.part_ml[(int64_t)s * a.rows + row];
        const float* src = a.part_o + ((int64_t)s * a.rows + row) * D + dc * 8;
        const float4 x0 = *reinterpret_cast<const float4*>(src), x1 = *reinterpret_cast<const float4*>(src + 4);
        if (!(ml.y != 0.f)) continue;  // a part without keys
        const float mn = fmaxf(m, ml.x);
        const float f0 = (m == -FTA_INF) ? 0.f : fta_exp2((m - mn) * a.c), f1 = fta_exp2((ml.x - mn) * a.c);
        m = mn;
        l = fmaf(l, f0, ml.y * f1);
        o[0] = fmaf(o[0], f0, x0.x * f1), o[1] = fmaf(o[1], f0, x0.y * f1);
        o[2] = fmaf(o[2], f0, x0.z * f1), o[3] = fmaf(o[3], f0, x0.w * f1);
        o[4] = fmaf(o[4], f0, x1.x * f1), o[5] = fmaf(o[5], f0, x1.y * f1);
        o[6] = fmaf(o[6], f0, x1.z * f1), o[7] = fmaf(o[7], f0, x1.w * f1);
    }
    *reinterpret_cast<float4*>(&so[sl][dc * 8]) = make_float4(o[0], o[1], o[2], o[3]);
    *reinterpret_cast<float4*>(&so[sl][dc * 8 + 4]) = make_float4(o[4], o[5], o[6], o[7]);
    if (dc == 0) sml[sl] = make_float2(m, l);
    __syncthreads();
    if (threadIdx.x >= D / 2) return;
    const int d = threadIdx.x * 2;
    m = -FTA_INF;
#pragma unroll
    for (int s = 0; s < NSL; ++s)
        if (sml[s].y != 0.f) m = fmaxf(m, sml[s].x);
    float y0 = 0.f, y1 = 0.f;
    l = 0.f;
#pragma unroll
    for (int s = 0; s < NSL; ++s) {
        const float2 ml = sml[s];
        const float f = ml.y != 0.f ? fta_exp2((ml.x - m) * a.c) : 0.f;
        if (ml.y != 0.f) {
            l = fmaf(ml.y, f, l);
            y0 = fmaf(so[s][d], f, y0);
            y1 = fmaf(so[s][d + 1], f, y1);
        }
    }
    const int64_t bhk = row / a.R;
    const int r = (int)(row - bhk * a.R), b = (int)(bhk / a.Hk), hk = (int)(bhk - (int64_t)b * a.Hk);
    const int t = r / a.G, h = hk * a.G + r - t * a.G;
    if (d == 0) a.lse[((int64_t)b * a.H + h) * a.T + t] = l != 0.f ? fmaf(m, a.c, fta_log2(l)) * kLn2 : -FTA_INF;
    if (d >= a.Dreal) return;
    const float f = l != 0.f ? 1.f / l : 0.f;
    *reinterpret_cast<uint32_t*>(a.o + b * a.o_sb + h * a.o_sh + t * a.o_sn + d) = E::pack2(y0 * f, y1 * f);
}

// ---------------------------------------------------------------------- host

int kernel_dim(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }
bool narrow(int64_t sn) { return sn >= 0 && sn <= (1 << 24); }

// Geometry and parts.
int cache_plan(CacheArgs& a, int B, int H, int Hk, int T, int S, int D, int P, int left, int sinks) {
    if (B <= 0 || H <= 0 || Hk <= 0 || T <= 0 || S <= 0 || D <= 0) return fta::arg_error("cache_attn: dims must be positive");
    if (H % Hk != 0) return fta::arg_error("cache_attn: num_heads must be a multiple of num_kv_heads");
    if (D % 16 != 0 || D > 256) return fta::arg_error("cache_attn: D must be a multiple of 16 up to 256");
    if (P < 0 || left < 0 || sinks < 0) return fta::arg_error("cache_attn: prefix, window and num_sinks must be non-negative");
    if (S > (1 << 29) || T > (1 << 20) || P > (1 << 29) || H > (1 << 20))
        return fta::unsupported("cache_attn: sizes past 2^29 keys, 2^20 new tokens or heads");
    if (!fta::size_fits(B, T, H, D)) return fta::unsupported("cache_attn: 2^60 elements and more");
    if (P > 0 && left < S) return fta::unsupported("cache_attn: a window behind a shared prefix");
    a = CacheArgs{};
    a.B = B, a.T = T, a.H = H, a.Hk = Hk, a.G = H / Hk, a.S = S, a.P = P, a.Dreal = D;
    if ((int64_t)T * a.G > (1 << 24)) return fta::unsupported("cache_attn: more than 2^24 rows per K/V head");
    a.R = T * a.G;
    a.left = std::min(left, S);
    a.sinks = a.left >= S - 1 ? 0 : std::min(sinks, S);
    a.rows = (int64_t)B * Hk * a.R;
    a.row_tiles = (a.R + 31) / 32;
    const int64_t wgs = (int64_t)B * Hk * a.row_tiles;
    // Keys a row tile can see, in 32-key tiles: at least one tile per wave and part.  About 512
    // workgroups in all (two a CU at D = 128), by shapes alone, as the lengths are on the device.
    // Target 256 / 512 / 1024 / 2048, us, 32 / 8 heads of 128, 4096 tokens each: 8 requests 27 / 28 /
    // 29 / 34, 64 requests 185 / 185 / 192 / 195, 65 (a second round of workgroups) 224 / 225 / 212
    // / 205, 128 362 / 362 / 362 / 374.  What it costs is a batch with one long request, whose
    // part is walked by one workgroup: 63 requests of 1024 tokens and one of 32768, 375 / 374 /
    // 223 / 146.
    const int64_t span = std::min<int64_t>(S, (int64_t)a.left + T + a.sinks);
    const int64_t tiles = (span + 31) / 32;
    a.ns = (int)std::max<int64_t>(1, std::min<int64_t>((512 + wgs - 1) / wgs, tiles / 4));
    if (P > 0) {
        const int64_t pt = ((int64_t)B * a.R + 127) / 128;
        if (pt > (1 << 24)) return fta::unsupported("cache_attn: too many rows");
        a.pre_tiles = (int)pt;
        a.pre_ns = (int)std::max<int64_t>(1, std::min<int64_t>((512 + pt * Hk - 1) / (pt * Hk), ((int64_t)P + 255) / 256));
    }
    // workgroups of 256 threads: fewer than 2^32 threads a launch
    const int64_t most = (1 << 24) - 1;
    if (a.rows > most || wgs * a.ns + (int64_t)Hk * a.pre_tiles * a.pre_ns > most)
        return fta::unsupported("cache_attn: too many rows");
    return FTA_OK;
}

int cache_slots(const CacheArgs& a) { return a.pre_ns + a.ns; }
size_t ml_bytes(const CacheArgs& a) { return fta::align_up((size_t)cache_slots(a) * a.rows * sizeof(float2)); }
size_t cache_bytes(const CacheArgs& a, int Dk) {
    if (cache_slots(a) <= 1) return 0;
    return ml_bytes(a) + fta::align_up((size_t)cache_slots(a) * a.rows * Dk * sizeof(float));
}

template <int DT, int D>
int launch_cache(CacheArgs& a, hipStream_t st) {
    int rc;
    a.pre_total = a.Hk * a.pre_tiles * a.pre_ns;
    a.total = a.B * a.Hk * a.row_tiles * a.ns;
    hipLaunchKernelGGL((fta_cache_attn_kernel<DT, D>), dim3((unsigned)(a.pre_total + a.total)), dim3(CacheShape<D>::NW * 64), 0,
                       st, a);
    if ((rc = fta::check_launch("fta_cache_attn_kernel")) != FTA_OK || cache_slots(a) <= 1) return rc;
    hipLaunchKernelGGL((fta_cache_combine_kernel<DT, D>), dim3((unsigned)a.rows), dim3(256), 0, st, a, cache_slots(a));
    return fta::check_launch("fta_cache_combine_kernel");
}

}  // namespace

extern "C" {

size_t fta_cache_attn_workspace_size(int B, int H, int Hk, int T, int S, int D, int P, int left, int num_sinks) {
    CacheArgs a;
    if (cache_plan(a, B, H, Hk, T, S, D, P, left, num_sinks) != FTA_OK) return 0;
    return cache_bytes(a, kernel_dim(D));
}

int fta_cache_attn(const void* q, const int64_t* q_strides, const void* k_cache, const int64_t* kc_strides,
                   const void* v_cache, const int64_t* vc_strides, int dtype, int B, int H, int Hk, int T, int S, int D,
                   const int32_t* cache_lens, const void* k_prefix, const int64_t* kp_strides, const void* v_prefix,
                   const int64_t* vp_strides, int P, int left, int num_sinks, float scale, void* o,
                   const int64_t* o_strides, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
    FTA_TRY_BEGIN
    CacheArgs a;
    int rc = cache_plan(a, B, H, Hk, T, S, D, P, left, num_sinks);
    if (rc != FTA_OK) return rc;
    if (dtype != FTA_DTYPE_BF16 && dtype != FTA_DTYPE_F16) return fta::arg_error("cache_attn: dtype must be bf16 or fp16");
    if (!(scale > 0.f) || scale > 2.0e38f)  // times log2(e) still finite
        return fta::arg_error("cache_attn: scale must be positive and at most 2e38");
    const size_t need = cache_bytes(a, kernel_dim(D));
    if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return fta::arg_error("cache_attn: workspace too small");
    if (!fta::all_set(q, q_strides, k_cache, kc_strides, v_cache, vc_strides, cache_lens, o, o_strides, lse) ||
        (P > 0 && !fta::all_set(k_prefix, kp_strides, v_prefix, vp_strides)))
        return fta::arg_error("cache_attn: a required pointer is null");
    a.q = (const uint16_t*)q, a.q_sb = q_strides[0], a.q_sh = q_strides[1], a.q_sn = q_strides[2];
    a.k = (const uint16_t*)k_cache, a.k_sb = kc_strides[0], a.k_sh = kc_strides[1], a.k_sn = kc_strides[2];
    a.v = (const uint16_t*)v_cache, a.v_sb = vc_strides[0], a.v_sh = vc_strides[1], a.v_sn = vc_strides[2];
    if (P > 0) {
        a.kp = (const uint16_t*)k_prefix, a.kp_sh = kp_strides[1], a.kp_sn = kp_strides[2];
        a.vp = (const uint16_t*)v_prefix, a.vp_sh = vp_strides[1], a.vp_sn = vp_strides[2];
        a.pre_narrow = narrow(a.kp_sn) && narrow(a.vp_sn);
    }
    a.narrow = narrow(a.k_sn) && narrow(a.v_sn);
    a.lens = cache_lens;
    a.o = (uint16_t*)o, a.o_sb = o_strides[0], a.o_sh = o_strides[1], a.o_sn = o_strides[2];
    a.lse = lse;
    a.c = scale * kLog2e;
    a.part_ml = (float2*)workspace;
    a.part_o = need > 0 ? (float*)((char*)workspace + ml_bytes(a)) : nullptr;
    hipStream_t st = (hipStream_t)stream;
    const bool bf = dtype == FTA_DTYPE_BF16;
    switch (kernel_dim(D)) {
        case 64: return bf ? launch_cache<FTA_DTYPE_BF16, 64>(a, st) : launch_cache<FTA_DTYPE_F16, 64>(a, st);
        case 128: return bf ? launch_cache<FTA_DTYPE_BF16, 128>(a, st) : launch_cache<FTA_DTYPE_F16, 128>(a, st);
        default: return bf ? launch_cache<FTA_DTYPE_BF16, 256>(a, st) : launch_cache<FTA_DTYPE_F16, 256>(a, st);
    }
    FTA_TRY_END
}

}  // extern "C"
