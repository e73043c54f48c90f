// What the attention kernels over K/V caches share, whatever the caches hold: the
// arguments, the merge of a workgroup's waves and the join of the parts that the keys of
// one request are cut into.
#pragma once

#include "fta_common.h"
#include "fta_host.h"

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
    int row_tiles, ns;        // own keys: tiles of R rows (32, or 16 over 4-bit caches), parts
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

// Merge of a workgroup's waves, then its rows r_lo .. r_lo + r_n - 1 of (b, hk) to the output, or as
// part sp.  Wave w holds the (unscaled) output of row r at so + (w * ROWS + r) * OROW and its running
// max and sum at sml[w * ROWS + r]; parts are DK columns wide.
template <int DT, int D, int DK, int ROWS, int OROW, int NW>
__device__ __forceinline__ void cache_merge(const CacheArgs& a, int bhk, int b, int hk, int r_lo, int r_n, int sp,
                                            const float* so, const float2* sml) {
    using E = Elem<DT>;
    const bool direct = a.ns == 1 && a.pre_ns == 0;
    for (int e = threadIdx.x; e < r_n * (D / 4); e += NW * 64) {
        const int rr = e / (D / 4), d = (e - rr * (D / 4)) * 4;
        float m = -FTA_INF, l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < NW; ++w)
            if (sml[w * ROWS + rr].y > 0.f) m = fmaxf(m, sml[w * ROWS + rr].x);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float2 ml = sml[w * ROWS + rr];
            if (!(ml.y != 0.f)) continue;  // this wave saw no key (a NaN sum goes on)
            const float f = fta_exp2((ml.x - m) * a.c);
            const float4 x = *reinterpret_cast<const float4*>(so + (w * ROWS + rr) * OROW + d);
            l = fmaf(ml.y, f, l);
            o.x = fmaf(x.x, f, o.x), o.y = fmaf(x.y, f, o.y), o.z = fmaf(x.z, f, o.z), o.w = fmaf(x.w, f, o.w);
        }
        const int row_r = r_lo + rr;
        const int64_t row = (int64_t)bhk * a.R + row_r;
        if (!direct) {
            write_row4(a, a.pre_ns + sp, row, DK, d, o);
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
int cache_slots(const CacheArgs& a) { return a.pre_ns + a.ns; }
size_t ml_bytes(const CacheArgs& a) { return fta::align_up((size_t)cache_slots(a) * a.rows * sizeof(float2)); }
size_t cache_bytes(const CacheArgs& a, int Dk) {
    if (cache_slots(a) <= 1) return 0;
    return ml_bytes(a) + fta::align_up((size_t)cache_slots(a) * a.rows * Dk * sizeof(float));
}

}  // namespace
