// Queries and keys in front of scoring and attention: the norm of every head and
// the rotation of its first columns by position in one pass, forward, backward and
// the serving form that also writes the new K / V rows into their caches.
//
// A row x is one head of one token (D columns).  With weights w and
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r,  u = n w,
// the first R columns of u are turned pair by pair by the angle of the token's
// position (pairs (i, i + R/2), or (2i, 2i + 1) when interleaved):
//   y_a = u_a cos - u_b sin,  y_b = u_b cos + u_a sin;
// the other columns pass.  Backward, with g = the transposed rotation of dy:
//   dw = sum over rows of g n,  h = g w,  dx = r (h - n mean(h n)).
//
// A row is held by LG = 2 .. 32 neighbouring lanes, 8 columns (16 bytes) each, so
// its sums are a few lane exchanges and a wave works on 64 / LG rows at once.  R is
// a multiple of 16: a lane's 8 columns are all turned or all passed, and with
// half-split pairs its partners are the 8 columns of one other lane, which are
// exchanged as packed 16-bit pairs (4 exchanges; r is the row's own and the
// partner's weights are held, so nothing is rounded on the way).  Every value is
// formed in fp32 and rounded once, when it is stored.
#include "fta_common.h"
#include "fta_host.h"
#include "fta_tile.h"

#include <algorithm>
#include <type_traits>

namespace {

// Codes and scales of a 4-bit cache ([B][Hk][S] rows, see fta_q4.hip); batch and head strides in elements.
struct Q4Out {
    uint32_t* codes;
    uint16_t* scales;
    int64_t c_sb, c_sh, s_sb, s_sh;
};

struct PrepArgs {
    const uint16_t *q, *k, *v;      // inputs (v: append only)
    const uint16_t *dqo, *dko;      // backward: gradients of the outputs
    uint16_t *qo, *ko, *vo;         // outputs (append: ko, vo are the caches; backward: dq, dk)
    int64_t q_sb, q_sh, q_sn, k_sb, k_sh, k_sn, v_sb, v_sh, v_sn;
    int64_t dq_sb, dq_sh, dq_sn, dk_sb, dk_sh, dk_sn;
    int64_t qo_sb, qo_sh, qo_sn, ko_sb, ko_sh, ko_sn, vo_sb, vo_sh, vo_sn;
    const void *qw, *kw;            // weights [D] or null (ones)
    int w_dtype;                    // 0 bf16, 1 fp16, 2 fp32
    const float *cos, *sin;         // [P][R / 2]
    const int32_t* positions;       // [B][N] (stride pos_sb between batches) or null: token index
    int64_t pos_sb;
    const int32_t* lens;            // append: tokens in the cache, the new ones included
    int S, pos_off;                 // append: rows of the cache, table row of cache row 0
    const int32_t* pos_offs;        // append: the same for each request, or null
    Q4Out qk, qv;                   // append to a 4-bit cache: in place of ko and vo
    float* part;                    // backward: [workgroup][2][D] partial weight gradients, or null
    int N, H, Hk, D, R, P, inter;
    int parts, per;                 // parts of a token's row groups, groups in each
    int64_t units;                  // (token, part) pairs
    float eps;
};

template <int DT>
__device__ __forceinline__ void unpack8(uint4 x, float* f) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = Elem<DT>::to_f32((uint16_t)(w[i] & 0xffffu));
        f[2 * i + 1] = Elem<DT>::to_f32((uint16_t)(w[i] >> 16));
    }
}
template <int DT>
__device__ __forceinline__ uint4 pack8(const float* f) {
    return make_uint4(Elem<DT>::pack2(f[0], f[1]), Elem<DT>::pack2(f[2], f[3]), Elem<DT>::pack2(f[4], f[5]),
                      Elem<DT>::pack2(f[6], f[7]));
}
__device__ __forceinline__ uint4 shfl4(uint4 x, int src) {
    return make_uint4(__shfl((int)x.x, src, 64), __shfl((int)x.y, src, 64), __shfl((int)x.z, src, 64),
                      __shfl((int)x.w, src, 64));
}
// Weights of columns d .. d + 7.
__device__ __forceinline__ void load_w8(const void* w, int dt, int d, float* f) {
    if (w == nullptr) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = 1.f;
    } else if (dt == FTA_DTYPE_F32) {
        const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(w) + d);
        const float4 y = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(w) + d + 4);
        f[0] = x.x, f[1] = x.y, f[2] = x.z, f[3] = x.w, f[4] = y.x, f[5] = y.y, f[6] = y.z, f[7] = y.w;
    } else {
        const uint4 x = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(w) + d);
        if (dt == FTA_DTYPE_BF16)
            unpack8<FTA_DTYPE_BF16>(x, f);
        else
            unpack8<FTA_DTYPE_F16>(x, f);
    }
}
// 16 bytes that are read or written once: past the caches where the call streams more than
// they hold (see kStream).
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
template <bool NT>
__device__ __forceinline__ uint4 load16(const uint16_t* p) {
    if constexpr (NT) return __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p)));
    return *reinterpret_cast<const uint4*>(p);
}
template <bool NT>
__device__ __forceinline__ void store16(uint16_t* p, uint4 v) {
    if constexpr (NT)
        __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v), reinterpret_cast<u32x4*>(p));
    else
        *reinterpret_cast<uint4*>(p) = v;
}
template <int LG>
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
    for (int o = 1; o < LG; o <<= 1) x += __shfl_xor(x, o, 64);
    return x;
}

// Whether any of a row's 16-bit values (8 to a lane) is not zero.  The lanes' votes are joined in
// scalar registers, where they cost nothing.
template <int LG>
__device__ __forceinline__ bool row_any(uint4 x) {
    constexpr uint64_t first = ~0ull / ((1ull << LG) - 1);  // the first lane of every row
    uint64_t v = __ballot(((x.x | x.y | x.z | x.w) & 0x7fff7fffu) != 0u);
#pragma unroll
    for (int o = 1; o < LG; o <<= 1) v |= v >> o;
    v &= first;
    return __builtin_amdgcn_inverse_ballot_w64((v << LG) - v);
}

// What a lane keeps for its 8 columns: where its partners are and the weights.
struct LaneCols {
    int d0, src;   // first column; lane that holds the partner columns (itself where there are none)
    bool live, turn;
    float sgn;     // half-split pairs: the sign of the partner's term, -1 in the first half
};
template <int LG>
__device__ __forceinline__ LaneCols lane_cols(const PrepArgs& a, int lane) {
    LaneCols c;
    const int li = lane & (LG - 1), half = a.R >> 4;
    c.d0 = li * 8;
    c.live = c.d0 < a.D;
    c.turn = c.d0 < a.R;
    c.sgn = li < half ? -1.f : 1.f;
    c.src = (!a.inter && c.turn) ? (li < half ? lane + half : lane - half) : lane;
    return c;
}

// The lane's 8 cos and sin of a table row (1 and 0 for columns that pass).
__device__ __forceinline__ void load_angles(const PrepArgs& a, const LaneCols& c, int pos, float* cs, float* sn) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        cs[e] = 1.f;
        sn[e] = 0.f;
    }
    if (!c.turn) return;
    const int64_t row = (int64_t)pos * (a.R >> 1);
    if (a.inter) {
        const float4 x = *reinterpret_cast<const float4*>(a.cos + row + (c.d0 >> 1));
        const float4 y = *reinterpret_cast<const float4*>(a.sin + row + (c.d0 >> 1));
        cs[0] = cs[1] = x.x, cs[2] = cs[3] = x.y, cs[4] = cs[5] = x.z, cs[6] = cs[7] = x.w;
        sn[0] = sn[1] = y.x, sn[2] = sn[3] = y.y, sn[4] = sn[5] = y.z, sn[6] = sn[7] = y.w;
    } else {
        const int i = c.d0 >= (a.R >> 1) ? c.d0 - (a.R >> 1) : c.d0;
        const float4 x0 = *reinterpret_cast<const float4*>(a.cos + row + i);
        const float4 x1 = *reinterpret_cast<const float4*>(a.cos + row + i + 4);
        const float4 y0 = *reinterpret_cast<const float4*>(a.sin + row + i);
        const float4 y1 = *reinterpret_cast<const float4*>(a.sin + row + i + 4);
        cs[0] = x0.x, cs[1] = x0.y, cs[2] = x0.z, cs[3] = x0.w, cs[4] = x1.x, cs[5] = x1.y, cs[6] = x1.z, cs[7] = x1.w;
        sn[0] = y0.x, sn[1] = y0.y, sn[2] = y0.z, sn[3] = y0.w, sn[4] = y1.x, sn[5] = y1.y, sn[6] = y1.z, sn[7] = y1.w;
    }
}

// ----------------------------------------------------------------------------
// Forward.  A wave strides over (token, part) pairs; a part is U groups of 64 / LG
// rows of one token, whose loads are issued together and share the token's angles.
// The weights (the lane's own and its partners') stay in registers.
// APPEND: rows past the query and key heads copy V; K and V go to cache row
// lens[b] - N + n (not written outside [0, S)).
// ----------------------------------------------------------------------------
template <int DT, int LG, int U, bool APPEND, bool NT>
__global__ __launch_bounds__(256) void fta_norm_rope_fwd_kernel(PrepArgs a) {
    constexpr int RW = 64 / LG;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const LaneCols c = lane_cols<LG>(a, lane);
    const int rows = a.H + a.Hk + (APPEND ? a.Hk : 0);
    const float inv_d = 1.f / (float)a.D;
    float wq[8], wk[8], pq[8], pk[8];
    {
        const int d = c.live ? c.d0 : 0, dp = c.live ? (c.src & (LG - 1)) * 8 : 0;
        load_w8(a.qw, a.w_dtype, d, wq);
        load_w8(a.kw, a.w_dtype, d, wk);
        load_w8(a.qw, a.w_dtype, dp, pq);
        load_w8(a.kw, a.w_dtype, dp, pk);
    }
    for (int64_t unit = (int64_t)blockIdx.x * 4 + wave; unit < a.units; unit += (int64_t)gridDim.x * 4) {
        const int64_t tok = unit / a.parts;
        const int part = (int)(unit - tok * a.parts);
        const int b = (int)(tok / a.N), n = (int)(tok - (int64_t)b * a.N);
        const int r0 = part * a.per * RW + lane / LG;

        int crow = 0, pos;
        if constexpr (APPEND) {
            const int64_t at = (int64_t)a.lens[b] - a.N + n;
            crow = (at < 0 || at >= a.S) ? -1 : (int)at;
            pos = (int)min(max(at + (a.pos_offs ? a.pos_offs[b] : a.pos_off), (int64_t)0), (int64_t)a.P - 1);
        } else {
            pos = a.positions ? a.positions[b * a.pos_sb + n] : n;
            pos = min(max(pos, 0), a.P - 1);
        }

        uint4 x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int row = r0 + u * RW;
            x[u] = fta_zero4();
            if (c.live && row < rows && u < a.per) {
                const uint16_t* p = row < a.H ? a.q + b * a.q_sb + row * a.q_sh + n * a.q_sn
                                              : a.k + b * a.k_sb + (row - a.H) * a.k_sh + n * a.k_sn;
                if (APPEND && row >= a.H + a.Hk) p = a.v + b * a.v_sb + (row - a.H - a.Hk) * a.v_sh + n * a.v_sn;
                x[u] = load16<NT>(p + c.d0);
            }
        }
        float cs[8], sn[8];
        load_angles(a, c, pos, cs, sn);
        if (!a.inter) {
#pragma unroll
            for (int e = 0; e < 8; ++e) sn[e] *= c.sgn;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int row = r0 + u * RW;
            const bool isq = row < a.H;
            float f[8], y[8];
            unpack8<DT>(x[u], f);
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = fmaf(f[e], f[e], ss);
            const float r = rsqrtf(fmaf(row_sum<LG>(ss), inv_d, a.eps));
            const uint4 xp = a.inter ? x[u] : shfl4(x[u], c.src);
            if (!c.live || row >= rows || u >= a.per) continue;
            uint16_t* out;
            if (APPEND && row >= a.H + a.Hk) {
                if (crow < 0) continue;
                out = a.vo + b * a.vo_sb + (row - a.H - a.Hk) * a.vo_sh + crow * a.vo_sn;
                store16<NT>(out + c.d0, x[u]);
                continue;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] *= r * (isq ? wq[e] : wk[e]);
            if (a.inter) {
#pragma unroll
                for (int e = 0; e < 8; e += 2) {  // written out: the append to a 4-bit cache forms the same bits
                    y[e] = fmaf(f[e], cs[e], -(f[e + 1] * sn[e]));
                    y[e + 1] = fmaf(f[e], sn[e], f[e + 1] * cs[e]);
                }
            } else {
                float g[8];
                unpack8<DT>(xp, g);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = fmaf(g[e] * (r * (isq ? pq[e] : pk[e])), sn[e], f[e] * cs[e]);
            }
            if (isq) {
                out = a.qo + b * a.qo_sb + row * a.qo_sh + n * a.qo_sn;
            } else if (APPEND) {
                if (crow < 0) continue;
                out = a.ko + b * a.ko_sb + (row - a.H) * a.ko_sh + crow * a.ko_sn;
            } else {
                out = a.ko + b * a.ko_sb + (row - a.H) * a.ko_sh + n * a.ko_sn;
            }
            store16<NT>(out + c.d0, pack8<DT>(y));
        }
    }
}

// ----------------------------------------------------------------------------
// Append to a 4-bit cache: the forward's tiling, K and V quantized.  K is rounded to its 16-bit type
// first, so that a cache holds the same whether its rows came prepared or not.  The groups of a part
// are of one kind (queries, keys, values) but where the kinds meet, and each kind has its own body.
// What bounds it: vector instructions, 190 a group of four rows; they take 63% of the cycles, 72% of those in which a
// CU has waves (32768 tokens, 32 / 8 heads of 128: 184 to 192 us, 708 MB).  One body for any row 227 us.  Held to
// four waves a SIMD 198 (128 vector registers, of which five groups spill 8 or 9; 67 scalar ones go to lanes), to
// three, with no vector register spilled, 206; through the caches 209; rows at 32-bit offsets 264 (more registers
// than there are); the queries by the forward's kernel and the rest by this one 121 + 84; one group at a time with
// the next one asked for ahead 373.
// ----------------------------------------------------------------------------

// x of lane ^ 1, ^ 2, and of lanes that hold the other halves of 8 and of 16 (equal within 4 and 8).
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
constexpr int kXor1 = 0xb1, kXor2 = 0x4e, kHalfMirror = 0x141, kMirror = 0x140;

// row_sum without LDS: the same additions
template <int LG>
__device__ __forceinline__ float row_sum_dpp(float x) {
    static_assert(LG >= 4, "");
    x += dpp<kXor1>(x);
    x += dpp<kXor2>(x);
    if constexpr (LG >= 8) x += dpp<kHalfMirror>(x);
    if constexpr (LG >= 16) x += dpp<kMirror>(x);
    if constexpr (LG >= 32) x += __shfl_xor(x, 16, 64);
    return x;
}

// Four bits of a row's values, this lane's eight columns of them: four lanes hold a group of 32,
// whose value of largest magnitude over -8 is its scale d (rounded to float16; the negative of two
// equal ones), and a value's code is round(x / d) + 8, ties to even, held to 0 .. 15.  x has at most 11
// bits and d as many, so a quotient that is no border between two codes is 2^-12 or more from
// the next, and the borders themselves are float32 numbers: x / d by a reciprocal and one
// step of correction, which is right to less than 2^-20 and exact on them, gives the same codes
// as an exact division.
__device__ __forceinline__ uint32_t quant8(const float* x, uint16_t& scale) {
    float hi = x[0], lo = x[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) {
        hi = fmaxf(hi, x[e]);
        lo = fminf(lo, x[e]);
    }
    hi = fmaxf(hi, dpp<kXor1>(hi));
    lo = fminf(lo, dpp<kXor1>(lo));
    hi = fmaxf(hi, dpp<kXor2>(hi));
    lo = fminf(lo, dpp<kXor2>(lo));
    const float top = (-lo >= hi ? lo : hi) * -0.125f;
    const _Float16 h = (_Float16)fminf(fmaxf(top, -65504.f), 65504.f);
    scale = __builtin_bit_cast(uint16_t, h);
    const float d = (float)h;
    if (d == 0.f) return 0x88888888u;
    const float r = __builtin_amdgcn_rcpf(d);
    float n[2] = {34952.f, 34952.f};  // 8 in each of four digits to base 16
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float q = x[e] * r;
        const float y = fmaf(fmaf(-q, d, x[e]), r, q);
        n[e >> 2] = fmaf(rintf(__builtin_amdgcn_fmed3f(y, -8.f, 7.f)), (float)(1 << (4 * (e & 3))), n[e >> 2]);
    }
    return (uint32_t)n[0] | (uint32_t)n[1] << 16;
}

template <int DT, int LG, int U, bool NT>
__global__ __launch_bounds__(256, 4) void fta_norm_rope_append_q4_kernel(PrepArgs a) {
    constexpr int RW = 64 / LG;
    static_assert(LG >= 4, "a group of 32 columns within a row's lanes");
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const LaneCols c = lane_cols<LG>(a, lane);
    const int rows = a.H + 2 * a.Hk, ng = (a.D + 31) >> 5;
    const float inv_d = 1.f / (float)a.D;
    float wq[8], wk[8], pq[8], pk[8];
    {
        const int d = c.live ? c.d0 : 0, dp = c.live ? (c.src & (LG - 1)) * 8 : 0;
        load_w8(a.qw, a.w_dtype, d, wq);
        load_w8(a.kw, a.w_dtype, d, wk);
        load_w8(a.qw, a.w_dtype, dp, pq);
        load_w8(a.kw, a.w_dtype, dp, pk);
    }
    const int oct = (c.d0 >> 3) & 3, grp = c.d0 >> 5;
    // rows of neighbouring tokens share cache lines: an XCD takes neighbouring tokens
    for (int64_t unit = (int64_t)fta_xcd_remap(blockIdx.x, gridDim.x) * 4 + wave; unit < a.units;
         unit += (int64_t)gridDim.x * 4) {
        int part, b, n;
        if (a.units <= 0x7fffffff) {  // 64-bit divisions were a third of the scalar instructions
            const uint32_t tok = (uint32_t)unit / (uint32_t)a.parts;
            part = (int)((uint32_t)unit - tok * (uint32_t)a.parts);
            b = (int)(tok / (uint32_t)a.N), n = (int)(tok - (uint32_t)b * (uint32_t)a.N);
        } else {
            const int64_t tok = unit / a.parts;
            part = (int)(unit - tok * a.parts);
            b = (int)(tok / a.N), n = (int)(tok - (int64_t)b * a.N);
        }
        part = fta_scalar(part), b = fta_scalar(b), n = fta_scalar(n);
        const int first = part * a.per * RW;
        const int64_t at = (int64_t)a.lens[b] - a.N + n;
        const bool in = at >= 0 && at < a.S;  // wave-uniform
        const int pos = (int)min(max(at + (a.pos_offs ? a.pos_offs[b] : a.pos_off), (int64_t)0), (int64_t)a.P - 1);
        // the token's rows of each kind, and the cache's
        const uint16_t* qp = a.q + b * a.q_sb + n * a.q_sn;
        const uint16_t* kp = a.k + b * a.k_sb + n * a.k_sn;
        const uint16_t* vp = a.v + b * a.v_sb + n * a.v_sn;
        uint16_t* op = a.qo + b * a.qo_sb + n * a.qo_sn;
        const int64_t crow = in ? at : 0;
        uint32_t* kc = a.qk.codes + b * a.qk.c_sb + crow * 4 * ng;
        uint32_t* vc = a.qv.codes + b * a.qv.c_sb + crow * 4 * ng;
        uint16_t* ks = a.qk.scales + b * a.qk.s_sb + crow * ng;
        uint16_t* vs = a.qv.scales + b * a.qv.s_sb + crow * ng;

        uint4 x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int row = first + u * RW + lane / LG;
            x[u] = fta_zero4();
            const int lo = first + u * RW, hi = lo + RW - 1;  // wave-uniform
            if (u >= a.per || lo >= rows) continue;
            if (c.live && row < rows) {
                const uint16_t* p;
                if (hi < a.H)
                    p = qp + row * a.q_sh;
                else if (lo >= a.H && hi < a.H + a.Hk)
                    p = kp + (row - a.H) * a.k_sh;
                else if (lo >= a.H + a.Hk)
                    p = vp + (row - a.H - a.Hk) * a.v_sh;
                else
                    p = row < a.H ? qp + row * a.q_sh : row < a.H + a.Hk ? kp + (row - a.H) * a.k_sh
                                                                         : vp + (row - a.H - a.Hk) * a.v_sh;
                x[u] = load16<NT>(p + c.d0);
            }
        }
        float cs[8], sn[8];
        load_angles(a, c, pos, cs, sn);
        if (!a.inter) {
#pragma unroll
            for (int e = 0; e < 8; ++e) sn[e] *= c.sgn;
        }
        // one group of rows.  KIND 0, 1, 2: queries, keys, values alone; 3: any of them
        auto group = [&](auto kind, int u) __attribute__((always_inline)) {
            constexpr int KIND = decltype(kind)::value;
            const int row = first + u * RW + lane / LG;
            const bool isq = KIND == 3 ? row < a.H : KIND == 0;
            const bool isv = KIND == 3 ? row >= a.H + a.Hk : KIND == 2;
            uint4 out = x[u];
            if constexpr (KIND != 2) {
                float f[8], g[8], y[8];
                unpack8<DT>(x[u], f);
                float ss = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) ss = fmaf(f[e], f[e], ss);
                const float r = rsqrtf(fmaf(row_sum_dpp<LG>(ss), inv_d, a.eps));
                const uint4 xp = a.inter ? x[u] : shfl4(x[u], c.src);
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] *= r * (isq ? wq[e] : wk[e]);
                if (a.inter) {
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        y[e] = fmaf(f[e], cs[e], -(f[e + 1] * sn[e]));
                        y[e + 1] = fmaf(f[e], sn[e], f[e + 1] * cs[e]);
                    }
                } else {
                    unpack8<DT>(xp, g);
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[e] = fmaf(g[e] * (r * (isq ? pq[e] : pk[e])), sn[e], f[e] * cs[e]);
                }
                const uint4 turned = pack8<DT>(y);
                if (KIND != 3 || !isv) out = turned;
            }
            if (row >= rows || u >= a.per) return;
            if (KIND == 0 || (KIND == 3 && isq)) {
                if (c.live) store16<NT>(op + row * a.qo_sh + c.d0, out);
                return;
            }
            float y[8];
            unpack8<DT>(out, y);  // columns behind D hold zeros
            if (!c.live) {
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = 0.f;
            }
            uint16_t scale;
            const uint32_t w = quant8(y, scale);  // a row's lanes are here together
            if (!in || grp >= ng) return;
            const int hk = row - a.H - (isv ? a.Hk : 0);
            uint32_t* codes = isv ? vc + hk * a.qv.c_sh + 4 * grp + oct : kc + hk * a.qk.c_sh + oct * ng + grp;
            *codes = w;
            if (oct == 0) *(isv ? vs + hk * a.qv.s_sh + grp : ks + hk * a.qk.s_sh + grp) = scale;
        };
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int lo = first + u * RW, hi = lo + RW - 1;  // wave-uniform
            if (u >= a.per || lo >= rows) break;
            if (hi < a.H)
                group(std::integral_constant<int, 0>{}, u);
            else if (lo >= a.H && hi < a.H + a.Hk)
                group(std::integral_constant<int, 1>{}, u);
            else if (lo >= a.H + a.Hk)
                group(std::integral_constant<int, 2>{}, u);
            else
                group(std::integral_constant<int, 3>{}, u);
        }
    }
}

// ----------------------------------------------------------------------------
// Backward.  The same tiling, a fixed grid that strides over the (token, part)
// pairs; each lane adds the weight gradients of its columns over all its rows, a
// workgroup adds its lanes' and writes one partial, and fta_norm_rope_dw_kernel
// adds the partials in order: no atomics, the same bits every run of a shape.
// A row whose gradient is zero is worked on as a row of zeros: its dx is zero and it adds
// nothing to dw, as the formulas say of any finite x, also where x is padding that holds
// NaN or infinities (0 * NaN would reach every weight's gradient).  Held to four waves a
// SIMD: one register more is three (32K tokens, 32 + 8 heads of 128: 205 -> 270 us).
// ----------------------------------------------------------------------------
template <int DT, int LG, int U, bool NT>
__global__ __launch_bounds__(256, 4) void fta_norm_rope_bwd_kernel(PrepArgs a) {
    constexpr int RW = 64 / LG;
    __shared__ float sw[4][2][LG * 8];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const LaneCols c = lane_cols<LG>(a, lane);
    const int rows = a.H + a.Hk;
    const float inv_d = 1.f / (float)a.D;
    float dwq[8], dwk[8], wq[8], wk[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) dwq[e] = dwk[e] = 0.f;
    load_w8(a.qw, a.w_dtype, c.live ? c.d0 : 0, wq);
    load_w8(a.kw, a.w_dtype, c.live ? c.d0 : 0, wk);
    for (int64_t unit = (int64_t)blockIdx.x * 4 + wave; unit < a.units; unit += (int64_t)gridDim.x * 4) {
        const int64_t tok = unit / a.parts;
        const int part = (int)(unit - tok * a.parts);
        const int b = (int)(tok / a.N), n = (int)(tok - (int64_t)b * a.N);
        int pos = a.positions ? a.positions[b * a.pos_sb + n] : n;
        pos = min(max(pos, 0), a.P - 1);
        const int r0 = part * a.per * RW + lane / LG;
        uint4 x[U], dy[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int row = r0 + u * RW;
            x[u] = dy[u] = fta_zero4();
            if (c.live && row < rows && u < a.per) {
                const bool isq = row < a.H;
                const int h = isq ? row : row - a.H;
                const uint16_t* p = isq ? a.q + b * a.q_sb + h * a.q_sh + n * a.q_sn
                                        : a.k + b * a.k_sb + h * a.k_sh + n * a.k_sn;
                const uint16_t* g = isq ? a.dqo + b * a.dq_sb + h * a.dq_sh + n * a.dq_sn
                                        : a.dko + b * a.dk_sb + h * a.dk_sh + n * a.dk_sn;
                x[u] = load16<NT>(p + c.d0);
                dy[u] = load16<NT>(g + c.d0);
            }
        }
        float cs[8], sn[8];
        load_angles(a, c, pos, cs, sn);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int row = r0 + u * RW;
            const bool isq = row < a.H;
            if (!row_any<LG>(dy[u])) x[u] = fta_zero4();
            float f[8], g[8], d[8];
            unpack8<DT>(x[u], f);
            unpack8<DT>(dy[u], d);
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = fmaf(f[e], f[e], ss);
            const float r = rsqrtf(fmaf(row_sum<LG>(ss), inv_d, a.eps));
            if (a.inter) {
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    g[e] = d[e] * cs[e] + d[e + 1] * sn[e];
                    g[e + 1] = d[e + 1] * cs[e] - d[e] * sn[e];
                }
            } else {
                float dp[8];
                unpack8<DT>(shfl4(dy[u], c.src), dp);
#pragma unroll
                for (int e = 0; e < 8; ++e) g[e] = fmaf(dp[e], -c.sgn * sn[e], d[e] * cs[e]);
            }
            float hn = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                f[e] *= r;  // n
                const float gn = g[e] * f[e];
                if (row < rows && u < a.per) {
                    dwq[e] += isq ? gn : 0.f;
                    dwk[e] += isq ? 0.f : gn;
                }
                g[e] *= isq ? wq[e] : wk[e];  // h
                hn = fmaf(g[e], f[e], hn);
            }
            const float m = row_sum<LG>(hn) * inv_d;
            if (!c.live || row >= rows || u >= a.per) continue;
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] = r * (g[e] - f[e] * m);
            const int h = isq ? row : row - a.H;
            uint16_t* out = isq ? a.qo + b * a.qo_sb + h * a.qo_sh + n * a.qo_sn
                                : a.ko + b * a.ko_sb + h * a.ko_sh + n * a.ko_sn;
            store16<NT>(out + c.d0, pack8<DT>(d));
        }
    }
    if (a.part == nullptr) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
#pragma unroll
        for (int o = LG; o < 64; o <<= 1) {
            dwq[e] += __shfl_xor(dwq[e], o, 64);
            dwk[e] += __shfl_xor(dwk[e], o, 64);
        }
        if (lane < LG) {
            sw[wave][0][lane * 8 + e] = dwq[e];
            sw[wave][1][lane * 8 + e] = dwk[e];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * a.D; i += 256) {
        const int t = i >= a.D, d = i - t * a.D;
        a.part[(int64_t)blockIdx.x * 2 * a.D + i] = (sw[0][t][d] + sw[1][t][d]) + (sw[2][t][d] + sw[3][t][d]);
    }
}

// Sum of the workgroups' partial weight gradients: 8 columns and 32 slices of the
// partials per workgroup; columns [0, D) are the query weights', the rest the keys'.
__global__ __launch_bounds__(256) void fta_norm_rope_dw_kernel(const float* part, int nwg, int D, void* dqw, void* dkw,
                                                               int w_dtype) {
    __shared__ float s[32][9];
    const int cx = threadIdx.x & 7, sy = threadIdx.x >> 3;
    const int col = blockIdx.x * 8 + cx;  // D is a multiple of 16
    float t[4] = {0.f, 0.f, 0.f, 0.f};
    int w = sy;
    for (; w + 96 < nwg; w += 128) {
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] += part[(int64_t)(w + 32 * i) * 2 * D + col];
    }
    for (; w < nwg; w += 32) t[0] += part[(int64_t)w * 2 * D + col];
    s[sy][cx] = (t[0] + t[1]) + (t[2] + t[3]);
    __syncthreads();
    if (sy != 0) return;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) sum += s[i][cx];
    void* out = col < D ? dqw : dkw;
    const int d = col < D ? col : col - D;
    if (out == nullptr) return;
    if (w_dtype == FTA_DTYPE_F32)
        reinterpret_cast<float*>(out)[d] = sum;
    else
        reinterpret_cast<uint16_t*>(out)[d] = (uint16_t)((w_dtype == FTA_DTYPE_BF16 ? Elem<FTA_DTYPE_BF16>::pack2(sum, 0.f)
                                                                                    : Elem<FTA_DTYPE_F16>::pack2(sum, 0.f)) &
                                                         0xffffu);
}

// ---------------------------------------------------------------------- host

int lanes_per_row(int D) {
    int l = 2;
    while (l * 8 < D) l <<= 1;
    return l;
}

int prep_geometry(int B, int H, int Hk, int N, int D, int R, int P) {
    if (B <= 0 || H <= 0 || Hk <= 0 || N <= 0 || D <= 0) return fta::arg_error("qk_norm_rope: dims must be positive");
    if (D % 16 != 0 || D > 256) return fta::arg_error("qk_norm_rope: D must be a multiple of 16 up to 256");
    if (R <= 0 || R % 16 != 0 || R > D)
        return fta::arg_error("qk_norm_rope: the rotated columns must be a positive multiple of 16 up to D");
    if (P <= 0) return fta::arg_error("qk_norm_rope: cos and sin must have rows");
    if (H > (1 << 20) || Hk > (1 << 20)) return fta::unsupported("qk_norm_rope: too many heads");
    if (!fta::size_fits(B, N, (int64_t)H + 2 * Hk, D)) return fta::unsupported("qk_norm_rope: 2^60 elements and more");
    return FTA_OK;
}

// The (token, part) pairs: the 64 / LG-row groups of a token in even parts of at most U.
void set_units(PrepArgs& a, int B, int U, int rows, int lanes = 0) {
    const int rw = 64 / (lanes > 0 ? lanes : lanes_per_row(a.D));
    const int groups = (rows + rw - 1) / rw;
    a.parts = (groups + U - 1) / U;
    a.per = (groups + a.parts - 1) / a.parts;
    a.units = (int64_t)B * a.N * a.parts;
}

// Groups per wave and grids, measured at 32K tokens, 32 + 8 heads of 128 (ten groups a token):
//  * forward, 671 MB: two groups a wave 166 us, four 150, five 132, ten 127; five with twice
//    the workgroups that run at once (the kernel strides over the rest) and past the caches
//    120 us, 5.6 TB/s.
//  * backward, 1.0 GB: one 328, two 229, four 260, five 252; past the caches two 204, three
//    203 (5.0 TB/s), five 197 with twice the partial sums.
// Few rows (a step of a serving batch, up to 4 kFwdGrid groups) take one group a wave, so that
// they spread over the CUs.  One group / five groups a wave, us of the kernel: 32 + 8 heads of
// 128, 16 tokens 3.3 / 5.3, 256 tokens 4.3 / 5.6, 512 tokens 6.2 / 6.9, 1228 tokens (the
// border) 12.0 / 9.6, 8192 tokens 53 / 35; 8 + 8 heads of 64, 1024 tokens 3.8 / 4.5, 2048
// tokens 5.5 / 5.8, 8192 tokens (past the border of 6144) 13.8 / 12.8.
constexpr int kFwdGroups = 5, kFwdGrid = 256 * 12, kBwdGroups = 3, kBwdGrid = 256 * 4;
// Bytes of q from which a call is taken to stream past the caches (4 MB of L2 a die, 256 MB
// behind them, shared with what the caller does next).  Past them / through them, us, every call
// on other tensors: forward and backward, 32 + 8 heads of 128, q of 32 MB 66 / 66, 64 MB
// 87 / 94, 128 MB 166 / 184, 256 MB 321 / 357; 16 + 16 heads of 64, 64 MB 142 / 155, 512 MB
// 1096 / 1196.  Forward with the window attention that reads its outputs: 16 MB 36.8 / 35.9
// (heads of 64, 32 MB: 74.9 / 73.0), 64 MB 94.9 / 94.8, 128 MB 176 / 178, 256 MB 336 / 340.
constexpr int64_t kStream = 64 << 20;

unsigned grid_of(int64_t units, int most) { return (unsigned)std::min<int64_t>((units + 3) / 4, most); }

bool streams(const PrepArgs& a, int B) { return (int64_t)B * a.N * a.H * a.D * 2 >= kStream; }

template <typename F>
int with_lanes(int D, F f) {
    switch (lanes_per_row(D)) {
        case 2: return f(std::integral_constant<int, 2>{});
        case 4: return f(std::integral_constant<int, 4>{});
        case 8: return f(std::integral_constant<int, 8>{});
        case 16: return f(std::integral_constant<int, 16>{});
        default: return f(std::integral_constant<int, 32>{});
    }
}

template <int DT, bool APPEND>
int launch_fwd(PrepArgs& a, int B, hipStream_t st) {
    const int rows = a.H + a.Hk + (APPEND ? a.Hk : 0);
    return with_lanes(a.D, [&](auto lg) {
        constexpr int LG = decltype(lg)::value;
        set_units(a, B, 1, rows);
        const bool few = a.units <= 4 * kFwdGrid, nt = streams(a, B);
        if (!few) set_units(a, B, kFwdGroups, rows);
        const dim3 g(grid_of(a.units, kFwdGrid)), t(256);
        if (few)
            hipLaunchKernelGGL((fta_norm_rope_fwd_kernel<DT, LG, 1, APPEND, false>), g, t, 0, st, a);
        else if (nt && !APPEND)
            hipLaunchKernelGGL((fta_norm_rope_fwd_kernel<DT, LG, kFwdGroups, APPEND, !APPEND>), g, t, 0, st, a);
        else
            hipLaunchKernelGGL((fta_norm_rope_fwd_kernel<DT, LG, kFwdGroups, APPEND, false>), g, t, 0, st, a);
        return fta::check_launch("fta_norm_rope_fwd_kernel");
    });
}

// One group a wave for as many waves as run at once (four a SIMD), five for more.  One / five, us of the kernel: 32 / 8
// heads of 128, 16 tokens 5.2 / 7.3, 256 6.0 / 7.9, 512 (6144 groups) 9.5 / 9.0, 1000 13.9 / 11.2, 2000 22.3 / 19.0,
// 8000 67.9 / 49.3; 8 / 8 heads of 64, 1000 tokens (3000 groups) 6.2 / 7.0, 2000 9.2 / 8.1; 12 / 4 of 80, 512
// tokens (2560) 6.0 / 7.7, 1000 (5000) 8.3 / 8.1, 4000 20.2 / 12.4; 16 / 2 of 256, 256 tokens (2560) 5.9 / 7.8, 512
// (5120) 8.7 / 8.3, 2000 21.2 / 15.0.
constexpr int kQ4Few = 4 * 1024;

template <int DT>
int launch_append_q4(PrepArgs& a, int B, hipStream_t st) {
    const int rows = a.H + 2 * a.Hk;
    return with_lanes(std::max(a.D, 32), [&](auto lg) {
        constexpr int LG = decltype(lg)::value < 4 ? 4 : decltype(lg)::value;
        set_units(a, B, 1, rows, LG);
        const bool few = a.units <= kQ4Few;
        if (!few) set_units(a, B, kFwdGroups, rows, LG);
        const dim3 g(grid_of(a.units, kFwdGrid)), t(256);
        if (few)
            hipLaunchKernelGGL((fta_norm_rope_append_q4_kernel<DT, LG, 1, false>), g, t, 0, st, a);
        else if (streams(a, B))
            hipLaunchKernelGGL((fta_norm_rope_append_q4_kernel<DT, LG, kFwdGroups, true>), g, t, 0, st, a);
        else
            hipLaunchKernelGGL((fta_norm_rope_append_q4_kernel<DT, LG, kFwdGroups, false>), g, t, 0, st, a);
        return fta::check_launch("fta_norm_rope_append_q4_kernel");
    });
}

template <int DT>
int launch_bwd(PrepArgs& a, int B, void* dqw, void* dkw, hipStream_t st) {
    return with_lanes(a.D, [&](auto lg) {
        constexpr int LG = decltype(lg)::value;
        set_units(a, B, kBwdGroups, a.H + a.Hk);
        const unsigned wgs = grid_of(a.units, kBwdGrid);
        if (streams(a, B))
            hipLaunchKernelGGL((fta_norm_rope_bwd_kernel<DT, LG, kBwdGroups, true>), dim3(wgs), dim3(256), 0, st, a);
        else
            hipLaunchKernelGGL((fta_norm_rope_bwd_kernel<DT, LG, kBwdGroups, false>), dim3(wgs), dim3(256), 0, st, a);
        int rc = fta::check_launch("fta_norm_rope_bwd_kernel");
        if (rc != FTA_OK || a.part == nullptr) return rc;
        hipLaunchKernelGGL(fta_norm_rope_dw_kernel, dim3(2 * a.D / 8), dim3(256), 0, st, a.part, (int)wgs, a.D, dqw, dkw,
                           a.w_dtype);
        return fta::check_launch("fta_norm_rope_dw_kernel");
    });
}

void set3(int64_t& sb, int64_t& sh, int64_t& sn, const int64_t* s) {
    sb = s[0];
    sh = s[1];
    sn = s[2];
}

int check_types(int dtype, int w_dtype) {
    if (dtype != FTA_DTYPE_BF16 && dtype != FTA_DTYPE_F16)
        return fta::arg_error("qk_norm_rope: dtype must be bf16 or fp16");
    if (w_dtype < 0 || w_dtype > FTA_DTYPE_F32) return fta::arg_error("qk_norm_rope: weights must be bf16, fp16 or fp32");
    return FTA_OK;
}

// What the appends to either cache have in common.
int append_args(PrepArgs& a, const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                const int64_t* v_strides, int dtype, int B, int H, int Hk, int T, int D, const void* q_weight,
                const void* k_weight, int weight_dtype, const float* cos, const float* sin, int P, int R, int position_offset,
                const int32_t* position_offsets, float eps, int interleaved, const int32_t* cache_lens, int S, void* q_out,
                const int64_t* qo_strides) {
    int rc = prep_geometry(B, H, Hk, T, D, R, P);
    if (rc != FTA_OK || (rc = check_types(dtype, weight_dtype)) != FTA_OK) return rc;
    if (!(eps > 0.f) || eps > 3.0e38f) return fta::arg_error("qk_norm_rope: eps must be positive and finite");
    if (S <= 0) return fta::arg_error("qk_norm_rope_append: the caches must have rows");
    if (!fta::all_set(q, q_strides, k, k_strides, v, v_strides, cos, sin, cache_lens, q_out, qo_strides))
        return fta::arg_error("qk_norm_rope_append: a required pointer is null");
    a.q = (const uint16_t*)q;
    a.k = (const uint16_t*)k;
    a.v = (const uint16_t*)v;
    a.qo = (uint16_t*)q_out;
    set3(a.q_sb, a.q_sh, a.q_sn, q_strides);
    set3(a.k_sb, a.k_sh, a.k_sn, k_strides);
    set3(a.v_sb, a.v_sh, a.v_sn, v_strides);
    set3(a.qo_sb, a.qo_sh, a.qo_sn, qo_strides);
    a.qw = q_weight, a.kw = k_weight, a.w_dtype = weight_dtype;
    a.cos = cos, a.sin = sin, a.P = P, a.R = R;
    a.lens = cache_lens, a.S = S, a.pos_off = position_offset, a.pos_offs = position_offsets;
    a.N = T, a.H = H, a.Hk = Hk, a.D = D, a.inter = interleaved != 0, a.eps = eps;
    return FTA_OK;
}

}  // namespace

extern "C" {

int fta_qk_norm_rope(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, int dtype, int B,
                     int H, int Hk, int N, int D, const void* q_weight, const void* k_weight, int weight_dtype,
                     const float* cos, const float* sin, int P, int R, const int32_t* positions,
                     int64_t positions_stride_b, float eps, int interleaved, void* q_out, const int64_t* qo_strides,
                     void* k_out, const int64_t* ko_strides, void* stream) {
    FTA_TRY_BEGIN
    int rc = prep_geometry(B, H, Hk, N, D, R, P);
    if (rc != FTA_OK || (rc = check_types(dtype, weight_dtype)) != FTA_OK) return rc;
    if (!(eps > 0.f) || eps > 3.0e38f) return fta::arg_error("qk_norm_rope: eps must be positive and finite");
    if (positions == nullptr && N > P) return fta::arg_error("qk_norm_rope: cos and sin have fewer rows than tokens");
    if (!fta::all_set(q, q_strides, k, k_strides, cos, sin, q_out, qo_strides, k_out, ko_strides))
        return fta::arg_error("qk_norm_rope: a required pointer is null");
    PrepArgs a = {};
    a.q = (const uint16_t*)q;
    a.k = (const uint16_t*)k;
    a.qo = (uint16_t*)q_out;
    a.ko = (uint16_t*)k_out;
    set3(a.q_sb, a.q_sh, a.q_sn, q_strides);
    set3(a.k_sb, a.k_sh, a.k_sn, k_strides);
    set3(a.qo_sb, a.qo_sh, a.qo_sn, qo_strides);
    set3(a.ko_sb, a.ko_sh, a.ko_sn, ko_strides);
    a.qw = q_weight, a.kw = k_weight, a.w_dtype = weight_dtype;
    a.cos = cos, a.sin = sin, a.P = P, a.R = R;
    a.positions = positions, a.pos_sb = positions_stride_b;
    a.N = N, a.H = H, a.Hk = Hk, a.D = D, a.inter = interleaved != 0, a.eps = eps;
    hipStream_t st = (hipStream_t)stream;
    return dtype == FTA_DTYPE_BF16 ? launch_fwd<FTA_DTYPE_BF16, false>(a, B, st) : launch_fwd<FTA_DTYPE_F16, false>(a, B, st);
    FTA_TRY_END
}

size_t fta_qk_norm_rope_bwd_workspace_size(int B, int H, int Hk, int N, int D) {
    if (prep_geometry(B, H, Hk, N, D, 16, 1) != FTA_OK) return 0;
    return fta::align_up((size_t)kBwdGrid * 2 * D * sizeof(float));
}

int fta_qk_norm_rope_bwd(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                         const void* dq_out, const int64_t* dqo_strides, const void* dk_out, const int64_t* dko_strides,
                         int dtype, int B, int H, int Hk, int N, int D, const void* q_weight, const void* k_weight,
                         int weight_dtype, const float* cos, const float* sin, int P, int R, const int32_t* positions,
                         int64_t positions_stride_b, float eps, int interleaved, void* dq, const int64_t* dq_strides,
                         void* dk, const int64_t* dk_strides, void* dq_weight, void* dk_weight, void* workspace,
                         size_t workspace_bytes, void* stream) {
    FTA_TRY_BEGIN
    int rc = prep_geometry(B, H, Hk, N, D, R, P);
    if (rc != FTA_OK || (rc = check_types(dtype, weight_dtype)) != FTA_OK) return rc;
    if (!(eps > 0.f) || eps > 3.0e38f) return fta::arg_error("qk_norm_rope: eps must be positive and finite");
    if (positions == nullptr && N > P) return fta::arg_error("qk_norm_rope: cos and sin have fewer rows than tokens");
    const bool dw = dq_weight != nullptr || dk_weight != nullptr;
    if (dw && (workspace == nullptr || workspace_bytes < fta_qk_norm_rope_bwd_workspace_size(B, H, Hk, N, D)))
        return fta::arg_error("qk_norm_rope_bwd: workspace too small");
    if (!fta::all_set(q, q_strides, k, k_strides, dq_out, dqo_strides, dk_out, dko_strides, cos, sin, dq, dq_strides, dk,
                      dk_strides))
        return fta::arg_error("qk_norm_rope_bwd: a required pointer is null");
    PrepArgs a = {};
    a.q = (const uint16_t*)q;
    a.k = (const uint16_t*)k;
    a.dqo = (const uint16_t*)dq_out;
    a.dko = (const uint16_t*)dk_out;
    a.qo = (uint16_t*)dq;
    a.ko = (uint16_t*)dk;
    set3(a.q_sb, a.q_sh, a.q_sn, q_strides);
    set3(a.k_sb, a.k_sh, a.k_sn, k_strides);
    set3(a.dq_sb, a.dq_sh, a.dq_sn, dqo_strides);
    set3(a.dk_sb, a.dk_sh, a.dk_sn, dko_strides);
    set3(a.qo_sb, a.qo_sh, a.qo_sn, dq_strides);
    set3(a.ko_sb, a.ko_sh, a.ko_sn, dk_strides);
    a.qw = q_weight, a.kw = k_weight, a.w_dtype = weight_dtype;
    a.cos = cos, a.sin = sin, a.P = P, a.R = R;
    a.positions = positions, a.pos_sb = positions_stride_b;
    a.N = N, a.H = H, a.Hk = Hk, a.D = D, a.inter = interleaved != 0, a.eps = eps;
    a.part = dw ? (float*)workspace : nullptr;
    hipStream_t st = (hipStream_t)stream;
    return dtype == FTA_DTYPE_BF16 ? launch_bwd<FTA_DTYPE_BF16>(a, B, dq_weight, dk_weight, st)
                                   : launch_bwd<FTA_DTYPE_F16>(a, B, dq_weight, dk_weight, st);
    FTA_TRY_END
}

int fta_qk_norm_rope_append(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                            const void* v, const int64_t* v_strides, int dtype, int B, int H, int Hk, int T, int D,
                            const void* q_weight, const void* k_weight, int weight_dtype, const float* cos,
                            const float* sin, int P, int R, int position_offset, float eps, int interleaved,
                            const int32_t* cache_lens, int S, void* q_out, const int64_t* qo_strides, void* k_cache,
                            const int64_t* kc_strides, void* v_cache, const int64_t* vc_strides, void* stream) {
    return fta_qk_norm_rope_append_at(q, q_strides, k, k_strides, v, v_strides, dtype, B, H, Hk, T, D, q_weight, k_weight,
                                      weight_dtype, cos, sin, P, R, position_offset, nullptr, eps, interleaved, cache_lens, S,
                                      q_out, qo_strides, k_cache, kc_strides, v_cache, vc_strides, stream);
}

int fta_qk_norm_rope_append_at(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                               const void* v, const int64_t* v_strides, int dtype, int B, int H, int Hk, int T, int D,
                               const void* q_weight, const void* k_weight, int weight_dtype, const float* cos,
                               const float* sin, int P, int R, int position_offset, const int32_t* position_offsets,
                               float eps, int interleaved, const int32_t* cache_lens, int S, void* q_out,
                               const int64_t* qo_strides, void* k_cache, const int64_t* kc_strides, void* v_cache,
                               const int64_t* vc_strides, void* stream) {
    FTA_TRY_BEGIN
    PrepArgs a = {};
    int rc = append_args(a, q, q_strides, k, k_strides, v, v_strides, dtype, B, H, Hk, T, D, q_weight, k_weight, weight_dtype,
                         cos, sin, P, R, position_offset, position_offsets, eps, interleaved, cache_lens, S, q_out, qo_strides);
    if (rc != FTA_OK) return rc;
    if (!fta::all_set(k_cache, kc_strides, v_cache, vc_strides))
        return fta::arg_error("qk_norm_rope_append: a required pointer is null");
    a.ko = (uint16_t*)k_cache;
    a.vo = (uint16_t*)v_cache;
    set3(a.ko_sb, a.ko_sh, a.ko_sn, kc_strides);
    set3(a.vo_sb, a.vo_sh, a.vo_sn, vc_strides);
    hipStream_t st = (hipStream_t)stream;
    return dtype == FTA_DTYPE_BF16 ? launch_fwd<FTA_DTYPE_BF16, true>(a, B, st) : launch_fwd<FTA_DTYPE_F16, true>(a, B, st);
    FTA_TRY_END
}

int fta_qk_norm_rope_append_q4(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                               const void* v, const int64_t* v_strides, int dtype, int B, int H, int Hk, int T, int D,
                               const void* q_weight, const void* k_weight, int weight_dtype, const float* cos,
                               const float* sin, int P, int R, int position_offset, const int32_t* position_offsets,
                               float eps, int interleaved, const int32_t* cache_lens, int S, void* q_out,
                               const int64_t* qo_strides, void* k_codes, const int64_t* kc_strides, void* k_scales,
                               const int64_t* ks_strides, void* v_codes, const int64_t* vc_strides, void* v_scales,
                               const int64_t* vs_strides, void* stream) {
    FTA_TRY_BEGIN
    PrepArgs a = {};
    int rc = append_args(a, q, q_strides, k, k_strides, v, v_strides, dtype, B, H, Hk, T, D, q_weight, k_weight, weight_dtype,
                         cos, sin, P, R, position_offset, position_offsets, eps, interleaved, cache_lens, S, q_out, qo_strides);
    if (rc != FTA_OK) return rc;
    if (!fta::all_set(k_codes, kc_strides, k_scales, ks_strides, v_codes, vc_strides, v_scales, vs_strides))
        return fta::arg_error("qk_norm_rope_append_q4: a required pointer is null");
    if ((((uintptr_t)k_codes | (uintptr_t)v_codes) & 3) != 0 || ((kc_strides[0] | kc_strides[1] | vc_strides[0] | vc_strides[1]) & 3) != 0)
        return fta::arg_error("qk_norm_rope_append_q4: codes must be 4-byte aligned");
    a.qk = {(uint32_t*)k_codes, (uint16_t*)k_scales, kc_strides[0] / 4, kc_strides[1] / 4, ks_strides[0], ks_strides[1]};
    a.qv = {(uint32_t*)v_codes, (uint16_t*)v_scales, vc_strides[0] / 4, vc_strides[1] / 4, vs_strides[0], vs_strides[1]};
    hipStream_t st = (hipStream_t)stream;
    return dtype == FTA_DTYPE_BF16 ? launch_append_q4<FTA_DTYPE_BF16>(a, B, st) : launch_append_q4<FTA_DTYPE_F16>(a, B, st);
    FTA_TRY_END
}

}  // extern "C"
