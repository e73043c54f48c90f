// Sliding-window attention with sinks, forward and backward.
//
// Query i of a sequence of len tokens sees key j when
//   j < len,  j <= i + right  and  (j >= i - left  or  j < sinks):
// a band around the diagonal and the first tokens, which stay visible to every later
// query.  o = sum_j p_ij v_j with p = softmax(scale q.k) over the visible keys, lse
// its log-sum; tokens at or past len give o = 0 and lse = -inf.  Backward, with
// delta = o . dO:  P = exp(scale q.k - lse),  dS = P (dO V^T - delta),
//   dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO.
//
// The walk of a workgroup is arithmetic, not a list: the 64-key tiles of the sinks,
// then those of its rows' band.  Per wave and tile the mask is one of three cases,
// told apart by scalar compares: nothing visible (skipped), everything (no mask), or,
// at the band's two edges, a word per row whose bits are the visible keys.
//
// Rows at or past len are never read: a tile that reaches them takes token len - 1 in
// their place (its scores are masked), so what padding holds cannot reach a result.
// Tiles inside the sequence are gathered whole, whether or not a row of the workgroup
// sees all their keys.
#include "fta_common.h"
#include "fta_host.h"
#include "fta_tile.h"

#include <algorithm>

namespace {

// Waves per workgroup of the forward and dQ.  Eight, whose K / V tiles serve twice the rows, keep
// a SIMD's two waves in step through each tile's barrier, so that both want the same pipe at
// the same time; two workgroups of four drift apart (32K tokens, 32 / 8 heads of 128, window
// 1024: forward 747 -> 733 us, dQ 1025 -> 944).  Two were slower on small grids too.
constexpr int kRowWaves = 4;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;

// The power of two that P carries into dV's product: the probabilities of long walks fall below
// fp16's normal range (2^-14) and would lose bits one by one; P <= 1 leaves room for 2^14 more.
// dK / dV read the lse less 14 and delta times 2^-14, so that P comes out scaled and dS does
// not; dV is scaled back in fp32.  bf16 has fp32's range.
template <int DT>
constexpr int kPBits = DT == FTA_DTYPE_F16 ? 14 : 0;
template <int DT>
constexpr float kPUnit = DT == FTA_DTYPE_F16 ? 0x1p-14f : 1.f;

struct WinArgs {
    const uint16_t *q, *k, *v, *o, *dout;
    int64_t q_sb, q_sh, q_sn, k_sb, k_sh, k_sn, v_sb, v_sh, v_sn, o_sb, o_sh, o_sn, d_sb, d_sh, d_sn;
    uint16_t *out0, *out1;  // o (forward), dq, or dk and dv
    int64_t o0_sb, o0_sh, o0_sn, o1_sb, o1_sh, o1_sn;
    const int32_t* lens;  // [B] or null
    float* lse;           // [B][H][N]: forward output, backward input
    float *lse2, *delta;  // [B][H][N] workspace: lse * log2(e) - kPBits and delta * kPUnit, from dQ to dK / dV
    float* part;          // dK / dV parts
    int B, N, H, Hk, G, Dreal;
    int left, right, sinks;
    float c, scale;
    int hw;               // forward, dQ: query heads per workgroup (they share K / V)
    int tiles;            // forward, dQ: token tiles per head; dK / dV: tiles of kt_keys keys
    int kt_keys;          // dK / dV: keys per tile
    int ts, nps, np;      // dK / dV: tiles that hold sinks, parts of each of them, parts of the others
    int total;
    bool kv_narrow, q_narrow, d_narrow;  // token strides that 32-bit lane offsets span
};

__device__ __forceinline__ int seq_len(const WinArgs& a, int b) {
    return a.lens ? __builtin_amdgcn_readfirstlane(min(max(a.lens[b], 0), a.N)) : a.N;
}

// The tiles of KEYS keys that rows [i_lo, i_hi] see: `ns` tiles of sinks, then the band's.
template <int KEYS>
struct WinWalk {
    int len, ns, c_lo, iters;
    __device__ __forceinline__ WinWalk(const WinArgs& a, int len_, int i_lo, int i_hi) : len(len_) {
        const int kb0 = max(0, i_lo - a.left), ke = min(len, i_hi + a.right + 1);  // the band's keys [kb0, ke)
        const int c_hi = (ke + KEYS - 1) / KEYS;
        c_lo = kb0 / KEYS;
        ns = (min(a.sinks, ke) + KEYS - 1) / KEYS;
        if (c_lo <= ns) c_lo = ns = 0;
        iters = ns + c_hi - c_lo;
    }
    // whether all rows of the tile at kb are tokens in front of len
    __device__ __forceinline__ bool whole(int kb) const { return kb + KEYS <= len; }
    // a token in front of len in place of one that is not
    __device__ __forceinline__ int seen(int t) const { return min(t, len - 1); }
};

// Walks the tiles in order: first key and its K and V rows, stepped (the multiplications were
// a good part of the scalar instructions of a tile).
template <int KEYS>
struct WinCursor {
    int it, kb;
    const uint16_t *k, *v;
    __device__ __forceinline__ WinCursor(const WinWalk<KEYS>& w, const WinArgs& a, const uint16_t* kp, const uint16_t* vp)
        : it(0), kb(w.ns > 0 ? 0 : w.c_lo * KEYS), k(kp + (int64_t)kb * a.k_sn), v(vp + (int64_t)kb * a.v_sn) {}
    __device__ __forceinline__ void next(const WinWalk<KEYS>& w, const WinArgs& a) {
        int d = KEYS;
        if (++it == w.ns) d = w.c_lo * KEYS - kb;  // from the sinks to the band
        kb += d;
        k += d * a.k_sn;
        v += d * a.v_sn;
    }
};

// What rows [i0, i0 + 31] see of the 32 keys at kb.
struct WinRows {
    int full_lo, full_hi;  // everything, for kb in [full_lo, full_hi]
    int any_lo, any_hi;    // something, for kb in [any_lo, any_hi] (or a sink)
    __device__ __forceinline__ WinRows(const WinArgs& a, int len, int i0) {
        full_lo = i0 + 31 - a.left;
        full_hi = min(i0 + a.right, len - 1) - 31;
        any_lo = i0 - a.left - 31;
        any_hi = min(i0 + 31, len - 1) + a.right;
        if (i0 >= len) full_hi = any_hi = -1;  // padding rows see nothing
    }
    __device__ __forceinline__ bool full(int kb) const { return kb >= full_lo && kb <= full_hi; }
    __device__ __forceinline__ bool none(const WinArgs& a, int kb) const { return kb > any_hi || (kb < any_lo && kb >= a.sinks); }
};

// Which of the 32 keys at kb row i sees (bit = key).
__device__ __forceinline__ uint32_t seen_keys(const WinArgs& a, int len, int i, int kb) {
    return fta_bits_below(min(i + a.right, len - 1) + 1 - kb) & (~fta_bits_below(i - a.left - kb) | fta_bits_below(a.sinks - kb));
}

// How many keys token i sees (sinks in front of the window and the window).
__device__ __forceinline__ int seen_count(const WinArgs& a, int len, int i) {
    return min(i + a.right, len - 1) - max(i - a.left, 0) + 1 + max(min(a.sinks, i - a.left), 0);
}
// Rows that see fewer keys than this take delta from their scores, see the dQ kernel.  Where all
// of them do (16384 tokens, 32 / 8 heads of 128, 41 tokens of window), forward and backward took
// 460 us without that walk and 462 with it; dQ's error falls from 1.5 to 2.3 roundings to 1.41.
constexpr int kFewKeys = 64;

// Workgroup -> (K/V head, b, head group, token tile).  An XCD takes an eighth of that order: heads
// outermost, so that it holds some of every sequence, however their lengths differ (8 sequences
// of 512 to 8192 tokens, 8 heads of 128, window 512: forward 216 -> 143 us, dQ 292 -> 196, dK /
// dV 409 -> 267 against sequences outermost).  Late tiles first: without a window they walk the
// most keys.
struct WinPlace {
    int b, h, hk, i0, i_lo, tok;  // batch, this wave's query head, its K/V head, its first row; the workgroup's first row, rows
    __device__ __forceinline__ WinPlace(const WinArgs& a, int wave) {
        const int wgi = fta_xcd_remap(blockIdx.x, a.total);
        const int per = fta_scalar(a.G / a.hw);  // head groups of a K/V head
        const int u = fta_scalar(wgi / a.tiles), tile = a.tiles - 1 - (wgi - u * a.tiles);
        const int kb = fta_scalar(u / per);
        const int wt = fta_scalar(wave / a.hw);
        hk = fta_scalar(kb / a.B);
        b = kb - hk * a.B;
        h = hk * a.G + (u - kb * per) * a.hw + wave - wt * a.hw;
        tok = 32 * fta_scalar(kRowWaves / a.hw);
        i_lo = tile * tok;
        i0 = i_lo + 32 * wt;
    }
};

// Stages of the forward and dQ: tiles of 32 NH keys of K and V, two in LDS.
template <int D, int NH>
struct WinShape {
    static constexpr int STAGE_B = 2 * NH * FtaTile<FTA_DTYPE_BF16, D>::TEN_B;
};
// waves per SIMD that the registers leave room for
constexpr int win_fwd_waves(int D) { return D <= 64 ? 4 : 2; }
constexpr int win_dq_waves(int D) { return D <= 64 ? 4 : D <= 128 ? 2 : 1; }

// ----------------------------------------------------------------------------
// Forward.  Four waves of 32 rows: hw query heads that share a K/V head, 4 / hw row
// tiles each; 64-key tiles of K and V (32 at D = 256), worked on 32 keys at a time so
// that the half tiles at the band's edges and the sinks' tile cost what they hold.
// What bounds it at D = 128: neither pipe alone, at a clock below the card's 2.4 GHz.  N32768, 32 / 8 heads of 128,
// window 1024, 4 sinks: 680 us, 845 TFLOP/s with the masked scores, 66% of a large library
// product on the same card; in one pass of 703 us at a clock of 1.88 GHz the matrix units
// were busy 44% of the cycles, the vector units 44%; more waves per SIMD (three, by 32-key stages)
// and other prefetch distances or wave priorities change it by under 4%.  Gathering the edge
// tiles whole took 74.6 -> 71.3 us at D = 64 (N10000 twice, 12 / 4 heads, 300 to both sides;
// 65 with the heads outermost) and 705 -> 681 here.  At D = 64 the vector instructions weigh
// most (67% of the cycles, the products 33%, so that the two hardly overlap): of 84 per 32
// x 32 scores (four cycles each, the 16 exp2 more) 64 are the fma, exp2, sum and packing of
// the softmax and 8 its maximum, against 8 MFMAs.
// D = 256 is held to 256 registers, two workgroups per CU: with 512 the compiler moved the
// whole accumulator through copies at every tile (N4096 twice, 16 / 2 heads, window 512: 150
// -> 94 us, 690 TFLOP/s without the masked scores).
// ----------------------------------------------------------------------------
template <int DT, int D, int NH>
__global__ __launch_bounds__(kRowWaves * 64, win_fwd_waves(D)) void fta_window_fwd_kernel(WinArgs a) {
    using T = FtaTile<DT, D>;
    using Sh = WinShape<D, NH>;
    constexpr int PD = D <= 128 ? 3 : 2;  // fragments read ahead
    constexpr int KEYS = 32 * NH;
    __shared__ __align__(1024) unsigned char sStage[2][Sh::STAGE_B];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const WinPlace p(a, wave);
    const int len = seq_len(a, p.b);
    const int row = p.i0 + (lane & 31);
    uint16_t* out = a.out0 + p.b * a.o0_sb + p.h * a.o0_sh + (int64_t)row * a.o0_sn;
    float* lse = a.lse + ((int64_t)p.b * a.H + p.h) * a.N;

    f32x16 oacc[T::DT32];
#pragma unroll
    for (int dt = 0; dt < T::DT32; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) oacc[dt][i] = 0.f;
    float m_run = -FTA_INF, l_run = 0.f;

    if (p.i_lo < len) {  // workgroup-uniform
        const uint16_t* kp = a.k + p.b * a.k_sb + p.hk * a.k_sh;
        const uint16_t* vp = a.v + p.b * a.v_sb + p.hk * a.v_sh;
        fta_frag qf[T::KS];
        T::load_rows(a.q + p.b * a.q_sb + p.h * a.q_sh + (int64_t)row * a.q_sn, row < len, a.Dreal, lane, qf);
        const WinWalk<KEYS> w(a, len, p.i_lo, min(p.i_lo + p.tok, len) - 1);
        const WinRows rows(a, len, p.i0);
        FtaGather<D, kRowWaves, KEYS> g;
        g.start(a.k_sn, a.v_sn, a.Dreal, wave, lane);
        const uint32_t lds0 = fta_lds_addr(&sStage[0][0]), ldsw = lds0 + 1024 * wave;
        const FtaAddr<D> ad0(lds0, lane);
        WinCursor<KEYS> at(w, a, kp, vp);  // the tile to gather
        auto issue = [&](int st) __attribute__((always_inline)) {
            const uint32_t lds = ldsw + st * Sh::STAGE_B;
            if (a.kv_narrow && w.whole(at.kb))
                g.whole(at.k, at.v, lds);
            else
                g.mapped(kp, vp, a.k_sn, a.v_sn, at.kb, a.Dreal, lds, wave, lane, [&](int t) { return w.seen(t); });
            at.next(w, a);
        };
        fta_wait_vmcnt<0>();  // register loads complete before the DMA stream, which the compiler does not count
        int kb = at.kb, it = 0;
        issue(0);
        // one tile, in stage ST: the stages alternate in the code, so that every LDS address is a
        // kept register and a constant
        auto tile = [&](auto st) __attribute__((always_inline)) {
            constexpr int ST = decltype(st)::value;
            fta_wait_vmcnt<0>();
            __syncthreads();  // tile `it` visible; every wave is past tile it - 1
            const int next = at.kb;
            if (++it < w.iters) issue(ST ^ 1);
#pragma unroll
            for (int sb = 0; sb < NH; ++sb) {
                const int kh = kb + 32 * sb;
                const bool full = rows.full(kh);
                if (!full && rows.none(a, kh)) continue;
                constexpr uint32_t KO = ST * Sh::STAGE_B, VO = KO + NH * T::TEN_B;
                const uint32_t ho = sb * T::TEN_B;
                const FtaAddr<D> ad = ad0.here();
                f32x16 s;
                T::template qk<PD>(ad, KO + ho, qf, s);
                if (!full) T::mask(seen_keys(a, len, row, kh), lane, s);
                T::template softmax_pv<PD>(ad, VO + ho, s, a.c, m_run, l_run, oacc);
            }
            kb = next;
        };
        while (it < w.iters) {
            tile(std::integral_constant<int, 0>{});
            if (it < w.iters) tile(std::integral_constant<int, 1>{});
        }
    }

    const float L = l_run + fta_xor32(l_run);
    if (row >= a.N) return;
    const bool live = row < len;
    if (lane < 32) lse[row] = live ? fmaf(m_run, a.c, fta_log2(L)) * kLn2 : -FTA_INF;
    if (!live) {  // a padding row: exact zeros, whatever the registers hold
#pragma unroll
        for (int dt = 0; dt < T::DT32; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) oacc[dt][i] = 0.f;
    }
    T::store_row(out, a.Dreal, lane, oacc, live ? 1.f / L : 0.f);
}

// ----------------------------------------------------------------------------
// dQ, with the forward's walk: S^T and dP^T = V dO^T of 32 keys at a time,
// dS^T = P^T (dP^T - delta), dQ^T += K^T dS^T.  It also forms delta and the lse in log2 units
// for dK / dV.
//
// delta = o . dO, summed in fp32 from the rounded o (both rows are at hand): its error, a rounding
// of o, is in every dS of the row alike and shrinks with the number n of keys that the row sees:
// dQ and dK are off by 2.3 times a rounding of the exact ones for n = 2, 1.6 for 8, 1.5 for 32
// and 1.43 to 1.47 from 64 on, of which 1.41 are the rounding of dS.  A workgroup with rows of
// fewer than 64 keys forms delta = sum_j P_ij dP_ij in fp32 instead, by a first walk over its keys
// without dQ's product (1.41 for every n); in a causal sequence that is the first tile of each head.
// dS is rounded to 16 bits for its product with K (in dK's kernel with Q), as P is in the forward.
// Bound as the forward is: N32768, 32 / 8 heads of 128, window 1024: 886 us, 973 TFLOP/s
// with the masked scores; N10000 twice, 12 / 4 heads of 64, 300 to both sides: 82 us.
// ----------------------------------------------------------------------------
template <int DT, int D, int NH>
__global__ __launch_bounds__(kRowWaves * 64, win_dq_waves(D)) void fta_window_dq_kernel(WinArgs a) {
    using E = Elem<DT>;
    using T = FtaTile<DT, D>;
    using Sh = WinShape<D, NH>;
    constexpr int KEYS = 32 * NH, KS = T::KS;
    __shared__ __align__(1024) unsigned char sStage[2][Sh::STAGE_B];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const WinPlace p(a, wave);
    const int len = seq_len(a, p.b);
    const int row = p.i0 + (lane & 31);
    const bool live = row < len;

    f32x16 acc[T::DT32];
#pragma unroll
    for (int dt = 0; dt < T::DT32; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[dt][i] = 0.f;

    if (p.i_lo < len) {  // workgroup-uniform
        const uint16_t* kp = a.k + p.b * a.k_sb + p.hk * a.k_sh;
        const uint16_t* vp = a.v + p.b * a.v_sb + p.hk * a.v_sh;
        fta_frag qf[KS], df[KS];
        T::load_rows(a.q + p.b * a.q_sb + p.h * a.q_sh + (int64_t)row * a.q_sn, live, a.Dreal, lane, qf);
        T::load_rows(a.dout + p.b * a.d_sb + p.h * a.d_sh + (int64_t)row * a.d_sn, live, a.Dreal, lane, df);
        const int64_t at_row = ((int64_t)p.b * a.H + p.h) * a.N + row;
        const float lse2 = live ? a.lse[at_row] * kLog2e : FTA_INF;  // a padding row: every exp is exactly 0
        float dl = 0.f;
        const int i_hi = min(p.i_lo + p.tok, len) - 1;
        const bool few = min(seen_count(a, len, p.i_lo), seen_count(a, len, i_hi)) < kFewKeys;  // workgroup-uniform
        if (!few) {
            const uint16_t* op = a.o + p.b * a.o_sb + p.h * a.o_sh + (int64_t)row * a.o_sn;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const int d = ks * 16 + (lane >> 5) * 8;
                const fta_frag of = (live && d < a.Dreal) ? *reinterpret_cast<const fta_frag*>(op + d) : fta_frag{0u, 0u, 0u, 0u};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    dl = fmaf(E::to_f32((uint16_t)(of[e] & 0xffffu)), E::to_f32((uint16_t)(df[ks][e] & 0xffffu)), dl);
                    dl = fmaf(E::to_f32((uint16_t)(of[e] >> 16)), E::to_f32((uint16_t)(df[ks][e] >> 16)), dl);
                }
            }
            dl += fta_xor32(dl);
        }
        const WinWalk<KEYS> w(a, len, p.i_lo, i_hi);
        const WinRows rows(a, len, p.i0);
        FtaGather<D, kRowWaves, KEYS> g;
        g.start(a.k_sn, a.v_sn, a.Dreal, wave, lane);
        const uint32_t lds0 = fta_lds_addr(&sStage[0][0]), ldsw = lds0 + 1024 * wave;
        const FtaAddr<D> ad0(lds0, lane);
        // the walk; FIRST: it only sums delta = sum over keys of P dP
        auto walk = [&](auto first) __attribute__((always_inline)) {
            constexpr bool FIRST = decltype(first)::value;
            WinCursor<KEYS> at(w, a, kp, vp);  // the tile to gather
            auto issue = [&](int st) __attribute__((always_inline)) {
                const uint32_t lds = ldsw + st * Sh::STAGE_B;
                if (a.kv_narrow && w.whole(at.kb))
                    g.whole(at.k, at.v, lds);
                else
                    g.mapped(kp, vp, a.k_sn, a.v_sn, at.kb, a.Dreal, lds, wave, lane, [&](int t) { return w.seen(t); });
                at.next(w, a);
            };
            fta_wait_vmcnt<0>();  // register loads and stores complete before the DMA stream, which the compiler does not count
            int kb = at.kb, it = 0;
            issue(0);
            // one tile, in stage ST: the stages alternate in the code, so that every LDS address is a
            // kept register and a constant
            auto tile = [&](auto st) __attribute__((always_inline)) {
                constexpr int ST = decltype(st)::value;
                fta_wait_vmcnt<0>();
                __syncthreads();  // tile `it` visible; every wave is past tile it - 1
                const int next = at.kb;
                if (++it < w.iters) issue(ST ^ 1);
#pragma unroll
                for (int sb = 0; sb < NH; ++sb) {
                    const int kh = kb + 32 * sb;
                    const bool full = rows.full(kh);
                    if (!full && rows.none(a, kh)) continue;
                    constexpr uint32_t KO = ST * Sh::STAGE_B, VO = KO + NH * T::TEN_B;
                    const uint32_t ho = sb * T::TEN_B;
                    const FtaAddr<D> ad = ad0.here();
                    f32x16 s, dp;
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[i] = dp[i] = 0.f;
                    fta_frag kf[2], vf[2], dsf[2];  // K and V fragments one MFMA pair ahead
                    kf[0] = ad.row(KO + ho, 0);
                    vf[0] = ad.row(VO + ho, 0);
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) {
                        if (ks + 1 < KS) {
                            kf[(ks + 1) & 1] = ad.row(KO + ho, ks + 1);
                            vf[(ks + 1) & 1] = ad.row(VO + ho, ks + 1);
                        }
                        s = fta_mma<DT>(kf[ks & 1], qf[ks], s);
                        dp = fta_mma<DT>(vf[ks & 1], df[ks], dp);
                    }
                    if (!full) T::mask(seen_keys(a, len, row, kh), lane, s);
                    if constexpr (FIRST) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) dl = fmaf(fta_exp2(fmaf(s[i], a.c, -lse2)), dp[i], dl);
                        continue;
                    }
#pragma unroll
                    for (int k2 = 0; k2 < 2; ++k2) {
                        float ds[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int i = 8 * k2 + e;
                            ds[e] = fta_exp2(fmaf(s[i], a.c, -lse2)) * (dp[i] - dl);
                        }
                        dsf[k2] = fta_pack_frag<DT>(ds);
                    }
#pragma unroll
                    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                        for (int dt = 0; dt < T::DT32; ++dt) acc[dt] = fta_mma<DT>(ad.tr(KO + ho, ks, dt), dsf[ks], acc[dt]);
                }
                kb = next;
            };
            while (it < w.iters) {
                tile(std::integral_constant<int, 0>{});
                if (it < w.iters) tile(std::integral_constant<int, 1>{});
            }
        };
        if (few) {
            walk(std::true_type{});
            dl += fta_xor32(dl);
            __syncthreads();  // every wave has read the last tile
        }
        if (live && lane < 32) {
            a.delta[at_row] = dl * kPUnit<DT>;
            a.lse2[at_row] = lse2 - kPBits<DT>;
        }
        walk(std::false_type{});
    }
    if (row < a.N)
        T::store_row(a.out0 + p.b * a.o0_sb + p.h * a.o0_sh + (int64_t)row * a.o0_sn, a.Dreal, lane, acc, a.scale);
}

// ----------------------------------------------------------------------------
// dK / dV at D = 256, where one wave's keys' rows and both accumulators would take every
// register: a workgroup owns 64 keys of one K/V head, wave (tt, 0) holds K of 32-key tile
// tt and accumulates dV, wave (tt, 1) holds V and accumulates dK one chunk behind; P
// crosses in fp32 through LDS:
//   wave (tt, 0):  S = Q K^T,  P = 2^{c S - lse2}  -> LDS;  dV += P^T dO
//   wave (tt, 1):  dP = dO V^T;  dS = P (dP - delta);  dK += dS^T Q
// One barrier per step; Q two steps ahead in four tiles, dO in three.  One workgroup per CU,
// so each step waits out its own barrier and LDS latencies: N4096, 8 heads of 256, window
// 512: 100 us; N8192, causal: 765 us, 720 TFLOP/s.
//
// This kernel and the next walk the 32-query chunks that see any of the workgroup's keys,
// through all query heads of the group in one sequence, so the sums over shared heads need
// neither atomics nor a second pass.  The tiles that hold sinks are seen by every later
// query: their walks are cut into nps parts as long as the other tiles' walks, and on small
// grids every walk into np parts; parts write fp32 sums that
// fta_window_dkv_combine_kernel adds in order.
// ----------------------------------------------------------------------------
template <int D>
struct WinDkvSplitShape {
    static constexpr int NW = 4, NTHR = 256, QSEG = D / 8;
    static constexpr int LQ = 32 * QSEG / NTHR;  // DMA instructions per wave and 32-row tile
    static constexpr int TILE_B = 32 * QSEG * 16;
    static constexpr int NQ = 4, ND = 3;
    static_assert((32 * QSEG) % NTHR == 0, "whole DMA instructions per wave");
};

template <int DT, int D>
__global__ __launch_bounds__(256, 1) void fta_window_dkv_split_kernel(WinArgs a) {
    using E = Elem<DT>;
    using Sh = WinDkvSplitShape<D>;
    constexpr int NW = Sh::NW, QSEG = Sh::QSEG, LQ = Sh::LQ, TILE_B = Sh::TILE_B;
    using SW = FtaSwz<QSEG>;
    constexpr int KS = D / 16, DT32 = D / 32;
    __shared__ __align__(1024) unsigned char sQ[Sh::NQ][TILE_B];
    __shared__ __align__(1024) unsigned char sD[Sh::ND][TILE_B];
    __shared__ __align__(1024) float sL[Sh::NQ][64];  // [lse of entry k, delta of entry k - 1] at k % 4
    __shared__ float4 sX[2][2][4][64];                // [step parity][tile][i / 4][lane]: P of the last two steps

    const int wgi = fta_xcd_remap(blockIdx.x, a.total);
    const int per = a.ts * a.nps + (a.tiles - a.ts) * a.np;  // workgroups per (b, K/V head)
    const int kbi = fta_scalar(wgi / per), slot = wgi - kbi * per;
    const bool sink = slot < a.ts * a.nps;
    const int parts = sink ? a.nps : a.np;
    const int off = sink ? slot : slot - a.ts * a.nps;
    const int tp = fta_scalar(off / parts);
    const int tile = sink ? tp : a.ts + tp;
    const int sp = off - tp * parts;
    const int hk = fta_scalar(kbi / a.B), b = kbi - hk * a.B;  // heads outermost, as in WinPlace
    const int bhk = b * a.Hk + hk;
    const int len = seq_len(a, b);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int hf = lane >> 5;
    const int tt = wave & 1;
    const bool hv = (wave >> 1) != 0;  // wave-uniform role: false = K / P / dV, true = V / dS / dK

    const int kb = 64 * tile, kt = kb + 32 * tt;  // first key of the workgroup, of this wave's tile
    const int key = kt + (lane & 31);             // this lane's column
    const bool kok = key < len;

    // entries [s0, s0 + U) of the sequence (query head, chunk of 32 queries)
    int c_lo = 0, nch = 0;
    if (kb < len) {
        c_lo = max(0, kb - a.right) >> 5;
        const int i_hi = kb < a.sinks ? len - 1 : min(len - 1, min(kb + 63, len - 1) + a.left);
        nch = (i_hi >> 5) + 1 - c_lo;
    }
    const int all = a.G * nch;
    const int s0 = fta_scalar((int)((int64_t)all * sp / parts));
    const int U = fta_scalar((int)((int64_t)all * (sp + 1) / parts)) - s0;

    fta_frag kv[KS];  // K (role 0) or V (role 1) rows of this tile
    {
        const uint16_t* src = hv ? a.v + b * a.v_sb + hk * a.v_sh + (int64_t)key * a.v_sn
                                 : a.k + b * a.k_sb + hk * a.k_sh + (int64_t)key * a.k_sn;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int d = ks * 16 + hf * 8;
            kv[ks] = (kok && d < a.Dreal) ? *reinterpret_cast<const fta_frag*>(src + d) : fta_frag{0u, 0u, 0u, 0u};
        }
    }
    fta_wait_vmcnt<0>();  // complete the register loads: the DMAs are invisible to the compiler

    uint32_t qoff[LQ], doff[LQ];
#pragma unroll
    for (int i = 0; i < LQ; ++i) {
        const int r2 = (i * NW + wave) * 64 + lane;
        const int row = r2 / QSEG;
        int j = SW::slot(row, r2 - row * QSEG);
        if (j * 8 >= a.Dreal) j = 0;  // columns past D: any finite data (never stored)
        qoff[i] = 2u * (row * (uint32_t)a.q_sn + j * 8);
        doff[i] = 2u * (row * (uint32_t)a.d_sn + j * 8);
    }
    const bool l_isd = (lane & 32) != 0;  // wave 0's DMA writes [lse2 32][delta 32]
    const uint32_t aro = 2u * SW::off(lane & 31, hf);
    const int br = 4 * hf + ((lane & 15) >> 2), bc = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    const uint32_t bro = 2u * (SW::off(br, bc >> 3) + (bc & 7));
    const uint32_t bro8 = 2u * (SW::off(br + 8, bc >> 3) + (bc & 7)) - bro;  // added: rows + 8
    const uint32_t ldq = fta_lds_addr(&sQ[0][0]), ldd = fta_lds_addr(&sD[0][0]), ldl = fta_lds_addr(&sL[0][0]);
    const uint16_t* q0 = a.q + b * a.q_sb + (int64_t)hk * a.G * a.q_sh;
    const uint16_t* d0 = a.dout + b * a.d_sb + (int64_t)hk * a.G * a.d_sh;
    const int64_t r0 = ((int64_t)b * a.H + (int64_t)hk * a.G) * a.N;

    // the rest runs in one copy per role, so each keeps only its own values live
    auto run = [&](auto role) {
        constexpr bool HV = decltype(role)::value;
        f32x16 acc[DT32];  // dV (role 0) or dK / scale (role 1): rows = keys, lane column = d
#pragma unroll
        for (int dt = 0; dt < DT32; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[dt][i] = 0.f;

        if (U > 0) {
            // the 32 rows from `base`, chunk c of their head
            auto tile_dma = [&](const uint16_t* base, int64_t sn, bool narrow, const uint32_t* o, int c, uint32_t lds)
                __attribute__((always_inline)) {
                if (narrow && 32 * c + 32 <= len) {
#pragma unroll
                    for (int i = 0; i < LQ; ++i) fta_dma16_so(base, o[i], lds + (i * NW + wave) * 1024);
                } else {  // the sequence's last chunk repeats its last row (masked)
                    int ln = lane;
                    asm volatile("" : "+v"(ln));
#pragma unroll
                    for (int i = 0; i < LQ; ++i) {
                        const int r2 = (i * NW + wave) * 64 + ln;
                        const int row = r2 / QSEG;
                        int j = SW::slot(row, r2 - row * QSEG);
                        if (j * 8 >= a.Dreal) j = 0;
                        const int64_t t = min(row, len - 1 - 32 * c);
                        fta_dma16_at(base + t * sn + j * 8, lds + (i * NW + wave) * 1024);
                    }
                }
            };
            // A (query head, chunk) entry of the walk: the chunk, its Q and dO rows, and the row of
            // its lse and delta.  The addresses are stepped, not multiplied out: at 128 scalar
            // instructions a step the scalar unit was as busy as the matrix unit.
            struct Entry {
                int c;
                const uint16_t *q, *d;
                int64_t r;
            };
            const int c_end = c_lo + nch, last = s0 + U - 1;
            const int64_t q_step = 32 * a.q_sn, d_step = 32 * a.d_sn;
            const int64_t q_turn = a.q_sh - (nch - 1) * q_step, d_turn = a.d_sh - (nch - 1) * d_step;
            const int64_t r_turn = a.N - 32 * (int64_t)(nch - 1);
            // entry s after entry s - 1 (past the end: the last one again, so every step issues the same number)
            auto next = [&](Entry e, int s) __attribute__((always_inline)) {
                if (s > last) return e;
                const bool turn = e.c + 1 == c_end;  // on to the next query head's first chunk
                return Entry{turn ? c_lo : e.c + 1, e.q + (turn ? q_turn : q_step), e.d + (turn ? d_turn : d_step),
                             e.r + (turn ? r_turn : 32)};
            };
            // step k - 2's gathers: Q and lse of entry eq (number kq), dO and delta of entry ed (kq - 1)
            auto issue = [&](int kq, int dslot, const Entry& eq, const Entry& ed) __attribute__((always_inline)) {
                tile_dma(eq.q, a.q_sn, a.q_narrow, qoff, eq.c, ldq + (kq & 3) * TILE_B);
                tile_dma(ed.d, a.d_sn, a.d_narrow, doff, ed.c, ldd + dslot * TILE_B);
                if (wave == 0) {
                    const int c = l_isd ? ed.c : eq.c;
                    const float* src = l_isd ? a.delta + ed.r : a.lse2 + eq.r;
                    fta_dma4_at(src + min(lane & 31, len - 1 - 32 * c), ldl + (kq & 3) * 256);
                }
            };
            // mask case of chunk c for this wave's keys
            auto mcase = [&](int c) __attribute__((always_inline)) {
                const int i0 = 32 * c;
                if (kt >= len || i0 + 31 < kt - a.right || (i0 > kt + 31 + a.left && kt >= a.sinks)) return 0;
                if (i0 >= kt + 31 - a.right && i0 + 31 < len && kt + 31 < len && (i0 + 31 <= kt + a.left || kt + 31 < a.sinks))
                    return 2;
                return 1;
            };
            const int g0 = fta_scalar(s0 / nch);
            const int c0 = c_lo + s0 - g0 * nch;
            Entry e1{c0, q0 + g0 * a.q_sh + c0 * q_step, d0 + g0 * a.d_sh + c0 * d_step, r0 + (int64_t)g0 * a.N + 32 * (int64_t)c0};
            int mk = mcase(c0), mkp = 0, ck = c0;
            issue(0, 2, e1, e1);
            Entry e2 = next(e1, s0 + 1);
            issue(1, 0, e2, e1);
            e1 = e2;                   // entry k + 1
            e2 = next(e1, s0 + 2);     // entry k + 2
            int ds = 2;                // dO slot of entry k - 1
            fta_frag af[2];               // role 0: P_{k-1}, A operand of dV_{k-1}
            for (int k = 0; k <= U; ++k) {
                // step k - 2's gathers complete (wave 0 issues the lse / delta DMA as well)
                if (wave == 0)
                    fta_wait_vmcnt<2 * LQ + 1>();
                else
                    fta_wait_vmcnt<2 * LQ>();
                // Q_k, dO_{k-1} and P_{k-1} visible; the slots of Q_{k-2}, dO_{k-2} and sX[k & 1] free
                __syncthreads();
                issue(k + 2, ds == 0 ? 2 : ds - 1, e2, e1);
                const float* ld = &sL[k & 3][0];
                const uint32_t dbase = ldd + ds * TILE_B;
                if constexpr (!HV) {
                    const uint32_t qb = ldq + (k & 3) * TILE_B + aro, ob = dbase + bro;
                    if (mkp == 0) af[0] = af[1] = fta_frag{0u, 0u, 0u, 0u};
                    // S_k (a dependent chain) interleaved with dV_{k-1} (independent MFMAs).
                    // One instruction stream for every case: without a pending accumulation P is
                    // zero and dO any finite tile; without a chain the S result is discarded.
                    if (mk | mkp) {
                        f32x16 own;  // S_k then P_k
#pragma unroll
                        for (int i = 0; i < 16; ++i) own[i] = 0.f;
                        fta_frag fs[2], fa2[2];
                        auto load = [&](int j, int sl) {
                            fs[sl] = fta_lds_frag(qb ^ (j * 32));
                            const uint32_t x = (j / DT32) * 16 * QSEG * 16;
                            fa2[sl] = fta_lds_tr_frag((ob ^ ((j % DT32) * 64)) + x, ((ob + bro8) ^ ((j % DT32) * 64)) + x);
                        };
                        load(0, 0);
#pragma unroll
                        for (int j = 0; j < KS; ++j) {  // KS = 2 * DT32: one accumulation MFMA per chain link
                            if (j + 1 < KS) load(j + 1, (j + 1) & 1);
                            own = fta_mma<DT>(fs[j & 1], kv[j], own);
                            acc[j % DT32] = fta_mma<DT>(af[j / DT32], fa2[j & 1], acc[j % DT32]);
                        }
                        __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
#pragma unroll
                        for (int j = 0; j < KS; ++j) {
                            if (j + 1 < KS) __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
                            __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
                        }
                        if (mk) {  // P_k = 2^{c S_k - lse2}: to LDS for role 1, packed for dV_k
#pragma unroll
                            for (int i = 0; i < 16; ++i) own[i] = fta_exp2(fmaf(own[i], a.c, -ld[c_row(i, lane)]));
                            if (mk == 1) {  // the lane's key is seen by rows [rlo, rhi] of the chunk
                                const int rlo = key - a.right - 32 * ck;
                                const int rhi = (kok ? min(key < a.sinks ? len - 1 : key + a.left, len - 1) : -1) - 32 * ck;
#pragma unroll
                                for (int i = 0; i < 16; ++i) {
                                    const int r = c_row(i, lane);
                                    own[i] = (r >= rlo && r <= rhi) ? own[i] : 0.f;
                                }
                            }
#pragma unroll
                            for (int i = 0; i < 16; i += 4)
                                sX[k & 1][tt][i / 4][lane] = make_float4(own[i], own[i + 1], own[i + 2], own[i + 3]);
#pragma unroll
                            for (int ks = 0; ks < 2; ++ks) {
                                float p8[8];
#pragma unroll
                                for (int e = 0; e < 8; ++e) p8[e] = own[8 * ks + e];
                                af[ks] = fta_pack_frag<DT>(p8);
                            }
                        }
                    }
                } else if (mkp) {
                    const uint32_t ob = dbase + aro, qb = ldq + ((k + 3) & 3) * TILE_B + bro;
                    f32x16 dpv;
#pragma unroll
                    for (int i = 0; i < 16; ++i) dpv[i] = 0.f;
                    {
                        constexpr int PD = 3;
                        fta_frag fr[PD + 1];
                        auto load = [&](auto nn) __attribute__((always_inline)) {
                            constexpr int n = decltype(nn)::value;
                            if constexpr (n < KS) fr[n % (PD + 1)] = fta_lds_frag(ob ^ (n * 32));
                        };
                        auto slot_ = [&](auto nn) __attribute__((always_inline)) {
                            constexpr int n = decltype(nn)::value;
                            load(std::integral_constant<int, n + PD>{});
                            dpv = fta_mma<DT>(fr[n % (PD + 1)], kv[n], dpv);
                        };
                        fta_static_for<0, PD>(load);
                        fta_static_for<0, KS>(slot_);
                    }
                    fta_frag ds2[2];  // dS = P (dP - delta)
#pragma unroll
                    for (int ks = 0; ks < 2; ++ks) {
                        float dv8[8];
#pragma unroll
                        for (int e = 0; e < 8; e += 4) {
                            const int i = 8 * ks + e;
                            const float4 pr = sX[(k + 1) & 1][tt][i / 4][lane];
                            const float4 dl = *reinterpret_cast<const float4*>(ld + 32 + c_row(i, lane));
                            dv8[e] = pr.x * fmaf(dpv[i], kPUnit<DT>, -dl.x);
                            dv8[e + 1] = pr.y * fmaf(dpv[i + 1], kPUnit<DT>, -dl.y);
                            dv8[e + 2] = pr.z * fmaf(dpv[i + 2], kPUnit<DT>, -dl.z);
                            dv8[e + 3] = pr.w * fmaf(dpv[i + 3], kPUnit<DT>, -dl.w);
                        }
                        ds2[ks] = fta_pack_frag<DT>(dv8);
                    }
                    {
                        constexpr int PD = 3;
                        fta_frag fr[PD + 1];
                        auto load = [&](auto nn) __attribute__((always_inline)) {
                            constexpr int n = decltype(nn)::value;
                            if constexpr (n < KS) {
                                constexpr int x = (n / DT32) * 16 * QSEG * 16;
                                fr[n % (PD + 1)] = fta_lds_tr_frag((qb ^ ((n % DT32) * 64)) + x, ((qb + bro8) ^ ((n % DT32) * 64)) + x);
                            }
                        };
                        auto slot_ = [&](auto nn) __attribute__((always_inline)) {
                            constexpr int n = decltype(nn)::value;
                            load(std::integral_constant<int, n + PD>{});
                            acc[n % DT32] = fta_mma<DT>(ds2[n / DT32], fr[n % (PD + 1)], acc[n % DT32]);
                        };
                        fta_static_for<0, PD>(load);
                        fta_static_for<0, KS>(slot_);
                    }
                }
                mkp = mk;
                mk = (k + 1 < U) ? mcase(e1.c) : 0;
                ck = e1.c;
                e1 = e2;
                e2 = next(e2, s0 + k + 3);
                ds = (ds == 2) ? 0 : ds + 1;
            }
            fta_wait_vmcnt<0>();  // the gathers past the walk's end
        }

        // C layout: lane column = d, rows = keys c_row(i, lane); role 0 stores dV, role 1 dK
        if (parts > 1) {
            float* po = a.part + ((((int64_t)(HV ? 0 : 1) * a.B * a.Hk + bhk) * (a.np > 1 ? per : a.ts * a.nps) + slot) * 64 + 32 * tt) * D;
#pragma unroll
            for (int dt = 0; dt < DT32; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) po[(int64_t)c_row(i, lane) * D + dt * 32 + (lane & 31)] = acc[dt][i];
            return;
        }
        uint16_t* out = HV ? a.out0 + b * a.o0_sb + hk * a.o0_sh : a.out1 + b * a.o1_sb + hk * a.o1_sh;
        const int64_t osn = HV ? a.o0_sn : a.o1_sn;
        const float osc = HV ? a.scale : kPUnit<DT>;
#pragma unroll
        for (int dt = 0; dt < DT32; ++dt) {
            const int d = dt * 32 + (lane & 31);
            if (d >= a.Dreal) continue;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int t = kt + c_row(i, lane);
                if (t < a.N) out[(int64_t)t * osn + d] = (uint16_t)(E::pack2(acc[dt][i] * osc, 0.f) & 0xffffu);
            }
        }
    };
    if (hv)
        run(std::true_type{});
    else
        run(std::false_type{});
}

// ----------------------------------------------------------------------------
// dK / dV up to D = 128: four waves of 32 keys, each with its keys' K and V rows and both
// accumulators in registers, so a 32-query chunk of Q and dO serves 128 keys and P never
// leaves the wave:
//   S = Q K^T,  dP = dO V^T,  P = 2^{c S - lse2},  dS = P (dP - delta)  (P and delta in kPUnit),
//   dV += P^T dO,  dK += dS^T Q.
// At D = 128 that is 250 registers, two workgroups per CU; 158 and three at D = 64.  Against
// 64 keys a workgroup with the work of a tile split over two waves (the kernel above):
// half the gathers and barriers, no exchange of P.  N32768, 32 / 8 heads of 128, window
// 1024: 1510 -> 1150 us, 1000 TFLOP/s with the masked scores; N10000 twice, 12 / 4 heads of 64,
// 300 to both sides: 175 -> 104.  Three stages instead of two change nothing.
// ----------------------------------------------------------------------------
template <int D>
struct WinDkvShape {
    static constexpr int NW = 4, KEYS = 128, QSEG = D / 8;
    static constexpr int LQ = 32 * QSEG / 256;
    static constexpr int TILE_B = 32 * QSEG * 16;
};

template <int DT, int D>
__global__ __launch_bounds__(256, D <= 64 ? 3 : 2) void fta_window_dkv_kernel(WinArgs a) {
    using E = Elem<DT>;
    using Sh = WinDkvShape<D>;
    using T = FtaTile<DT, D>;
    constexpr int NW = Sh::NW, QSEG = Sh::QSEG, LQ = Sh::LQ, TILE_B = Sh::TILE_B;
    using SW = FtaSwz<QSEG>;
    constexpr int KS = D / 16, DT32 = D / 32;
    __shared__ __align__(1024) unsigned char sStage[2][2 * TILE_B];  // Q, dO
    __shared__ __align__(1024) float sL[2][64];                       // lse2, delta

    const int wgi = fta_xcd_remap(blockIdx.x, a.total);
    const int per = a.ts * a.nps + (a.tiles - a.ts) * a.np;  // workgroups per (b, K/V head)
    const int kbi = fta_scalar(wgi / per), slot = wgi - kbi * per;
    const bool sink = slot < a.ts * a.nps;
    const int parts = sink ? a.nps : a.np;
    const int off = sink ? slot : slot - a.ts * a.nps;
    const int tp = fta_scalar(off / parts);
    const int tile = sink ? tp : a.ts + tp;
    const int sp = off - tp * parts;
    const int hk = fta_scalar(kbi / a.B), b = kbi - hk * a.B;  // heads outermost, as in WinPlace
    const int bhk = b * a.Hk + hk;
    const int len = seq_len(a, b);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kb = Sh::KEYS * tile, kt = kb + 32 * wave;

    int c_lo = 0, nch = 0;
    if (kb < len) {
        c_lo = max(0, kb - a.right) >> 5;
        const int i_hi = kb < a.sinks ? len - 1 : min(len - 1, min(kb + Sh::KEYS - 1, len - 1) + a.left);
        nch = (i_hi >> 5) + 1 - c_lo;
    }
    const int all = a.G * nch;
    const int s0 = fta_scalar((int)((int64_t)all * sp / parts));
    const int U = fta_scalar((int)((int64_t)all * (sp + 1) / parts)) - s0;

    f32x16 dk[DT32], dv[DT32];
#pragma unroll
    for (int dt = 0; dt < DT32; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) dk[dt][i] = dv[dt][i] = 0.f;

    if (U > 0) {
        fta_frag kf[KS], vf[KS];
        const int key = kt + (lane & 31);
        const bool kok = key < len;
        T::load_rows(a.k + b * a.k_sb + hk * a.k_sh + (int64_t)key * a.k_sn, kok, a.Dreal, lane, kf);
        T::load_rows(a.v + b * a.v_sb + hk * a.v_sh + (int64_t)key * a.v_sn, kok, a.Dreal, lane, vf);
        fta_wait_vmcnt<0>();
        // Per-lane DMA source: instruction 0 fills row drow; the others lie 256 / QSEG rows down
        // each, a multiple of 16, where the swizzle repeats: the same lane offset from a base
        // further down.
        constexpr int STEP = 256 / QSEG;
        static_assert(STEP % 16 == 0, "the swizzle repeats");
        const int drow = (wave * 64 + lane) / QSEG;
        int dcol = SW::slot(drow, (wave * 64 + lane) % QSEG) * 8;
        if (dcol >= a.Dreal) dcol = 0;  // columns past D: any finite data (never stored)
        const uint32_t qoff = 2u * (drow * (uint32_t)a.q_sn + dcol), doff = 2u * (drow * (uint32_t)a.d_sn + dcol);
        const bool l_isd = (lane & 32) != 0;
        const uint32_t lds0 = fta_lds_addr(&sStage[0][0]), ldsw = lds0 + 1024 * wave, ldl = fta_lds_addr(&sL[0][0]);
        const FtaAddr<D, (D <= 64)> ad0(lds0, lane);
        const int64_t q_step = 32 * a.q_sn, d_step = 32 * a.d_sn;
        const int64_t q_turn = a.q_sh - (nch - 1) * q_step, d_turn = a.d_sh - (nch - 1) * d_step;
        const int64_t r_turn = a.N - 32 * (int64_t)(nch - 1);
        const int g0 = fta_scalar(s0 / nch), c_end = c_lo + nch;
        int ci = c_lo + s0 - g0 * nch, cc = ci;  // chunk to gather, chunk to work on
        const uint16_t* qp = a.q + b * a.q_sb + ((int64_t)hk * a.G + g0) * a.q_sh + ci * q_step;
        const uint16_t* dp = a.dout + b * a.d_sb + ((int64_t)hk * a.G + g0) * a.d_sh + ci * d_step;
        int64_t rp = ((int64_t)b * a.H + (int64_t)hk * a.G + g0) * a.N + 32 * (int64_t)ci;

        // 32 rows of chunk ci from `base`
        auto tile_dma = [&](const uint16_t* base, int64_t sn, bool narrow, uint32_t o, uint32_t lds)
            __attribute__((always_inline)) {
            if (narrow && 32 * ci + 32 <= len) {
                auto one = [&](auto ii) __attribute__((always_inline)) {
                    constexpr int i = decltype(ii)::value;
                    fta_dma16_to<i * NW * 1024>(base + i * STEP * sn, o, lds);
                };
                fta_static_for<0, LQ>(one);
            } else {  // the sequence's last chunk repeats its last row (masked); formed here, kept nowhere
                int ln = lane;
                asm volatile("" : "+v"(ln));
#pragma unroll
                for (int i = 0; i < LQ; ++i) {
                    const int r2 = (i * NW + wave) * 64 + ln;
                    const int row = r2 / QSEG;
                    int j = SW::slot(row, r2 - row * QSEG);
                    if (j * 8 >= a.Dreal) j = 0;
                    const int64_t t = min(row, len - 1 - 32 * ci);
                    fta_dma16_at(base + t * sn + j * 8, lds + i * NW * 1024);
                }
            }
        };
        auto issue = [&](int st) __attribute__((always_inline)) {
            tile_dma(qp, a.q_sn, a.q_narrow, qoff, ldsw + st * 2 * TILE_B);
            tile_dma(dp, a.d_sn, a.d_narrow, doff, ldsw + st * 2 * TILE_B + TILE_B);
            if (wave == 0) {
                const float* src = l_isd ? a.delta + rp : a.lse2 + rp;
                fta_dma4_at(src + min(lane & 31, len - 1 - 32 * ci), ldl + st * 256);
            }
            const bool turn = ci + 1 == c_end;  // on to the next query head's first chunk
            ci = turn ? c_lo : ci + 1;
            qp += turn ? q_turn : q_step;
            dp += turn ? d_turn : d_step;
            rp += turn ? r_turn : 32;
        };
        // rows [32 c, 32 c + 31] see all of this wave's keys for c in [full_lo, full_hi], some of them
        // for c in [any_lo, any_hi] (any later ones too where the keys hold sinks)
        const int full_lo = (max(kt + 31 - a.right, 0) + 31) >> 5, any_lo = max(kt - a.right, 0) >> 5;
        const int full_hi = kt + 31 < len ? (min(kt + 31 < a.sinks ? len - 1 : kt + a.left, len - 1) - 31) >> 5 : -1;
        const int any_hi = kt >= len ? -1 : kt < a.sinks ? len >> 5 : (kt + 31 + a.left) >> 5;
        int k = 0;
        issue(0);
        auto chunk = [&](auto st_) __attribute__((always_inline)) {
            constexpr int ST = decltype(st_)::value;
            constexpr uint32_t QO = ST * 2 * TILE_B, OO = QO + TILE_B;
            fta_wait_vmcnt<0>();
            __syncthreads();  // chunk k visible; every wave is past chunk k - 1
            const int c = cc;
            cc = ci;
            if (++k < U) issue(ST ^ 1);
            if (c >= any_lo && c <= any_hi) {
                const bool whole = c >= full_lo && c <= full_hi;
                const int i0 = 32 * c;
                const float* ld = &sL[ST][0];
                const auto ad = ad0.here();
                f32x16 s, dpv;
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = dpv[i] = 0.f;
                {
                    fta_frag fq[2], fo[2];
                    fq[0] = ad.row(QO, 0);
                    fo[0] = ad.row(OO, 0);
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) {
                        if (ks + 1 < KS) {
                            fq[(ks + 1) & 1] = ad.row(QO, ks + 1);
                            fo[(ks + 1) & 1] = ad.row(OO, ks + 1);
                        }
                        s = fta_mma<DT>(fq[ks & 1], kf[ks], s);
                        dpv = fta_mma<DT>(fo[ks & 1], vf[ks], dpv);
                    }
                }
                if (!whole) {
                    // query rows [rlo, rhi] of the chunk see this lane's key: bit = row
                    int ln = lane;
                    asm volatile("" : "+v"(ln));
                    const int key = kt + (ln & 31);
                    const int rlo = key - a.right - i0;
                    const int rhi = (key < len ? min(key < a.sinks ? len - 1 : key + a.left, len - 1) : -1) - i0;
                    T::mask(fta_bits_below(rhi + 1) & ~fta_bits_below(rlo), lane, s);
                }
                fta_frag pf[2], df[2];
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
                    float p8[8], d8[8];
#pragma unroll
                    for (int e = 0; e < 8; e += 4) {
                        const int i = 8 * ks + e;
                        const float4 l4 = *reinterpret_cast<const float4*>(ld + c_row(i, lane));
                        const float4 e4 = *reinterpret_cast<const float4*>(ld + 32 + c_row(i, lane));
                        p8[e] = fta_exp2(fmaf(s[i], a.c, -l4.x));
                        p8[e + 1] = fta_exp2(fmaf(s[i + 1], a.c, -l4.y));
                        p8[e + 2] = fta_exp2(fmaf(s[i + 2], a.c, -l4.z));
                        p8[e + 3] = fta_exp2(fmaf(s[i + 3], a.c, -l4.w));
                        d8[e] = p8[e] * fmaf(dpv[i], kPUnit<DT>, -e4.x);
                        d8[e + 1] = p8[e + 1] * fmaf(dpv[i + 1], kPUnit<DT>, -e4.y);
                        d8[e + 2] = p8[e + 2] * fmaf(dpv[i + 2], kPUnit<DT>, -e4.z);
                        d8[e + 3] = p8[e + 3] * fmaf(dpv[i + 3], kPUnit<DT>, -e4.w);
                    }
                    pf[ks] = fta_pack_frag<DT>(p8);
                    df[ks] = fta_pack_frag<DT>(d8);
                }
                {
                    constexpr int PD = 2, NM = 4 * DT32;  // dV and dK in turn
                    fta_frag fr[PD + 1];
                    auto load = [&](auto nn) __attribute__((always_inline)) {
                        constexpr int n = decltype(nn)::value;
                        if constexpr (n < NM) fr[n % (PD + 1)] = ad.tr((n & 1) ? QO : OO, n / 2 / DT32, n / 2 % DT32);
                    };
                    auto slot_ = [&](auto nn) __attribute__((always_inline)) {
                        constexpr int n = decltype(nn)::value, ks = n / 2 / DT32, dt = n / 2 % DT32;
                        if constexpr (n % 2 == 0) __builtin_amdgcn_sched_barrier(0);
                        load(std::integral_constant<int, n + PD>{});
                        if constexpr ((n & 1) == 0)
                            dv[dt] = fta_mma<DT>(pf[ks], fr[n % (PD + 1)], dv[dt]);
                        else
                            dk[dt] = fta_mma<DT>(df[ks], fr[n % (PD + 1)], dk[dt]);
                    };
                    fta_static_for<0, PD>(load);
                    fta_static_for<0, NM>(slot_);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        };
        while (k < U) {
            chunk(std::integral_constant<int, 0>{});
            if (k < U) chunk(std::integral_constant<int, 1>{});
        }
    }

    // C layout: lane column = d, rows = keys c_row(i, lane)
    if (parts > 1) {
        const int64_t slots = a.np > 1 ? per : a.ts * a.nps;
        float* pk = a.part + (((int64_t)bhk * slots + slot) * Sh::KEYS + 32 * wave) * D;
        float* pv = pk + (int64_t)a.B * a.Hk * slots * Sh::KEYS * D;
#pragma unroll
        for (int dt = 0; dt < DT32; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int64_t at = (int64_t)c_row(i, lane) * D + dt * 32 + (lane & 31);
                pk[at] = dk[dt][i];
                pv[at] = dv[dt][i];
            }
        return;
    }
    uint16_t* ok = a.out0 + b * a.o0_sb + hk * a.o0_sh;
    uint16_t* ov = a.out1 + b * a.o1_sb + hk * a.o1_sh;
#pragma unroll
    for (int dt = 0; dt < DT32; ++dt) {
        const int d = dt * 32 + (lane & 31);
        if (d >= a.Dreal) continue;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int t = kt + c_row(i, lane);
            if (t >= a.N) continue;
            const uint32_t pk = E::pack2(dk[dt][i] * a.scale, dv[dt][i] * kPUnit<DT>);
            ok[(int64_t)t * a.o0_sn + d] = (uint16_t)(pk & 0xffffu);
            ov[(int64_t)t * a.o1_sn + d] = (uint16_t)(pk >> 16);
        }
    }
}

// Sum of the dK / dV parts: SL threads per (tensor, b, K/V head, key of a tile with parts,
// 8 columns) add every SL-th part and then their sums, always in the same order; dK takes
// the scale here.  (One thread for all parts of a tile took 17.6 us for 58 parts.)
template <int DT, int D, int SL>
__global__ __launch_bounds__(256) void fta_window_dkv_combine_kernel(WinArgs a, int keys) {
    using E = Elem<DT>;
    constexpr int DC = D / 8, ROWS = 256 / (DC * SL);
    __shared__ float so[SL][ROWS * D];
    const int dc = threadIdx.x % DC, sl = threadIdx.x / DC % SL, rr = threadIdx.x / (DC * SL);
    const int64_t rows = (int64_t)a.B * a.Hk * keys;
    int64_t row = (int64_t)blockIdx.x * ROWS + rr;
    const bool ok = row < 2 * rows;
    const int ten = row >= rows;  // 0: dK, 1: dV
    row = ok ? row - ten * rows : 0;
    const int t = (int)(row % keys), bhk = (int)(row / keys);
    constexpr int KEYS = D <= 128 ? 128 : 64;  // of a tile
    const int tile = t / KEYS, d0 = dc * 8;
    const int slots = a.ts * a.nps + (a.np > 1 ? (a.tiles - a.ts) * a.np : 0);
    const int n = tile < a.ts ? a.nps : a.np;
    const int first = tile < a.ts ? tile * a.nps : a.ts * a.nps + (tile - a.ts) * a.np;
    float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (ok && n > 1) {
        const float* src = a.part + ((((int64_t)ten * a.B * a.Hk + bhk) * slots + first) * KEYS + t % KEYS) * D + d0;
        for (int p = sl; p < n; p += SL) {
            const float4 x0 = *reinterpret_cast<const float4*>(src + (int64_t)p * KEYS * D);
            const float4 x1 = *reinterpret_cast<const float4*>(src + (int64_t)p * KEYS * D + 4);
            o[0] += x0.x, o[1] += x0.y, o[2] += x0.z, o[3] += x0.w;
            o[4] += x1.x, o[5] += x1.y, o[6] += x1.z, o[7] += x1.w;
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) so[sl][rr * D + d0 + e] = o[e];
    __syncthreads();
    if (sl != 0 || !ok || n <= 1 || d0 >= a.Dreal) return;  // n <= 1: written by the kernel itself
    const float f = ten ? kPUnit<DT> : a.scale;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
#pragma unroll
        for (int i = 1; i < SL; ++i) o[e] += so[i][rr * D + d0 + e];
        o[e] *= f;
    }
    const int b = bhk / a.Hk, hk = bhk - b * a.Hk;
    uint16_t* op = ten ? a.out1 + b * a.o1_sb + hk * a.o1_sh + (int64_t)t * a.o1_sn + d0
                       : a.out0 + b * a.o0_sb + hk * a.o0_sh + (int64_t)t * a.o0_sn + d0;
    *reinterpret_cast<uint4*>(op) = make_uint4(E::pack2(o[0], o[1]), E::pack2(o[2], o[3]), E::pack2(o[4], o[5]),
                                               E::pack2(o[6], o[7]));
}

// ---------------------------------------------------------------------- host

constexpr int64_t kMaxGrid = (1 << 24) - 1;  // workgroups of 256 threads: fewer than 2^32 threads a launch

int kernel_dim(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }
bool narrow(int64_t sn) { return sn >= 0 && sn <= (1 << 24); }

// Arguments that forward and backward share; the window is clamped to the sequence.
int win_common(WinArgs& a, const void* q, const int64_t* qs, const void* k, const int64_t* ks, const void* v,
               const int64_t* vs, int dtype, int B, int H, int Hk, int N, int D, const int32_t* lens, int left, int right,
               int sinks, float scale) {
    if (B <= 0 || H <= 0 || Hk <= 0 || N <= 0 || D <= 0) return fta::arg_error("window_attn: dims must be positive");
    if (H % Hk != 0) return fta::arg_error("window_attn: num_heads must be a multiple of num_kv_heads");
    if (D % 16 != 0 || D > 256) return fta::arg_error("window_attn: D must be a multiple of 16 up to 256");
    if (left < 0 || right < 0 || sinks < 0) return fta::arg_error("window_attn: window and num_sinks must be non-negative");
    if (!(scale > 0.f) || scale > 2.0e38f)  // times log2(e) still finite
        return fta::arg_error("window_attn: scale must be positive and at most 2e38");
    if (dtype != FTA_DTYPE_BF16 && dtype != FTA_DTYPE_F16) return fta::arg_error("window_attn: dtype must be bf16 or fp16");
    if (N > (1 << 29)) return fta::unsupported("window_attn: more than 2^29 tokens");
    if (!fta::size_fits(B, N, H, D)) return fta::unsupported("window_attn: 2^60 elements and more");
    if (!fta::all_set(qs, ks, vs)) return fta::arg_error("window_attn: strides are null");
    a = WinArgs{};
    a.q = (const uint16_t*)q, a.q_sb = qs[0], a.q_sh = qs[1], a.q_sn = qs[2];
    a.k = (const uint16_t*)k, a.k_sb = ks[0], a.k_sh = ks[1], a.k_sn = ks[2];
    a.v = (const uint16_t*)v, a.v_sb = vs[0], a.v_sh = vs[1], a.v_sn = vs[2];
    a.lens = lens;
    a.B = B, a.N = N, a.H = H, a.Hk = Hk, a.G = H / Hk, a.Dreal = D;
    a.left = std::min(left, N), a.right = std::min(right, N);
    a.sinks = a.left >= N - 1 ? 0 : std::min(sinks, N);  // a window of everything has no sinks left
    a.scale = scale;
    a.c = scale * kLog2e;
    a.kv_narrow = narrow(a.k_sn) && narrow(a.v_sn);
    a.q_narrow = narrow(a.q_sn);
    return FTA_OK;
}

// Grid of the forward and dQ: a workgroup takes as many query heads of a K/V head as
// divide both its waves and the group.
int64_t row_grid(WinArgs& a) {
    a.hw = 1;
    while (a.hw * 2 <= kRowWaves && a.G % (a.hw * 2) == 0) a.hw *= 2;
    const int tok = 32 * (kRowWaves / a.hw);
    a.tiles = (a.N + tok - 1) / tok;
    return (int64_t)a.B * (a.H / a.hw) * a.tiles;
}

template <int DT, int D>
int launch_rows(WinArgs& a, bool dq, hipStream_t st) {
    const int64_t grid = row_grid(a);
    if (grid > kMaxGrid) return fta::unsupported("window_attn: too many tokens");
    a.total = (int)grid;
    if (dq)
        hipLaunchKernelGGL((fta_window_dq_kernel<DT, D, 2>), dim3((unsigned)grid), dim3(kRowWaves * 64), 0, st, a);
    else
        hipLaunchKernelGGL((fta_window_fwd_kernel<DT, D, (D <= 128 ? 2 : 1)>), dim3((unsigned)grid), dim3(kRowWaves * 64), 0, st, a);
    return fta::check_launch(dq ? "fta_window_dq_kernel" : "fta_window_fwd_kernel");
}

// Parts of the dK / dV walks.  Grids that leave CUs idle cut every walk into up to 4 parts of
// at least 8 steps (N1024, 4 heads of 128, causal: 47 us whole, 19.4 + 5 with their sum in
// 4; N2048, 8 on 2 heads of 64, window 256: 52 + 4.6 -> 18.4 + 5.4), but not shorter ones
// (N2048, 8 heads of 128, window 256, 13 steps: 26.9 + 4.8 whole, 21.4 + 12.4 in 2).  The
// tiles with sinks get parts as long as the other walks, 2048 in all (268 MB of parts at D =
// 128), which is what fills the card several times over.
void dkv_parts(WinArgs& a) {
    a.kt_keys = a.Dreal <= 128 ? 128 : 64;
    a.tiles = (a.N + a.kt_keys - 1) / a.kt_keys;
    a.ts = (a.sinks + a.kt_keys - 1) / a.kt_keys;
    const int64_t wgs = (int64_t)a.tiles * a.B * a.Hk;
    const int64_t nall = (a.N + 31) / 32;
    const int64_t steps = a.G * std::min<int64_t>(nall, ((int64_t)a.kt_keys + a.left + a.right + 31) / 32 + 1);
    const int64_t np = std::max<int64_t>(1, std::min<int64_t>({4, 256 / wgs, steps / 8}));
    a.np = (int)np;
    const int64_t own = std::max<int64_t>(8, steps / np);
    const int64_t sink_wgs = (int64_t)a.ts * a.B * a.Hk;
    a.nps = a.ts == 0 ? 1
                      : (int)std::max<int64_t>(np, std::min<int64_t>({128, (a.G * nall + own - 1) / own, 2048 / sink_wgs}));
}

int64_t dkv_slots(const WinArgs& a) {
    return (a.nps > 1 ? (int64_t)a.ts * a.nps : 0) + (a.np > 1 ? (int64_t)(a.tiles - a.ts) * a.np : 0);
}
size_t rows_bytes(int B, int H, int N) { return fta::align_up((size_t)B * H * N * sizeof(float)); }
size_t part_bytes(const WinArgs& a, int Dk) {
    return fta::align_up((size_t)2 * a.B * a.Hk * dkv_slots(a) * a.kt_keys * Dk * sizeof(float));
}

template <int DT, int D>
int launch_dkv(WinArgs& a, hipStream_t st) {
    const int64_t grid = ((int64_t)a.ts * a.nps + (int64_t)(a.tiles - a.ts) * a.np) * a.B * a.Hk;
    if (grid > kMaxGrid) return fta::unsupported("window_attn: too many tokens");
    a.total = (int)grid;
    if constexpr (D <= 128)
        hipLaunchKernelGGL((fta_window_dkv_kernel<DT, D>), dim3((unsigned)grid), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((fta_window_dkv_split_kernel<DT, D>), dim3((unsigned)grid), dim3(256), 0, st, a);
    int rc = fta::check_launch("fta_window_dkv_kernel");
    if (rc != FTA_OK || (a.np <= 1 && (a.ts == 0 || a.nps <= 1))) return rc;
    const int keys = a.np > 1 ? a.N : std::min(a.N, a.ts * a.kt_keys);
    // many parts of few keys (the sinks alone), or a few parts of every key
    constexpr int SLF = 256 / (D / 8) < 16 ? 256 / (D / 8) : 16;
    const int sl = a.np > 1 ? 4 : SLF, per = 256 / (D / 8 * sl);
    const int64_t wgs = (2 * (int64_t)a.B * a.Hk * keys + per - 1) / per;
    if (wgs > kMaxGrid) return fta::unsupported("window_attn: too many tokens");
    if (a.np > 1)
        hipLaunchKernelGGL((fta_window_dkv_combine_kernel<DT, D, 4>), dim3((unsigned)wgs), dim3(256), 0, st, a, keys);
    else
        hipLaunchKernelGGL((fta_window_dkv_combine_kernel<DT, D, SLF>), dim3((unsigned)wgs), dim3(256), 0, st, a, keys);
    return fta::check_launch("fta_window_dkv_combine_kernel");
}

template <typename F>
int with_shape(int dtype, int D, F f) {
    auto dim = [&](auto dt) {
        switch (kernel_dim(D)) {
            case 64: return f(dt, std::integral_constant<int, 64>{});
            case 128: return f(dt, std::integral_constant<int, 128>{});
            default: return f(dt, std::integral_constant<int, 256>{});
        }
    };
    return dtype == FTA_DTYPE_BF16 ? dim(std::integral_constant<int, FTA_DTYPE_BF16>{})
                                   : dim(std::integral_constant<int, FTA_DTYPE_F16>{});
}

}  // namespace

extern "C" {

int fta_window_attn_fwd(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                        const int64_t* v_strides, int dtype, int B, int H, int Hk, int N, int D, const int32_t* seq_lens,
                        int left, int right, int num_sinks, float scale, void* o, const int64_t* o_strides, float* lse,
                        void* stream) {
    FTA_TRY_BEGIN
    WinArgs a;
    int rc = win_common(a, q, q_strides, k, k_strides, v, v_strides, dtype, B, H, Hk, N, D, seq_lens, left, right,
                        num_sinks, scale);
    if (rc != FTA_OK) return rc;
    if (!fta::all_set(q, k, v, o, o_strides, lse))
        return fta::arg_error("window_attn: a required pointer is null");
    a.out0 = (uint16_t*)o, a.o0_sb = o_strides[0], a.o0_sh = o_strides[1], a.o0_sn = o_strides[2];
    a.lse = lse;
    return with_shape(dtype, D, [&](auto dt, auto dk) {
        return launch_rows<decltype(dt)::value, decltype(dk)::value>(a, false, (hipStream_t)stream);
    });
    FTA_TRY_END
}

size_t fta_window_attn_bwd_workspace_size(int B, int H, int Hk, int N, int D, int left, int right, int num_sinks) {
    const int64_t none[3] = {0, 0, 0};
    WinArgs a;
    if (win_common(a, nullptr, none, nullptr, none, nullptr, none, FTA_DTYPE_BF16, B, H, Hk, N, D, nullptr, left, right,
                   num_sinks, 1.f) != FTA_OK)
        return 0;
    dkv_parts(a);
    return 2 * rows_bytes(B, H, N) + part_bytes(a, kernel_dim(D));
}

int fta_window_attn_bwd(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                        const int64_t* v_strides, const void* o, const int64_t* o_strides, const void* dout,
                        const int64_t* do_strides, int dtype, int B, int H, int Hk, int N, int D, const int32_t* seq_lens,
                        int left, int right, int num_sinks, float scale, const float* lse, void* dq,
                        const int64_t* dq_strides, void* dk, const int64_t* dk_strides, void* dv,
                        const int64_t* dv_strides, void* workspace, size_t workspace_bytes, void* stream) {
    FTA_TRY_BEGIN
    WinArgs a;
    int rc = win_common(a, q, q_strides, k, k_strides, v, v_strides, dtype, B, H, Hk, N, D, seq_lens, left, right,
                        num_sinks, scale);
    if (rc != FTA_OK) return rc;
    if (workspace == nullptr || workspace_bytes < fta_window_attn_bwd_workspace_size(B, H, Hk, N, D, left, right, num_sinks))
        return fta::arg_error("window_attn_bwd: workspace too small");
    if (!fta::all_set(q, k, v, o, o_strides, dout, do_strides, lse, dq, dq_strides, dk, dk_strides, dv, dv_strides))
        return fta::arg_error("window_attn_bwd: a required pointer is null");
    a.o = (const uint16_t*)o, a.o_sb = o_strides[0], a.o_sh = o_strides[1], a.o_sn = o_strides[2];
    a.dout = (const uint16_t*)dout, a.d_sb = do_strides[0], a.d_sh = do_strides[1], a.d_sn = do_strides[2];
    a.d_narrow = narrow(a.d_sn);
    a.lse = const_cast<float*>(lse);
    a.lse2 = (float*)workspace;
    a.delta = (float*)((char*)workspace + rows_bytes(B, H, N));
    a.part = (float*)((char*)workspace + 2 * rows_bytes(B, H, N));
    hipStream_t st = (hipStream_t)stream;
    // dQ first: it leaves delta and the lse in log2 units for dK / dV
    a.out0 = (uint16_t*)dq, a.o0_sb = dq_strides[0], a.o0_sh = dq_strides[1], a.o0_sn = dq_strides[2];
    rc = with_shape(dtype, D, [&](auto dt, auto dkk) {
        return launch_rows<decltype(dt)::value, decltype(dkk)::value>(a, true, st);
    });
    if (rc != FTA_OK) return rc;
    a.out0 = (uint16_t*)dk, a.o0_sb = dk_strides[0], a.o0_sh = dk_strides[1], a.o0_sn = dk_strides[2];
    a.out1 = (uint16_t*)dv, a.o1_sb = dv_strides[0], a.o1_sh = dv_strides[1], a.o1_sn = dv_strides[2];
    dkv_parts(a);
    return with_shape(dtype, D, [&](auto dt, auto dkk) { return launch_dkv<decltype(dt)::value, decltype(dkk)::value>(a, st); });
    FTA_TRY_END
}

}  // extern "C"
