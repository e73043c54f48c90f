// How much attention each cached key received, added to a running sum:
//   w[b][hk][j] += sum over new tokens t and the query heads of hk of exp(scale q_t . k_j - lse_t)
// for the tokens that see key j (as in fta_cache_attn: the last T of len_b tokens, token t at
// p = len_b - T + t sees j <= p with j >= p - left or j < sinks).  lse is the attention's own
// log-sum, so nothing is normalised here.  T is 1 for a step of a serving batch and the prompt's
// length for a prompt; keys are 16-bit rows or rows of a 4-bit cache (see fta_q4.hip).
//
// S = Q K^T with the keys as columns: a wave keeps 32 keys in registers, one to a lane and its
// mirror, and walks over all the rows that see them, 32 at a time; a key's terms stay in these lanes, two
// (of few rows, four), whose sums are added in a fixed order at the end of a walk or tile.
// So a key is read once and there are no atomics (the same bits every run).
// Many rows come through LDS, shared by the four waves: TT tokens x GG query heads of the group,
// as many heads as it takes to fill 32 rows where there are few tokens.
#include "fta_common.h"
#include "fta_host.h"
#include "fta_q4.h"
#include "fta_tile.h"

#include <algorithm>

namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct WeighArgs {
    const uint16_t* q;
    int64_t q_sb, q_sh, q_sn;
    const uint8_t* k;  // 16-bit rows, or codes
    int64_t k_sb, k_sh, k_sn;  // bytes
    const uint16_t* ks;  // scales of 4-bit rows
    int64_t ks_sb, ks_sh;
    const float* lse;  // [B][H][T]
    const int32_t* lens;
    float* w;
    int64_t w_sb, w_sh;
    float* part;  // [part][B * Hk][S]
    int B, T, H, Hk, G, S, Dreal, left, sinks;
    int GG, TT, groups;  // query heads and tokens of 32 rows; head groups of a K/V head
    int tiles, per, np, total;  // key tiles; chunks of 32 rows in a part, parts of the longest walk
    float c;
    int chunks;   // of 32 rows, where they all stay in LDS; else 0
    bool few;     // the rows stay in registers
    bool narrow;  // a chunk's rows are within 32-bit offsets
};

constexpr int kWeighWaves = 4, kWeighKeys = 32 * kWeighWaves;

// The walk of a workgroup's keys from k_lo: chunks [c_lo, c_lo + nct) of TT tokens that see any of them,
// for each head group.
struct WeighWalk {
    int c_lo = 0, nct = 0;
    __device__ __forceinline__ WeighWalk(const WeighArgs& a, int len, int k_lo) {
        if (k_lo >= len) return;
        const int p0 = len - a.T;  // position of the first new token
        const int t_lo = max(0, k_lo - p0);
        const int64_t far = (int64_t)min(k_lo + kWeighKeys, len) - 1 + a.left - p0;
        const int t_hi = k_lo < a.sinks ? a.T - 1 : (int)min(far, (int64_t)a.T - 1);
        c_lo = fta_scalar(t_lo / a.TT);
        if (t_hi >= t_lo) nct = fta_scalar(t_hi / a.TT) + 1 - c_lo;
    }
};

// 32 keys, one to a lane and its mirror, as they are loaded, and as B operands.
template <int DT, int KD, bool Q4>
struct KeyRows {
    static constexpr int KS = KD / 16, NG = KD / 32;
    uint32_t w[Q4 ? 2 * NG : 4 * KS];
    uint16_t d[Q4 ? NG : 1];
    __device__ __forceinline__ void load(const WeighArgs& a, int b, int hk, int64_t row, bool ok, int lane) {
        const int hf = lane >> 5;
        const uint8_t* p = a.k + b * a.k_sb + hk * a.k_sh + row * a.k_sn;
        if constexpr (Q4) {
            const uint32_t* kp = reinterpret_cast<const uint32_t*>(p);
            const uint16_t* scales = a.ks + b * a.ks_sb + hk * a.ks_sh + row * NG;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                d[g] = scales[g];
#pragma unroll
                for (int m = 0; m < 2; ++m) w[2 * g + m] = kp[(2 * hf + m) * NG + g];  // octet 2 hf + m of the group
            }
        } else {
            fta_frag f[KS];
            FtaTile<DT, KD>::load_rows(reinterpret_cast<const uint16_t*>(p), ok, a.Dreal, lane, f);
#pragma unroll
            for (int i = 0; i < KS; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) w[4 * i + e] = f[i][e];
        }
    }
    __device__ __forceinline__ void operands(const WeighArgs& a, int lane, fta_frag (&kf)[KS], float (&ds)[NG]) const {
        const int hf = lane >> 5;
        if constexpr (Q4) {
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                ds[g] = (float)__builtin_bit_cast(_Float16, d[g]);
#pragma unroll
                for (int m = 0; m < 2; ++m) {  // the group's first or second product
                    float n[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) n[e] = (float)((int)((w[2 * g + m] >> (4 * e)) & 15u) - 8);
                    kf[2 * g + m] = 32 * g + 16 * hf + 8 * m < a.Dreal ? fta_pack_frag<DT>(n) : fta_frag{0u, 0u, 0u, 0u};
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < KS; ++i) kf[i] = fta_frag{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
        }
    }
};

// The rows of a chunk, its first token at position q_lo, whose tokens see a key.
__device__ __forceinline__ uint32_t rows_that_see(const WeighArgs& a, int q_lo, int key) {
    const int64_t t_hi = key < a.sinks ? a.TT - 1 : min((int64_t)key + a.left - q_lo, (int64_t)a.TT - 1);
    const int rlo = max(key - q_lo, 0) >= a.TT ? 32 : max(key - q_lo, 0) * a.GG;
    const int rhi = (int)max(t_hi + 1, (int64_t)0) * a.GG;
    return fta_bits_below(rhi) & ~fta_bits_below(rlo);
}

// -lse log2(e), or -inf for what gives nothing: a row that saw nothing (lse = -inf) or does not exist (inf).  A NaN
// would outlast a masked score and reach keys that its token does not see: it gives nothing here, and
// makes the sums of its own keys NaN in the end.
__device__ __forceinline__ float row_offset(float lse) { return fabsf(lse) < FTA_INF ? -lse * kLog2e : -FTA_INF; }

// What chunk c's 32 rows, in LDS at `rows` with their row_offset at sl, add to this lane's key kt + (lane & 31).
template <int DT, int KD, bool Q4>
__device__ __forceinline__ float chunk_sum(const WeighArgs& a, const fta_frag (&kf)[KD / 16], const float (&ds)[KD / 32],
                                           uint32_t rows, const float* sl, int c, int kt, int len, int lane) {
    constexpr int QSEG = KD / 8, KS = KD / 16, NG = KD / 32;
    using SW = FtaSwz<QSEG>;
    const int hf = lane >> 5, key = kt + (lane & 31);
    const int q_lo = len - a.T + c * a.TT, q_hi = min(q_lo + a.TT, len) - 1;  // positions of the chunk's tokens
    if (q_hi < kt || (kt + 31 < q_lo - a.left && kt >= a.sinks)) return 0.f;  // wave-uniform
    const uint32_t ro = rows + (lane & 31) * QSEG * 16u;
    auto frag = [&](int slot) { return fta_lds_frag(ro + 16u * (slot ^ SW::x(lane & 31))); };
    f32x16 x;
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = 0.f;
    if constexpr (Q4) {
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            f32x16 y;
#pragma unroll
            for (int i = 0; i < 16; ++i) y[i] = 0.f;
            y = fta_mma<DT>(frag(4 * g + 2 * hf), kf[2 * g], y);
            y = fta_mma<DT>(frag(4 * g + 2 * hf + 1), kf[2 * g + 1], y);
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = fmaf(ds[g], y[i], x[i]);
        }
    } else {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) x = fta_mma<DT>(frag(2 * ks + hf), kf[ks], x);
    }
    if (!(q_lo >= kt + 31 && (q_hi - a.left <= kt || kt + 31 < a.sinks))) {
        asm volatile("");  // an edge: kept apart, or every chunk pays for it
        FtaTile<DT, KD>::mask(rows_that_see(a, q_lo, key), lane, x);
    }
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
        const float4 l = *reinterpret_cast<const float4*>(&sl[c_row(i, lane)]);
        x[i] = fta_exp2(fmaf(x[i], a.c, l.x));
        x[i + 1] = fta_exp2(fmaf(x[i + 1], a.c, l.y));
        x[i + 2] = fta_exp2(fmaf(x[i + 2], a.c, l.z));
        x[i + 3] = fta_exp2(fmaf(x[i + 3], a.c, l.w));
    }
    return ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7])) +
           (((x[8] + x[9]) + (x[10] + x[11])) + ((x[12] + x[13]) + (x[14] + x[15])));
}

// ----------------------------------------------------------------------------
// Many rows.  KD: columns (16-bit keys: 64, 128 or 256; 4-bit keys: 32 per group).
// What bounds it: matrix and vector instructions (of these the 16 exp2 of a tile most), at a clock that
// their power lowers.  A prompt of 8192 tokens, 32 / 8 heads of 128: 334 to 364 us by run, 750 to 820 TFLOP/s at 2.0 GHz, the
// matrix units busy 36% of the cycles, the vector units 56%: 104% together of the cycles in which a CU has waves,
// so they hardly overlap.  Four stages with all of a part's lse loaded ahead (367 beside 360), two key tiles a
// wave (411), and the last chunk's exp2 between this one's products (357 to 374) gained nothing: what overlaps
// more runs at a lower clock.  The weights so far loaded with the keys instead of at the end changed nothing.
// 4-bit keys are expanded once for a walk, and every group's product is scaled by itself: 64 more multiply-adds a tile
// at 128 columns, 456 us for the same prompt; 4096 tokens, 16 / 4 heads of 256, 318 us beside 130 on 16-bit keys (256
// registers, 9 more spilled).
// ----------------------------------------------------------------------------
template <int DT, int KD, bool Q4>
__global__ __launch_bounds__(kWeighWaves * 64, KD <= 128 ? 3 : 2) void fta_cache_weights_kernel(WeighArgs a) {
    constexpr int QSEG = KD / 8, KS = KD / 16, NG = KD / 32, BLOCKS = QSEG / 2, TILE_B = 32 * QSEG * 16;
    using SW = FtaSwz<QSEG>;
    __shared__ __align__(1024) unsigned char sQ[2][TILE_B];
    __shared__ __align__(16) float sL[2][32];  // row_offset
    __shared__ int sNan;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wgi = fta_xcd_remap(blockIdx.x, a.total);
    const int u = fta_scalar(wgi / a.np), sp = wgi - u * a.np;
    const int bhk = fta_scalar(u / a.tiles), tile = u - bhk * a.tiles;  // the first keys, which most rows see, first
    const int b = fta_scalar(bhk / a.Hk), hk = bhk - b * a.Hk;
    const int len = __builtin_amdgcn_readfirstlane(min(max(a.lens[b], 0), a.S));
    const int kt = kWeighKeys * tile + 32 * wave, key = kt + (lane & 31);  // this wave's first key, this lane's
    const WeighWalk walk(a, len, kWeighKeys * tile);
    const int c_lo = walk.c_lo, nct = walk.nct;
    const int64_t all = (int64_t)nct * a.groups;
    if ((int64_t)sp * a.per >= all) return;  // a walk of fewer parts
    const int s0 = sp * a.per, s1 = (int)min(all, (int64_t)s0 + a.per);

    const uint16_t* qp = a.q + b * a.q_sb + (int64_t)hk * a.G * a.q_sh;
    const float* lp = a.lse + ((int64_t)b * a.H + (int64_t)hk * a.G) * a.T;
    // this lane's rows of a chunk: token and head within it, 16-byte slot
    constexpr int MINE = (BLOCKS + kWeighWaves - 1) / kWeighWaves;
    int tt[MINE], gg[MINE], col[MINE];
    uint32_t off[MINE];  // bytes, where strides let 32 bits hold them
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
        const int s = (i * kWeighWaves + wave) * 64 + lane, row = (s / QSEG) & 31;
        const int j = SW::slot(row, s - (s / QSEG) * QSEG);
        const bool has = row < a.TT * a.GG;  // the last rows of a chunk that heads do not fill repeat its first
        tt[i] = has ? row / a.GG : 0;
        gg[i] = has ? row - tt[i] * a.GG : 0;
        col[i] = j * 8 < a.Dreal ? j * 8 : 0;  // columns past D: they meet zero key columns
        off[i] = 2u * (tt[i] * (uint32_t)a.q_sn + gg[i] * (uint32_t)a.q_sh + col[i]);
    }
    const bool lhas = (lane & 31) < a.TT * a.GG;
    const int ltt = lhas ? (lane & 31) / a.GG : 0, lgg = lhas ? (lane & 31) - ltt * a.GG : 0;
    const int64_t loff = (int64_t)lgg * a.T + ltt;
    const uint32_t ldq = fta_lds_addr(&sQ[0][0]);
    float lv = 0.f;  // lse of the next chunk's row `lane` (wave 0)
    auto issue = [&](int ct, int cg, int st) __attribute__((always_inline)) {
        const int t0 = ct * a.TT, g0 = cg * a.GG;
        if (a.narrow && t0 + a.TT <= a.T && g0 + a.GG <= a.G) {  // every row is there
            const uint16_t* base = qp + t0 * a.q_sn + g0 * a.q_sh;
#pragma unroll
            for (int i = 0; i < MINE; ++i) {
                const int blk = i * kWeighWaves + wave;
                if (blk < BLOCKS) fta_dma16_so(base, off[i], ldq + st * TILE_B + blk * 1024);  // wave-uniform
            }
            if (wave == 0) {
                const float x = lp[(int64_t)g0 * a.T + t0 + loff];
                lv = lhas ? x : FTA_INF;
            }
        } else {
#pragma unroll
            for (int i = 0; i < MINE; ++i) {
                const int blk = i * kWeighWaves + wave;
                const int64_t t = min(t0 + tt[i], a.T - 1), g = min(g0 + gg[i], a.G - 1);
                if (blk < BLOCKS) fta_dma16_at(qp + t * a.q_sn + g * a.q_sh + col[i], ldq + st * TILE_B + blk * 1024);
            }
            if (wave == 0) {
                const bool ok = t0 + ltt < a.T && g0 + lgg < a.G && lhas;
                const float x = lp[ok ? (int64_t)g0 * a.T + t0 + loff : 0];
                lv = ok ? x : FTA_INF;
            }
        }
    };
    int cg = fta_scalar(s0 / nct), ct = c_lo + s0 - cg * nct;
    issue(ct, cg, 0);
    fta_frag kf[KS];
    float ds[NG];
    {
        KeyRows<DT, KD, Q4> keys;
        const bool kok = key < a.S;
        keys.load(a, b, hk, kok ? key : 0, kok, lane);
        keys.operands(a, lane, kf, ds);
    }
    float run = 0.f, sum = 0.f;
    bool nans = false;  // wave 0: a row's lse was
    int st = 0;
    for (int s = s0; s < s1; ++s, st ^= 1) {
        fta_wait_vmcnt<0>();
        if (wave == 0 && lane < 32) sL[st][lane] = row_offset(lv);
        nans |= lv != lv;
        __syncthreads();  // this chunk visible; every wave is past the last one
        const int c = ct;
        if (++ct == c_lo + nct) {
            ct = c_lo;
            ++cg;
        }
        if (s + 1 < s1) issue(ct, cg, st ^ 1);
        // sums of a chunk, of 64 chunks, of all: their rounding errors stay small on long walks
        if (((s - s0) & 63) == 63) {
            sum += run;
            run = 0.f;
        }
        run += chunk_sum<DT, KD, Q4>(a, kf, ds, ldq + st * TILE_B, sL[st], c, kt, len, lane);
    }
    sum += run;
    sum += fta_xor32(sum);
    if (wave == 0) sNan = __ballot(nans) != 0ull;
    __syncthreads();
    if (sNan) {
        for (int s = s0; s < s1; ++s) {
            const int g0 = s / nct * a.GG, t0 = (c_lo + s % nct) * a.TT, r = lane & 31, t = t0 + r / a.GG, g = g0 + r % a.GG;
            const bool ok = r < a.TT * a.GG && t < a.T && g < a.G;
            const float x = lp[ok ? (int64_t)g * a.T + t : 0];
            if ((uint32_t)__ballot(ok && x != x) & rows_that_see(a, len - a.T + t0, key)) sum = __builtin_nanf("");
        }
    }
    if (lane >= 32 || key >= len) return;
    if (a.np > 1)
        a.part[((int64_t)sp * a.B * a.Hk + bhk) * a.S + key] = sum;
    else
        a.w[b * a.w_sb + hk * a.w_sh + key] += sum;
}

// ----------------------------------------------------------------------------
// Rows that stay in LDS, up to kHeld chunks of 32: the last tokens of a prompt, or several tokens of a step. They are
// loaded once, and the keys stream past: a workgroup takes a run of keys, its waves 32-key tiles in turn, the
// next tile's asked for ahead.
// What bounds it: memory for 16-bit keys (64 requests x 12 tokens on 4096 to 8192, 32 / 8 heads of 128: 190 to 207 us, 4.2
// TB/s), vector instructions for 4-bit ones (153 to 161 us; more than a third of them turn codes into 16-bit numbers
// one by one; at 256 columns 45 registers are spilled).  The kernel of many rows, which starts anew for every 128
// keys, takes 216 and 273; 2 x 32 tokens on up to 32768 4-bit keys, 16 / 4 heads of 64, 17.5 and 19.5.  Eight chunks,
// which leave two waves a SIMD at 128 columns, are slower than it: 64 tokens, 40 us and 32.
// ----------------------------------------------------------------------------
constexpr int kHeld = 4;
template <int DT, int KD, bool Q4>
__global__ __launch_bounds__(256, KD <= 128 ? 3 : 2) void fta_cache_weights_rows_kernel(WeighArgs a) {
    constexpr int QSEG = KD / 8, KS = KD / 16, NG = KD / 32, BLOCKS = QSEG / 2, TILE_B = 32 * QSEG * 16, NW = 4;
    using SW = FtaSwz<QSEG>;
    __shared__ __align__(1024) unsigned char sQ[kHeld][TILE_B];
    __shared__ __align__(16) float sL[kHeld][32];
    __shared__ uint32_t sNan[kHeld];  // rows of a chunk whose lse is
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int bhk = fta_scalar(blockIdx.x / a.np), sp = blockIdx.x - bhk * a.np;
    const int b = fta_scalar(bhk / a.Hk), hk = bhk - b * a.Hk;
    const int len = __builtin_amdgcn_readfirstlane(min(max(a.lens[b], 0), a.S));
    // 32-key tiles: the sinks', then the band's
    const int kb0 = max(0, len - a.T - a.left);
    int ns = (min(a.sinks, len) + 31) >> 5, c_lo = kb0 >> 5;
    const int c_hi = (len + 31) >> 5;
    if (c_lo <= ns) c_lo = ns = 0;
    const int all = max(ns + c_hi - c_lo, 0);
    const int it0 = fta_scalar((int)((int64_t)all * sp / a.np)), it1 = fta_scalar((int)((int64_t)all * (sp + 1) / a.np));
    if (it0 >= it1) return;  // all waves

    const uint16_t* qp = a.q + b * a.q_sb + (int64_t)hk * a.G * a.q_sh;
    const float* lp = a.lse + ((int64_t)b * a.H + (int64_t)hk * a.G) * a.T;
    const uint32_t ldq = fta_lds_addr(&sQ[0][0]);
    const int nct = a.chunks / a.groups;  // chunk = head group * nct + tokens / TT
    for (int i = wave; i < a.chunks * BLOCKS; i += NW) {
        const int ch = i / BLOCKS, blk = i - ch * BLOCKS, cg = ch / nct, ct = ch - cg * nct;  // wave-uniform
        const int s = blk * 64 + lane, row = s / QSEG, j = SW::slot(row, s - row * QSEG);
        const bool has = row < a.TT * a.GG;
        const int tt = has ? row / a.GG : 0, gg = has ? row - tt * a.GG : 0;  // rows that are not there repeat others
        const int64_t t = min(ct * a.TT + tt, a.T - 1), g = min(cg * a.GG + gg, a.G - 1);
        fta_dma16_at(qp + t * a.q_sn + g * a.q_sh + (j * 8 < a.Dreal ? j * 8 : 0), ldq + i * 1024);
    }
    for (int i = threadIdx.x; i < a.chunks * 32; i += 256) {
        const int ch = i >> 5, row = i & 31, cg = ch / nct, ct = ch - cg * nct;
        const int t = ct * a.TT + row / a.GG, g = cg * a.GG + row % a.GG;
        const bool ok = row < a.TT * a.GG && t < a.T && g < a.G;
        const float x = lp[ok ? (int64_t)g * a.T + t : 0];
        sL[ch][row] = row_offset(ok ? x : FTA_INF);
        const uint64_t n = __ballot(ok && x != x);  // of two chunks, or of the last
        if (row == 0) sNan[ch] = (uint32_t)(n >> (lane & 32));
    }
    float* wp = a.w + b * a.w_sb + hk * a.w_sh;
    auto tile = [&](int it) { return 32 * (it < ns ? it : c_lo + it - ns); };
    struct Tile {
        KeyRows<DT, KD, Q4> keys;
        float before;
    };
    auto ask = [&](int it, Tile& x) __attribute__((always_inline)) {
        const int j = min(tile(it) + (lane & 31), len - 1);  // behind the last token: masked, and not written
        x.keys.load(a, b, hk, j, true, lane);
        x.before = wp[j];
    };
    Tile cur, nxt;
    if (it0 + wave < it1) ask(it0 + wave, cur);
    fta_wait_vmcnt<0>();
    __syncthreads();
    for (int it = it0 + wave; it < it1; it += NW) {
        if (it + NW < it1) ask(it + NW, nxt);
        fta_frag kf[KS];
        float ds[NG];
        cur.keys.operands(a, lane, kf, ds);
        const int kt = tile(it), key = kt + (lane & 31);
        float sum = 0.f;
        for (int cg = 0, ch = 0; cg < a.groups; ++cg)
            for (int ct = 0; ct < nct; ++ct, ++ch) sum += chunk_sum<DT, KD, Q4>(a, kf, ds, ldq + ch * TILE_B, sL[ch], ct, kt, len, lane);
        sum += fta_xor32(sum);
        if (lane < 32 && key < len) wp[key] = cur.before + sum;
        cur = nxt;
    }
    for (int ch = 0; ch < a.chunks; ++ch) {
        const uint32_t n = fta_scalar((int)sNan[ch]);
        if (n == 0) continue;
        for (int it = it0 + wave; it < it1; it += NW) {
            const int key = tile(it) + (lane & 31);
            if (lane < 32 && key < len && (n & rows_that_see(a, len - a.T + ch % nct * a.TT, key))) wp[key] = __builtin_nanf("");
        }
    }
}

// ----------------------------------------------------------------------------
// Few rows (T * G of at most 32): a serving step.  A workgroup takes a run of keys, its waves 32-key tiles
// in turn, the next tile's asked for ahead; the rows, 16 or 32, stay in registers.  16 x 16 x 32 products,
// S = Q K^T: lane (k, q) = (l & 15, l >> 4) holds rows 4 q + i of its key k.  4-bit keys enter as 16 + n,
// after a product of the rows with -24 (see fta_q4.hip).
// What bounds it: memory.  64 requests of 4096 to 8192 tokens, 32 / 8 heads of 128: 154 us, 5.4 TB/s; with 4-bit keys
// 61 to 68 us, 3.4 TB/s, where vector instructions weigh as much.  Two tiles of rows: 64 requests x 8 tokens 207 us, with
// 4-bit keys 117 (12 registers spilled); 32 x 8 tokens, 16 / 4 heads of 256 in 4 bits, 176 (68 spilled; 35 at 224
// columns).
// ----------------------------------------------------------------------------
template <int KD, bool Q4>
struct KeyTile {  // 32 keys as B operands: of keys 16 t + k, this lane's words
    uint32_t w[2][Q4 ? KD / 32 : KD / 8];
    uint16_t d[2][KD / 32];
    float before[2];
};

template <int DT, int KD, bool Q4, int RT>
__global__ __launch_bounds__(256, KD <= 128 ? 3 : 2) void fta_cache_weights_step_kernel(WeighArgs a) {
    constexpr int NG = KD / 32, NW = 4;
    const int lane = threadIdx.x & 63, r16 = lane & 15, qt = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int bhk = fta_scalar(blockIdx.x / a.np), sp = blockIdx.x - bhk * a.np;
    const int b = fta_scalar(bhk / a.Hk), hk = bhk - b * a.Hk;
    const int len = __builtin_amdgcn_readfirstlane(min(max(a.lens[b], 0), a.S));
    const int R = a.T * a.G, p0 = len - a.T, p1 = len - 1;  // rows; first and last position
    // 32-key tiles: the sinks', then the band's
    const int kb0 = max(0, p0 - a.left);
    int ns = (min(a.sinks, len) + 31) >> 5, c_lo = kb0 >> 5;
    const int c_hi = (len + 31) >> 5;
    if (c_lo <= ns) c_lo = ns = 0;
    const int all = max(ns + c_hi - c_lo, 0);
    const int it0 = fta_scalar((int)((int64_t)all * sp / a.np)), it1 = fta_scalar((int)((int64_t)all * (sp + 1) / a.np));
    if (it0 + wave >= it1) return;

    const uint8_t* kp = a.k + b * a.k_sb + hk * a.k_sh;
    const uint16_t* ks = a.ks + b * a.ks_sb + hk * a.ks_sh;
    float* wp = a.w + b * a.w_sb + hk * a.w_sh;
    auto key = [&](int it) { return 32 * (it < ns ? it : c_lo + it - ns); };
    using Tile = KeyTile<KD, Q4>;
    auto ask = [&](int it, Tile& x) __attribute__((always_inline)) {
        const int kb = key(it);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int j = min(kb + 16 * t + r16, len - 1);  // behind the last token: masked, and not written
            if constexpr (Q4) {
                __builtin_memcpy(x.w[t], __builtin_assume_aligned(kp + (int64_t)j * (16 * NG) + qt * 4 * NG, 4), 4 * NG);
#pragma unroll
                for (int g = 0; g < NG; ++g) x.d[t][g] = ks[(int64_t)j * NG + g];
            } else {
                const uint8_t* row = kp + (int64_t)j * a.k_sn;
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const int d = 32 * g + 8 * qt;
                    const fta_frag f = d < a.Dreal ? *reinterpret_cast<const fta_frag*>(row + 2 * d) : fta_frag{0u, 0u, 0u, 0u};
#pragma unroll
                    for (int e = 0; e < 4; ++e) x.w[t][4 * g + e] = f[e];
                }
            }
            x.before[t] = wp[j];
        }
    };
    Tile cur, nxt;
    ask(it0 + wave, cur);

    fta_frag qf[RT][NG];
    float nl[RT][4];  // of rows 4 qt + i
    int pos[RT][4];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = 16 * rt + r16, t = min(r, R - 1) / a.G, g = min(r, R - 1) - t * a.G;
        const uint16_t* qp = a.q + b * a.q_sb + (int64_t)(hk * a.G + g) * a.q_sh + t * a.q_sn;
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            const int d = 32 * n + 8 * qt;
            const fta_frag x = (r < R && d < a.Dreal) ? *reinterpret_cast<const fta_frag*>(qp + d) : fta_frag{0u, 0u, 0u, 0u};
            qf[rt][n] = Q4 ? fta_paired(x) : x;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int rr = 16 * rt + 4 * qt + i, tr = min(rr, R - 1) / a.G, gr = min(rr, R - 1) - tr * a.G;
            const float x = a.lse[((int64_t)b * a.H + hk * a.G + gr) * a.T + tr];
            nl[rt][i] = rr < R && x != -FTA_INF ? -x * kLog2e : -FTA_INF;  // a row that saw nothing gives nothing
            pos[rt][i] = p0 + tr;
        }
    }
    f32x4 first[RT][Q4 ? NG : 1];
    if constexpr (Q4) {
        constexpr uint32_t m24 = DT == FTA_DTYPE_BF16 ? 0xc1c0c1c0u : 0xce00ce00u;  // -24
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int g = 0; g < NG; ++g)
                first[rt][g] = fta_mma16<DT>(qf[rt][g], fta_frag{m24, m24, m24, m24}, f32x4{0.f, 0.f, 0.f, 0.f});
    }
    const uint32_t sixteen = fta_in_vgpr(kFtaSixteen<DT>);
    const float zero = __builtin_bit_cast(float, fta_in_vgpr(0u));

    for (int it = it0 + wave; it < it1; it += NW) {
        if (it + NW < it1) ask(it + NW, nxt);
        const int kb = key(it);
        const bool full = kb + 31 <= p0 && (kb >= p1 - a.left || kb + 31 < a.sinks);
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                f32x4 x = f32x4{zero, zero, zero, zero};
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    if constexpr (Q4) {
                        const f32x4 y = fta_mma16<DT>(qf[rt][g], fta_codes16<DT>(cur.w[t][g], sixteen), first[rt][g]);
                        const float d = (float)__builtin_bit_cast(_Float16, cur.d[t][g]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) x[i] = fmaf(d, y[i], x[i]);
                    } else {
                        x = fta_mma16<DT>(qf[rt][g], fta_frag{cur.w[t][4 * g], cur.w[t][4 * g + 1], cur.w[t][4 * g + 2], cur.w[t][4 * g + 3]}, x);
                    }
                }
                const int j = kb + 16 * t + r16;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool seen = full || (j <= pos[rt][i] && (j >= pos[rt][i] - a.left || j < a.sinks));
                    const float p = fta_exp2(fmaf(x[i], a.c, nl[rt][i]));
                    sum[t] += seen ? p : 0.f;
                }
            }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const float s = fta_sum_quarters(sum[t]);
            const int j = kb + 16 * t + r16;
            if (qt == 0 && j < len) wp[j] = cur.before[t] + s;
        }
        cur = nxt;
    }
}

// Sum of the parts that a key's walk has.
__global__ __launch_bounds__(256) void fta_cache_weights_join_kernel(WeighArgs a) {
    const int bhk = blockIdx.y, b = bhk / a.Hk, hk = bhk - b * a.Hk;
    const int j = blockIdx.x * 256 + threadIdx.x;
    const int len = min(max(a.lens[b], 0), a.S);
    const int tile = fta_scalar((blockIdx.x * 256 + (threadIdx.x & ~63)) / kWeighKeys);  // a wave's 64 keys lie in one tile
    if (j >= len) return;
    const WeighWalk w(a, len, kWeighKeys * tile);
    const int parts = (int)(((int64_t)w.nct * a.groups + a.per - 1) / a.per);
    const int64_t n = (int64_t)a.B * a.Hk * a.S;
    const float* p = a.part + (int64_t)bhk * a.S + j;
    float s = 0.f;
    for (int i = 0; i < parts; ++i) s += p[i * n];
    a.w[b * a.w_sb + hk * a.w_sh + j] += s;
}

// ---------------------------------------------------------------------- host

int weigh_plan(WeighArgs& a, bool q4, int B, int H, int Hk, int T, int S, int D, int left, int sinks) {
    if (B <= 0 || H <= 0 || Hk <= 0 || T <= 0 || S <= 0 || D <= 0) return fta::arg_error("cache_weights: dims must be positive");
    if (H % Hk != 0) return fta::arg_error("cache_weights: num_heads must be a multiple of num_kv_heads");
    if (D % 16 != 0 || D > 256) return fta::arg_error("cache_weights: D must be a multiple of 16 up to 256");
    if (left < 0 || sinks < 0) return fta::arg_error("cache_weights: window and num_sinks must be non-negative");
    if (S > (1 << 29) || T > (1 << 29) || H > (1 << 20))
        return fta::unsupported("cache_weights: sizes past 2^29 tokens or 2^20 heads");
    if (!fta::size_fits(B, T, H, D) || !fta::size_fits(B, S, Hk, D)) return fta::unsupported("cache_weights: 2^60 elements and more");
    a = WeighArgs{};
    a.B = B, a.T = T, a.H = H, a.Hk = Hk, a.G = H / Hk, a.S = S, a.Dreal = D;
    a.left = std::min(left, S);
    a.sinks = a.left >= S - 1 ? 0 : std::min(sinks, S);
    // Heads x tokens of a chunk, so that rows and the mask are a division by GG away.  T = 17 .. 31 leaves up to 15 of
    // 32 rows unused, T = 33 gives every head a second chunk of one token, and such rows may take the kernel of many where
    // as many others are held: 16 requests of 4096 to 8192 tokens, four K/V heads of 128, 32 tokens x 4 heads (held) 41 us,
    // 20 x 5 53, 33 x 3 57.
    a.GG = std::min(a.G, std::max(1, 32 / std::min(T, 32)));
    a.TT = 32 / a.GG;
    a.groups = (a.G + a.GG - 1) / a.GG;
    const int64_t most = (1 << 24) - 1, heads = (int64_t)B * Hk;
    a.few = (int64_t)T * a.G <= 32;
    const int64_t tiles = (std::min<int64_t>(S, (int64_t)a.left + T + a.sinks + 62) + 31) / 32;  // of 32 keys
    auto parts = [&](int64_t target, int64_t least) { return std::min<int64_t>((target + heads - 1) / heads, tiles / least); };
    if (a.few) {
        // Parts cost nothing but a workgroup's start (every key is its own): enough to fill the chip, down to one
        // tile of a wave, and about 16384 of two tiles and more, whose starts overlap with others' ends; 4-bit tiles
        // are shorter, 2048 of four.  Target 2048 / 8192 / 16384 / 65536 (the last down to one tile), us, 64 requests
        // of 4096 to 8192 tokens, 32 / 8 heads: of 128 193 / 161 / 154 / 158, of 64 123 / 89 / 85 / 90, of 128 in 4
        // bits 66 / 71 / 83 / 113.
        const int64_t np = std::max<int64_t>(1, std::max(parts(1024, 4), q4 ? parts(2048, 16) : parts(16384, 8)));
        if (heads * np > most) return fta::unsupported("cache_weights: too many heads");
        a.np = (int)np;
        a.total = (int)(heads * np);
        return FTA_OK;
    }
    const int64_t held = (int64_t)((T + a.TT - 1) / a.TT) * a.groups;
    if (held <= kHeld) {
        // Parts as above, of two tiles a wave and more.  Target 1024 / 2048 / 4096 / 16384, us, 32 / 8 heads of 128, 4096
        // to 8192 tokens: 64 requests x 12 246 / 243 / 226 / 196, 16 x 16 69 / 63 / 62 / 61; 64 x 12 in 4 bits
        // 177 / 156 / 155 / 205, 18 x 16 of up to 16028, 16 / 4 heads of 256 in 4 bits, 126 / 132 / 149 / 149.
        const int64_t np = std::max<int64_t>(1, std::max(parts(1024, 8), q4 ? parts(2048, 16) : parts(16384, 8)));
        if (heads * np > most) return fta::unsupported("cache_weights: too many heads");
        a.chunks = (int)held;
        a.np = (int)np;
        a.total = (int)(heads * np);
        return FTA_OK;
    }
    a.tiles = (S + kWeighKeys - 1) / kWeighKeys;
    const int64_t wgs = heads * a.tiles;
    // walks in chunks: the longest, and all of them, of sequences that fill the cache
    const int64_t span = (int64_t)a.left + kWeighKeys + 1;
    auto chunks = [&](int64_t tokens) { return ((tokens + a.TT - 1) / a.TT + 1) * a.groups; };
    const int64_t longest = chunks(std::min<int64_t>(T, a.sinks > 0 ? T : span));
    if (longest > (1 << 30)) return fta::unsupported("cache_weights: too many rows");
    const int64_t mean = chunks(std::min<int64_t>(span, T - std::max<int64_t>(0, T - ((int64_t)S - T)) / 2));
    // Parts of 32 chunks and more, about 4096 of them: causal walks shorten with the key, and tiles of sinks
    // walk every token.  Target 1024 / 2048 / 4096 / 8192, us: 8192 tokens 523 / 440 / 361 / 361; least 32 / 64
    // chunks: 2048 tokens 46 / 66.  Down to 8 chunks where they would not be 1024 parts, least 32 / 16 / 8 / 4, us of
    // both kernels: 6 x 456 tokens, 8 heads on one, 39 / 24 / 19 / 21, 8 x 512, 32 / 8 heads, 41 / 35 / 35 / 36.
    const int64_t work = wgs * mean;
    a.per = (int)std::min(longest, std::max(std::clamp<int64_t>(work / 1024, 8, 32), work / 4096));
    a.np = (int)((longest + a.per - 1) / a.per);
    if (wgs * a.np > most || heads > 65535 || heads * ((S + 255) / 256) > most)
        return fta::unsupported("cache_weights: too many keys");
    a.total = (int)(wgs * a.np);
    return FTA_OK;
}

size_t weigh_bytes(const WeighArgs& a) { return a.few || a.chunks > 0 || a.np <= 1 ? 0 : fta::align_up((size_t)a.np * a.B * a.Hk * a.S * sizeof(float)); }

template <int DT, int KD, bool Q4>
int launch_weigh(const WeighArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)a.total), t(256);
    if (a.few) {
        if (a.T * a.G <= 16)
            hipLaunchKernelGGL((fta_cache_weights_step_kernel<DT, KD, Q4, 1>), grid, t, 0, st, a);
        else
            hipLaunchKernelGGL((fta_cache_weights_step_kernel<DT, KD, Q4, 2>), grid, t, 0, st, a);
        return fta::check_launch("fta_cache_weights_step_kernel");
    }
    if (a.chunks > 0) {
        hipLaunchKernelGGL((fta_cache_weights_rows_kernel<DT, KD, Q4>), grid, t, 0, st, a);
        return fta::check_launch("fta_cache_weights_rows_kernel");
    }
    hipLaunchKernelGGL((fta_cache_weights_kernel<DT, KD, Q4>), grid, t, 0, st, a);
    int rc = fta::check_launch("fta_cache_weights_kernel");
    if (rc != FTA_OK || a.np <= 1) return rc;
    const dim3 g((unsigned)((a.S + 255) / 256), (unsigned)(a.B * a.Hk));
    hipLaunchKernelGGL(fta_cache_weights_join_kernel, g, t, 0, st, a);
    return fta::check_launch("fta_cache_weights_join_kernel");
}

template <int DT>
int launch_weigh_dims(const WeighArgs& a, bool q4, hipStream_t st) {
    if (!q4) {
        if (a.Dreal <= 64) return launch_weigh<DT, 64, false>(a, st);
        if (a.Dreal <= 128) return launch_weigh<DT, 128, false>(a, st);
        return launch_weigh<DT, 256, false>(a, st);
    }
    switch ((a.Dreal + 31) / 32) {
        case 1: return launch_weigh<DT, 32, true>(a, st);
        case 2: return launch_weigh<DT, 64, true>(a, st);
        case 3: return launch_weigh<DT, 96, true>(a, st);
        case 4: return launch_weigh<DT, 128, true>(a, st);
        case 5: return launch_weigh<DT, 160, true>(a, st);
        case 6: return launch_weigh<DT, 192, true>(a, st);
        case 7: return launch_weigh<DT, 224, true>(a, st);
        default: return launch_weigh<DT, 256, true>(a, st);
    }
}

}  // namespace

extern "C" {

size_t fta_cache_weights_workspace_size(int B, int H, int Hk, int T, int S, int D, int left, int num_sinks) {
    WeighArgs a;
    if (weigh_plan(a, false, B, H, Hk, T, S, D, left, num_sinks) != FTA_OK) return 0;
    return weigh_bytes(a);
}

int fta_cache_weights(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* k_scales,
                      const int64_t* ks_strides, int dtype, int B, int H, int Hk, int T, int S, int D,
                      const int32_t* cache_lens, int left, int num_sinks, float scale, const float* lse, float* weights,
                      const int64_t* w_strides, void* workspace, size_t workspace_bytes, void* stream) {
    FTA_TRY_BEGIN
    WeighArgs a;
    const bool q4 = k_scales != nullptr;
    int rc = weigh_plan(a, q4, B, H, Hk, T, S, D, left, num_sinks);
    if (rc != FTA_OK) return rc;
    if (dtype != FTA_DTYPE_BF16 && dtype != FTA_DTYPE_F16) return fta::arg_error("cache_weights: dtype must be bf16 or fp16");
    if (!(scale > 0.f) || scale > 2.0e38f)  // times log2(e) still finite
        return fta::arg_error("cache_weights: scale must be positive and at most 2e38");
    const size_t need = weigh_bytes(a);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return fta::arg_error("cache_weights: workspace too small");
    if (!fta::all_set(q, q_strides, k, k_strides, cache_lens, lse, weights, w_strides) || (k_scales != nullptr && ks_strides == nullptr))
        return fta::arg_error("cache_weights: a required pointer is null");
    a.q = (const uint16_t*)q, a.q_sb = q_strides[0], a.q_sh = q_strides[1], a.q_sn = q_strides[2];
    a.k = (const uint8_t*)k;
    if (q4) {
        if ((((uintptr_t)k) & 15) != 0 || ((k_strides[0] | k_strides[1]) & 15) != 0)
            return fta::arg_error("cache_weights: the heads' codes must be 16-byte aligned");
        a.k_sb = k_strides[0], a.k_sh = k_strides[1], a.k_sn = (D + 31) / 32 * 16;
        a.ks = (const uint16_t*)k_scales, a.ks_sb = ks_strides[0], a.ks_sh = ks_strides[1];
    } else {
        a.k_sb = 2 * k_strides[0], a.k_sh = 2 * k_strides[1], a.k_sn = 2 * k_strides[2];
    }
    a.lse = lse;
    a.lens = cache_lens;
    a.w = weights, a.w_sb = w_strides[0], a.w_sh = w_strides[1];
    a.part = (float*)workspace;
    a.c = scale * kLog2e;
    auto fits = [](int64_t stride, int n) { return stride >= 0 && stride <= (1 << 29) / n; };
    a.narrow = fits(a.q_sn, 32) && fits(a.q_sh, 32);
    hipStream_t st = (hipStream_t)stream;
    return dtype == FTA_DTYPE_BF16 ? launch_weigh_dims<FTA_DTYPE_BF16>(a, q4, st) : launch_weigh_dims<FTA_DTYPE_F16>(a, q4, st);
    FTA_TRY_END
}

}  // extern "C"
