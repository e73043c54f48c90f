// Caches of 4-bit keys and values: the attention of new tokens over them, and reading
// them back in 16 bits (the append that writes them is in fta_prep.hip).
//
// A row is one head of one token, NG = ceil(D / 32) groups of 32 columns (the last one
// filled up with zeros).  A group has a float16 scale d, its value of largest magnitude
// over -8, and a code n = 0 .. 15 for each column, which stands for d (n - 8).  Eight codes
// make a 32-bit word, column 8 o + i of group g at bits 4 i .. 4 i + 3 of
//   word 4 g + o   of a value row (columns in order),
//   word o NG + g  of a key row (octet o of every group side by side).
// Codes are [B][Hk][S][16 NG] bytes, scales [B][Hk][S][NG]: the rows of one head follow each
// other, so a tile of keys is one run of memory.
//
// Attention, visibility and rows that see nothing as in fta_cache_attn.  Nothing is
// expanded to 16-bit values: the codes go to the matrix units as they stand and the scales
// are applied in fp32,
//   s_j = sum_g d_jg sum_{c in g} (n_jc - 8) q_c,
//   o_c = sum_j (p_j d_jg) (n_jc - 8)               for c in group g,
// so that what 4 bits hold is multiplied without a further rounding, but for that of p d.
#include "fta_cache.h"
#include "fta_q4.h"
#include "fta_tile.h"

#include <algorithm>

namespace {

struct Q4Args {
    CacheArgs c;
    const uint8_t *kc, *vc;            // codes
    const uint16_t *ks, *vs;           // scales
    int64_t kc_sb, kc_sh, vc_sb, vc_sh;  // bytes
    int64_t ks_sb, ks_sh, vs_sb, vs_sh;  // elements
};

template <int N>
struct Words {
    uint32_t w[N];
};
// N words from a 4-byte aligned address
template <int N>
__device__ __forceinline__ Words<N> load_words(const uint8_t* p) {
    Words<N> x;
    __builtin_memcpy(&x, __builtin_assume_aligned(p, 4), 4 * N);
    return x;
}
// The scales of one row (2-byte aligned where there is an odd number), two in a word.
template <int NG>
__device__ __forceinline__ Words<(NG + 1) / 2> load_scales(const uint16_t* p) {
    if constexpr (NG % 2 == 0) {
        return load_words<NG / 2>(reinterpret_cast<const uint8_t*>(p));
    } else {
        Words<(NG + 1) / 2> x;
#pragma unroll
        for (int g = 0; g < NG; g += 2) x.w[g / 2] = p[g] | (g + 1 < NG ? (uint32_t)p[g + 1] << 16 : 0u);
        return x;
    }
}
__device__ __forceinline__ float half_of(uint32_t w, int hi) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(hi ? w >> 16 : w & 0xffffu));
}

template <int NG>
struct Q4Shape {
    static constexpr int NW = 4, KEYS = 64, ROWS = 16;
    static constexpr int ROW_B = 16 * NG, TILE_B = KEYS * ROW_B, SC_B = 2 * KEYS * NG * 2;
    static constexpr int STAGE_B = 2 * TILE_B + 2 * SC_B;  // a tile of key and of value codes, both's scales twice
    static constexpr int OROW = 32 * NG + 4;
    static constexpr int MERGE_B = NW * ROWS * OROW * 4, ML_B = NW * ROWS * 8;
    static constexpr int LDS_B = NW * STAGE_B > MERGE_B + ML_B ? NW * STAGE_B : MERGE_B + ML_B;
    // waves per SIMD that LDS leaves room for, and registers but for eight groups: they want more than 256, and spill 16
    static constexpr int WAVES = NG <= 2 ? 4 : NG <= 4 ? 3 : 2;
    // A row's 16-byte slots are exchanged by row so that the reads of 16 rows (one slot each) spread
    // over the banks: transpose reads take rows 16 q + e of the values, operand reads rows
    // 16 a + 4 t + e (a, e = 0 .. 3) of the keys.
    __device__ static __forceinline__ int vslot(int row, int p) {
        if constexpr (NG == 2 || NG == 6)
            return p ^ ((row >> 3) & 1);
        else if constexpr (NG == 4)
            return p ^ ((row >> 2) & 3);
        else if constexpr (NG == 8)
            return p ^ ((row >> 1) & 7);
        else
            return p;  // an odd number of slots spreads by itself
    }
    __device__ static __forceinline__ int kslot(int row, int p) {
        if constexpr (NG == 2)
            return p ^ ((row >> 4) & 1);
        else if constexpr (NG == 4)
            return p ^ ((row >> 4) & 3);
        else if constexpr (NG == 8)
            return p ^ (((row >> 1) & 1) | ((row >> 3) & 6));
        else
            return p;
    }
};

// ----------------------------------------------------------------------------
// Attention.  Workgroup = (b, K/V head, 16 rows, part); each wave takes 64-key tiles of its own.
// 16 x 16 x 32 products: a group's 32 columns are one of them, and few rows (a K/V head's query
// heads times its new tokens) waste little.
//   S^T = K Q^T: lane (r, q) = (l & 15, l >> 4) holds row r's scores of keys 16 q + 4 t + i
//   (register i of product t; the key rows are handed to the products in that order), and so the
//   16 keys whose value codes one transpose read gives lane (c, q) for its column c.
// The codes enter as 16 + n; -24 sum_{c in g} q_c is the key products' first addend, and every value
// product is followed by one of the same p d with -24 in every column.
// bf16: p d is rounded to bf16 as P is in the 16-bit kernels; o is off by 0.0023 of itself (root mean square) where
// its own rounding alone is 0.0017.  fp16: it would leave fp16's range for the scales that caches hold, so it goes
// as two bf16 numbers, hi + lo, 16 bits of it, which takes about a tenth of the time for what bf16 could not hold.
// A wave has one stage for a tile's key codes and one for its value codes: the next tile's keys are
// asked for before this one's values are multiplied, the next values after it.  Three waves per
// SIMD cover the rest of the wait.
// What bounds it: memory where there are many requests.  128 of 4096 to 8192 tokens, 32 / 8 heads of 128,
// bf16: 185 us, 906 MB, 5.0 TB/s (a large copy 5.1); with two stages each and two waves per SIMD 245.
// 64 requests: bf16 98 to 109 us, fp16, whose values take twice the products, 114 to 122.  One request of 4096: 9.5 us, the
// latency of a wave's start, its one tile and the merge.  Four requests of a window of 2000, three tokens each,
// 16 / 2 heads of 256, fp16: 24 us, latency again (a wave's one tile is 2480 vector and 167 matrix instructions).
// Many tokens: vector and matrix instructions, since each 16 rows unpack their keys and values anew and half of the
// value products take the 24 off again.  One request, 32 / 8 heads of 128, a call, bf16 / fp16: 128 tokens on 8192 73 / 85
// us, 512 on 8192 201 / 251, a prompt of 2048 140 / 165, of 8192 1252 / 1621 (window attention of 16-bit rows: 68 and 556).
// ----------------------------------------------------------------------------
template <int DT, int NG>
__global__ __launch_bounds__(256, Q4Shape<NG>::WAVES) void fta_q4_attn_kernel(Q4Args A) {
    using Sh = Q4Shape<NG>;
    constexpr int NW = Sh::NW, ROW_B = Sh::ROW_B, TILE_B = Sh::TILE_B, NS = (NG + 1) / 2;
    __shared__ __align__(1024) unsigned char sStage[Sh::LDS_B];
    const CacheArgs& a = A.c;
    const int lane = threadIdx.x & 63, r16 = lane & 15, qt = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wgi = blockIdx.x;
    const int rest = fta_scalar(wgi / a.ns), sp = wgi - rest * a.ns;
    const int bhk = fta_scalar(rest / a.row_tiles), rt = rest - bhk * a.row_tiles;
    const int b = fta_scalar(bhk / a.Hk), hk = bhk - b * a.Hk;
    const int r_lo = 16 * rt, r_n = min(16, a.R - r_lo);
    const int len = __builtin_amdgcn_readfirstlane(min(max(a.lens[b], 0), a.S));
    const int p0 = len - a.T + fta_scalar(r_lo / a.G), p1 = len - a.T + fta_scalar((r_lo + r_n - 1) / a.G);  // first and last position
    const int r = r_lo + r16;
    const int pos = (r < a.R) ? len - a.T + r / a.G : -1;  // this lane's row

    // 64-key tiles: the sinks', then the band's
    const int ke = max(p1 + 1, 0), kb0 = max(0, p0 - a.left);
    int ns = (min(a.sinks, ke) + 63) >> 6, c_lo = kb0 >> 6;
    const int c_hi = (ke + 63) >> 6;
    if (c_lo <= ns) c_lo = ns = 0;
    const int all = max(ns + c_hi - c_lo, 0);
    const int it0 = fta_scalar((int)((int64_t)all * sp / a.ns)), it1 = fta_scalar((int)((int64_t)all * (sp + 1) / a.ns));

    f32x4 oacc[2 * NG];
#pragma unroll
    for (int i = 0; i < 2 * NG; ++i) oacc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m_run = -FTA_INF, l_run = 0.f;

    if (it0 + wave < it1) {  // wave-uniform
        const uint8_t* kc = A.kc + b * A.kc_sb + hk * A.kc_sh;
        const uint8_t* vc = A.vc + b * A.vc_sb + hk * A.vc_sh;
        const uint16_t* ks = A.ks + b * A.ks_sb + hk * A.ks_sh;
        const uint16_t* vs = A.vs + b * A.vs_sb + hk * A.vs_sh;
        unsigned char* stage = sStage + wave * Sh::STAGE_B;
        uint16_t* sc0 = reinterpret_cast<uint16_t*>(stage + 2 * TILE_B);  // [tile parity][keys, values][NG][64]
        const uint32_t ldk = fta_lds_addr(stage), ldv = ldk + TILE_B;

        fta_frag qf[NG];
        f32x4 first[NG];  // -24 sum q over the group, the key products' first addend
        {
            const uint16_t* qp = a.q + q_offset(a, b, hk, min(r, a.R - 1));
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const int d = 32 * g + 8 * qt;
                const fta_frag x = (r < a.R && d < a.Dreal) ? *reinterpret_cast<const fta_frag*>(qp + d) : fta_frag{0u, 0u, 0u, 0u};
                float s = 0.f;
#pragma unroll
                for (int e = 0; e < 4; ++e) s += Elem<DT>::to_f32((uint16_t)(x[e] & 0xffffu)) + Elem<DT>::to_f32((uint16_t)(x[e] >> 16));
                s = -24.f * fta_sum_quarters(s);
                first[g] = f32x4{s, s, s, s};
                qf[g] = fta_paired(x);
            }
        }
        auto key = [&](int it) { return 64 * (it < ns ? it : c_lo + it - ns); };
        auto whole = [&](int kb) { return kb + 64 <= ke && (kb >= kb0 || kb + 64 <= a.sinks); };
        // keys that no row sees are taken from one that is seen (masked)
        auto seen = [&](int t) -> int64_t { return t >= ke ? ke - 1 : (t < kb0 && t >= a.sinks) ? kb0 : t; };
        uint32_t koff[NG], voff[NG];  // of this lane's 16 bytes of a tile
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const int s = i * 64 + lane, row = s / NG, p = s - row * NG;
            koff[i] = row * ROW_B + Sh::kslot(row, p) * 16;
            voff[i] = row * ROW_B + Sh::vslot(row, p) * 16;
        }
        auto codes = [&](const uint8_t* base, const uint32_t* off, int kb, uint32_t lds) __attribute__((always_inline)) {
            if (whole(kb)) {
                const uint8_t* tile = base + (int64_t)kb * ROW_B;
#pragma unroll
                for (int i = 0; i < NG; ++i) fta_dma16_so(tile, off[i], lds + i * 1024);
            } else {
#pragma unroll
                for (int i = 0; i < NG; ++i) {
                    const int row = (i * 64 + lane) / NG;
                    fta_dma16_at(base + seen(kb + row) * ROW_B + (off[i] - row * ROW_B), lds + i * 1024);
                }
            }
        };
        struct Scales {
            Words<NS> k, v;
        };
        auto scales = [&](int kb) __attribute__((always_inline)) {  // of key kb + lane
            const int64_t row = whole(kb) ? kb + lane : seen(kb + lane);
            return Scales{load_scales<NG>(ks + row * NG), load_scales<NG>(vs + row * NG)};
        };
        auto put_scales = [&](const Scales& x, uint16_t* sc) __attribute__((always_inline)) {
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                sc[64 * g + lane] = (uint16_t)(x.k.w[g / 2] >> (16 * (g & 1)));
                sc[64 * (NG + g) + lane] = (uint16_t)(x.v.w[g / 2] >> (16 * (g & 1)));
            }
        };
        // this lane's key words: row 16 (r16 >> 2) + 4 t + (r16 & 3) of product t, its words qt NG ..
        const int krow = 16 * (r16 >> 2) + (r16 & 3);
        auto key_words = [&](int t) __attribute__((always_inline)) {
            const unsigned char* row = stage + (krow + 4 * t) * ROW_B;
            Words<NG> x;
            if constexpr (NG == 8) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    __builtin_memcpy(&x.w[4 * h], __builtin_assume_aligned(row + Sh::kslot(krow + 4 * t, 2 * qt + h) * 16, 16), 16);
            } else if constexpr (NG == 4) {
                __builtin_memcpy(&x, __builtin_assume_aligned(row + Sh::kslot(krow + 4 * t, qt) * 16, 16), 16);
            } else if constexpr (NG == 2) {
                __builtin_memcpy(&x, __builtin_assume_aligned(row + Sh::kslot(krow + 4 * t, qt >> 1) * 16 + 8 * (qt & 1), 8), 8);
            } else {
                __builtin_memcpy(&x, __builtin_assume_aligned(row + qt * 4 * NG, 4), 4 * NG);
            }
            return x;
        };
        const uint32_t vrow = ldv + (16 * qt + r16) * ROW_B;
        const uint32_t sixteen_k = fta_in_vgpr(kFtaSixteen<DT>), sixteen_v = fta_in_vgpr(kFtaSixteen<FTA_DTYPE_BF16>);
        const float zero = __builtin_bit_cast(float, fta_in_vgpr(0u));  // products of fp16 and fp32 numbers are one instruction as multiply-adds
        const fta_frag less24 = fta_frag{0xc1c0c1c0u, 0xc1c0c1c0u, 0xc1c0c1c0u, 0xc1c0c1c0u};  // bf16

        fta_wait_vmcnt<0>();  // the Q loads: the DMAs are invisible to the compiler's wait counting
        int it = it0 + wave, kb = key(it);
        Scales sreg = scales(kb);
        codes(kc, koff, kb, ldk);
        codes(vc, voff, kb, ldv);
        put_scales(sreg, sc0);
        if (it + NW < it1) sreg = scales(key(it + NW));
        fta_wait_vmcnt<0>();
        int odd = 0;
        while (true) {
            fta_wait_vmcnt<NG>();  // the key codes are there; the last NG, the value codes, may be on their way
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("" ::: "memory");
            const uint16_t* sks = sc0 + odd * (Sh::SC_B / 2);
            const uint16_t* svs = sks + 64 * NG;
            f32x4 s[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const Words<NG> kw = key_words(t);
#pragma unroll
                for (int i = 0; i < 4; ++i) s[t][i] = zero;
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const f32x4 x = fta_mma16<DT>(fta_codes16<DT>(kw.w[g], sixteen_k), qf[g], first[g]);
                    Words<2> d;  // scales of keys 16 qt + 4 t + i
                    __builtin_memcpy(&d, __builtin_assume_aligned(sks + 64 * g + 16 * qt + 4 * t, 8), 8);
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[t][i] = fmaf(half_of(d.w[i >> 1], i & 1), x[i], s[t][i]);
                }
            }
            if (!(kb + 63 <= p0 && (kb >= p1 - a.left || kb + 63 < a.sinks))) {  // (rows past R are never written)
                const int k0 = kb + 16 * qt;
                const uint32_t m = fta_bits_below(pos + 1 - k0) & (~fta_bits_below(pos - a.left - k0) | fta_bits_below(a.sinks - k0));
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e >> 2][e & 3] = (m >> e) & 1u ? s[e >> 2][e & 3] : -FTA_INF;
            }
            float mx = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3]));
#pragma unroll
            for (int t = 1; t < 4; ++t) mx = fmaxf(mx, fmaxf(fmaxf(s[t][0], s[t][1]), fmaxf(s[t][2], s[t][3])));
            mx = fta_max_quarters(mx);
            const float mn = fmaxf(m_run, mx);
            const bool grow = (mn - m_run) * a.c > 8.f;  // rescaled only where P could pass 2^8
            if (__ballot(grow) != 0ull) {
                const float alpha = grow ? fta_exp2((m_run - mn) * a.c) : 1.f;
#pragma unroll
                for (int i = 0; i < 2 * NG; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) oacc[i][e] *= alpha;
                l_run *= alpha;
                if (grow) m_run = mn;
            }
            const float mc = (m_run == -FTA_INF) ? 0.f : m_run * a.c;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[t][i] = fta_exp2(fmaf(s[t][i], a.c, -mc));
                    l_run += s[t][i];
                }
            // the value codes and the next tile's scales are there, and every read of the key codes has returned
            const bool more = it + NW < it1;
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
            asm volatile("" ::: "memory");
            const int kn = key(it + NW);
            if (more) {
                put_scales(sreg, sc0 + (odd ^ 1) * (Sh::SC_B / 2));
                if (it + 2 * NW < it1) sreg = scales(key(it + 2 * NW));
                codes(kc, koff, kn, ldk);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                Words<8> d;  // scales of the lane's keys 16 qt + 4 t + i
                __builtin_memcpy(&d, __builtin_assume_aligned(svs + 64 * g + 16 * qt, 16), 32);
                fta_frag hi[2], lo[2];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float x = fmaf(half_of(d.w[4 * h + (i >> 1)], i & 1), s[2 * h][i], zero);
                        const float y = fmaf(half_of(d.w[4 * h + 2 + (i >> 1)], i & 1), s[2 * h + 1][i], zero);
                        hi[h][i] = Elem<FTA_DTYPE_BF16>::pack2(x, y);
                        if constexpr (DT == FTA_DTYPE_F16)
                            lo[h][i] = Elem<FTA_DTYPE_BF16>::pack2(x - __builtin_bit_cast(float, hi[h][i] << 16),
                                                                   y - __builtin_bit_cast(float, hi[h][i] & 0xffff0000u));
                    }
#pragma unroll
                for (int ct = 0; ct < 2; ++ct) {  // 16 columns
                    typedef int v2i __attribute__((ext_vector_type(2)));
                    const uint32_t at = vrow + Sh::vslot(16 * qt + r16, g) * 16 + 8 * ct;
                    const v2i w = __builtin_amdgcn_ds_read_tr4_b64_v2i32((__attribute__((address_space(3))) v2i*)at);
                    f32x4& o = oacc[2 * g + ct];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const fta_frag v = fta_codes16<FTA_DTYPE_BF16>((uint32_t)w[h], sixteen_v);
                        o = fta_mma16<FTA_DTYPE_BF16>(v, hi[h], o);
                        o = fta_mma16<FTA_DTYPE_BF16>(less24, hi[h], o);
                        if constexpr (DT == FTA_DTYPE_F16) {
                            o = fta_mma16<FTA_DTYPE_BF16>(v, lo[h], o);
                            o = fta_mma16<FTA_DTYPE_BF16>(less24, lo[h], o);
                        }
                    }
                }
            }
            if (!more) break;
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): every read of the value codes has returned
            asm volatile("" ::: "memory");
            codes(vc, voff, kn, ldv);
            kb = kn;
            it += NW;
            odd ^= 1;
        }
    }

    // merge of the waves through LDS (the stages are done with)
    const float L = fta_sum_quarters(l_run);
    __syncthreads();
    float* so = reinterpret_cast<float*>(sStage);
    float2* sml = reinterpret_cast<float2*>(sStage + Sh::MERGE_B);
    if (lane < 16) sml[wave * 16 + lane] = make_float2(m_run, L);
#pragma unroll
    for (int i = 0; i < 2 * NG; ++i)
        *reinterpret_cast<float4*>(so + (wave * 16 + r16) * Sh::OROW + 16 * i + 4 * qt) =
            make_float4(oacc[i][0], oacc[i][1], oacc[i][2], oacc[i][3]);
    __syncthreads();
    cache_merge<DT, 32 * NG, (NG <= 2 ? 64 : NG <= 4 ? 128 : 256), 16, Sh::OROW, NW>(a, bhk, b, hk, r_lo, r_n, sp, so, sml);
}

// ----------------------------------------------------------------------------
// A cache's rows in 16 bits: a thread expands eight codes of a key or value row (one word, one
// scale) to 16 bytes.  What bounds it: memory, 32768 rows of 8 heads of 128 in 32 us (172 MB, 5.3 TB/s).
// ----------------------------------------------------------------------------
struct Q4Read {
    const uint8_t *kc, *vc;
    const uint16_t *ks, *vs;
    int64_t kc_sb, kc_sh, vc_sb, vc_sh, ks_sb, ks_sh, vs_sb, vs_sh;
    uint16_t *k, *v;  // [B][S][Hk][D]
    int Hk, S, D, NG;
    int64_t total;    // B * S * Hk * (D / 8)
};

template <int DT>
__global__ __launch_bounds__(256) void fta_q4_read_kernel(Q4Read a) {
    const int oct = a.D / 8;
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < a.total; e += (int64_t)gridDim.x * 256) {
        const int64_t row = e / oct;
        const int c = (int)(e - row * oct), g = c >> 2, o = c & 3;
        const int64_t tok = row / a.Hk;
        const int hk = (int)(row - tok * a.Hk), b = (int)(tok / a.S);
        const int64_t t = tok - (int64_t)b * a.S;
        const int rb = 16 * a.NG;
        const uint32_t wk = *reinterpret_cast<const uint32_t*>(a.kc + b * a.kc_sb + hk * a.kc_sh + t * rb + 4 * (o * a.NG + g));
        const uint32_t wv = *reinterpret_cast<const uint32_t*>(a.vc + b * a.vc_sb + hk * a.vc_sh + t * rb + 4 * c);
        const float dk = half_of(a.ks[b * a.ks_sb + hk * a.ks_sh + t * a.NG + g], 0);
        const float dv = half_of(a.vs[b * a.vs_sb + hk * a.vs_sh + t * a.NG + g], 0);
        uint4 xk, xv;
        uint32_t* pk = &xk.x;
        uint32_t* pv = &xv.x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            auto val = [](uint32_t w, int n, float d) { return d * (float)((int)((w >> (4 * n)) & 15u) - 8); };
            pk[i] = Elem<DT>::pack2(val(wk, 2 * i, dk), val(wk, 2 * i + 1, dk));
            pv[i] = Elem<DT>::pack2(val(wv, 2 * i, dv), val(wv, 2 * i + 1, dv));
        }
        *reinterpret_cast<uint4*>(a.k + e * 8) = xk;
        *reinterpret_cast<uint4*>(a.v + e * 8) = xv;
    }
}

// ---------------------------------------------------------------------- host

int q4_dims(int B, int Hk, int S, int D) {
    if (B <= 0 || Hk <= 0 || S <= 0 || D <= 0) return fta::arg_error("q4 cache: dims must be positive");
    if (D % 16 != 0 || D > 256) return fta::arg_error("q4 cache: D must be a multiple of 16 up to 256");
    if (S > (1 << 29) || Hk > (1 << 20)) return fta::unsupported("q4 cache: sizes past 2^29 keys or 2^20 heads");
    if (!fta::size_fits(B, S, Hk, D)) return fta::unsupported("q4 cache: 2^60 elements and more");
    return FTA_OK;
}

// Geometry and parts.
int q4_plan(CacheArgs& a, int B, int H, int Hk, int T, int S, int D, int left, int sinks) {
    int rc = q4_dims(B, Hk, S, D);
    if (rc != FTA_OK) return rc;
    if (H <= 0 || T <= 0) return fta::arg_error("q4_attn: dims must be positive");
    if (H % Hk != 0) return fta::arg_error("q4_attn: num_heads must be a multiple of num_kv_heads");
    if (left < 0 || sinks < 0) return fta::arg_error("q4_attn: window and num_sinks must be non-negative");
    if (T > (1 << 20) || H > (1 << 20)) return fta::unsupported("q4_attn: more than 2^20 new tokens or heads");
    if (!fta::size_fits(B, T, H, D)) return fta::unsupported("q4_attn: 2^60 elements and more");
    a = CacheArgs{};
    a.B = B, a.T = T, a.H = H, a.Hk = Hk, a.G = H / Hk, a.S = S, a.Dreal = D;
    if ((int64_t)T * a.G > (1 << 24)) return fta::unsupported("q4_attn: more than 2^24 rows per K/V head");
    a.R = T * a.G;
    a.left = std::min(left, S);
    a.sinks = a.left >= S - 1 ? 0 : std::min(sinks, S);
    a.rows = (int64_t)B * Hk * a.R;
    a.row_tiles = (a.R + 15) / 16;
    const int64_t wgs = (int64_t)B * Hk * a.row_tiles;
    const int64_t span = std::min<int64_t>(S, (int64_t)a.left + T + a.sinks);
    const int64_t tiles = (span + 63) / 64;
    // At least 512 workgroups, down to a tile for each wave and part; and about 2048, where a wave still
    // has eight tiles of its own: three workgroups of 128 columns fit a CU, and 768 at a time leave a
    // long tail of a call of, say, 1024.  Target 512 / 1024 / 2048 / 4096, us of both kernels, 32 / 8 heads of
    // 128, 4096 to 8192 tokens: 8 requests 24 / 26 / 30 / 29, 64 requests 100 / 117 / 104 / 109, 100 requests 168 /
    // 156 / 150 / 154, 128 requests 218 / 212 / 189 / 185; 64 requests of 2048 to 4096, 16 / 4 heads of 256 118 /
    // 131 / 157 / 197.
    auto parts = [&](int64_t target, int64_t least) { return std::min<int64_t>((target + wgs - 1) / wgs, tiles / least); };
    a.ns = (int)std::max<int64_t>(1, std::max(parts(512, 4), parts(2048, 32)));
    // workgroups of 256 threads: fewer than 2^32 threads a launch
    const int64_t most = (1 << 24) - 1;
    if (a.rows > most || wgs * a.ns > most) return fta::unsupported("q4_attn: too many rows");
    return FTA_OK;
}

template <int DT, int NG>
int launch_q4(Q4Args& A, hipStream_t st) {
    CacheArgs& a = A.c;
    a.total = a.B * a.Hk * a.row_tiles * a.ns;
    hipLaunchKernelGGL((fta_q4_attn_kernel<DT, NG>), dim3((unsigned)a.total), dim3(256), 0, st, A);
    int rc = fta::check_launch("fta_q4_attn_kernel");
    if (rc != FTA_OK || cache_slots(a) <= 1) return rc;
    hipLaunchKernelGGL((fta_cache_combine_kernel<DT, (NG <= 2 ? 64 : NG <= 4 ? 128 : 256)>), dim3((unsigned)a.rows), dim3(256), 0,
                       st, a, cache_slots(a));
    return fta::check_launch("fta_cache_combine_kernel");
}

template <int DT>
int launch_q4_groups(Q4Args& A, hipStream_t st) {
    switch ((A.c.Dreal + 31) / 32) {
        case 1: return launch_q4<DT, 1>(A, st);
        case 2: return launch_q4<DT, 2>(A, st);
        case 3: return launch_q4<DT, 3>(A, st);
        case 4: return launch_q4<DT, 4>(A, st);
        case 5: return launch_q4<DT, 5>(A, st);
        case 6: return launch_q4<DT, 6>(A, st);
        case 7: return launch_q4<DT, 7>(A, st);
        default: return launch_q4<DT, 8>(A, st);
    }
}

// 16-byte steps of the codes; of the scales 4-byte steps where a row has an even number of them
bool q4_aligned(const void* codes, const int64_t* cs, const void* scales, const int64_t* ss, int D) {
    const int even = (D + 31) / 32 % 2 == 0;
    return ((uintptr_t)codes & 15) == 0 && ((cs[0] | cs[1]) & 15) == 0 && ((uintptr_t)scales & (even ? 3 : 1)) == 0 &&
           ((ss[0] | ss[1]) & even) == 0;
}

}  // namespace

extern "C" {

size_t fta_q4_attn_workspace_size(int B, int H, int Hk, int T, int S, int D, int left, int num_sinks) {
    CacheArgs a;
    if (q4_plan(a, B, H, Hk, T, S, D, left, num_sinks) != FTA_OK) return 0;
    return cache_bytes(a, kernel_dim(D));
}

int fta_q4_attn(const void* q, const int64_t* q_strides, const void* k_codes, const int64_t* kc_strides, const void* k_scales,
                const int64_t* ks_strides, const void* v_codes, const int64_t* vc_strides, const void* v_scales,
                const int64_t* vs_strides, int dtype, int B, int H, int Hk, int T, int S, int D, const int32_t* cache_lens,
                int left, int num_sinks, float scale, void* o, const int64_t* o_strides, float* lse, void* workspace,
                size_t workspace_bytes, void* stream) {
    FTA_TRY_BEGIN
    Q4Args A = {};
    CacheArgs& a = A.c;
    int rc = q4_plan(a, B, H, Hk, T, S, D, left, num_sinks);
    if (rc != FTA_OK) return rc;
    if (dtype != FTA_DTYPE_BF16 && dtype != FTA_DTYPE_F16) return fta::arg_error("q4_attn: dtype must be bf16 or fp16");
    if (!(scale > 0.f) || scale > 2.0e38f)  // times log2(e) still finite
        return fta::arg_error("q4_attn: scale must be positive and at most 2e38");
    const size_t need = cache_bytes(a, kernel_dim(D));
    if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return fta::arg_error("q4_attn: workspace too small");
    if (!fta::all_set(q, q_strides, k_codes, kc_strides, k_scales, ks_strides, v_codes, vc_strides, v_scales, vs_strides,
                      cache_lens, o, o_strides, lse))
        return fta::arg_error("q4_attn: a required pointer is null");
    if (!q4_aligned(k_codes, kc_strides, k_scales, ks_strides, D) || !q4_aligned(v_codes, vc_strides, v_scales, vs_strides, D))
        return fta::arg_error("q4_attn: the heads' codes must be 16-byte aligned, their scales 4-byte");
    a.q = (const uint16_t*)q, a.q_sb = q_strides[0], a.q_sh = q_strides[1], a.q_sn = q_strides[2];
    A.kc = (const uint8_t*)k_codes, A.kc_sb = kc_strides[0], A.kc_sh = kc_strides[1];
    A.vc = (const uint8_t*)v_codes, A.vc_sb = vc_strides[0], A.vc_sh = vc_strides[1];
    A.ks = (const uint16_t*)k_scales, A.ks_sb = ks_strides[0], A.ks_sh = ks_strides[1];
    A.vs = (const uint16_t*)v_scales, A.vs_sb = vs_strides[0], A.vs_sh = vs_strides[1];
    a.lens = cache_lens;
    a.o = (uint16_t*)o, a.o_sb = o_strides[0], a.o_sh = o_strides[1], a.o_sn = o_strides[2];
    a.lse = lse;
    a.c = scale * kLog2e;
    a.part_ml = (float2*)workspace;
    a.part_o = need > 0 ? (float*)((char*)workspace + ml_bytes(a)) : nullptr;
    hipStream_t st = (hipStream_t)stream;
    return dtype == FTA_DTYPE_BF16 ? launch_q4_groups<FTA_DTYPE_BF16>(A, st) : launch_q4_groups<FTA_DTYPE_F16>(A, st);
    FTA_TRY_END
}

int fta_q4_read(const void* k_codes, const int64_t* kc_strides, const void* k_scales, const int64_t* ks_strides,
                const void* v_codes, const int64_t* vc_strides, const void* v_scales, const int64_t* vs_strides, int dtype,
                int B, int Hk, int S, int D, void* k, void* v, void* stream) {
    FTA_TRY_BEGIN
    int rc = q4_dims(B, Hk, S, D);
    if (rc != FTA_OK) return rc;
    if (dtype != FTA_DTYPE_BF16 && dtype != FTA_DTYPE_F16) return fta::arg_error("q4_read: dtype must be bf16 or fp16");
    if (!fta::all_set(k_codes, kc_strides, k_scales, ks_strides, v_codes, vc_strides, v_scales, vs_strides, k, v))
        return fta::arg_error("q4_read: a required pointer is null");
    if (!q4_aligned(k_codes, kc_strides, k_scales, ks_strides, D) || !q4_aligned(v_codes, vc_strides, v_scales, vs_strides, D))
        return fta::arg_error("q4_read: the heads' codes must be 16-byte aligned, their scales 4-byte");
    Q4Read a = {};
    a.kc = (const uint8_t*)k_codes, a.kc_sb = kc_strides[0], a.kc_sh = kc_strides[1];
    a.vc = (const uint8_t*)v_codes, a.vc_sb = vc_strides[0], a.vc_sh = vc_strides[1];
    a.ks = (const uint16_t*)k_scales, a.ks_sb = ks_strides[0], a.ks_sh = ks_strides[1];
    a.vs = (const uint16_t*)v_scales, a.vs_sb = vs_strides[0], a.vs_sh = vs_strides[1];
    a.k = (uint16_t*)k, a.v = (uint16_t*)v;
    a.Hk = Hk, a.S = S, a.D = D, a.NG = (D + 31) / 32;
    a.total = (int64_t)B * S * Hk * (D / 8);
    const dim3 g((unsigned)std::min<int64_t>((a.total + 255) / 256, 256 * 32));
    hipStream_t st = (hipStream_t)stream;
    if (dtype == FTA_DTYPE_BF16)
        hipLaunchKernelGGL((fta_q4_read_kernel<FTA_DTYPE_BF16>), g, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((fta_q4_read_kernel<FTA_DTYPE_F16>), g, dim3(256), 0, st, a);
    return fta::check_launch("fta_q4_read_kernel");
    FTA_TRY_END
}

}  // extern "C"
