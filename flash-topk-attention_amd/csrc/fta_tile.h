// Attention of 32 query rows against tiles of 32 NH keys in LDS: the inner step of the
// window and cache kernels.
//
// K and V tiles are row-major ([32 NH][D], rows swizzled by FtaSwz) and filled by LDS
// DMA.  A wave owns 32 query rows as the columns of S^T = K Q^T (32x32x16 MFMA, NH
// 32-key parts), so a row's scores are 16 registers each of lanes l and l + 32 and
// its maximum and sum are lane values; P^T in that layout is the B operand of
// O^T += V^T P^T as it stands, V^T coming from LDS transpose reads.
#pragma once

#include <type_traits>

#include "fta_common.h"

// f(integral_constant<int, I>) for I = I0 .. N - 1
template <int I, int N, typename F>
__device__ __forceinline__ void fta_static_for(F& f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        fta_static_for<I + 1, N>(f);
    }
}

// A wave-uniform value in a scalar register (integer divisions leave theirs in vector
// registers, and the DMA's base address has to be formed by scalar instructions: a
// VMEM instruction may not read a scalar register in the five cycles after a vector
// instruction wrote it, and nothing sees that distance into inline asm).
__device__ __forceinline__ int fta_scalar(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Bits [lo, hi) of a 32-bit mask; lo and hi may lie anywhere.
__device__ __forceinline__ uint32_t fta_bits_below(int hi) { return hi >= 32 ? 0xffffffffu : hi <= 0 ? 0u : (1u << hi) - 1u; }
__device__ __forceinline__ uint32_t fta_bits(int lo, int hi) { return fta_bits_below(hi) & ~fta_bits_below(lo); }

// An MFMA operand fragment.  A vector type all the way from its load: as a struct of four
// words the compiler may read it word by word (two ds_read2_b32 instead of one
// ds_read_b128, which conflict in LDS: the D = 256 forward spent two thirds of its LDS
// cycles on that).
typedef unsigned int fta_frag __attribute__((ext_vector_type(4)));

template <int DT>
__device__ __forceinline__ f32x16 fta_mma(fta_frag a, fta_frag b, f32x16 c) {
    if constexpr (DT == FTA_DTYPE_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(fta_bf16x8, a), __builtin_bit_cast(fta_bf16x8, b), c,
                                                       0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(fta_f16x8, a), __builtin_bit_cast(fta_f16x8, b), c, 0,
                                                      0, 0);
}
// 16 bytes of LDS, and two 8-byte transpose reads, by byte address
__device__ __forceinline__ fta_frag fta_lds_frag(uint32_t addr) {
    return *(__attribute__((address_space(3))) const fta_frag*)addr;
}
__device__ __forceinline__ fta_frag fta_lds_tr_frag(uint32_t lo, uint32_t hi) {
    const fta_s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((fta_lds_s16x4*)lo);
    const fta_s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((fta_lds_s16x4*)hi);
    return __builtin_bit_cast(fta_frag, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}
// eight fp32 values rounded to a fragment
template <int DT>
__device__ __forceinline__ fta_frag fta_pack_frag(const float* f) {
    return fta_frag{Elem<DT>::pack2(f[0], f[1]), Elem<DT>::pack2(f[2], f[3]), Elem<DT>::pack2(f[4], f[5]),
                    Elem<DT>::pack2(f[6], f[7])};
}

// Per-lane byte offsets of the operand fragments in a tile of D columns: K (or V) rows,
// and the two halves of a transposed fragment.  Other k slices and column tiles differ by
// an XOR of their slot bits, 16 or 32 rows down by a constant.
struct FtaLane {
    uint32_t row, tr0, tr1;
};
template <int D>
__device__ __forceinline__ FtaLane fta_lane_offsets(int lane) {
    using SW = FtaSwz<D / 8>;
    const int vr = 4 * (lane >> 5) + ((lane & 15) >> 2), vc = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    return {2u * SW::off(lane & 31, lane >> 5), 2u * (SW::off(vr, vc >> 3) + (vc & 7)),
            2u * (SW::off(vr + 8, vc >> 3) + (vc & 7))};
}

template <int DT, int D, int NH>
struct FtaTile {
    using E = Elem<DT>;
    static constexpr int QSEG = D / 8;         // 16-byte slots per row
    static constexpr int KEYS = 32 * NH;
    static constexpr int SLOTS = KEYS * QSEG;  // per tile
    static constexpr int TEN_B = SLOTS * 16;   // bytes per tile
    static constexpr int KS = D / 16, DT32 = D / 32;
    using SW = FtaSwz<QSEG>;

    __device__ static __forceinline__ fta_frag row_frag(uint32_t base, const FtaLane& l, int half, int ks) {
        return fta_lds_frag(((base + l.row) ^ (ks * 32)) + half * 32 * QSEG * 16);
    }
    __device__ static __forceinline__ fta_frag tr_frag(uint32_t base, const FtaLane& l, int ks, int dt) {
        const uint32_t x = ks * 16 * QSEG * 16;
        return fta_lds_tr_frag(((base + l.tr0) ^ (dt * 64)) + x, ((base + l.tr1) ^ (dt * 64)) + x);
    }

    // s[half] = (K Q^T)[32 half .. + 31][row], fragments read PD MFMAs ahead.
    template <int PD>
    __device__ static __forceinline__ void qk(uint32_t kbase, const FtaLane& l, const fta_frag* qf, f32x16* s) {
        fta_frag fr[PD + 1];
        auto load = [&](auto nn) __attribute__((always_inline)) {
            constexpr int n = decltype(nn)::value;
            if constexpr (n < NH * KS) fr[n % (PD + 1)] = row_frag(kbase, l, n % NH, n / NH);
        };
        auto slot = [&](auto nn) __attribute__((always_inline)) {
            constexpr int n = decltype(nn)::value;
            if constexpr (n % 2 == 0) __builtin_amdgcn_sched_barrier(0);
            load(std::integral_constant<int, n + PD>{});
            if constexpr (n < NH) {
#pragma unroll
                for (int i = 0; i < 16; ++i) s[n][i] = 0.f;
            }
            s[n % NH] = fta_mma<DT>(fr[n % (PD + 1)], qf[n / NH], s[n % NH]);
        };
        fta_static_for<0, PD>(load);
        fta_static_for<0, NH * KS>(slot);
        __builtin_amdgcn_sched_barrier(0);
    }

    // Online softmax of the tile's scores (masked ones are -inf) and O^T += V^T P^T.
    // The accumulators are rescaled only when a row's maximum grows by more than 2^8:
    // P stays below 2^8 and its 16-bit rounding keeps the same relative error.  A row
    // that has seen no key yet keeps m = -inf and adds exact zeros.
    template <int PD>
    __device__ static __forceinline__ void softmax_pv(uint32_t vbase, const FtaLane& l, const f32x16* s, float c,
                                                      float& m_run, float& l_run, f32x16* oacc) {
        float mx = s[0][0];
#pragma unroll
        for (int sb = 0; sb < NH; ++sb)
#pragma unroll
            for (int i = (sb == 0); i < 16; ++i) mx = fmaxf(mx, s[sb][i]);
        {
            float x = mx, y = mx;  // the row's other half of the keys is in lane ^ 32
            fta_swap32(x, y);
            mx = fmaxf(x, y);
        }
        const float mn = fmaxf(m_run, mx);
        const bool grow = (mn - m_run) * c > 8.f;
        if (__ballot(grow) != 0ull) {
            const float alpha = grow ? fta_exp2((m_run - mn) * c) : 1.f;
#pragma unroll
            for (int dt = 0; dt < DT32; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) oacc[dt][i] *= alpha;
            l_run *= alpha;
            if (grow) m_run = mn;
        }
        const float mc = (m_run == -FTA_INF) ? 0.f : m_run * c;
        float ls = 0.f;
        constexpr int NM = 2 * NH * DT32;
        fta_frag fr[PD + 1];
        fta_frag pf;
        auto load = [&](auto nn) __attribute__((always_inline)) {
            constexpr int n = decltype(nn)::value;
            if constexpr (n < NM) fr[n % (PD + 1)] = tr_frag(vbase, l, n / DT32, n % DT32);
        };
        auto slot = [&](auto nn) __attribute__((always_inline)) {
            constexpr int n = decltype(nn)::value, ks = n / DT32;
            if constexpr (n % 2 == 0) __builtin_amdgcn_sched_barrier(0);
            load(std::integral_constant<int, n + PD>{});
            if constexpr (n % DT32 == 0) {
                float pv[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    pv[e] = fta_exp2(fmaf(s[ks >> 1][8 * (ks & 1) + e], c, -mc));
                    ls += pv[e];
                }
                pf = fta_pack_frag<DT>(pv);
            }
            oacc[n % DT32] = fta_mma<DT>(fr[n % (PD + 1)], pf, oacc[n % DT32]);
        };
        fta_static_for<0, PD>(load);
        fta_static_for<0, NM>(slot);
        __builtin_amdgcn_sched_barrier(0);
        l_run += ls;
    }

    // -inf for the scores of 32 keys whose bit of `seen` (bit = key) is clear.
    __device__ static __forceinline__ void mask(uint32_t seen, int lane, f32x16& s) {
        const uint32_t m = seen >> (4 * (lane >> 5));  // register r holds key (r >> 2) * 8 + (r & 3) of these
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const uint32_t k = (uint32_t)(((int)(m << (31 - ((r >> 2) * 8 + (r & 3))))) >> 31);
            const float v = s[r];
            s[r] = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, v) & k) | (0xff800000u & ~k));
        }
    }

    // A wave's Q (or dO) rows as B operands: row `ok ? p : none` of this lane, zero past Dreal.
    __device__ static __forceinline__ void load_rows(const uint16_t* p, bool ok, int Dreal, int lane, fta_frag* f) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int d = ks * 16 + (lane >> 5) * 8;
            f[ks] = (ok && d < Dreal) ? *reinterpret_cast<const fta_frag*>(p + d) : fta_frag{0u, 0u, 0u, 0u};
        }
    }
    // One row of O^T (this lane's column), scaled and rounded once.
    __device__ static __forceinline__ void store_row(uint16_t* p, int Dreal, int lane, const f32x16* acc, float f) {
#pragma unroll
        for (int dt = 0; dt < DT32; ++dt)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int d = dt * 32 + c_row(i, lane);
                if (d < Dreal)
                    *reinterpret_cast<uint2*>(p + d) =
                        make_uint2(E::pack2(acc[dt][i] * f, acc[dt][i + 1] * f), E::pack2(acc[dt][i + 2] * f, acc[dt][i + 3] * f));
            }
    }
};

// Fills one K and one V tile of KEYS rows by LDS DMA, NW waves together: LQ instructions
// per wave and tensor, instruction i of a wave writing the 1 KB block i * NW + wave.
template <int D, int NW, int KEYS>
struct FtaGather {
    static constexpr int QSEG = D / 8, LQ = KEYS * QSEG / (64 * NW), TEN_B = KEYS * QSEG * 16;
    static_assert((KEYS * QSEG) % (64 * NW) == 0, "whole DMA instructions per wave");
    using SW = FtaSwz<QSEG>;

    uint32_t koff[LQ], voff[LQ];  // row * stride + column, in bytes (token strides up to 2^24 elements)

    __device__ __forceinline__ void start(int64_t k_sn, int64_t v_sn, int Dreal, int wave, int lane) {
#pragma unroll
        for (int i = 0; i < LQ; ++i) {
            const int sidx = (i * NW + wave) * 64 + lane;
            const int row = sidx / QSEG;
            int j = SW::slot(row, sidx - row * QSEG);
            if (j * 8 >= Dreal) j = 0;  // columns past D: they meet zero Q columns or are never stored
            koff[i] = 2u * (row * (uint32_t)k_sn + j * 8);
            voff[i] = 2u * (row * (uint32_t)v_sn + j * 8);
        }
    }
    // rows kb .. kb + KEYS - 1, all of them inside the tensor
    __device__ __forceinline__ void whole(const uint16_t* kp, const uint16_t* vp, int64_t k_sn, int64_t v_sn, int kb,
                                          uint32_t lds, int wave) const {
        const uint16_t* kbp = kp + (int64_t)kb * k_sn;
        const uint16_t* vbp = vp + (int64_t)kb * v_sn;
#pragma unroll
        for (int i = 0; i < LQ; ++i) fta_dma16_so(kbp, koff[i], lds + (i * NW + wave) * 1024);
#pragma unroll
        for (int i = 0; i < LQ; ++i) fta_dma16_so(vbp, voff[i], lds + TEN_B + (i * NW + wave) * 1024);
    }
    // rows row_of(kb), row_of(kb + 1), ...: 64-bit addresses, formed here so that this
    // rarer case keeps nothing live
    template <typename F>
    __device__ __forceinline__ void mapped(const uint16_t* kp, const uint16_t* vp, int64_t k_sn, int64_t v_sn, int kb,
                                           int Dreal, uint32_t lds, int wave, int lane, F row_of) const {
        asm volatile("" : "+v"(lane));
#pragma unroll
        for (int i = 0; i < LQ; ++i) {
            const int sidx = (i * NW + wave) * 64 + lane;
            const int row = sidx / QSEG;
            int j = SW::slot(row, sidx - row * QSEG);
            if (j * 8 >= Dreal) j = 0;
            const int64_t t = row_of(kb + row);
            fta_dma16_at(kp + t * k_sn + j * 8, lds + (i * NW + wave) * 1024);
            fta_dma16_at(vp + t * v_sn + j * 8, lds + TEN_B + (i * NW + wave) * 1024);
        }
    }
};
