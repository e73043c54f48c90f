// Attention of 32 query rows against tiles of 32 keys in LDS: the inner step of the
// window and cache kernels.
//
// K and V tiles are row-major ([32][D], rows swizzled by FtaSwz) and filled by LDS
// DMA.  A wave owns 32 query rows as the columns of S^T = K Q^T (32x32x16 MFMA),
// so a row's scores are 16 registers each of lanes l and l + 32 and
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

// A 32-bit mask of the bits below hi, which may lie anywhere.
__device__ __forceinline__ uint32_t fta_bits_below(int hi) { return hi >= 32 ? 0xffffffffu : hi <= 0 ? 0u : (1u << hi) - 1u; }

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

// Per-lane LDS addresses of the operand fragments of a 32-row tile of D columns at `base`
// (a multiple of 1024): rows (K or V as they stand), and the two halves of a transposed
// fragment.  k slices and column tiles differ by an XOR of their slot bits; 16 rows, other
// tiles and other stages by constants that go into the instructions' offsets.  KEPT: every
// XOR is formed once and held; else at each use, where registers are short.
template <int D, bool KEPT = (D <= 128)>
struct FtaAddr {
    static constexpr int KS = D / 16, DT32 = D / 32;
    uint32_t row_[KEPT ? KS : 1], tr0_[KEPT ? DT32 : 1], tr1_[KEPT ? DT32 : 1];

    __device__ __forceinline__ FtaAddr(uint32_t base, int lane) {
        using SW = FtaSwz<D / 8>;
        const int vr = 4 * (lane >> 5) + ((lane & 15) >> 2), vc = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
        const uint32_t r = base + 2u * SW::off(lane & 31, lane >> 5);
        const uint32_t t0 = base + 2u * (SW::off(vr, vc >> 3) + (vc & 7));
        const uint32_t t1 = base + 2u * (SW::off(vr + 8, vc >> 3) + (vc & 7));
#pragma unroll
        for (int k = 0; k < (KEPT ? KS : 1); ++k) row_[k] = r ^ (k * 32);
#pragma unroll
        for (int d = 0; d < (KEPT ? DT32 : 1); ++d) {
            tr0_[d] = t0 ^ (d * 64);
            tr1_[d] = t1 ^ (d * 64);
        }
    }
    // Where the XORs are not kept: the same addresses, opaque to the compiler, which would else
    // form every XOR ahead of the loop all the same, and spill.
    __device__ __forceinline__ FtaAddr here() const {
        FtaAddr x = *this;
        if constexpr (!KEPT) asm volatile("" : "+v"(x.row_[0]), "+v"(x.tr0_[0]), "+v"(x.tr1_[0]));
        return x;
    }
    // rows 0 .. 31 of the tile `off` bytes further on, columns 16 ks .. 16 ks + 15
    __device__ __forceinline__ fta_frag row(uint32_t off, int ks) const {
        return fta_lds_frag((KEPT ? row_[KEPT ? ks : 0] : row_[0] ^ (ks * 32)) + off);
    }
    // its rows 16 ks .. 16 ks + 15 transposed, columns 32 dt .. 32 dt + 31
    __device__ __forceinline__ fta_frag tr(uint32_t off, int ks, int dt) const {
        const uint32_t x = off + ks * 16 * (D / 8) * 16;
        return fta_lds_tr_frag((KEPT ? tr0_[KEPT ? dt : 0] : tr0_[0] ^ (dt * 64)) + x,
                               (KEPT ? tr1_[KEPT ? dt : 0] : tr1_[0] ^ (dt * 64)) + x);
    }
};

template <int DT, int D>
struct FtaTile {
    using E = Elem<DT>;
    static constexpr int QSEG = D / 8;            // 16-byte slots per row
    static constexpr int TEN_B = 32 * QSEG * 16;  // bytes per 32-row tile
    static constexpr int KS = D / 16, DT32 = D / 32;

    // s = (K Q^T)[key][row] of the 32 keys at `off`, fragments read PD MFMAs ahead.
    template <int PD, typename A>
    __device__ static __forceinline__ void qk(const A& ad, uint32_t off, const fta_frag* qf, f32x16& s) {
        fta_frag fr[PD + 1];
        auto load = [&](auto nn) __attribute__((always_inline)) {
            constexpr int n = decltype(nn)::value;
            if constexpr (n < KS) fr[n % (PD + 1)] = ad.row(off, n);
        };
        auto slot = [&](auto nn) __attribute__((always_inline)) {
            constexpr int n = decltype(nn)::value;
            if constexpr (n % 2 == 0) __builtin_amdgcn_sched_barrier(0);
            load(std::integral_constant<int, n + PD>{});
            s = fta_mma<DT>(fr[n % (PD + 1)], qf[n], s);
        };
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 0.f;
        fta_static_for<0, PD>(load);
        fta_static_for<0, KS>(slot);
        __builtin_amdgcn_sched_barrier(0);
    }

    // Online softmax of those scores (masked ones are -inf) and O^T += V^T P^T, V at `off`.
    // The accumulators are rescaled only when a row's maximum grows by more than 2^8:
    // P stays below 2^8 and its 16-bit rounding keeps the same relative error.  That rounding
    // is what the matrix instructions of 16-bit V take, and as large as the rounding of o
    // itself: o is off by up to sqrt(2) times the latter (the sum l adds the unrounded P; P as
    // a sum of two 16-bit numbers would be half as many products again).  A row that has seen
    // no key yet keeps m = -inf and adds exact zeros.
    template <int PD, typename A>
    __device__ static __forceinline__ void softmax_pv(const A& ad, uint32_t off, const f32x16& s, float c, float& m_run,
                                                      float& l_run, f32x16* oacc) {
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
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
        constexpr int NM = 2 * DT32;
        fta_frag fr[PD + 1];
        fta_frag pf;
        auto load = [&](auto nn) __attribute__((always_inline)) {
            constexpr int n = decltype(nn)::value;
            if constexpr (n < NM) fr[n % (PD + 1)] = ad.tr(off, n / DT32, n % DT32);
        };
        auto slot = [&](auto nn) __attribute__((always_inline)) {
            constexpr int n = decltype(nn)::value, ks = n / DT32;
            if constexpr (n % 2 == 0) __builtin_amdgcn_sched_barrier(0);
            load(std::integral_constant<int, n + PD>{});
            if constexpr (n % DT32 == 0) {
                float pv[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    pv[e] = fta_exp2(fmaf(s[8 * ks + e], c, -mc));
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

    // -inf for the scores whose bit of `seen` (bit = key, or query row) is clear.
    __device__ static __forceinline__ void mask(uint32_t seen, int lane, f32x16& s) {
        const uint32_t m = seen >> (4 * (lane >> 5));  // register r holds (r >> 2) * 8 + (r & 3) of these
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const uint32_t k = (uint32_t)(((int)(m << (31 - ((r >> 2) * 8 + (r & 3))))) >> 31);
            const float v = s[r];
            s[r] = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, v) & k) | (0xff800000u & ~k));
        }
    }

    // A wave's Q (or dO) rows as B operands: this lane's row at p, zero past Dreal and where !ok.
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

// One wave-wide LDS DMA (fta_dma16_so) to `lds` + a constant, the sum formed in M0 itself.
template <int OFF>
__device__ __forceinline__ void fta_dma16_to(const void* base, uint32_t voff, uint32_t lds) {
    asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(base),
                 "s"(__builtin_amdgcn_readfirstlane(lds)), "i"(OFF) : "memory", "m0", "scc");
}

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
    // the KEYS rows from kp and vp, all of them inside the tensor; lds: this wave's first block
    // (the tile's address + 1024 * wave)
    __device__ __forceinline__ void whole(const uint16_t* kp, const uint16_t* vp, uint32_t lds) const {
        auto one = [&](auto ii) __attribute__((always_inline)) {
            constexpr int i = decltype(ii)::value;
            if constexpr (i < LQ)
                fta_dma16_to<i * NW * 1024>(kp, koff[i], lds);
            else
                fta_dma16_to<TEN_B + (i - LQ) * NW * 1024>(vp, voff[i - LQ], lds);
        };
        fta_static_for<0, 2 * LQ>(one);
    }
    // rows row_of(kb), row_of(kb + 1), ... of the sequence at kp and vp: 64-bit addresses,
    // formed here so that this rarer case keeps nothing live
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
            fta_dma16_at(kp + t * k_sn + j * 8, lds + i * NW * 1024);
            fta_dma16_at(vp + t * v_sn + j * 8, lds + TEN_B + i * NW * 1024);
        }
    }
};
