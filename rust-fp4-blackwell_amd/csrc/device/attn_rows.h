// Attention of query rows over an 8-bit or fp16 KV cache on the matrix cores
// (gfx950): one query row, causal prompt rows, or one row for each sequence of
// a batch over keys that all of them share and keys of their own.
//
//   out[i][h] = sum_t softmax_t(q[i][h] . k_t / sqrt(HD)) v_t
//
// over the shared keys t < len0 (causal: t <= pos0 + i) and the row's own keys
// t < lens[i].  A KV head's query rows (i, g), g < group, are packed i * group
// + g into tiles of 16, so a wave's matrix instructions serve 16 of them,
// whatever the group.  A workgroup of 4 waves takes 16 MT (4 / WK) rows and a
// chunk of keys; its WK key groups take alternate blocks of 32 keys and merge
// their softmax states through LDS.  Where the keys are split over several
// workgroups each writes its state (m, l, acc) to the caller's workspace and a
// second kernel merges them (stream order, nothing that must start at zero).
//
// K and V go from memory to registers, with no LDS:
//   S^T (32 x 16) = K . Q^T      lane (q4 = l / 16, l16 = l % 16) holds K row
//                                l16 of each 16-key half, 16 bytes at a time
//   O^T (HD x 16) += V^T . P^T   lane holds, for the 8 keys whose scores the
//                                S^T accumulators gave it, dimensions
//                                l16 HD/16 .. +HD/16 - 1: a row of 16 lanes
//                                reads whole V rows, and dimension l16 HD/16 + n
//                                is row l16 of tile n
// q and p enter as hi + lo fp16 terms (about 2^-22 relative: outputs within
// 1e-6 of exact ones; one term would leave 1e-4), e4m3 values are exact in
// fp16, products are exact and sums f32.
//
// Scales of the 8-bit cache, 2^(byte - 127) for each key: they go into the
// conversion to fp16, less a reference exponent of the wave (kref, vref), which
// keeps every value in fp16's range: the reference is raised when a byte
// exceeds it by more than 7 (codes to 448 * 2^7 = 57344), so values are exact
// down to scales 2^15 below it, and off by at most 2^-41 of the largest value
// below that.  2^kref is part of the scores' factor, 2^vref of O's.  A byte of
// 255 makes its key NaN for every row that sees it, and for no other.
#pragma once
#include "common.h"

RFP4_DEV float pow2_int(int e) // 2^e, e of -126 .. 127; smaller e count as -126
{
    return __uint_as_float((uint32_t)(max(e, -126) + 127) << 23);
}

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Keys t0 .. of one cache for one KV head: what attn_rows_keys walks.
struct AttnRowsKeys {
    const uint8_t *k, *v;   // the head's token 0
    const uint8_t *ks, *vs; // its scale byte (8-bit caches)
    uint64_t ts;            // token stride (elements)
    uint32_t lo, hi;        // keys of this workgroup, lo a multiple of 32
    uint32_t end;           // keys that exist, at least hi
};

// A wave's MT tiles of 16 query rows: lane (q4, l16) works for row l16 of each.
template <int HD, int MT>
struct AttnRowsState {
    static constexpr int KS = HD / 32; // K steps of S
    static constexpr int NN = HD / 16; // dimension tiles of O

    uint32_t l16, q4, lane;
    f16x8 qa[MT][KS], ql[MT][KS];
    f32x4 o[MT][NN];
    float m[MT], l[MT], f[MT]; // running maximum and sum, the scores' factor less 2^kref
    uint32_t lim[MT];          // keys that the lane's row sees

    // q of the lane's row of each tile, scaled by a power of two of its own to
    // at most 256, and that scale's inverse into the scores' factor.  PAIRED:
    // the dimensions of K step k in this lane as 16-byte loads of 8-bit K rows
    // hold them, two steps a load
    template <bool PAIRED>
    RFP4_DEV void load_q(const AttnRowsArgs &a, uint32_t kvh, uint32_t row0, uint32_t row_end, uint32_t limit0)
    {
        // log2(e) / sqrt(HD) in two factors: the score's factor a power of two,
        // so that a scaled score less the maximum is exact to one rounding and 0
        // for the maximum itself; the rest into q
        const float c = __fmul_rn(1.4426950408889634f, __fdiv_rn(1.0f, __fsqrt_rn((float)HD)));
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            const uint32_t rho = row0 + 16u * (uint32_t)mt + l16;
            const bool in = rho < row_end;
            const uint32_t i = min(rho, row_end - 1u) / a.group, g = min(rho, row_end - 1u) % a.group;
            lim[mt] = a.causal ? min(a.pos0 + i + 1u, limit0) : limit0;
            const float *qp = a.q + (size_t)i * a.q_rs + (size_t)(kvh * a.group + g) * HD;
            float x[KS][8];
            float amax = 0.0f;
#pragma unroll
            for (int k = 0; k < KS; k++) {
                const uint32_t d = PAIRED ? 64u * (uint32_t)(k / 2) + 16u * q4 + 8u * (uint32_t)(k % 2) : 32u * (uint32_t)k + 8u * q4;
                const float4 x0 = *(const float4 *)(qp + d), x1 = *(const float4 *)(qp + d + 4);
                x[k][0] = x0.x; x[k][1] = x0.y; x[k][2] = x0.z; x[k][3] = x0.w;
                x[k][4] = x1.x; x[k][5] = x1.y; x[k][6] = x1.z; x[k][7] = x1.w;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    x[k][j] = in ? x[k][j] : 0.0f;
                    amax = fmaxf(amax, fabsf(x[k][j]));
                }
            }
            amax = xor32_max(xor16_max(amax));
            const int e = amax > 0.0f ? min(max((int)(__float_as_uint(amax) >> 23) - 127, -110), 127) : 0; // 2^e <= amax < 2^(e+1), or smaller
            const float up = pow2_int(max(-e, -120)), up2 = pow2_int(7 - e - max(-e, -120));
#pragma unroll
            for (int k = 0; k < KS; k++) {
#pragma unroll
                for (int j = 0; j < 8; j++) x[k][j] = __fmul_rn(__fmul_rn(__fmul_rn(x[k][j], up), up2), 4.0f * c);
                // (not split_hi_lo8: of a product the compiler takes hi twice, rounded from
                // the product for the operand and from its f32 for lo, which near a tie of
                // the two leaves lo an fp16 step off: 1e-4 of such a row, one row in 250)
                split_hi_lo8_mix(x[k], qa[mt][k], ql[mt][k]);
            }
            f[mt] = __fmul_rn(pow2_int(e), 0.25f / 128.0f);
            m[mt] = -3.402823466e38f;
            l[mt] = 0.0f;
#pragma unroll
            for (int n = 0; n < NN; n++) o[mt][n] = {0.0f, 0.0f, 0.0f, 0.0f};
        }
    }

    // The scores of tile mt over the 32 keys from key0 (st: S^T of the two
    // 16-key halves, the lane's keys 4 q4 .. +3 of each; nan: the keys of scale
    // byte 255) to probabilities as two fp16 terms; keys at and past `hi` are
    // masked.  fk: the scores' factor.
    template <bool F8>
    RFP4_DEV void probabilities(int mt, const f32x4 (&st)[2], uint32_t key0, uint32_t hi, uint32_t nan, float fk, f16x8 &ph, f16x8 &pl)
    {
        float p[8];
#pragma unroll
        for (int j = 0; j < 8; j++) p[j] = st[j / 4][j % 4];
        // (the empty asm keeps what these rare branches compute out of the loop's registers)
        if (F8 && nan) {
            uint32_t k0 = 4u * q4;
            asm volatile("" : "+v"(k0));
#pragma unroll
            for (int j = 0; j < 8; j++)
                if ((nan >> (k0 + (uint32_t)(j < 4 ? j : 12 + j))) & 1u) p[j] = __uint_as_float(0x7FC00000u);
        }
        // masked scores at -infinity (p = 0 whatever maximum is subtracted)
        const uint32_t last = min(lim[mt], hi);
        if (__any(key0 + 32u > last)) {
            uint32_t k0 = key0 + 4u * q4;
            asm volatile("" : "+v"(k0));
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (k0 + (uint32_t)(j < 4 ? j : 12 + j) >= last) p[j] = -INFINITY;
        }
        // online softmax in base 2; the subtracted maximum is raised only when
        // a score of the row exceeds it by more than 8 (p at most 2^8), so the
        // common block has no cross-lane step
        float mx = p[0];
#pragma unroll
        for (int j = 1; j < 8; j++) mx = fmaxf(mx, p[j]);
        mx *= fk;
        if (__any(mx > m[mt] + 8.0f)) {
            const float top = xor32_max(xor16_max(mx));
            const float mnew = top > m[mt] + 8.0f ? top : m[mt];
            const float alpha = __builtin_amdgcn_exp2f(m[mt] - mnew);
            m[mt] = mnew;
            l[mt] *= alpha;
#pragma unroll
            for (int n = 0; n < NN; n++) o[mt][n] *= alpha;
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
            p[j] = __builtin_amdgcn_exp2f(fmaf(p[j], fk, -m[mt]));
            l[mt] += p[j];
        }
        split_hi_lo8_mix(p, ph, pl);
    }

    // f * 2^(kref - 127), never 0 or infinite: a masked score times it stays -infinity
    RFP4_DEV float factor(int mt, int kref) const
    {
        return fminf(fmaxf(ldexpf(f[mt], kref - 127), 1.17549435e-38f), 3.402823466e38f);
    }
    RFP4_DEV void scale_o(float by)
    {
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int n = 0; n < NN; n++) o[mt][n] *= by;
    }
};

// Key groups whose K and V go to the registers.
template <int HD, bool F8, int MT, int WK>
struct AttnRows : AttnRowsState<HD, MT> {
    typedef AttnRowsState<HD, MT> State;
    using State::KS;
    using State::NN;
    using State::l16;
    using State::q4;
    using State::lane;
    using State::qa;
    using State::ql;
    using State::o;
    using State::f;
    static constexpr int EB = F8 ? 1 : 2;       // bytes of an element
    static constexpr int NKL = HD * EB / 64;    // 16-byte K loads of a lane per 16-key half
    static constexpr int VW = NN * EB / 4;      // dwords of a lane per V row
    static constexpr int ROWS = 16 * MT * (4 / WK); // query rows of a workgroup
    int wave, kgrp;

    uint4 kr[2][NKL];    // raw K rows l16 and 16 + l16 of a block
    uint32_t vr[8][VW];  // raw V of the lane's 8 keys
    uint32_t sb;         // scale byte of key lane % 32, K's in lanes 0..31, V's in the others

    RFP4_DEV void load_vrow(uint32_t (&r)[VW], const uint8_t *p)
    {
        if constexpr (VW == 1) {
            r[0] = *(const uint32_t *)p;
        } else if constexpr (VW == 2) {
            const uint2 x = *(const uint2 *)p;
            r[0] = x.x; r[1] = x.y;
        } else {
            const uint4 x = *(const uint4 *)p;
            r[0] = x.x; r[1] = x.y; r[2] = x.z; r[3] = x.w;
        }
    }
    // Blocks inside the cache take 32-bit lane offsets from uniform bases; the
    // last one, and strides past 4 GB, clamp each key to the last that exists
    // (finite or not, a key at or past `hi` is masked).
    RFP4_DEV bool whole(const AttnRowsKeys &s, uint32_t key0) const { return s.ts < (1ull << 24) && key0 + 32u <= s.end; }
    RFP4_DEV void load_k(const AttnRowsKeys &s, uint32_t key0)
    {
        if (whole(s, key0)) {
            const uint32_t off = (uint32_t)EB * l16 * (uint32_t)s.ts + 16u * q4;
            const uint8_t *b = s.k + (uint64_t)key0 * s.ts * EB;
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int i = 0; i < NKL; i++) kr[h][i] = *(const uint4 *)(b + (uint64_t)(16 * h) * s.ts * EB + off + 64 * i);
        } else {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint8_t *b = s.k + (uint64_t)min(key0 + 16u * (uint32_t)h + l16, s.end - 1u) * s.ts * EB + 16u * q4;
#pragma unroll
                for (int i = 0; i < NKL; i++) kr[h][i] = *(const uint4 *)(b + 64 * i);
            }
        }
        if constexpr (F8) {
            const uint32_t t = min(key0 + (lane & 31u), s.end - 1u);
            sb = (lane < 32u ? s.ks : s.vs)[(uint64_t)t * (s.ts / HD)];
        }
    }
    RFP4_DEV void load_v(const AttnRowsKeys &s, uint32_t key0)
    {
        if (whole(s, key0)) {
            const uint32_t off = (uint32_t)EB * (4u * q4 * (uint32_t)s.ts + (uint32_t)NN * l16);
            const uint8_t *b = s.v + (uint64_t)key0 * s.ts * EB;
#pragma unroll
            for (int j = 0; j < 8; j++) load_vrow(vr[j], b + (uint64_t)(j < 4 ? j : 12 + j) * s.ts * EB + off);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint32_t t = min(key0 + 4u * q4 + (uint32_t)(j < 4 ? j : 12 + j), s.end - 1u);
                load_vrow(vr[j], s.v + ((uint64_t)t * s.ts + (uint32_t)NN * l16) * EB);
            }
        }
    }

    // The wave's keys of s, blocks of 32 from lo + 32 kgrp on, every WK-th.
    // whi: keys that some row of the wave sees.  sc: 64 floats of LDS of the wave.
    RFP4_DEV void walk(const AttnRowsKeys &s, uint32_t whi, float *sc)
    {
        uint32_t key0 = s.lo + 32u * (uint32_t)kgrp;
        if (key0 >= whi) return;
        load_k(s, key0);
        load_v(s, key0);
        int kref = -1000, vref = -1000;
        float fk[MT];
#pragma unroll
        for (int mt = 0; mt < MT; mt++) fk[mt] = f[mt];
        for (;;) {
            const uint32_t next = key0 + 32u * WK;
            const bool more = next < whi && next > key0;
            uint32_t nan = 0;
            float ksc[2] = {1.0f, 1.0f}, vsc[8] = {1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f};
            if constexpr (F8) {
                const bool bad = sb == 255u;
                const uint64_t nans = __ballot(bad);
                const int ref = lane < 32u ? kref : vref;
                if (__any(!bad && (int)sb > ref + 7)) {
                    float top = bad ? -2000.0f : (float)sb; // bytes are exact in f32
                    top = xor16_max(row16_max(top));
                    const int kt = __builtin_amdgcn_readfirstlane((int)top), vt = __builtin_amdgcn_readlane((int)top, 32);
                    if (kt > kref + 7) {
                        kref = kt;
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) fk[mt] = this->factor(mt, kref);
                    }
                    if (vt > vref + 7) {
                        this->scale_o(pow2_int(vref - vt)); // 2^-126 for the first block, whose O is 0
                        vref = vt;
                    }
                }
                sc[lane] = bad ? 1.0f : pow2_int((int)sb - (lane < 32u ? kref : vref));
                nan = (uint32_t)nans | (uint32_t)(nans >> 32);
                __builtin_amdgcn_wave_barrier();
                ksc[0] = sc[l16];
                ksc[1] = sc[16u + l16];
                const float4 v0 = *(const float4 *)&sc[32u + 4u * q4], v1 = *(const float4 *)&sc[48u + 4u * q4];
                vsc[0] = v0.x; vsc[1] = v0.y; vsc[2] = v0.z; vsc[3] = v0.w;
                vsc[4] = v1.x; vsc[5] = v1.y; vsc[6] = v1.z; vsc[7] = v1.w;
                __builtin_amdgcn_wave_barrier();
            }
            // ---- S^T: accumulator r of half h is key 16 h + 4 q4 + r of row l16
            f32x4 st[MT][2];
#pragma unroll
            for (int mt = 0; mt < MT; mt++) st[mt][0] = st[mt][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < KS; k++) {
                f16x8 ka[2];
#pragma unroll
                for (int h = 0; h < 2; h++) ka[h] = k_operand(h, k, ksc[h]);
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
#pragma unroll
                    for (int h = 0; h < 2; h++) st[mt][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[h], qa[mt][k], st[mt][h], 0, 0, 0);
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
#pragma unroll
                    for (int h = 0; h < 2; h++) st[mt][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[h], ql[mt][k], st[mt][h], 0, 0, 0);
            }
            if (more) load_k(s, next);
            f16x8 ph[MT], pl[MT];
#pragma unroll
            for (int mt = 0; mt < MT; mt++) this->template probabilities<F8>(mt, st[mt], key0, s.hi, nan, fk[mt], ph[mt], pl[mt]);
            // ---- O^T += V^T P^T, dimension tiles NB at a time
            constexpr int NB = F8 ? 4 : 2; // tiles of a V dword
#pragma unroll
            for (int w = 0; w < VW; w++) {
                f16x8 va[NB];
                v_operands(w, vsc, va);
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
#pragma unroll
                    for (int n = 0; n < NB; n++)
                        o[mt][NB * w + n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va[n], ph[mt], o[mt][NB * w + n], 0, 0, 0);
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
#pragma unroll
                    for (int n = 0; n < NB; n++)
                        o[mt][NB * w + n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va[n], pl[mt], o[mt][NB * w + n], 0, 0, 0);
            }
            if (!more) break;
            load_v(s, next);
            key0 = next;
        }
        if constexpr (F8) {
            this->scale_o(ldexpf(1.0f, vref - 127));
        }
    }

    // K row l16 of half h at K step k as fp16
    RFP4_DEV f16x8 k_operand(int h, int k, float scale)
    {
        typedef uint32_t u32x4v __attribute__((ext_vector_type(4)));
        if constexpr (F8) {
            const uint4 r = kr[h][k / 2];
            const uint32_t w0 = k % 2 ? r.z : r.x, w1 = k % 2 ? r.w : r.y;
            const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, scale, true);
            const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, scale, true);
            return f16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
        } else {
            const uint4 r = kr[h][k];
            return __builtin_bit_cast(f16x8, u32x4v{r.x, r.y, r.z, r.w});
        }
    }

    // V^T operands of the tiles of V dword w: row l16 of each tile at the lane's 8 keys
    template <int NB>
    RFP4_DEV void v_operands(int w, const float (&vsc)[8], f16x8 (&va)[NB])
    {
        typedef uint32_t u32x4v __attribute__((ext_vector_type(4)));
        u32x4v t[NB];
#pragma unroll
        for (int jp = 0; jp < 4; jp++) {
            uint32_t a[NB / 2], b[NB / 2]; // pairs of dimensions of keys 2 jp and 2 jp + 1
#pragma unroll
            for (int i = 0; i < NB / 2; i++) {
                if constexpr (F8) {
                    if (i == 0) {
                        a[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(vr[2 * jp][w], vsc[2 * jp], false));
                        b[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(vr[2 * jp + 1][w], vsc[2 * jp + 1], false));
                    } else {
                        a[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(vr[2 * jp][w], vsc[2 * jp], true));
                        b[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(vr[2 * jp + 1][w], vsc[2 * jp + 1], true));
                    }
                } else {
                    a[i] = vr[2 * jp][w];
                    b[i] = vr[2 * jp + 1][w];
                }
                t[2 * i][jp] = __builtin_amdgcn_perm(b[i], a[i], 0x05040100u);
                t[2 * i + 1][jp] = __builtin_amdgcn_perm(b[i], a[i], 0x07060302u);
            }
        }
#pragma unroll
        for (int n = 0; n < NB; n++) va[n] = __builtin_bit_cast(f16x8, t[n]);
    }
};

// Query rows enough for 4 waves of MT tiles each: all of them take every key,
// which the workgroup stages in LDS as fp16 rows, block by block, two stages:
// while a block's scores and P V are computed from one, the next block goes
// from registers (loaded a block earlier) through the conversion into the
// other, so a key is converted once for 64 MT rows.  V^T operands come out of
// the rows through the transposing LDS read.  Rows are padded (K by 16 bytes:
// read 16 rows at a time, 16 bytes each; V by 32: 8 rows, 32 bytes), so reads
// cover the banks once and every address is one register and a constant.
// Dimension 16 n + 4 q4 + r is accumulator r of tile n.
template <int HD, bool F8, int MT>
struct AttnRowsTile : AttnRowsState<HD, MT> {
    typedef AttnRowsState<HD, MT> State;
    using State::KS;
    using State::NN;
    using State::l16;
    using State::q4;
    using State::lane;
    using State::qa;
    using State::ql;
    using State::o;
    static constexpr uint32_t EB = F8 ? 1 : 2;
    static constexpr uint32_t BK = 4096 / HD;   // keys of a block: 32 of 128 dimensions, 64 of 64
    static constexpr uint32_t KRB = 2 * HD + 16, VRB = 2 * HD + 32; // bytes of a staged K and V row
    static constexpr uint32_t NL = EB;          // 16-byte loads of a thread for a block's K (and V)
    static constexpr uint32_t CPR = HD * EB / 16; // 16-byte pieces of a cache row
    static constexpr uint32_t VOFF = BK * KRB, STAGE = VOFF + BK * VRB; // a block's K rows, then its V rows
    typedef short i16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
    typedef __attribute__((address_space(3))) uint8_t lds_u8;

    uint4 kraw[NL], vraw[NL];
    uint32_t kb, vb;        // scale bytes of key lane % BK of the block in the registers
    int kref = -1000, vref = -1000;
    uint64_t nan = 0;       // its keys of byte 255

    // Piece i of thread t: row and 16-byte piece of a block's K or V
    RFP4_DEV static uint32_t piece_row(uint32_t t, uint32_t i) { return (t + 256u * i) / CPR; }
    RFP4_DEV static uint32_t piece_col(uint32_t t, uint32_t i) { return (t + 256u * i) % CPR; }

    RFP4_DEV void load(const AttnRowsKeys &s, uint32_t key0)
    {
        if (s.ts < (1ull << 24) && key0 + BK <= s.end) { // 32-bit lane offsets from uniform bases
            const uint8_t *k = s.k + (uint64_t)key0 * s.ts * EB, *v = s.v + (uint64_t)key0 * s.ts * EB;
#pragma unroll
            for (uint32_t i = 0; i < NL; i++) {
                const uint32_t off = piece_row(threadIdx.x, i) * (uint32_t)s.ts * EB + 16u * piece_col(threadIdx.x, i);
                kraw[i] = *(const uint4 *)(k + off);
                vraw[i] = *(const uint4 *)(v + off);
            }
            if constexpr (F8) {
                const uint64_t t = (uint64_t)key0 * (s.ts / HD);
                const uint32_t off = lane % BK * (uint32_t)(s.ts / HD);
                kb = (s.ks + t)[off];
                vb = (s.vs + t)[off];
            }
        } else { // keys past the last that exists re-read it; they are masked
            uint32_t tid = threadIdx.x;
            asm volatile("" : "+v"(tid)); // nothing of this path is held over the loop
#pragma unroll
            for (uint32_t i = 0; i < NL; i++) {
                const uint64_t off = (uint64_t)min(key0 + piece_row(tid, i), s.end - 1u) * s.ts * EB + 16u * piece_col(tid, i);
                kraw[i] = *(const uint4 *)(s.k + off);
                vraw[i] = *(const uint4 *)(s.v + off);
            }
            if constexpr (F8) {
                const uint64_t t = (uint64_t)min(key0 + tid % BK, s.end - 1u) * (s.ts / HD);
                kb = s.ks[t];
                vb = s.vs[t];
            }
        }
    }

    // The block in the registers as fp16 rows of the stage at st; moves the
    // references (the same in every wave: all hold the same bytes)
    RFP4_DEV void stage(lds_u8 *st)
    {
        if constexpr (F8) {
            const bool bad = kb == 255u || vb == 255u;
            nan = __ballot(bad);
            if (__any(!bad && ((int)kb > kref + 7 || (int)vb > vref + 7))) {
                const int kt = __builtin_amdgcn_readfirstlane((int)wave_max(bad ? -2000.0f : (float)kb)); // exact in f32
                const int vt = __builtin_amdgcn_readfirstlane((int)wave_max(bad ? -2000.0f : (float)vb));
                kref = kt > kref + 7 ? kt : kref;
                vref = vt > vref + 7 ? vt : vref;
            }
            const uint32_t r = piece_row(threadIdx.x, 0), c = piece_col(threadIdx.x, 0);
            const float ks = __shfl(bad ? 1.0f : pow2_int((int)kb - kref), (int)r, 64), vs = __shfl(bad ? 1.0f : pow2_int((int)vb - vref), (int)r, 64);
            uint4 w[2];
            widen(kraw[0], ks, w);
            put(st + r * KRB + 32u * c, w[0]);
            put(st + r * KRB + 32u * c + 16u, w[1]);
            widen(vraw[0], vs, w);
            put(st + VOFF + r * VRB + 32u * c, w[0]);
            put(st + VOFF + r * VRB + 32u * c + 16u, w[1]);
        } else {
#pragma unroll
            for (uint32_t i = 0; i < NL; i++) {
                const uint32_t r = piece_row(threadIdx.x, i), c = piece_col(threadIdx.x, i);
                put(st + r * KRB + 16u * c, kraw[i]);
                put(st + VOFF + r * VRB + 16u * c, vraw[i]);
            }
        }
    }
    RFP4_DEV static void put(lds_u8 *p, uint4 v) { *(__attribute__((address_space(3))) uint4 *)p = v; }
    RFP4_DEV static void widen(uint4 r, float scale, uint4 (&w)[2])
    {
        const uint32_t x[4] = {r.x, r.y, r.z, r.w};
        uint32_t y[8];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            y[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[i], scale, false));
            y[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[i], scale, true));
        }
        w[0] = make_uint4(y[0], y[1], y[2], y[3]);
        w[1] = make_uint4(y[4], y[5], y[6], y[7]);
    }

    // Keys s.lo .. s.hi of the workgroup, of which this wave's rows see those below whi
    RFP4_DEV void walk(const AttnRowsKeys &s, uint32_t whi, lds_u8 *lds)
    {
        // the transposing read: lane j of 16 gives the address of 4 halves, row
        // j / 4 of 4, columns 4 (j % 4) .. +3 of 16, and gets column j of the 4 rows
        const uint32_t kaddr = l16 * KRB + 16u * q4, vaddr = VOFF + (4u * q4 + (l16 >> 2)) * VRB + 8u * (l16 & 3u);
        load(s, s.lo);
        stage(lds);
        float fk[MT];
#pragma unroll
        for (int mt = 0; mt < MT; mt++) fk[mt] = F8 ? this->factor(mt, kref) : this->f[mt];
        int kcur = kref, vcur = vref; // the references of the block that is computed
        uint64_t nan_now = nan;
        uint32_t buf = 0;
        if (s.lo + BK < s.hi) load(s, s.lo + BK);
        __syncthreads();
        for (uint32_t key0 = s.lo;; key0 += BK) {
            if constexpr (F8) {
                if (kref != kcur || vref != vcur) {
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) fk[mt] = this->factor(mt, kref);
                    this->scale_o(pow2_int(vcur - vref));
                    kcur = kref;
                    vcur = vref;
                }
                nan_now = nan;
            }
            const bool more = s.hi - key0 > BK;
            if (more) {
                stage(lds + (buf ^ 1u) * STAGE);
                if (s.hi - key0 > 2u * BK) load(s, key0 + 2u * BK);
            }
            lds_u8 *st = lds + buf * STAGE;
#pragma unroll
            for (uint32_t c = 0; c < BK / 32u; c++) {
                if (key0 + 32u * c >= whi) break; // the same for the whole wave
                f32x4 sc[MT][2];
#pragma unroll
                for (int mt = 0; mt < MT; mt++) sc[mt][0] = sc[mt][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int k = 0; k < KS; k++) {
                    f16x8 ka[2];
#pragma unroll
                    for (uint32_t h = 0; h < 2; h++)
                        ka[h] = *(const __attribute__((address_space(3))) f16x8 *)(st + kaddr + 64u * (uint32_t)k + (32u * c + 16u * h) * KRB);
#pragma unroll
                    for (int mt = 0; mt < MT; mt++)
#pragma unroll
                        for (int h = 0; h < 2; h++) sc[mt][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[h], qa[mt][k], sc[mt][h], 0, 0, 0);
#pragma unroll
                    for (int mt = 0; mt < MT; mt++)
#pragma unroll
                        for (int h = 0; h < 2; h++) sc[mt][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[h], ql[mt][k], sc[mt][h], 0, 0, 0);
                }
                f16x8 ph[MT], pl[MT];
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
                    this->template probabilities<F8>(mt, sc[mt], key0 + 32u * c, s.hi, (uint32_t)(nan_now >> (32u * c)), fk[mt], ph[mt], pl[mt]);
#pragma unroll
                for (int n = 0; n < NN; n++) {
                    const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(st + vaddr + 32u * (uint32_t)n + 32u * c * VRB));
                    const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(st + vaddr + 32u * (uint32_t)n + (32u * c + 16u) * VRB));
                    typedef short i16x8 __attribute__((ext_vector_type(8)));
                    const f16x8 va = __builtin_bit_cast(f16x8, i16x8{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w});
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) o[mt][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, ph[mt], o[mt][n], 0, 0, 0);
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) o[mt][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl[mt], o[mt][n], 0, 0, 0);
                }
            }
            if (!more) break;
            __syncthreads();
            buf ^= 1u;
        }
        if constexpr (F8) this->scale_o(ldexpf(1.0f, vcur - 127));
    }
};

// Dimensions d .. d + 3 of (row i, head): the output, or of a split's state
// (first: with the row's maximum and sum)
template <int HD>
RFP4_DEV void attn_rows_put(const AttnRowsArgs &a, uint32_t i, uint32_t head, uint32_t S, uint32_t split, uint32_t d, bool first, float M, float L,
                            f32x4 acc)
{
    if (S > 1u) {
        float *dst = a.part + ((size_t)((size_t)i * a.n_heads + head) * S + split) * (HD + 4);
        if (first) {
            dst[0] = M;
            dst[1] = L;
        }
        *(f32x4 *)(dst + 4 + d) = acc;
    } else { // no key: 0, not 0 / 0; a NaN sum stays NaN
        const bool none = L == 0.0f;
        f32x4 y;
#pragma unroll
        for (int j = 0; j < 4; j++) y[j] = none ? 0.0f : __fdiv_rn(acc[j], L);
        *(f32x4 *)(a.out + (size_t)i * a.out_rs + (size_t)head * HD + d) = y;
    }
}

// One item of a workgroup with few rows: the query rows row0 .. row_end (at
// most 16 MT) of KV head kvh over s by 4 key groups, written as outputs, or as
// split `split`'s states.
template <int HD, bool F8, int MT>
RFP4_DEV void attn_rows_few(const AttnRowsArgs &a, uint32_t kvh, uint32_t row0, uint32_t row_end, const AttnRowsKeys &s, uint32_t split)
{
    constexpr int WK = 4;
    typedef AttnRows<HD, F8, MT, WK> R;
    __shared__ __align__(16) float sc[WK][64];
    R r;
    r.lane = threadIdx.x & 63u;
    r.l16 = r.lane & 15u;
    r.q4 = r.lane >> 4;
    r.kgrp = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    r.template load_q<F8>(a, kvh, row0, row_end, s.hi);
    r.walk(s, s.hi, sc[r.kgrp]);
#pragma unroll
    for (int mt = 0; mt < MT; mt++) r.l[mt] = xor32_sum(xor16_sum(r.l[mt]));
    const uint32_t S = a.splits0 + a.splits1;

    // the key groups' states through LDS
    constexpr int RW = 16 * MT, LD = HD + 4;
    __shared__ __align__(16) float ro[WK][RW][LD];
    __shared__ float rm[WK][RW], rl[WK][RW];
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        const uint32_t row = 16u * (uint32_t)mt + r.l16;
        if (r.q4 == 0u) {
            rm[r.kgrp][row] = r.m[mt];
            rl[r.kgrp][row] = r.l[mt];
        }
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int n = 0; n < R::NN; n += 4)
                *(float4 *)&ro[r.kgrp][row][(4u * r.q4 + (uint32_t)t) * R::NN + n] =
                    make_float4(r.o[mt][n][t], r.o[mt][n + 1][t], r.o[mt][n + 2][t], r.o[mt][n + 3][t]);
    }
    __syncthreads();
    constexpr uint32_t LPR = HD / 4; // lanes of a row, 4 dimensions each
    for (uint32_t u = threadIdx.x; u < (uint32_t)RW * LPR; u += 256u) {
        const uint32_t row = u / LPR, d = 4u * (u % LPR), rho = row0 + row;
        if (rho >= row_end) break;
        float M = rm[0][row];
#pragma unroll
        for (int g = 1; g < WK; g++) M = fmaxf(M, rm[g][row]);
        float L = 0.0f;
        f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int g = 0; g < WK; g++) {
            const float w = __builtin_amdgcn_exp2f(rm[g][row] - M);
            L = fmaf(rl[g][row], w, L);
            const f32x4 x = *(const f32x4 *)&ro[g][row][d];
#pragma unroll
            for (int j = 0; j < 4; j++) acc[j] = fmaf(x[j], w, acc[j]);
        }
        attn_rows_put<HD>(a, rho / a.group, kvh * a.group + rho % a.group, S, split, d, d == 0u, M, L, acc);
    }
}

// The same for up to 64 MT rows, whose waves take all keys each.
template <int HD, bool F8, int MT>
RFP4_DEV void attn_rows_many(const AttnRowsArgs &a, uint32_t kvh, uint32_t row0, uint32_t row_end, const AttnRowsKeys &s, uint32_t split)
{
    typedef AttnRowsTile<HD, F8, MT> R;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * R::STAGE];
    R r;
    r.lane = threadIdx.x & 63u;
    r.l16 = r.lane & 15u;
    r.q4 = r.lane >> 4;
    const uint32_t wrow = row0 + 16u * MT * (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    r.template load_q<false>(a, kvh, wrow, row_end, s.hi);
    uint32_t whi = wrow < row_end ? s.hi : 0u; // waves without rows stage and wait only
    if (a.causal) whi = min(whi, a.pos0 + min(wrow + 16u * MT - 1u, row_end - 1u) / a.group + 1u);
    r.walk(s, whi, (typename R::lds_u8 *)lds);
    const uint32_t S = a.splits0 + a.splits1;
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        const float L = xor32_sum(xor16_sum(r.l[mt]));
        const uint32_t rho = wrow + 16u * (uint32_t)mt + r.l16;
        if (rho >= row_end) continue;
#pragma unroll
        for (int n = 0; n < R::NN; n++)
            attn_rows_put<HD>(a, rho / a.group, kvh * a.group + rho % a.group, S, split, 16u * (uint32_t)n + 4u * r.q4, n == 0 && r.q4 == 0u, r.m[mt], L,
                              r.o[mt][n]);
    }
}

// Workgroup (kvh, item), kvh = blockIdx.x % n_kv_heads (with 8 KV heads each
// XCD, workgroup id % 8, keeps one head's K and V in its L2): the shared keys'
// items (row tile, split) first, the longest causal ranges leading, then the
// own keys' (row, split).
template <int HD, bool F8, int MT, bool MANY, bool OWN>
RFP4_DEV void attn_rows_body(const AttnRowsArgs &a)
{
    constexpr uint32_t EB = F8 ? 1u : 2u;
    constexpr uint32_t RW = MANY ? 64u * MT : 16u * MT;
    const uint32_t kvh = blockIdx.x % a.n_kv_heads, item = blockIdx.x / a.n_kv_heads;
    uint32_t row0, row_end, split;
    const void *k, *v;
    const uint8_t *ks, *vs;
    uint64_t base;
    AttnRowsKeys s;
    const bool own = OWN && item >= a.tiles0 * a.splits0;
    if (!own) {
        const uint32_t tile = a.tiles0 - 1u - item / a.splits0;
        split = item % a.splits0;
        row0 = tile * RW;
        row_end = min(row0 + RW, a.rows * a.group);
        s.lo = split * a.chunk0;
        s.end = a.len0;
        s.hi = min(s.lo + a.chunk0, a.len0);
        if (a.causal) s.hi = min(s.hi, a.pos0 + (row_end - 1u) / a.group + 1u);
        if (s.lo >= s.hi) return;
        s.ts = a.ts0;
        base = (uint64_t)kvh * a.hs0;
        k = a.k0; v = a.v0; ks = a.ks0; vs = a.vs0;
    } else {
        const uint32_t x = item - a.tiles0 * a.splits0, row = x / a.splits1, part = x % a.splits1;
        s.end = (uint32_t)__builtin_amdgcn_readfirstlane((int)min(a.lens[row], a.cap1));
        split = a.splits0 + part;
        row0 = row * a.group;
        row_end = row0 + a.group;
        s.lo = part * a.chunk1;
        s.hi = min(s.lo + a.chunk1, s.end);
        // a split past the row's last key is not merged; with one split in all, the row is 0
        if (s.lo >= s.end && a.splits0 + a.splits1 > 1u) return;
        s.ts = a.ts1;
        base = (uint64_t)row * a.ss1 + (uint64_t)kvh * a.hs1;
        k = a.k1; v = a.v1; ks = a.ks1; vs = a.vs1;
    }
    s.k = (const uint8_t *)k + base * EB;
    s.v = (const uint8_t *)v + base * EB;
    s.ks = F8 ? ks + base / HD : nullptr;
    s.vs = F8 ? vs + base / HD : nullptr;
    if constexpr (MANY) {
        if (!own) attn_rows_many<HD, F8, MT>(a, kvh, row0, row_end, s, split);
        else attn_rows_few<HD, F8, 1>(a, kvh, row0, row_end, s, split);
    } else {
        attn_rows_few<HD, F8, MT>(a, kvh, row0, row_end, s, split);
    }
}

// The states of query row i, head h, merged: M = max m, out = sum acc 2^(m - M)
// / sum l 2^(m - M); 0 for a row without keys.  256 / HD parts of the splits,
// a dimension per lane.
template <int HD>
RFP4_DEV void attn_rows_merge_body(const AttnRowsArgs &a)
{
    constexpr uint32_t P = 256u / HD;
    __shared__ float pm[P], pl[P], pacc[P][HD];
    const uint32_t h = blockIdx.x % a.n_heads, i = blockIdx.x / a.n_heads;
    const uint32_t d = threadIdx.x % HD, p = threadIdx.x / HD, S = a.splits0 + a.splits1;
    const uint32_t keys0 = a.causal ? a.pos0 + i + 1u : a.len0, keys1 = a.splits1 ? min(a.lens[i], a.cap1) : 0u;
    const uint32_t n0 = a.splits0 ? (keys0 + a.chunk0 - 1u) / a.chunk0 : 0u;
    const uint32_t n = n0 + (a.splits1 ? (keys1 + a.chunk1 - 1u) / a.chunk1 : 0u);
    const float *st = a.part + (size_t)((size_t)i * a.n_heads + h) * S * (HD + 4);
    float M = -3.402823466e38f, L = 0.0f, acc = 0.0f;
    for (uint32_t x = p; x < n; x += P) {
        const float *w = st + (size_t)(x < n0 ? x : a.splits0 + (x - n0)) * (HD + 4);
        const float m = w[0], l = w[1], v = w[4 + d];
        const float top = fmaxf(M, m);
        const float c0 = __builtin_amdgcn_exp2f(M - top), c1 = __builtin_amdgcn_exp2f(m - top);
        L = fmaf(L, c0, l * c1);
        acc = fmaf(acc, c0, v * c1);
        M = top;
    }
    pacc[p][d] = acc;
    if (d == 0u) {
        pm[p] = M;
        pl[p] = L;
    }
    __syncthreads();
    if (p) return;
    for (uint32_t x = 1; x < P; x++) {
        const float top = fmaxf(M, pm[x]);
        const float c0 = __builtin_amdgcn_exp2f(M - top), c1 = __builtin_amdgcn_exp2f(pm[x] - top);
        L = fmaf(L, c0, pl[x] * c1);
        acc = fmaf(acc, c0, pacc[x][d] * c1);
        M = top;
    }
    a.out[(size_t)i * a.out_rs + (size_t)h * HD + d] = L == 0.0f ? 0.0f : __fdiv_rn(acc, L);
}
