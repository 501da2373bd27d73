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

template <int HD, bool F8, int MT, int WK>
struct AttnRows {
    static constexpr int KS = HD / 32;          // K steps of S
    static constexpr int NN = HD / 16;          // dimension tiles of O
    static constexpr int EB = F8 ? 1 : 2;       // bytes of an element
    static constexpr int NKL = HD * EB / 64;    // 16-byte K loads of a lane per 16-key half
    static constexpr int VW = NN * EB / 4;      // dwords of a lane per V row
    static constexpr int ROWS = 16 * MT * (4 / WK); // query rows of a workgroup

    uint32_t l16, q4, lane;
    int wave, kgrp;
    f16x8 qa[MT][KS], ql[MT][KS];
    f32x4 o[MT][NN];
    float m[MT], l[MT], f[MT]; // running maximum and sum, the scores' factor less 2^kref
    uint32_t lim[MT];          // keys that the lane's row sees

    // q of the lane's row of each tile, scaled by a power of two of its own to
    // at most 256, and that scale's inverse into the scores' factor
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
                // the dimensions of K step k in this lane: an 8-bit load of 16 covers two steps
                const uint32_t d = F8 ? 64u * (uint32_t)(k / 2) + 16u * q4 + 8u * (uint32_t)(k % 2) : 32u * (uint32_t)k + 8u * q4;
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
                        for (int mt = 0; mt < MT; mt++) // never 0 or infinite: a masked score times it stays -infinity
                            fk[mt] = fminf(fmaxf(ldexpf(f[mt], kref - 127), 1.17549435e-38f), 3.402823466e38f);
                    }
                    if (vt > vref + 7) {
                        const float down = pow2_int(vref - vt); // 2^-126 for the first block, whose O is 0
                        vref = vt;
#pragma unroll
                        for (int mt = 0; mt < MT; mt++)
#pragma unroll
                            for (int n = 0; n < NN; n++) o[mt][n] *= down;
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
            for (int mt = 0; mt < MT; mt++) {
                float p[8];
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int r = 0; r < 4; r++) p[4 * h + r] = st[mt][h][r];
                if (F8 && nan) {
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        if ((nan >> (4u * q4 + (uint32_t)(j < 4 ? j : 12 + j))) & 1u) p[j] = __uint_as_float(0x7FC00000u);
                }
                // masked scores at -infinity (p = 0 whatever maximum is subtracted)
                if (__any(key0 + 32u > min(lim[mt], s.hi))) {
                    const uint32_t last = min(lim[mt], s.hi);
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        if (key0 + 4u * q4 + (uint32_t)(j < 4 ? j : 12 + j) >= last) p[j] = -INFINITY;
                }
                // online softmax in base 2; the subtracted maximum is raised
                // only when a score of the row exceeds it by more than 8 (p at
                // most 2^8), so the common block has no cross-lane step
                float mx = p[0];
#pragma unroll
                for (int j = 1; j < 8; j++) mx = fmaxf(mx, p[j]);
                mx *= fk[mt];
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
                    p[j] = __builtin_amdgcn_exp2f(fmaf(p[j], fk[mt], -m[mt]));
                    l[mt] += p[j];
                }
                split_hi_lo8_mix(p, ph[mt], pl[mt]);
            }
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
            const float up = ldexpf(1.0f, vref - 127);
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int n = 0; n < NN; n++) o[mt][n] *= up;
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

// One (rows, keys) item of a workgroup: the query rows row0 .. row_end of KV
// head kvh over s, written as outputs, or as split `split`'s states.
template <int HD, bool F8, int MT, int WK>
RFP4_DEV void attn_rows_item(const AttnRowsArgs &a, uint32_t kvh, uint32_t row0, uint32_t row_end, const AttnRowsKeys &s,
                             uint32_t limit0, uint32_t split)
{
    typedef AttnRows<HD, F8, MT, WK> R;
    __shared__ __align__(16) float sc[4][64];
    R r;
    r.lane = threadIdx.x & 63u;
    r.l16 = r.lane & 15u;
    r.q4 = r.lane >> 4;
    r.wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    r.kgrp = r.wave % WK;
    const uint32_t wrow = row0 + 16u * MT * (uint32_t)(r.wave / WK);
    if (WK == 1 && wrow >= row_end) return; // no barrier with one key group
    r.load_q(a, kvh, wrow, row_end, limit0);
    uint32_t whi = s.hi;
    if (a.causal) whi = min(whi, a.pos0 + min(wrow + 16u * MT - 1u, row_end - 1u) / a.group + 1u);
    if (wrow < row_end) r.walk(s, whi, sc[r.wave]);
#pragma unroll
    for (int mt = 0; mt < MT; mt++) r.l[mt] = xor32_sum(xor16_sum(r.l[mt]));
    const uint32_t S = a.splits0 + a.splits1;

    if constexpr (WK == 1) {
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            const uint32_t rho = wrow + 16u * (uint32_t)mt + r.l16;
            if (rho >= row_end) continue;
            const uint32_t i = rho / a.group, head = kvh * a.group + rho % a.group;
            float *dst;
            float inv = 1.0f;
            if (S > 1u) {
                dst = a.part + ((size_t)((size_t)i * a.n_heads + head) * S + split) * (HD + 4) + 4;
                if (r.q4 == 0u) {
                    dst[-4] = r.m[mt];
                    dst[-3] = r.l[mt];
                }
            } else {
                dst = a.out + (size_t)i * a.out_rs + (size_t)head * HD;
                inv = r.l[mt];
            }
            // (no key: 0, not 0 / 0; a NaN sum stays NaN)
            const bool none = inv == 0.0f;
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int n = 0; n < R::NN; n += 4) {
                    float y[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) y[j] = none ? 0.0f : __fdiv_rn(r.o[mt][n + j][t], inv);
                    *(float4 *)(dst + (4u * r.q4 + (uint32_t)t) * R::NN + n) = make_float4(y[0], y[1], y[2], y[3]);
                }
        }
    } else {
        // the key groups' states through LDS
        constexpr int RW = R::ROWS, LD = HD + 4;
        __shared__ __align__(16) float ro[WK][RW][LD];
        __shared__ float rm[WK][RW], rl[WK][RW];
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            const uint32_t row = 16u * (uint32_t)(MT * (r.wave / WK) + mt) + r.l16;
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
            const uint32_t i = rho / a.group, head = kvh * a.group + rho % a.group;
            if (S > 1u) {
                float *dst = a.part + ((size_t)((size_t)i * a.n_heads + head) * S + split) * (HD + 4);
                if (d == 0u) {
                    dst[0] = M;
                    dst[1] = L;
                }
                *(f32x4 *)(dst + 4 + d) = acc;
            } else {
                const bool none = L == 0.0f;
                f32x4 y;
#pragma unroll
                for (int j = 0; j < 4; j++) y[j] = none ? 0.0f : __fdiv_rn(acc[j], L);
                *(f32x4 *)(a.out + (size_t)i * a.out_rs + (size_t)head * HD + d) = y;
            }
        }
    }
}

// Workgroup (kvh, item), kvh = blockIdx.x % n_kv_heads (with 8 KV heads each
// XCD, workgroup id % 8, keeps one head's K and V in its L2): the shared keys'
// items (row tile, split) first, the longest causal ranges leading, then the
// own keys' (row, split).
template <int HD, bool F8, int MT, int WK>
RFP4_DEV void attn_rows_body(const AttnRowsArgs &a)
{
    constexpr uint32_t EB = F8 ? 1u : 2u;
    constexpr uint32_t RW = 16u * MT * (4 / WK);
    const uint32_t kvh = blockIdx.x % a.n_kv_heads, item = blockIdx.x / a.n_kv_heads;
    const uint32_t flat = a.rows * a.group;
    AttnRowsKeys s;
    if (item < a.tiles0 * a.splits0) {
        const uint32_t tile = a.tiles0 - 1u - item / a.splits0, split = item % a.splits0;
        const uint32_t row0 = tile * RW, row_end = flat;
        s.lo = split * a.chunk0;
        s.end = a.len0;
        s.hi = min(s.lo + a.chunk0, a.len0);
        if (a.causal) s.hi = min(s.hi, a.pos0 + (min(row0 + RW, flat) - 1u) / a.group + 1u);
        if (s.lo >= s.hi) return;
        s.ts = a.ts0;
        s.k = (const uint8_t *)a.k0 + (uint64_t)kvh * a.hs0 * EB;
        s.v = (const uint8_t *)a.v0 + (uint64_t)kvh * a.hs0 * EB;
        s.ks = F8 ? a.ks0 + (uint64_t)kvh * (a.hs0 / HD) : nullptr;
        s.vs = F8 ? a.vs0 + (uint64_t)kvh * (a.hs0 / HD) : nullptr;
        attn_rows_item<HD, F8, MT, WK>(a, kvh, row0, row_end, s, s.hi, split);
    } else {
        const uint32_t own = item - a.tiles0 * a.splits0, row = own / a.splits1, split = own % a.splits1;
        const uint32_t len = (uint32_t)__builtin_amdgcn_readfirstlane((int)min(a.lens[row], a.cap1));
        s.lo = split * a.chunk1;
        s.end = len;
        s.hi = min(s.lo + a.chunk1, len);
        // a split past the row's last key is not merged; with one split in all, the row is 0
        if (s.lo >= len && a.splits0 + a.splits1 > 1u) return;
        const uint64_t base = (uint64_t)row * a.ss1 + (uint64_t)kvh * a.hs1;
        s.ts = a.ts1;
        s.k = (const uint8_t *)a.k1 + base * EB;
        s.v = (const uint8_t *)a.v1 + base * EB;
        s.ks = F8 ? a.ks1 + base / HD : nullptr;
        s.vs = F8 ? a.vs1 + base / HD : nullptr;
        attn_rows_item<HD, F8, 1, 4>(a, kvh, row * a.group, (row + 1u) * a.group, s, s.hi, a.splits0 + split);
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
