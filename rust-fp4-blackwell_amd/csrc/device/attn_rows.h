// Attention of query rows over an 8-bit or fp16 KV cache on the matrix cores
// (gfx950): one query row, causal prompt rows, or one row for each sequence of
// a batch over keys that all of them share and keys of their own.
//
//   out[i][h] = sum_t softmax_t(q[i][h] . k_t / sqrt(HD)) v_t
//
// over the shared keys t < len0 (causal: t <= pos0 + i) and the row's own keys
// t < lens[i].  A KV head's query rows (i, g), g < group, are packed i * group
// + g into tiles of 16, so a wave's matrix instructions serve 16 of them,
// whatever the group.  Two kernels: for few rows a tile for a workgroup, whose
// 4 waves take alternate key blocks straight into registers (AttnRowsFew); for
// more, 4 tiles for a workgroup, which stages the keys in LDS (AttnRowsMany).
// Where the keys are split over several workgroups each writes its state (m, l,
// acc) to the caller's workspace and a second kernel merges them (stream order,
// nothing that must start at zero).
//
// The products are transposed, so that a score stays in the lane that needs its
// probability (lane l: q4 = l / 16, l16 = l % 16):
//   S^T (32 x 16) = K . Q^T      accumulator r of 16-key half h is key 16 h +
//                                4 q4 + r of row l16: 8 keys of the lane
//   O^T (HD x 16) += V^T . P^T   whose operands take those 8 keys
// q and p enter as hi + lo fp16 terms (about 2^-22 relative: outputs within
// 1e-6 of exact ones; one term would leave 1e-4), e4m3 values are exact in
// fp16, products are exact and sums f32.
//
// Scales of the 8-bit cache, 2^(byte - 127) for each key: they go into the
// conversion to fp16, less a reference exponent (kref, vref), which keeps every
// value in fp16's range: the reference is raised when a byte exceeds it by more
// than 7 (codes to 448 * 2^7 = 57344), so values are exact down to scales 2^15
// below it, and off by at most 2^-41 of the largest value below that.  2^kref is
// part of the scores' factor, 2^vref of O's.  A byte of 255 makes its key NaN
// for every row that sees it, and for no other.
#pragma once
#include "common.h"

RFP4_DEV float pow2_int(int e) // 2^e, e of -126 .. 127; smaller e count as -126
{
    return __uint_as_float((uint32_t)(max(e, -126) + 127) << 23);
}

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4v __attribute__((ext_vector_type(4)));

// Two e4m3 codes (the low or high half of w) times 2^exponent(scale) as fp16
template <bool HIGH>
RFP4_DEV uint32_t fp8x2_to_f16(uint32_t w, float scale)
{
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, HIGH));
}

// split_hi_lo8_mix for values that a matrix instruction takes next: what reads a
// register that a vector instruction wrote waits two states, which the compiler
// does not count from inside an asm
RFP4_DEV void attn_split8(const float *v, f16x8 &hi, f16x8 &lo)
{
    split_hi_lo8_mix(v, hi, lo);
    asm("s_nop 2" : "+v"(lo));
}

RFP4_DEV f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// One cache for one KV head, and a workgroup's keys of it.
struct AttnRowsKeys {
    const uint8_t *k, *v;   // the head's token 0
    const uint8_t *ks, *vs; // its scale byte (8-bit caches)
    uint64_t ts;            // token stride (elements)
    uint32_t lo, hi;        // the keys, lo a multiple of 128
    uint32_t end;           // keys that exist, at least hi
};

// A wave's tile of 16 query rows; the lane works for row l16.
template <int HD>
struct AttnRowsState {
    static constexpr int KS = HD / 32; // K steps of S
    static constexpr int NN = HD / 16; // dimension tiles of O

    uint32_t l16, q4, lane;
    f16x8 qa[KS], ql[KS];
    f32x4 o[NN];
    float m, l;   // running maximum (in base-2 units, as split states hold it) and sum
    float f, fk;  // the scores' factor less 2^kref, and with the current one
    float thr;    // the score above which the maximum is raised, (m + 8) / fk
    uint32_t lim; // keys that the row sees

    RFP4_DEV AttnRowsState()
    {
        lane = threadIdx.x & 63u;
        l16 = lane & 15u;
        q4 = lane >> 4;
    }

    // q of the row (row0 + l16 of row_end), scaled by a power of two of its own
    // to at most 256, and that scale's inverse into the scores' factor.  PAIRED:
    // the dimensions of K step k in this lane as 16-byte loads of 8-bit K rows
    // hold them, two steps a load.
    template <bool PAIRED>
    RFP4_DEV void load_q(const AttnRowsArgs &a, uint32_t kvh, uint32_t row0, uint32_t row_end, uint32_t limit0)
    {
        // log2(e) / sqrt(HD) in two factors: the score's factor a power of two,
        // so that a scaled score less the maximum is exact to one rounding and 0
        // for the maximum itself; the rest into q
        const float c = __fmul_rn(1.4426950408889634f, __fdiv_rn(1.0f, __fsqrt_rn((float)HD)));
        const uint32_t rho = row0 + l16;
        const bool in = rho < row_end;
        const uint32_t i = min(rho, row_end - 1u) / a.group, g = min(rho, row_end - 1u) % a.group;
        lim = a.causal ? min(a.pos0 + i + 1u, limit0) : limit0;
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
            attn_split8(x[k], qa[k], ql[k]);
        }
        f = __fmul_rn(pow2_int(e), 0.25f / 128.0f);
        m = -3.402823466e38f;
        l = 0.0f;
        set_factor(127);
#pragma unroll
        for (int n = 0; n < NN; n++) o[n] = {0.0f, 0.0f, 0.0f, 0.0f};
    }

    RFP4_DEV void threshold() { thr = __fdiv_rn(m + 8.0f, fk); }
    // The scores' factor with K of reference kref: f * 2^(kref - 127), never 0
    // or infinite, so that a masked score times it stays -infinity
    RFP4_DEV void set_factor(int kref)
    {
        fk = fminf(fmaxf(ldexpf(f, kref - 127), 1.17549435e-38f), 3.402823466e38f);
        threshold();
    }
    RFP4_DEV void scale_o(float by)
    {
#pragma unroll
        for (int n = 0; n < NN; n++) o[n] *= by;
    }

    // Scores st of 32 keys.  The common block takes a maximum of eight and one
    // comparison: the subtracted maximum is raised only when a score of the row
    // exceeds it by more than 8 (p at most 2^8).
    RFP4_DEV static float largest(const f32x4 (&st)[2])
    {
        // v_maximum3: fmaxf would first quiet each matrix result; a NaN makes
        // the maximum NaN, which exceeds nothing (its row is NaN by l and O)
        auto max3 = [](float a, float b, float c) { return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c); };
        const float x = max3(st[0][0], st[0][1], st[0][2]), y = max3(st[0][3], st[1][0], st[1][1]);
        return __builtin_elementwise_maximum(max3(x, st[1][2], st[1][3]), y);
    }
    RFP4_DEV bool exceeds(const f32x4 (&st)[2]) const { return largest(st) > thr; }
    // For blocks with NaN or masked keys or such a score: NaN for the keys of
    // scale byte 255 (nan), -infinity for those at and past `hi` or the row's
    // last (p = 0 whatever maximum is subtracted), and the maximum moved.
    RFP4_DEV void settle(f32x4 (&st)[2], uint32_t key0, uint32_t hi, uint32_t nan)
    {
        uint32_t k0 = 4u * q4; // (the empty asm keeps what this path computes out of the loop's registers)
        asm volatile("" : "+v"(k0));
        const uint32_t last = min(lim, hi);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t t = k0 + (uint32_t)(j < 4 ? j : 12 + j);
            if ((nan >> t) & 1u) st[j / 4][j % 4] = __uint_as_float(0x7FC00000u);
            if (key0 + t >= last) st[j / 4][j % 4] = -INFINITY;
        }
        const float mx = largest(st) * fk;
        if (__any(mx > m + 8.0f)) {
            const float top = xor32_max(xor16_max(mx));
            const float mnew = top > m + 8.0f ? top : m;
            const float alpha = __builtin_amdgcn_exp2f(m - mnew);
            m = mnew;
            l *= alpha;
            scale_o(alpha);
            threshold();
        }
    }
    // Settled scores to probabilities as two fp16 terms
    RFP4_DEV void probabilities(const f32x4 (&st)[2], f16x8 &ph, f16x8 &pl)
    {
        float p[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            p[j] = __builtin_amdgcn_exp2f(fmaf(st[j / 4][j % 4], fk, -m));
            l += p[j];
        }
        attn_split8(p, ph, pl);
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

// ---- few rows: one tile, key groups of a wave each, K and V from memory to
// registers with no LDS.  K operands are 16-byte pieces of rows l16 and 16 +
// l16; for V^T a lane loads dimensions l16 HD/16 .. +HD/16 - 1 of its 8 keys, so
// a row of 16 lanes reads whole V rows, and dimension l16 HD/16 + n is row l16
// of tile n.  A wave holds two blocks, and refills a block's registers as soon as
// its operands are through them.
//
// Bound by HBM where the keys are many, else by the chain of a launch: loads,
// scores, softmax, P V, the groups' merge.  One row of 32 heads of 128 over 8, 8
// bits: 32769 keys (68 MB) 15.5-16.4 us, 4.1-4.4 TB/s; 4096 keys 6.2-6.5 us; 77 keys
// of 4 heads of 64 over one 4.1 us (the whole chain once).  16 rows over 4096 shared
// fp16 keys read them four times, once for every 4 rows, out of L2: 14.3-15.0 us with
// their own 200 keys, and from there 1.2 us for every 32 keys of a wave.
template <int HD, bool F8, int WK>
struct AttnRowsFew : AttnRowsState<HD> {
    typedef AttnRowsState<HD> State;
    using State::KS;
    using State::NN;
    using State::l16;
    using State::q4;
    using State::lane;
    using State::qa;
    using State::ql;
    using State::o;
    static constexpr int EB = F8 ? 1 : 2;    // bytes of an element
    static constexpr int NKL = HD * EB / 64; // 16-byte K loads of a lane per 16-key half
    static constexpr int VW = NN * EB / 4;   // dwords of a lane per V row

    struct Block {
        u32x4v kr[2][NKL];   // raw K rows l16 and 16 + l16
        uint32_t vr[8][VW];  // raw V of the lane's 8 keys
        uint32_t sb;         // scale byte of key lane % 32, K's in lanes 0..31, V's in the others
    };
    Block even, odd;
    int kref = -1000, vref = -1000;

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
    RFP4_DEV void load_k(Block &x, const AttnRowsKeys &s, uint32_t key0)
    {
        if (whole(s, key0)) {
            const uint32_t off = (uint32_t)EB * l16 * (uint32_t)s.ts + 16u * q4;
            const uint8_t *b = s.k + (uint64_t)key0 * s.ts * EB;
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int i = 0; i < NKL; i++) x.kr[h][i] = *(const u32x4v *)(b + (uint64_t)(16 * h) * s.ts * EB + off + 64 * i);
        } else {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint8_t *b = s.k + (uint64_t)min(key0 + 16u * (uint32_t)h + l16, s.end - 1u) * s.ts * EB + 16u * q4;
#pragma unroll
                for (int i = 0; i < NKL; i++) x.kr[h][i] = *(const u32x4v *)(b + 64 * i);
            }
        }
        if constexpr (F8) {
            const uint32_t t = min(key0 + (lane & 31u), s.end - 1u);
            x.sb = (lane < 32u ? s.ks : s.vs)[(uint64_t)t * (s.ts / HD)];
        }
    }
    RFP4_DEV void load_v(Block &x, const AttnRowsKeys &s, uint32_t key0)
    {
        if (whole(s, key0)) {
            const uint32_t off = (uint32_t)EB * (4u * q4 * (uint32_t)s.ts + (uint32_t)NN * l16);
            const uint8_t *b = s.v + (uint64_t)key0 * s.ts * EB;
#pragma unroll
            for (int j = 0; j < 8; j++) load_vrow(x.vr[j], b + (uint64_t)(j < 4 ? j : 12 + j) * s.ts * EB + off);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint32_t t = min(key0 + 4u * q4 + (uint32_t)(j < 4 ? j : 12 + j), s.end - 1u);
                load_vrow(x.vr[j], s.v + ((uint64_t)t * s.ts + (uint32_t)NN * l16) * EB);
            }
        }
    }

    // The wave's blocks of s: 32 keys from key0 on, every WK-th; the loads of the
    // first two are out (key0 < s.hi).  sc: 64 floats of LDS of the wave.
    RFP4_DEV void walk(const AttnRowsKeys &s, uint32_t key0, float *sc)
    {
        for (;; key0 += 64u * WK) {
            block(even, s, key0, sc);
            if (key0 + 32u * WK >= s.hi) break;
            block(odd, s, key0 + 32u * WK, sc);
            if (key0 + 64u * WK >= s.hi) break;
        }
        if constexpr (F8) this->scale_o(ldexpf(1.0f, vref - 127));
    }
    // The block at key0 in x, whose registers then load the one after next
    RFP4_DEV void block(Block &x, const AttnRowsKeys &s, uint32_t key0, float *sc)
    {
        const uint32_t next = key0 + 64u * WK;
        const bool more = next < s.hi;
        uint32_t nan = 0;
        float ksc[2] = {1.0f, 1.0f}, vsc[8] = {1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f};
        if constexpr (F8) {
            const bool bad = x.sb == 255u;
            const int ref = lane < 32u ? kref : vref;
            if (__builtin_expect(__any(bad || (int)x.sb > ref + 7), 0)) {
                const uint64_t nans = __ballot(bad);
                nan = (uint32_t)nans | (uint32_t)(nans >> 32);
                float top = bad ? -2000.0f : (float)x.sb; // bytes are exact in f32
                top = xor16_max(row16_max(top));
                const int kt = __builtin_amdgcn_readfirstlane((int)top), vt = __builtin_amdgcn_readlane((int)top, 32);
                if (kt > kref + 7) {
                    kref = kt;
                    this->set_factor(kref);
                }
                if (vt > vref + 7) {
                    this->scale_o(pow2_int(vref - vt)); // 2^-126 for the first block, whose O is 0
                    vref = vt;
                }
            }
            sc[lane] = bad ? 1.0f : pow2_int((int)x.sb - (lane < 32u ? kref : vref));
            __builtin_amdgcn_wave_barrier();
            ksc[0] = sc[l16];
            ksc[1] = sc[16u + l16];
            const float4 v0 = *(const float4 *)&sc[32u + 4u * q4], v1 = *(const float4 *)&sc[48u + 4u * q4];
            vsc[0] = v0.x; vsc[1] = v0.y; vsc[2] = v0.z; vsc[3] = v0.w;
            vsc[4] = v1.x; vsc[5] = v1.y; vsc[6] = v1.z; vsc[7] = v1.w;
            __builtin_amdgcn_wave_barrier();
        }
        f32x4 st[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
        for (int k = 0; k < KS; k++) {
            const f16x8 k0 = k_operand(x, 0, k, ksc[0]), k1 = k_operand(x, 1, k, ksc[1]);
            st[0] = mfma16(k0, qa[k], st[0]);
            st[1] = mfma16(k1, qa[k], st[1]);
            st[0] = mfma16(k0, ql[k], st[0]);
            st[1] = mfma16(k1, ql[k], st[1]);
        }
        if (more) load_k(x, s, next);
        if (nan || __any(key0 + 32u > min(this->lim, s.hi) || this->exceeds(st))) this->settle(st, key0, s.hi, nan);
        f16x8 ph, pl;
        this->probabilities(st, ph, pl);
        constexpr int NB = F8 ? 4 : 2; // tiles of a V dword
#pragma unroll
        for (int w = 0; w < VW; w++) {
            f16x8 va[NB];
            v_operands(x, w, vsc, va);
#pragma unroll
            for (int n = 0; n < NB; n++) o[NB * w + n] = mfma16(va[n], ph, o[NB * w + n]);
#pragma unroll
            for (int n = 0; n < NB; n++) o[NB * w + n] = mfma16(va[n], pl, o[NB * w + n]);
        }
        if (more) load_v(x, s, next);
    }

    // K row l16 of half h at K step k as fp16
    RFP4_DEV static f16x8 k_operand(const Block &x, int h, int k, float scale)
    {
        if constexpr (F8) {
            const u32x4v r = x.kr[h][k / 2];
            const uint32_t w0 = k % 2 ? r.z : r.x, w1 = k % 2 ? r.w : r.y;
            return __builtin_bit_cast(f16x8, u32x4v{fp8x2_to_f16<false>(w0, scale), fp8x2_to_f16<true>(w0, scale), fp8x2_to_f16<false>(w1, scale),
                                                    fp8x2_to_f16<true>(w1, scale)});
        } else {
            return __builtin_bit_cast(f16x8, x.kr[h][k]);
        }
    }

    // V^T operands of the tiles of V dword w: row l16 of each tile at the lane's 8 keys
    template <int NB>
    RFP4_DEV static void v_operands(const Block &x, int w, const float (&vsc)[8], f16x8 (&va)[NB])
    {
        u32x4v t[NB];
#pragma unroll
        for (int jp = 0; jp < 4; jp++) {
            uint32_t a[NB / 2], b[NB / 2]; // pairs of dimensions of keys 2 jp and 2 jp + 1
            if constexpr (F8) {
                a[0] = fp8x2_to_f16<false>(x.vr[2 * jp][w], vsc[2 * jp]);
                a[1] = fp8x2_to_f16<true>(x.vr[2 * jp][w], vsc[2 * jp]);
                b[0] = fp8x2_to_f16<false>(x.vr[2 * jp + 1][w], vsc[2 * jp + 1]);
                b[1] = fp8x2_to_f16<true>(x.vr[2 * jp + 1][w], vsc[2 * jp + 1]);
            } else {
                a[0] = x.vr[2 * jp][w];
                b[0] = x.vr[2 * jp + 1][w];
            }
#pragma unroll
            for (int i = 0; i < NB / 2; i++) {
                t[2 * i][jp] = __builtin_amdgcn_perm(b[i], a[i], 0x05040100u);
                t[2 * i + 1][jp] = __builtin_amdgcn_perm(b[i], a[i], 0x07060302u);
            }
        }
#pragma unroll
        for (int n = 0; n < NB; n++) va[n] = __builtin_bit_cast(f16x8, t[n]);
    }
};

// The query rows row0 .. row_end (at most 16) of KV head kvh over s, written as
// outputs, or as split `split`'s states.
template <int HD, bool F8>
RFP4_DEV void attn_rows_few(const AttnRowsArgs &a, uint32_t kvh, uint32_t row0, uint32_t row_end, const AttnRowsKeys &s, uint32_t split)
{
    constexpr int WK = 4, NN = HD / 16;
    __shared__ __align__(16) float sc[WK][64];
    __shared__ __align__(16) float ro[WK][16][HD + 4];
    __shared__ float rm[WK][16], rl[WK][16];
    AttnRowsFew<HD, F8, WK> r;
    const uint32_t kgrp = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), key0 = s.lo + 32u * kgrp;
    const bool any = key0 < s.hi;
    if (any) { // before q: its scaling runs under these loads
        r.load_k(r.even, s, key0);
        r.load_v(r.even, s, key0);
        if (key0 + 32u * WK < s.hi) {
            r.load_k(r.odd, s, key0 + 32u * WK);
            r.load_v(r.odd, s, key0 + 32u * WK);
        }
    }
    r.template load_q<F8>(a, kvh, row0, row_end, s.hi);
    if (any) r.walk(s, key0, sc[kgrp]);
    r.l = xor32_sum(xor16_sum(r.l));

    // the key groups' states through LDS
    if (r.q4 == 0u) {
        rm[kgrp][r.l16] = r.m;
        rl[kgrp][r.l16] = r.l;
    }
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int n = 0; n < NN; n += 4)
            *(float4 *)&ro[kgrp][r.l16][(4u * r.q4 + (uint32_t)t) * NN + n] = make_float4(r.o[n][t], r.o[n + 1][t], r.o[n + 2][t], r.o[n + 3][t]);
    __syncthreads();
    const uint32_t S = a.splits0 + a.splits1;
    constexpr uint32_t LPR = HD / 4; // lanes of a row, 4 dimensions each
    for (uint32_t u = threadIdx.x; u < 16u * LPR; u += 64u * WK) {
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

// ---- many rows: 4 tiles, a wave each, and two groups of 4 waves that take the
// same 64 rows and alternate key blocks (group g blocks g, g + 2, ...).  A group
// stages its block in LDS as fp16 rows, so a key is read and converted once for
// 64 rows.  V^T operands come out of the rows through the transposing LDS read.
// Rows are padded (K by 16 bytes: read 16 rows at a time, 16 bytes each; V by
// 32: 8 rows, 32 bytes), so reads cover the banks once and every address is one
// register and a constant.  Dimension 16 n + 4 q4 + r is accumulator r of tile n.
//
// The groups run half a step apart between common barriers: while one loads and does
// its matrix instructions (P V of its block, then the scores of its next one), the
// other takes exponentials, converts and stages; 4 waves a SIMD (128 registers),
// two workgroups a CU.  At 2048 rows after 2048 keys of 32
// heads of 128 over 8 (206 GFLOP with the second terms) 186 us in a row of
// calls, 1.11 PFLOP/s, where a large fp16 product reaches 1.15; under the
// profiler 207 us, the matrix cores busy 47 % of the cycles.  64 rows over 16384
// keys: 49-54 us.  What bounds it there: a vector half takes 1500-1650 cycles, a
// matrix half 1600-1750 with 550 of loads and their addresses (in the vector half
// those took it to 1800, the whole 188 us), and the waits between 200-450 each.  Alone
// on a SIMD a wave's vector instruction takes 5.4 cycles, its exponential or mixed
// fma 9.4, beside another's matrix instructions 6.8 and 11.
// Measured there and not better: 32 rows a wave (210 us; free-running 212; with
// the conversion between the matrix instructions 241), 8 waves of 16 rows and
// one group (222), 4 groups (259), 32 rows a wave without the rare paths moved
// out of the loop's way (305).  In a row of calls (188-198 at the time): staging and loads
// between the matrix instructions, with two buffers (V half 900 cycles, M half 2050:
// 205), staged rows permuted so that no write meets a bank twice (the same), 16-byte
// loads and each scale byte loaded once (187).
template <int HD, bool F8>
struct AttnRowsMany : AttnRowsState<HD> {
    typedef AttnRowsState<HD> State;
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
    static constexpr uint32_t STEP = 2 * BK;    // of both groups
    static constexpr int NC = (int)BK / 32;
    static constexpr uint32_t KRB = 2 * HD + 16, VRB = 2 * HD + 32; // bytes of a staged K and V row
    static constexpr uint32_t NL = EB;          // 16-byte loads of a thread for a block's K (and V)
    static constexpr uint32_t CPR = HD * EB / 16; // 16-byte pieces of a cache row
    static constexpr uint32_t KBUF = BK * KRB, GROUP = KBUF + BK * VRB, LDS = 2 * GROUP; // a group's K rows, then its V rows
    typedef short i16x4 __attribute__((ext_vector_type(4)));
    typedef short i16x8 __attribute__((ext_vector_type(8)));
    typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
    typedef __attribute__((address_space(3))) uint8_t lds_u8;

    // What this thread loads of a block's K (and V): 16 bytes of fp16 rows twice,
    // 8 bytes of 8-bit rows twice, so that its two 16-byte pieces of the staged
    // rows lie beside its neighbours' (no bank conflicts), and the scale byte of
    // its row (own) and of key lane % BK (all: what moves the reference)
    struct Raw {
        u32x4v x[NL];
        uint32_t own, all;
    };
    uint32_t tid;           // thread of the group
    Raw kraw, vraw;
    int kref = -1000, vref = -1000; // references of the latest staged K and V
    f32x4 sc[NC][2];
    f16x8 ph[NC], pl[NC];

    RFP4_DEV static uint32_t row(uint32_t t, uint32_t i) { return F8 ? t / (HD / 16) : (t + 256u * i) / CPR; }
    RFP4_DEV static uint32_t col(uint32_t t, uint32_t i) { return F8 ? t % (HD / 16) : (t + 256u * i) % CPR; }
    // A 32-bit value as the loop holds it: an offset is not widened to 64 bits, nor
    // anything computed from it, outside of the loop
    RFP4_DEV static uint32_t fixed(uint32_t x)
    {
        asm volatile("" : "+v"(x));
        return x;
    }
    // K (or V) rows of a block inside the cache, x its first row and xs its first
    // scale byte: 32-bit lane offsets from uniform bases
    RFP4_DEV void load_whole(const AttnRowsKeys &s, const uint8_t *x, const uint8_t *xs, Raw &raw)
    {
        const uint32_t ts = (uint32_t)s.ts;
        if constexpr (F8) {
            const uint32_t at = fixed(row(tid, 0) * ts + 8u * col(tid, 0));
            const uint2 a = *(const uint2 *)(x + at), b = *(const uint2 *)(x + at + HD / 2);
            raw.x[0] = u32x4v{a.x, a.y, b.x, b.y};
            raw.own = xs[fixed(row(tid, 0) * (ts / HD))];
            raw.all = xs[fixed(lane % BK * (ts / HD))];
        } else {
#pragma unroll
            for (uint32_t i = 0; i < NL; i++) raw.x[i] = *(const u32x4v *)(x + fixed(row(tid, i) * ts * EB + 16u * col(tid, i)));
        }
    }
    // Those of any block at key0: keys past the last that exists re-read it; they are masked
    RFP4_DEV void load_any(const AttnRowsKeys &s, const uint8_t *x, const uint8_t *xs, uint32_t key0, Raw &raw)
    {
        const uint32_t t = fixed(tid);
        if constexpr (F8) {
            const uint64_t at = (uint64_t)min(key0 + row(t, 0), s.end - 1u) * s.ts;
            const uint2 a = *(const uint2 *)(x + at + 8u * col(t, 0)), b = *(const uint2 *)(x + at + 8u * col(t, 0) + HD / 2);
            raw.x[0] = u32x4v{a.x, a.y, b.x, b.y};
            raw.own = xs[at / HD];
            raw.all = xs[(uint64_t)min(key0 + t % BK, s.end - 1u) * (s.ts / HD)];
        } else {
#pragma unroll
            for (uint32_t i = 0; i < NL; i++)
                raw.x[i] = *(const u32x4v *)(x + ((uint64_t)min(key0 + row(t, i), s.end - 1u) * s.ts * EB + 16u * col(t, i)));
        }
    }

    // Whether a key of the block in the registers has a scale that the reference
    // does not cover, or byte 255
    RFP4_DEV static bool uncovered(const Raw &raw, int ref) { return (int)raw.all > min(ref + 7, 254); }
    // Then moves the reference (the same in every wave of the group: all hold the
    // same bytes); a byte of 255 counts as a scale of 1.  The keys that have it.
    RFP4_DEV uint64_t refer(Raw &raw, int &ref)
    {
        const bool bad = raw.all == 255u;
        const int top = __builtin_amdgcn_readfirstlane((int)wave_max(bad ? -2000.0f : (float)raw.all)); // exact in f32
        ref = top > ref + 7 ? top : ref;
        if (raw.own == 255u) raw.own = (uint32_t)ref;
        return __ballot(bad);
    }
    // The block in the registers as fp16 rows of RB bytes at `to`
    template <uint32_t RB>
    RFP4_DEV void stage(lds_u8 *to, const Raw &raw, int ref)
    {
        if constexpr (F8) {
            const float scale = __uint_as_float((uint32_t)max((int)raw.own + (127 - ref), 1) << 23);
            lds_u8 *p = to + row(tid, 0) * RB + 16u * col(tid, 0);
            put(p, raw.x[0].x, raw.x[0].y, scale);
            put(p + HD, raw.x[0].z, raw.x[0].w, scale);
        } else {
#pragma unroll
            for (uint32_t i = 0; i < NL; i++) *(__attribute__((address_space(3))) u32x4v *)(to + row(tid, i) * RB + 16u * col(tid, i)) = raw.x[i];
        }
    }
    RFP4_DEV static void put(lds_u8 *p, uint32_t w0, uint32_t w1, float scale)
    {
        *(__attribute__((address_space(3))) u32x4v *)p =
            u32x4v{fp8x2_to_f16<false>(w0, scale), fp8x2_to_f16<true>(w0, scale), fp8x2_to_f16<false>(w1, scale), fp8x2_to_f16<true>(w1, scale)};
    }

    // O^T += V^T P^T of the staged V (PV), then S^T of the staged K; kbuf and vbuf:
    // this lane's addresses in them.  An operand of 16 bytes feeds two
    // instructions, 32 cycles, and takes over 100 from LDS: it is read AHEAD
    // operands before its use (the scheduling barriers keep that order).
    template <bool PV>
    RFP4_DEV void matrix(const lds_u8 *vbuf, const lds_u8 *kbuf)
    {
        constexpr int NPV = PV ? NC * NN : 0, N = NPV + NC * KS * 2, AHEAD = 2;
        f16x8 x[AHEAD + 1];
        auto fetch = [&](int j) {
            if (j < NPV) {
                const lds_u8 *const at = vbuf + 32u * (uint32_t)(j % NN) + 32u * (uint32_t)(j / NN) * VRB;
                const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)at);
                const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(at + 16u * VRB));
                return __builtin_bit_cast(f16x8, i16x8{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w});
            }
            const int i = j - NPV, c = i / (2 * KS), k = i / 2 % KS, h = i % 2;
            return *(const __attribute__((address_space(3))) f16x8 *)(kbuf + 64u * (uint32_t)k + (32u * (uint32_t)c + 16u * (uint32_t)h) * KRB);
        };
#pragma unroll
        for (int j = 0; j < AHEAD; j++) x[j] = fetch(j);
#pragma unroll
        for (int j = 0; j < N; j++) {
            if (j + AHEAD < N) x[(j + AHEAD) % (AHEAD + 1)] = fetch(j + AHEAD);
            __builtin_amdgcn_sched_barrier(0);
            const f16x8 y = x[j % (AHEAD + 1)];
            if (j < NPV) {
                const int c = j / NN, d = j % NN;
                o[d] = mfma16(y, ph[c], o[d]);
                o[d] = mfma16(y, pl[c], o[d]);
            } else {
                const int i = j - NPV, c = i / (2 * KS), k = i / 2 % KS, h = i % 2;
                sc[c][h] = mfma16(y, qa[k], k ? sc[c][h] : f32x4{0.0f, 0.0f, 0.0f, 0.0f});
                sc[c][h] = mfma16(y, ql[k], sc[c][h]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    RFP4_DEV static void barrier() // with this wave's LDS accesses done; global loads stay in flight
    {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    }

    // Group `group`'s blocks of the keys s.lo .. s.hi (at least one key), of which
    // this wave's rows see those below whi, and all of them those below wlo.  Every
    // wave of the workgroup passes the same barriers.
    RFP4_DEV void walk(const AttnRowsKeys &s, uint32_t wlo, uint32_t whi, uint32_t group, lds_u8 *lds)
    {
        lds_u8 *const kbuf = lds + group * GROUP, *const vbuf = kbuf + KBUF;
        // the transposing read: lane j of 16 gives the address of 4 halves, row
        // j / 4 of 4, columns 4 (j % 4) .. +3 of 16, and gets column j of the 4 rows
        const lds_u8 *const kl = kbuf + l16 * KRB + 16u * q4, *const vl = vbuf + (4u * q4 + (l16 >> 2)) * VRB + 8u * (l16 & 3u);
        const uint32_t steps = (s.hi - s.lo + STEP - 1u) / STEP; // of either group; the second's last block may lie past the keys
        uint32_t key0 = s.lo + group * BK;
        load_any(s, s.k, s.ks, key0, kraw);
        load_any(s, s.v, s.vs, key0, vraw);
        uint64_t knan = 0; // keys of byte 255 of the K in LDS
        if constexpr (F8) knan = refer(kraw, kref);
        stage<KRB>(kbuf, kraw, kref);
        load_any(s, s.k, s.ks, key0 + STEP, kraw);
        barrier();
        if (group) barrier(); // half a step behind
        matrix<false>(vl, kl);
        barrier();
        int kcur = -1001, vcur = -1000; // references of the factor (the first block always sets it) and of O
        // the blocks to load next: V of the next step, K of the one after it
        const uint64_t step = (uint64_t)STEP * s.ts, ofs = (uint64_t)(key0 + STEP) * s.ts;
        const uint8_t *vn = s.v + ofs * EB, *kn = s.k + (ofs + step) * EB, *vsn = s.vs + (F8 ? ofs / HD : 0u), *ksn = s.ks + (F8 ? (ofs + step) / HD : 0u);
        const uint32_t in = s.ts < (1ull << 24) ? s.end : 0u; // keys that the 32-bit offsets reach
        for (uint32_t i = 0;; i++, key0 += STEP) {
            // ---- vector half: its V and the next block's K to LDS; the block's probabilities
            // (expected branches fall through: a taken one costs the wave a fetch)
            uint64_t nan = 0;
            if constexpr (F8) {
                if (__builtin_expect(kref != kcur, 0)) {
                    this->set_factor(kref);
                    kcur = kref;
                }
                nan = knan;
                knan = 0;
                if (__builtin_expect(__any(uncovered(vraw, vref) || uncovered(kraw, kref)), 0)) {
                    nan |= refer(vraw, vref);
                    knan = refer(kraw, kref); // (a stale block after the last)
                    this->scale_o(pow2_int(vcur - vref)); // 2^-126 for the first block, whose O is 0
                    vcur = vref;
                }
            }
            stage<VRB>(vbuf, vraw, vref);
            stage<KRB>(kbuf, kraw, kref);
            const bool live = key0 < whi; // the same for the whole wave
            if (__builtin_expect(live, 1)) {
                bool rare = false;
#pragma unroll
                for (int c = 0; c < NC; c++) rare = rare || this->exceeds(sc[c]);
                if (__builtin_expect(nan || key0 + BK > wlo || __any(rare), 0)) {
#pragma unroll
                    for (int c = 0; c < NC; c++) this->settle(sc[c], key0 + 32u * (uint32_t)c, s.hi, (uint32_t)(nan >> (32 * c)));
                }
#pragma unroll
                for (int c = 0; c < NC; c++) this->probabilities(sc[c], ph[c], pl[c]);
            }
            barrier();
            // ---- matrix half: the next loads; P V of the block, the scores of the next
            if (__builtin_expect(key0 + 2u * STEP + BK <= in, 1)) {
                load_whole(s, vn, vsn, vraw);
                load_whole(s, kn, ksn, kraw);
            } else {
                load_any(s, s.v, s.vs, key0 + STEP, vraw);
                load_any(s, s.k, s.ks, key0 + 2u * STEP, kraw);
            }
            vn += step * EB;
            kn += step * EB;
            if constexpr (F8) {
                vsn += step / HD;
                ksn += step / HD;
            }
            if (__builtin_expect(live, 1)) {
                __builtin_amdgcn_s_setprio(1);
                matrix<true>(vl, kl);
                __builtin_amdgcn_s_setprio(0);
            }
            if (i + 1u == steps) break;
            barrier();
        }
        if (!group) barrier(); // the other group's last half step
        if constexpr (F8) this->scale_o(ldexpf(1.0f, vcur - 127));
    }
};

// The query rows row0 .. row_end (at most 64) of KV head kvh over s by the two
// groups, whose states are merged through LDS.
template <int HD, bool F8>
RFP4_DEV void attn_rows_many(const AttnRowsArgs &a, uint32_t kvh, uint32_t row0, uint32_t row_end, const AttnRowsKeys &s, uint32_t split)
{
    typedef AttnRowsMany<HD, F8> R;
    typedef float Merge[4][R::NN * 4 + 2][64]; // the second group's O, m, l, by wave and lane
    constexpr uint32_t LDS = R::LDS > sizeof(Merge) ? R::LDS : sizeof(Merge);
    __shared__ __attribute__((aligned(1024))) uint8_t lds[LDS];
    R r;
    r.tid = threadIdx.x & 255u;
    const uint32_t wid = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), group = wid >> 2, wave = wid & 3u;
    const uint32_t wrow = row0 + 16u * wave;
    r.template load_q<false>(a, kvh, wrow, row_end, s.hi);
    uint32_t whi = wrow < row_end ? s.hi : 0u, wlo = s.hi; // waves without rows stage and wait only
    if (a.causal) {
        whi = min(whi, a.pos0 + min(wrow + 15u, row_end - 1u) / a.group + 1u);
        wlo = min(wlo, a.pos0 + wrow / a.group + 1u);
    }
    if (s.lo < s.hi) r.walk(s, wlo, whi, group, (typename R::lds_u8 *)lds); // the same for the whole workgroup
    __syncthreads();
    r.l = xor32_sum(xor16_sum(r.l));
    float(*const w)[64] = (*(Merge *)lds)[wave];
    if (group) {
#pragma unroll
        for (int n = 0; n < R::NN; n++)
#pragma unroll
            for (int t = 0; t < 4; t++) w[4 * n + t][r.lane] = r.o[n][t];
        w[4 * R::NN][r.lane] = r.m;
        w[4 * R::NN + 1][r.lane] = r.l;
    }
    __syncthreads();
    const uint32_t rho = wrow + r.l16;
    if (group || rho >= row_end) return;
    const float m1 = w[4 * R::NN][r.lane], M = fmaxf(r.m, m1);
    const float c0 = __builtin_amdgcn_exp2f(r.m - M), c1 = __builtin_amdgcn_exp2f(m1 - M);
    const float L = fmaf(r.l, c0, w[4 * R::NN + 1][r.lane] * c1);
    const uint32_t i = rho / a.group, head = kvh * a.group + rho % a.group, S = a.splits0 + a.splits1;
#pragma unroll
    for (int n = 0; n < R::NN; n++) {
        f32x4 acc;
#pragma unroll
        for (int t = 0; t < 4; t++) acc[t] = fmaf(r.o[n][t], c0, w[4 * n + t][r.lane] * c1);
        attn_rows_put<HD>(a, i, head, S, split, 16u * (uint32_t)n + 4u * r.q4, n == 0 && r.q4 == 0u, M, L, acc);
    }
}

// Workgroup (kvh, item), kvh = blockIdx.x % n_kv_heads (with 8 KV heads each
// XCD, workgroup id % 8, keeps one head's K and V in its L2): the shared keys'
// items (row tile, split) first, the longest causal ranges leading, then the
// own keys' (row, split).
template <int HD, bool F8, bool MANY>
RFP4_DEV void attn_rows_body(const AttnRowsArgs &a)
{
    constexpr uint32_t EB = F8 ? 1u : 2u, RW = MANY ? 64u : 16u;
    const uint32_t kvh = blockIdx.x % a.n_kv_heads, item = a.first + blockIdx.x / a.n_kv_heads;
    uint32_t row0, row_end, split;
    const void *k, *v;
    const uint8_t *ks, *vs;
    uint64_t base;
    AttnRowsKeys s;
    if (item < a.tiles0 * a.splits0) {
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
    if constexpr (MANY) attn_rows_many<HD, F8>(a, kvh, row0, row_end, s, split);
    else attn_rows_few<HD, F8>(a, kvh, row0, row_end, s, split);
}

// The states of query row i, head h, merged: M = max m, out = sum acc 2^(m - M)
// / sum l 2^(m - M); 0 for a row without keys.  HD / 4 lanes take the dimensions
// of a state, the workgroup's 1024 / HD parts every so many of the splits; the
// first four of each part are loaded beside the (m, l) that their weights need,
// so up to 4096 / HD splits take one round trip of memory: 32 heads of 32 splits
// 2.6-3.8 us, most of it the launch (9.3 us with a round trip for every 8 of 52).
template <int HD>
RFP4_DEV void attn_rows_merge_body(const AttnRowsArgs &a)
{
    constexpr uint32_t P = 1024u / HD, LPR = HD / 4, AHEAD = 4;
    __shared__ float w[kAttnRowsMaxSplits], red[8];
    __shared__ __align__(16) float acc_p[P][HD];
    const uint32_t h = blockIdx.x % a.n_heads, i = blockIdx.x / a.n_heads;
    const uint32_t tid = threadIdx.x, d = 4u * (tid % LPR), p = tid / LPR, S = a.splits0 + a.splits1;
    const uint32_t keys0 = a.causal ? a.pos0 + i + 1u : a.len0, keys1 = a.splits1 ? min(a.lens[i], a.cap1) : 0u;
    const uint32_t n0 = a.splits0 ? (keys0 + a.chunk0 - 1u) / a.chunk0 : 0u;
    const uint32_t n = n0 + (a.splits1 ? (keys1 + a.chunk1 - 1u) / a.chunk1 : 0u);
    const float *st = a.part + (size_t)((size_t)i * a.n_heads + h) * S * (HD + 4);
    auto state = [&](uint32_t x) { return st + (size_t)(x < n0 ? x : a.splits0 + (x - n0)) * (HD + 4); };
    f32x4 v[AHEAD];
#pragma unroll
    for (uint32_t j = 0; j < AHEAD; j++) {
        const uint32_t x = p + P * j;
        v[j] = x < n ? *(const f32x4 *)(state(x) + 4 + d) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    constexpr uint32_t ML = kAttnRowsMaxSplits / 256u; // (m, l) of a thread
    float m[ML], l[ML];
    float M = -3.402823466e38f;
#pragma unroll
    for (uint32_t j = 0; j < ML; j++) {
        const uint32_t x = tid + 256u * j;
        m[j] = x < n ? state(x)[0] : -3.402823466e38f;
        l[j] = x < n ? state(x)[1] : 0.0f;
        M = fmaxf(M, m[j]);
    }
    M = wave_max(M);
    if ((tid & 63u) == 0u) red[tid >> 6] = M;
    __syncthreads();
    M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    float L = 0.0f;
#pragma unroll
    for (uint32_t j = 0; j < ML; j++) {
        const uint32_t x = tid + 256u * j;
        const float c = __builtin_amdgcn_exp2f(m[j] - M);
        if (x < n) w[x] = c;
        L = fmaf(l[j], x < n ? c : 0.0f, L);
    }
    L = wave_sum(L);
    if ((tid & 63u) == 0u) red[4 + (tid >> 6)] = L;
    __syncthreads();
    L = (red[4] + red[5]) + (red[6] + red[7]);
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (uint32_t j = 0; j < AHEAD; j++) {
        const uint32_t x = p + P * j;
        const float c = x < n ? w[x] : 0.0f;
#pragma unroll
        for (int t = 0; t < 4; t++) acc[t] = fmaf(v[j][t], c, acc[t]);
    }
    for (uint32_t x = p + P * AHEAD; x < n; x += P) {
        const f32x4 y = *(const f32x4 *)(state(x) + 4 + d);
        const float c = w[x];
#pragma unroll
        for (int t = 0; t < 4; t++) acc[t] = fmaf(y[t], c, acc[t]);
    }
    *(f32x4 *)&acc_p[p][d] = acc;
    __syncthreads();
    if (tid >= LPR) return;
#pragma unroll
    for (uint32_t x = 1; x < P; x++) acc += *(const f32x4 *)&acc_p[x][d];
    const bool none = L == 0.0f;
#pragma unroll
    for (int t = 0; t < 4; t++) acc[t] = none ? 0.0f : __fdiv_rn(acc[t], L);
    *(f32x4 *)(a.out + (size_t)i * a.out_rs + (size_t)h * HD + d) = acc;
}
