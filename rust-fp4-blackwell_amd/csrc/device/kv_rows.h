// New K and V rows into a cache (gfx950): fp16, or e4m3 codes with one
// power-of-two scale for each token and KV head.
//
// 8-bit row x of head_dim values, amax = max |x|: se = the smallest integer
// >= -127 with amax * 2^-se <= 448 (the largest e4m3 value), scale byte
// se + 127, code = e4m3(x * 2^-se) to nearest even.  e4m3 is a floating format,
// so a finer scale than a power of two would add precision nowhere but below
// 2^-6 of the scaled row; with it x * 2^-se is exact, a code is x rounded once
// (at most half a step, 2^-4 relative, where |x| >= 2^(se - 6)), and the scale
// costs one byte.  A row of zeros has byte 0; a row with a value that is not
// finite has byte 255 (E8M0's NaN) and codes 0, so that it reads as NaN as a
// whole and a code is always finite.
//
// HD / 8 lanes take a row, 8 values each, so that a lane reads 32 bytes and writes
// 8 codes, and its row's maximum takes 3 or 4 DPP steps.  Bound by HBM (5 bytes a
// value): 2048 rows of 8 heads of 128 (21 MB) 4.5-4.9 us, 4.3-4.6 TB/s, where a
// large copy reaches 4.7.  A single token's rows by the launch: 1.9 us.
#pragma once
#include "common.h"

// Largest value (as an unsigned word) of aligned groups of N lanes, N = 8, 16.
template <int CTRL>
RFP4_DEV uint32_t dpp_max_u32(uint32_t v)
{
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false));
}
template <int N>
RFP4_DEV uint32_t group_max_u32(uint32_t v)
{
    v = dpp_max_u32<DPP_QUAD_1032>(v);
    v = dpp_max_u32<DPP_QUAD_2301>(v);
    v = dpp_max_u32<DPP_ROW_HALF_MIRROR>(v);
    return N == 16 ? dpp_max_u32<DPP_ROW_MIRROR>(v) : v;
}

template <int HD, bool F8>
RFP4_DEV void kv_rows_body(const KvRowsArgs &a)
{
    constexpr uint32_t LPR = HD / 8;
    const uint32_t unit = blockIdx.x * (256u / LPR) + threadIdx.x / LPR, lane = threadIdx.x % LPR;
    if (unit >= a.rows * 2u * a.n_kv_heads) return; // whole lane groups
    const uint32_t row = unit / (2u * a.n_kv_heads), r = unit % (2u * a.n_kv_heads);
    const bool is_v = r >= a.n_kv_heads;
    const uint32_t h = is_v ? r - a.n_kv_heads : r;
    const uint32_t t = a.positions ? a.positions[row] : a.pos0 + row;
    const float *src = (is_v ? a.v + (size_t)row * a.v_rs : a.k + (size_t)row * a.k_rs) + h * HD + 8u * lane;
    const float4 x0 = *(const float4 *)src, x1 = *(const float4 *)(src + 4);
    const float x[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
    const uint64_t at = (a.positions ? (uint64_t)row * a.ss : 0u) + (uint64_t)t * a.ts + (uint64_t)h * a.hs;
    if constexpr (F8) {
        uint32_t m = 0; // |x| as ordered bits: infinities and NaNs above every finite value
#pragma unroll
        for (int i = 0; i < 8; i++) m = max(m, __float_as_uint(x[i]) & 0x7FFFFFFFu);
        m = group_max_u32<LPR>(m);
        if (t >= a.capacity) return;
        // amax = 1.f * 2^(E - 127): amax 2^-se <= 448 = 1.75 * 2^8 gives se + 127 = E - 8, one more where 1.f > 1.75
        const int byte = max((int)(m >> 23) - 8 + ((m & 0x7FFFFFu) > 0x600000u ? 1 : 0), 0);
        const bool bad = m >= 0x7F800000u;
        const float inv = __uint_as_float((uint32_t)(254 - byte) << 23); // 2^-se, a normal number for every byte
        int c[2];
#pragma unroll
        for (int w = 0; w < 2; w++) {
            int v = 0;
            v = __builtin_amdgcn_cvt_pk_fp8_f32(__fmul_rn(x[4 * w], inv), __fmul_rn(x[4 * w + 1], inv), v, false);
            v = __builtin_amdgcn_cvt_pk_fp8_f32(__fmul_rn(x[4 * w + 2], inv), __fmul_rn(x[4 * w + 3], inv), v, true);
            c[w] = bad ? 0 : v;
        }
        *(uint2 *)((uint8_t *)(is_v ? a.vc : a.kc) + at + 8u * lane) = make_uint2((uint32_t)c[0], (uint32_t)c[1]);
        if (lane == 0u) (is_v ? a.vs : a.ks)[at / HD] = bad ? 255u : (uint8_t)byte;
    } else {
        if (t >= a.capacity) return;
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++)
            w[i] = (uint32_t)f32_to_f16_bits(x[2 * i]) | (uint32_t)f32_to_f16_bits(x[2 * i + 1]) << 16;
        *(uint4 *)((uint16_t *)(is_v ? a.vc : a.kc) + at + 8u * lane) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}
