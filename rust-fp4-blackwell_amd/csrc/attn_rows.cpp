// C-ABI entry points of the 8-bit KV cache, of the attention over it, and of
// attention of a batch that shares a prefix (include/rfp4.h): argument checks
// and launch plans.  Nothing of the library's is shared between calls: split
// states live in the caller's workspace.
#include "runtime.h"

#include <algorithm>

using namespace rfp4;

namespace {

bool aligned(const void *p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

// Keys and rows a call may have: 32-bit key and row counts with room for a
// block past the end.
constexpr uint64_t kMaxKeys = (uint64_t)1 << 31;
constexpr uint64_t kMaxStride = (uint64_t)1 << 48; // elements

struct Cache {
    const void *k, *v;
    const uint8_t *ks, *vs;
    uint64_t ts, hs, ss;
};

// A cache of `what`'s: pointers, 16-byte aligned rows, and for the 8-bit one
// strides of whole rows (a row's scale is at its element offset / head_dim).
int check_cache(const char *what, const Cache &c, bool fp8, uint32_t hd)
{
    if (!c.k || !c.v || (fp8 && (!c.ks || !c.vs))) return set_error(RFP4_E_INVALID, "%s: null cache pointer", what);
    const uint64_t unit = fp8 ? hd : 8u;
    if (!aligned(c.k, 16) || !aligned(c.v, 16) || c.ts % unit || c.hs % unit || c.ss % unit)
        return set_error(RFP4_E_ALIGN, "%s: cache rows must start 16-byte aligned, strides (%llu, %llu, %llu) be multiples of %llu", what,
                         (unsigned long long)c.ss, (unsigned long long)c.ts, (unsigned long long)c.hs, (unsigned long long)unit);
    if (c.ts >= kMaxStride || c.hs >= kMaxStride || c.ss >= kMaxStride) return set_error(RFP4_E_SHAPE, "%s: stride over 2^48", what);
    return RFP4_OK;
}

int check_heads(const char *what, uint32_t nh, uint32_t nkv, uint32_t hd)
{
    if (hd != 64 && hd != 128) return set_error(RFP4_E_SHAPE, "%s: head_dim %u unsupported (64 or 128)", what, hd);
    if (nkv == 0 || nh == 0 || nh % nkv || nh / nkv > 8)
        return set_error(RFP4_E_SHAPE, "%s: %u query heads over %u KV heads (group of at most 8)", what, nh, nkv);
    return RFP4_OK;
}

int check_rows(const char *what, const float *q, uint32_t q_rs, const float *out, uint32_t out_rs, uint32_t rows, uint32_t nh, uint32_t hd)
{
    if (!q || !out) return set_error(RFP4_E_INVALID, "%s: null pointer", what);
    if (!aligned(q, 16) || !aligned(out, 16) || q_rs % 4u || out_rs % 4u)
        return set_error(RFP4_E_ALIGN, "%s: q and out rows must start 16-byte aligned", what);
    if ((uint64_t)nh * hd > UINT32_MAX || (rows > 1 && (q_rs < nh * hd || out_rs < nh * hd)))
        return set_error(RFP4_E_SHAPE, "%s: row strides %u, %u < %u heads x %u", what, q_rs, out_rs, nh, hd);
    return RFP4_OK;
}

thread_local int t_mode = 0; // 0 planned, 1 attn_rows_few, 2 attn_rows_many

// How a call is cut: the kernel by its query rows of a KV head, the keys into
// splits.
struct Plan {
    bool many;
    uint32_t tiles0, splits0, chunk0, splits1, chunk1;
    uint32_t splits() const { return splits0 + splits1; }
};

// n splits or fewer, in chunks of a multiple of 128 keys (a workgroup's step).
void cut(uint64_t keys, uint64_t n, uint32_t *splits, uint32_t *chunk)
{
    const uint64_t c = ((keys + n - 1) / n + 127) / 128 * 128;
    *chunk = (uint32_t)c;
    *splits = (uint32_t)((keys + c - 1) / c);
}

// Splits of `keys` shared keys at most, for `tiles` row tiles: as many as make a
// workgroup for each of 256 CUs, of at least 128 keys (a block for each wave; 8
// heads x 4096 keys: 128 keys 6.2 us and 2.7 to merge, 256 7.2 and 2.5), and 256
// for the staging kernel (64 rows over 4096 keys: 128 keys 15.8 + 4.0, 256 13.8 +
// 3.4, 512 25.3 + 4.5); for that two workgroups a CU where a split keeps 2048 keys
// (256 rows after 16384 keys 165 -> 141 us; with 1024 left 64 rows over 16384 50.9
// -> 52.8, with 256 over 4096 25.6 -> 31.5).  Never fewer for more keys; 512 and
// 256 of the rows' own at most, within the merge's kAttnRowsMaxSplits.
uint64_t splits_of(bool many, uint64_t keys, uint64_t tiles, uint32_t nkv)
{
    const uint64_t wgs = tiles * nkv;
    uint64_t n = std::min<uint64_t>(256u / wgs, keys / (many ? 256u : 128u));
    if (many) n = std::max(n, std::min<uint64_t>(512u / wgs, keys / 2048u));
    return std::max<uint64_t>(1, n);
}
uint64_t splits_of_own(uint64_t keys, uint32_t rows, uint32_t nkv)
{
    return std::max<uint64_t>(1, std::min<uint64_t>(256u / ((uint64_t)rows * nkv), keys / 128u));
}
uint64_t tiles_of(bool many, uint64_t flat) { return many ? (flat + 63) / 64 : (flat + 15) / 16; }

Plan plan(bool causal, bool fp8, uint32_t nkv, uint32_t group, uint32_t hd, uint32_t rows, uint64_t len0, uint64_t cap1)
{
    Plan p{};
    const uint64_t flat = (uint64_t)rows * group;
    // 16 query rows for a workgroup whose waves read keys of their own, or 64 for
    // one that stages them: the first reads and converts a key for every 16 rows
    // and starts sooner, so few rows or keys are its.  Up to 32 rows of a KV head the
    // second wastes half its waves (20 rows of 64 over 4096 keys 12.3 / 14.9 us, few
    // / many).  Prompts that give it a workgroup for most CUs without splits, by the
    // scores (query heads x keys): heads of 128, 320 rows (160 workgroups) 14.6 / 15.7,
    // 400 18.6 / 17.5 (2.6e6), 512 20.4 / 18.8, 700 29.5 / 23.8, 512 after 2048 63.1 /
    // 50.7; heads of 64, 700 15.4 / 16.9 (7.8e6), 1024 23.8 / 22.1 (1.7e7), 512 after
    // 2048 35.6 / 32.9.  Else splits have to be long, by the keys: 8 bits, heads of 128,
    // 64 rows over 4096 25.3 / 29.2, 6144 32.7 / 31.3, 16384 67.6 / 47.5, 128 after 4096
    // 32.8 / 36.7, 8192 58.6 / 52.8, 256 after 4096 53.6 / 56.7, 8192 96.9 / 82.2; of
    // 64, 64 over 8192 30.5 / 26.3, 256 after 4096 32.9 / 40.5; fp16, which needs no
    // conversion, 64 over 2048 21.2 / 25.1, 4096 29.1 / 26.9, 16384 83.0 / 44.8; 16 rows
    // over 8192 (4.2e6 scores) are the first's.
    const uint64_t keys = causal ? (uint64_t)rows * (len0 - rows) + (uint64_t)rows * (rows + 1u) / 2u : (uint64_t)rows * len0;
    const uint64_t scores = keys * group * nkv;
    const bool full = causal && tiles_of(true, flat) * nkv >= 192u, full_scores = scores > (hd == 128 ? 2500000u : 12000000u);
    const bool split = len0 >= (fp8 ? 6000u : 4000u) && scores > (hd == 128 ? 6000000u : 12000000u);
    p.many = flat > 32 && (full ? full_scores : split);
    if (t_mode) p.many = t_mode == 2;
    if (len0) {
        p.tiles0 = (uint32_t)tiles_of(p.many, flat);
        cut(len0, splits_of(p.many, len0, p.tiles0, nkv), &p.splits0, &p.chunk0);
    }
    // The rows' own keys, a workgroup for each row's query heads: the first kernel's,
    // in a launch of its own where the second takes the shared ones, unless they are
    // few (run()).
    if (cap1) cut(cap1, splits_of_own(cap1, rows, nkv), &p.splits1, &p.chunk1);
    return p;
}

size_t state_bytes(uint64_t splits, uint32_t rows, uint32_t nh, uint32_t hd)
{
    return splits > 1 ? (size_t)rows * nh * splits * (hd + 4) * sizeof(float) : 0;
}

// A workspace for the split states of up to len0 shared and cap1 own keys: a chunk
// is a whole number of steps, so fewer keys can take more splits.
size_t workspace_bytes_of(uint32_t nkv, uint32_t nh, uint32_t hd, uint32_t rows, uint64_t len0, uint64_t cap1)
{
    const uint64_t flat = (uint64_t)rows * (nh / nkv);
    const bool either = flat > 32 && !t_mode, many = t_mode == 2;
    uint64_t n = 0;
    if (len0) n = splits_of(many, len0, tiles_of(many, flat), nkv);
    if (len0 && either) n = std::max(n, splits_of(true, len0, tiles_of(true, flat), nkv));
    if (cap1) n += splits_of_own(cap1, rows, nkv);
    return state_bytes(n, rows, nh, hd);
}

int run(const char *what, const Plan &p, AttnRowsArgs &a, bool fp8, uint32_t hd, void *workspace, size_t workspace_bytes, hipStream_t s)
{
    const size_t need = state_bytes(p.splits(), a.rows, a.n_heads, hd);
    if (need && !workspace) return set_error(RFP4_E_INVALID, "%s: null workspace (%zu bytes)", what, need);
    if (need && !aligned(workspace, 16)) return set_error(RFP4_E_ALIGN, "%s: workspace must be 16-byte aligned", what);
    if (need > workspace_bytes)
        return set_error(RFP4_E_CAPACITY, "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, need);
    a.part = (float *)workspace;
    a.group = a.n_heads / a.n_kv_heads;
    a.tiles0 = p.tiles0;
    a.splits0 = p.splits0;
    a.chunk0 = p.chunk0;
    a.splits1 = p.splits1;
    a.chunk1 = p.chunk1;
    const uint64_t shared = (uint64_t)p.tiles0 * p.splits0 * a.n_kv_heads, own = (uint64_t)a.rows * p.splits1 * a.n_kv_heads;
    const uint64_t merges = (uint64_t)a.rows * a.n_heads, most = std::max(shared + own, merges);
    if (most > ((uint64_t)1 << 22))
        return set_error(RFP4_E_CAPACITY, "%s: %llu workgroups (at most 2^22)", what, (unsigned long long)most);
    static const char *const kNames[2][2][2] = { // [head dim 128][8 bits][many]
        {{"rfp4_attn_rows_hd64_f16_few", "rfp4_attn_rows_hd64_f16_many"}, {"rfp4_attn_rows_hd64_fp8_few", "rfp4_attn_rows_hd64_fp8_many"}},
        {{"rfp4_attn_rows_hd128_f16_few", "rfp4_attn_rows_hd128_f16_many"}, {"rfp4_attn_rows_hd128_fp8_few", "rfp4_attn_rows_hd128_fp8_many"}}};
    const char *const *const names = kNames[hd == 128][fp8];
    // few own keys beside the shared ones of the second kernel, in its launch: 64
    // rows of up to 300 own keys over 16384 shared 51.8 us, in two launches 58.3
    const uint64_t many = !p.many ? 0u : a.cap1 <= 512u ? shared + own : shared;
    if (many) {
        if (int rc = launch(names[1], dim3((unsigned)many), dim3(512), s, &a)) return rc;
    }
    a.first = (uint32_t)(many / a.n_kv_heads);
    if (const uint64_t items = shared + own - many) {
        if (int rc = launch(names[0], dim3((unsigned)items), dim3(256), s, &a)) return rc;
    }
    if (p.splits() == 1) return RFP4_OK;
    // the splits' states, or the zeros of rows that have no keys at all
    return launch(hd == 64 ? "rfp4_attn_rows_merge_hd64" : "rfp4_attn_rows_merge_hd128", dim3((unsigned)merges), dim3(256), s, &a);
}

int append_rows(const char *what, bool fp8, hipStream_t s, uint32_t rows, uint32_t nkv, uint32_t hd, uint32_t pos0, const uint32_t *positions,
                const float *k, uint32_t k_rs, const float *v, uint32_t v_rs, void *kc, uint8_t *ks, void *vc, uint8_t *vs, uint64_t ss,
                uint64_t ts, uint64_t hs, uint32_t capacity)
{
    if (hd != 64 && hd != 128) return set_error(RFP4_E_SHAPE, "%s: head_dim %u unsupported (64 or 128)", what, hd);
    if (nkv == 0) return set_error(RFP4_E_SHAPE, "%s: n_kv_heads must be > 0", what);
    if (rows == 0) return RFP4_OK;
    if (!k || !v) return set_error(RFP4_E_INVALID, "%s: null pointer", what);
    const Cache c{kc, vc, ks, vs, ts, hs, positions ? ss : 0};
    if (int rc = check_cache(what, c, fp8, hd)) return rc;
    if (!aligned(k, 16) || !aligned(v, 16) || k_rs % 4u || v_rs % 4u)
        return set_error(RFP4_E_ALIGN, "%s: k and v rows must start 16-byte aligned", what);
    if ((uint64_t)nkv * hd > UINT32_MAX || (rows > 1 && (k_rs < nkv * hd || v_rs < nkv * hd)))
        return set_error(RFP4_E_SHAPE, "%s: row strides %u, %u < %u heads x %u", what, k_rs, v_rs, nkv, hd);
    if (!positions && (uint64_t)pos0 + rows > capacity)
        return set_error(RFP4_E_KV_OVERFLOW, "%s: positions %u .. %llu of a cache of %u", what, pos0, (unsigned long long)pos0 + rows - 1, capacity);
    // no two rows may share memory: by stride, each dimension spans what the smaller ones cover
    struct { uint64_t n, stride; } dim[3] = {{capacity, ts}, {nkv, hs}, {positions ? rows : 1u, ss}};
    std::sort(dim, dim + 3, [](const auto &x, const auto &y) { return x.stride < y.stride; });
    unsigned __int128 span = hd;
    for (const auto &d : dim) {
        if (d.n <= 1) continue;
        if (d.stride < span) return set_error(RFP4_E_SHAPE, "%s: strides (%llu, %llu, %llu) make cache rows overlap", what, (unsigned long long)ss,
                                              (unsigned long long)ts, (unsigned long long)hs);
        span += (unsigned __int128)d.stride * (d.n - 1);
    }
    const uint64_t units = (uint64_t)rows * 2u * nkv, per = 256u / (hd / 8u);
    if (units > ((uint64_t)1 << 27)) return set_error(RFP4_E_CAPACITY, "%s: %u rows of %u heads in one call", what, rows, nkv);
    KvRowsArgs a{k, v, kc, vc, ks, vs, positions, positions ? ss : 0, ts, hs, k_rs, v_rs, rows, nkv, pos0, capacity};
    static const char *const kNames[2][2] = {{"rfp4_kv_rows_hd64_f16", "rfp4_kv_rows_hd64_fp8"}, {"rfp4_kv_rows_hd128_f16", "rfp4_kv_rows_hd128_fp8"}};
    return launch(kNames[hd == 128][fp8], dim3((unsigned)((units + per - 1) / per)), dim3(256), s, &a);
}

int causal(const char *what, hipStream_t s, uint32_t nh, uint32_t nkv, uint32_t hd, uint32_t pos0, uint32_t rows, const float *q, uint32_t q_rs,
           const Cache &c, void *workspace, size_t workspace_bytes, float *out, uint32_t out_rs)
{
    if (int rc = check_heads(what, nh, nkv, hd)) return rc;
    if (rows == 0) return RFP4_OK;
    if (int rc = check_rows(what, q, q_rs, out, out_rs, rows, nh, hd)) return rc;
    if (int rc = check_cache(what, c, true, hd)) return rc;
    const uint64_t keys = (uint64_t)pos0 + rows;
    if (keys > kMaxKeys || (uint64_t)rows * nh > kMaxKeys) return set_error(RFP4_E_SHAPE, "%s: %llu keys, %u rows", what, (unsigned long long)keys, rows);
    AttnRowsArgs a{};
    a.q = q; a.out = out;
    a.k0 = c.k; a.v0 = c.v; a.ks0 = c.ks; a.vs0 = c.vs;
    a.ts0 = c.ts; a.hs0 = c.hs;
    a.q_rs = q_rs; a.out_rs = out_rs;
    a.n_heads = nh; a.n_kv_heads = nkv;
    a.rows = rows; a.causal = 1; a.pos0 = pos0; a.len0 = (uint32_t)keys;
    return run(what, plan(true, true, nkv, nh / nkv, hd, rows, keys, 0), a, true, hd, workspace, workspace_bytes, s);
}

int prefix_rows(const char *what, bool fp8, hipStream_t s, uint32_t batch, uint32_t nh, uint32_t nkv, uint32_t hd, const float *q, uint32_t q_rs,
                uint32_t prefix, const Cache &p, uint32_t max_suffix, const uint32_t *lens, const Cache &own, void *workspace,
                size_t workspace_bytes, float *out, uint32_t out_rs)
{
    if (int rc = check_heads(what, nh, nkv, hd)) return rc;
    if (batch == 0) return RFP4_OK;
    if (int rc = check_rows(what, q, q_rs, out, out_rs, batch, nh, hd)) return rc;
    if (prefix)
        if (int rc = check_cache(what, p, fp8, hd)) return rc;
    if (max_suffix) {
        if (!lens) return set_error(RFP4_E_INVALID, "%s: null suffix lengths", what);
        if (int rc = check_cache(what, own, fp8, hd)) return rc;
    }
    if (prefix > kMaxKeys || max_suffix > kMaxKeys || (uint64_t)batch * nh > kMaxKeys)
        return set_error(RFP4_E_SHAPE, "%s: prefix %u, suffix %u, batch %u", what, prefix, max_suffix, batch);
    AttnRowsArgs a{};
    a.q = q; a.out = out;
    a.k0 = p.k; a.v0 = p.v; a.ks0 = p.ks; a.vs0 = p.vs;
    a.ts0 = p.ts; a.hs0 = p.hs;
    a.k1 = own.k; a.v1 = own.v; a.ks1 = own.ks; a.vs1 = own.vs;
    a.ts1 = own.ts; a.hs1 = own.hs; a.ss1 = own.ss;
    a.lens = lens;
    a.q_rs = q_rs; a.out_rs = out_rs;
    a.n_heads = nh; a.n_kv_heads = nkv;
    a.rows = batch; a.len0 = prefix; a.cap1 = max_suffix;
    return run(what, plan(false, fp8, nkv, nh / nkv, hd, batch, prefix, max_suffix), a, fp8, hd, workspace, workspace_bytes, s);
}

} // namespace

extern "C" {

int rfp4_debug_attn_rows(int mode)
{
    if (mode < 0 || mode > 2) return set_error(RFP4_E_INVALID, "attention of rows: mode %d (0, 1 or 2)", mode);
    t_mode = mode;
    return RFP4_OK;
}

int kv_append_rows_f16(rfp4_stream_t stream, uint32_t rows, uint32_t n_kv_heads, uint32_t head_dim, uint32_t pos0, const uint32_t *positions,
                       const float *k, uint32_t k_row_stride, const float *v, uint32_t v_row_stride, uint16_t *kc, uint16_t *vc,
                       uint64_t seq_stride, uint64_t token_stride, uint64_t head_stride, uint32_t capacity)
{
    return append_rows("kv_append_rows_f16", false, (hipStream_t)stream, rows, n_kv_heads, head_dim, pos0, positions, k, k_row_stride, v,
                       v_row_stride, kc, nullptr, vc, nullptr, seq_stride, token_stride, head_stride, capacity);
}

int kv_append_rows_fp8(rfp4_stream_t stream, uint32_t rows, uint32_t n_kv_heads, uint32_t head_dim, uint32_t pos0, const uint32_t *positions,
                       const float *k, uint32_t k_row_stride, const float *v, uint32_t v_row_stride, uint8_t *kc, uint8_t *k_scales, uint8_t *vc,
                       uint8_t *v_scales, uint64_t seq_stride, uint64_t token_stride, uint64_t head_stride, uint32_t capacity)
{
    return append_rows("kv_append_rows_fp8", true, (hipStream_t)stream, rows, n_kv_heads, head_dim, pos0, positions, k, k_row_stride, v,
                       v_row_stride, kc, k_scales, vc, v_scales, seq_stride, token_stride, head_stride, capacity);
}

size_t attn_prefill_fp8_workspace(uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim, uint32_t pos0, uint32_t rows)
{
    if (check_heads("attn_prefill_fp8_workspace", n_heads, n_kv_heads, head_dim) || rows == 0) return 0;
    return workspace_bytes_of(n_kv_heads, n_heads, head_dim, rows, (uint64_t)pos0 + rows, 0);
}

size_t attn_decode_fp8_workspace(uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim, uint32_t seq)
{
    return seq ? attn_prefill_fp8_workspace(n_heads, n_kv_heads, head_dim, seq - 1u, 1) : 0;
}

size_t attn_decode_prefix_workspace(uint32_t batch, uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim, uint32_t prefix, uint32_t max_suffix)
{
    if (check_heads("attn_decode_prefix_workspace", n_heads, n_kv_heads, head_dim) || batch == 0) return 0;
    return workspace_bytes_of(n_kv_heads, n_heads, head_dim, batch, prefix, max_suffix);
}

int attn_decode_fp8(rfp4_stream_t stream, uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim, uint32_t seq, const float *q,
                    const uint8_t *kc, const uint8_t *k_scales, const uint8_t *vc, const uint8_t *v_scales, uint64_t token_stride,
                    uint64_t head_stride, void *workspace, size_t workspace_bytes, float *out)
{
    if (seq == 0) return set_error(RFP4_E_SHAPE, "attn_decode_fp8: seq must be >= 1");
    return causal("attn_decode_fp8", (hipStream_t)stream, n_heads, n_kv_heads, head_dim, seq - 1u, 1, q, 0,
                  Cache{kc, vc, k_scales, v_scales, token_stride, head_stride, 0}, workspace, workspace_bytes, out, 0);
}

int attn_prefill_fp8(rfp4_stream_t stream, uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim, uint32_t pos0, uint32_t rows, const float *q,
                     uint32_t q_row_stride, const uint8_t *kc, const uint8_t *k_scales, const uint8_t *vc, const uint8_t *v_scales,
                     uint64_t token_stride, uint64_t head_stride, void *workspace, size_t workspace_bytes, float *out, uint32_t out_row_stride)
{
    return causal("attn_prefill_fp8", (hipStream_t)stream, n_heads, n_kv_heads, head_dim, pos0, rows, q, q_row_stride,
                  Cache{kc, vc, k_scales, v_scales, token_stride, head_stride, 0}, workspace, workspace_bytes, out, out_row_stride);
}

int attn_decode_prefix_f16(rfp4_stream_t stream, uint32_t batch, uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim, const float *q,
                           uint32_t q_row_stride, uint32_t prefix, const uint16_t *pk, const uint16_t *pv, uint64_t p_token_stride,
                           uint64_t p_head_stride, uint32_t max_suffix, const uint32_t *suffix_lens, const uint16_t *sk, const uint16_t *sv,
                           uint64_t s_seq_stride, uint64_t s_token_stride, uint64_t s_head_stride, void *workspace, size_t workspace_bytes,
                           float *out, uint32_t out_row_stride)
{
    return prefix_rows("attn_decode_prefix_f16", false, (hipStream_t)stream, batch, n_heads, n_kv_heads, head_dim, q, q_row_stride, prefix,
                       Cache{pk, pv, nullptr, nullptr, p_token_stride, p_head_stride, 0}, max_suffix, suffix_lens,
                       Cache{sk, sv, nullptr, nullptr, s_token_stride, s_head_stride, s_seq_stride}, workspace, workspace_bytes, out, out_row_stride);
}

int attn_decode_prefix_fp8(rfp4_stream_t stream, uint32_t batch, uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim, const float *q,
                           uint32_t q_row_stride, uint32_t prefix, const uint8_t *pk, const uint8_t *pk_scales, const uint8_t *pv,
                           const uint8_t *pv_scales, uint64_t p_token_stride, uint64_t p_head_stride, uint32_t max_suffix,
                           const uint32_t *suffix_lens, const uint8_t *sk, const uint8_t *sk_scales, const uint8_t *sv, const uint8_t *sv_scales,
                           uint64_t s_seq_stride, uint64_t s_token_stride, uint64_t s_head_stride, void *workspace, size_t workspace_bytes,
                           float *out, uint32_t out_row_stride)
{
    return prefix_rows("attn_decode_prefix_fp8", true, (hipStream_t)stream, batch, n_heads, n_kv_heads, head_dim, q, q_row_stride, prefix,
                       Cache{pk, pv, pk_scales, pv_scales, p_token_stride, p_head_stride, 0}, max_suffix, suffix_lens,
                       Cache{sk, sv, sk_scales, sv_scales, s_token_stride, s_head_stride, s_seq_stride}, workspace, workspace_bytes, out,
                       out_row_stride);
}

} // extern "C"
