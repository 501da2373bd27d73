"""kv_append_rows_*, attn_decode_fp8, attn_prefill_fp8 and attn_decode_prefix_*
on the device against float64 (kv8.py: the definitions, and the bound of an
output with its derivation)."""
import ctypes as C

import numpy as np
import pytest

import kv8
from test_gpu_kernels import _dev

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[1, 2], ids=["few", "many"])
def kernel(rf, request):
    """Both kernels of the attention calls at every size (the planner gives the second large ones only)."""
    rf.check(rf.load().rfp4_debug_attn_rows(request.param))
    yield request.param
    rf.check(rf.load().rfp4_debug_attn_rows(0))


HEAD, TOKEN = "head", "token"


def strides(layout, nkv, cap, hd):
    return (hd, cap * hd) if layout == HEAD else (nkv * hd, hd)


def lay(x, layout):
    """[..., token, head, dim] as the layout stores it."""
    return np.ascontiguousarray(np.swapaxes(x, -3, -2) if layout == HEAD else x)


class Cache:
    """`cap` tokens of which the first `keys` (per sequence of `lead`) hold values, the others garbage that reads as NaN."""

    def __init__(self, rf, stream, rng, layout, nkv, keys, cap, hd, fp8, lead=(), kscale=1.0, vscale=0.4):
        self.layout, self.fp8 = layout, fp8
        self.ts, self.hs = strides(layout, nkv, cap, hd)
        self.ss = nkv * cap * hd
        self.val, self.dev = [], []
        for sc in (kscale, vscale):
            x = (sc * rng.standard_normal((*lead, cap, nkv, hd))).astype(np.float32)
            if fp8:
                c, s = kv8.encode(x)
                c[..., keys:, :, :], s[..., keys:, :] = 127, 255
                self.val.append(kv8.decode(c, s))
                self.dev += [_dev(rf, lay(c, layout), stream), _dev(rf, np.ascontiguousarray(np.swapaxes(s, -2, -1)) if layout == HEAD else s, stream)]
            else:
                x = x.astype(np.float16)
                x[..., keys:, :, :] = np.nan
                self.val.append(x.astype(np.float64))
                self.dev.append(_dev(rf, lay(x, layout).view(np.uint16), stream))


def work(rf, stream, size):
    """A workspace of exactly the size asked for, full of NaNs; guarded by 64 words that must stay."""
    host = np.full(size // 4 + 64, np.nan, np.float32)
    return _dev(rf, host, stream)


def guard(buf, size, stream):
    assert np.isnan(buf.to_host(size // 4 + 64, np.float32, stream)[size // 4:]).all()


def check(got, want, A, keys, vmax):
    assert np.isfinite(got).all()
    err, tol = np.abs(got - want).max(), kv8.bound(A, keys, vmax)
    assert err <= tol, f"error {err:.3g}, bound {tol:.3g}"


# ------------------------------------------------------------------ the cache's rows
def special_rows(rng, n, hd):
    """Rows of every magnitude, ties of the format, zeros, subnormals, huge values, infinities and NaNs."""
    x = rng.standard_normal((n, hd)).astype(np.float32)
    x *= (2.0 ** rng.integers(-30, 30, (n, 1))).astype(np.float32)
    mid = ((kv8.LEVELS[1:] + kv8.LEVELS[:-1]) / 2).astype(np.float32)
    for i in range(0, n, 3):  # values at and next to the borders between two codes, under a power of two
        t = rng.choice(mid, hd) * rng.choice([-1, 1], hd)
        t[0] = 448
        x[i] = np.nextafter(t, rng.choice([-np.inf, 0, np.inf], hd).astype(np.float32) * t + t, dtype=np.float32) * np.float32(2.0 ** rng.integers(-40, 40))
    special = [np.zeros(hd), np.full(hd, 2.0 ** -149), np.full(hd, 2.0 ** -120), np.full(hd, 3.4e38), np.full(hd, 448.0), np.full(hd, 448.0001),
               np.full(hd, -0.0)]
    for j, s in enumerate(special):
        x[(5 * j + 1) % n] = s
    if n > 40:
        x[37, 3], x[38, hd - 1], x[39, 0] = np.inf, np.nan, -np.inf
    return x


@pytest.mark.parametrize("layout", [HEAD, TOKEN])
@pytest.mark.parametrize("rows,nkv,hd,pos0,cap", [(1, 1, 64, 0, 1), (1, 8, 128, 5, 9), (33, 3, 64, 7, 41), (130, 2, 128, 0, 131), (257, 1, 128, 3, 260)])
def test_append_fp8(rf, stream, layout, rows, nkv, hd, pos0, cap):
    rng = np.random.default_rng(rows * hd + nkv)
    rs = nkv * hd + 8  # rows of a wider buffer
    src = [np.full((rows, rs), 7, np.float32) for _ in range(2)]
    x = [special_rows(rng, rows * nkv, hd).reshape(rows, nkv, hd) for _ in range(2)]
    for s, v in zip(src, x):
        s[:, :nkv * hd] = v.reshape(rows, -1)
    codes = [np.full((cap, nkv, hd), 0xA5, np.uint8) for _ in range(2)]
    scales = [np.full((cap, nkv), 0x5A, np.uint8) for _ in range(2)]
    dev = [_dev(rf, a, stream) for a in codes + scales]
    ts, hs = strides(layout, nkv, cap, hd)
    rf.kv_append_rows_fp8(stream, rows, nkv, hd, pos0, None, _dev(rf, src[0], stream), rs, _dev(rf, src[1], stream), rs, dev[0], dev[2],
                          dev[1], dev[3], 0, ts, hs, cap)
    for i in range(2):
        codes[i][pos0:pos0 + rows], scales[i][pos0:pos0 + rows] = kv8.encode(x[i])
        got = dev[i].to_host(cap * nkv * hd, np.uint8, stream)
        np.testing.assert_array_equal(got, lay(codes[i], layout).reshape(-1))
        got = dev[2 + i].to_host(cap * nkv, np.uint8, stream)
        np.testing.assert_array_equal(got, (scales[i].T if layout == HEAD else scales[i]).reshape(-1))


@pytest.mark.parametrize("layout", [HEAD, TOKEN])
@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("batch,nkv,hd,cap", [(1, 1, 64, 1), (5, 2, 128, 4), (48, 4, 64, 17)])
def test_append_batch(rf, stream, layout, fp8, batch, nkv, hd, cap):
    """Row b at positions[b] of sequence b; positions at and past the capacity are padding."""
    rng = np.random.default_rng(batch)
    pos = rng.integers(0, cap, batch).astype(np.uint32)
    pos[1::4] = rng.choice([cap, cap + 1, 0xFFFFFFFF], len(pos[1::4]))
    x = [rng.standard_normal((batch, nkv, hd)).astype(np.float32) for _ in range(2)]
    want = [np.full((batch, cap, nkv, hd), 0x21 if fp8 else 0x2121, np.uint8 if fp8 else np.uint16) for _ in range(2)]
    scales = [np.full((batch, cap, nkv), 0x5A, np.uint8) for _ in range(2)]
    dev, sdev = [_dev(rf, w, stream) for w in want], [_dev(rf, s, stream) for s in scales]
    ts, hs = strides(layout, nkv, cap, hd)
    dpos, dk, dv = _dev(rf, pos, stream), _dev(rf, x[0], stream), _dev(rf, x[1], stream)
    args = (stream, batch, nkv, hd, 0, dpos, dk, nkv * hd, dv, nkv * hd)
    if fp8:
        rf.kv_append_rows_fp8(*args, dev[0], sdev[0], dev[1], sdev[1], nkv * cap * hd, ts, hs, cap)
    else:
        rf.kv_append_rows_f16(*args, dev[0], dev[1], nkv * cap * hd, ts, hs, cap)
    for i in range(2):
        c, s = kv8.encode(x[i]) if fp8 else (x[i].astype(np.float16).view(np.uint16), None)
        for b in range(batch):
            if pos[b] < cap:
                want[i][b, pos[b]] = c[b]
                if fp8:
                    scales[i][b, pos[b]] = s[b]
        np.testing.assert_array_equal(dev[i].to_host(want[i].size, want[i].dtype, stream), lay(want[i], layout).reshape(-1))
        got = sdev[i].to_host(scales[i].size, np.uint8, stream)
        np.testing.assert_array_equal(got, (np.swapaxes(scales[i], -2, -1) if layout == HEAD else scales[i]).reshape(-1))


@pytest.mark.parametrize("layout", [HEAD, TOKEN])
def test_append_f16_rows(rf, stream, layout):
    rng = np.random.default_rng(3)
    rows, nkv, hd, pos0, cap = 19, 3, 128, 2, 30
    x = [(rng.standard_normal((rows, nkv, hd)) * 10.0 ** rng.integers(-8, 6, (rows, nkv, 1))).astype(np.float32) for _ in range(2)]
    want = [np.full((cap, nkv, hd), 0x2121, np.uint16) for _ in range(2)]
    dev = [_dev(rf, w, stream) for w in want]
    rf.kv_append_rows_f16(stream, rows, nkv, hd, pos0, None, _dev(rf, x[0], stream), nkv * hd, _dev(rf, x[1], stream), nkv * hd, dev[0], dev[1],
                          0, *strides(layout, nkv, cap, hd), cap)
    for i in range(2):
        with np.errstate(over="ignore"):
            want[i][pos0:pos0 + rows] = x[i].astype(np.float16).view(np.uint16)
        np.testing.assert_array_equal(dev[i].to_host(want[i].size, np.uint16, stream), lay(want[i], layout).reshape(-1))


# ------------------------------------------------------------------ one query row
def run_decode(rf, stream, c, q, nh, nkv, hd, seq):
    size = rf.attn_decode_fp8_workspace(nh, nkv, hd, seq)
    ws = work(rf, stream, size)
    out = _dev(rf, np.full(nh * hd + 16, 5, np.float32), stream)
    rf.attn_decode_fp8(stream, nh, nkv, hd, seq, _dev(rf, q, stream), *c.dev, c.ts, c.hs, ws, size, out)
    got = out.to_host(nh * hd + 16, np.float32, stream)
    assert (got[nh * hd:] == 5).all()
    guard(ws, size, stream)
    return got[:nh * hd].reshape(nh, hd)


def decode_want(c, q, group, keys):
    """Each query head over its KV head's first `keys` tokens, the largest A, and |v|'s largest."""
    res = [attend_head(c, q[h], h // group, keys) for h in range(len(q))]
    return np.stack([r[0] for r in res]), max(r[1] for r in res), np.abs(c.val[1][..., :keys, :, :]).max()


def attend_head(c, q, kvh, keys):
    o, A = kv8.attend(q[None], c.val[0][:keys, kvh], c.val[1][:keys, kvh])
    return o[0], A


@pytest.mark.parametrize("seq", [1, 2, 31, 32, 33, 96, 127, 128, 129, 255, 256, 257, 511, 513, 1000, 4097, 20000])
@pytest.mark.parametrize("nh,nkv,hd,layout", [(8, 2, 128, HEAD), (8, 1, 64, TOKEN), (3, 3, 128, TOKEN), (10, 2, 64, HEAD), (32, 8, 128, HEAD)])
def test_decode_fp8(rf, stream, kernel, nh, nkv, hd, layout, seq):
    if seq > 5000 and nh > 8:
        seq = 5003
    rng = np.random.default_rng(seq + nh)
    c = Cache(rf, stream, rng, layout, nkv, seq, seq + 37, hd, True)
    q = rng.standard_normal((nh, hd)).astype(np.float32)
    want, A, vmax = decode_want(c, q, nh // nkv, seq)
    check(run_decode(rf, stream, c, q, nh, nkv, hd, seq), want, A, seq, vmax)


@pytest.mark.parametrize("mag", [1e-30, 1e-12, 1e-4, 1e3, 1e15, 1e30])
@pytest.mark.parametrize("hd", [64, 128])
def test_decode_fp8_magnitudes(rf, stream, kernel, hd, mag):
    """q and K of any size whose products are ordinary scores, and tiny q over a cache with rows of zeros."""
    nh, nkv, seq = 4, 2, 301
    rng = np.random.default_rng(hd)
    c = Cache(rf, stream, rng, HEAD, nkv, seq, seq + 3, hd, True, kscale=1 / mag, vscale=mag)
    q = (mag * rng.standard_normal((nh, hd))).astype(np.float32)
    want, A, vmax = decode_want(c, q, 2, seq)
    got = run_decode(rf, stream, c, q, nh, nkv, hd, seq)
    check(got, want, A, seq, vmax)
    z = Cache(rf, stream, rng, HEAD, nkv, seq, seq + 3, hd, True, kscale=0.0)
    want, A, vmax = decode_want(z, q * np.float32(1e-8 if mag < 1 else 1), 2, seq)
    check(run_decode(rf, stream, z, q * np.float32(1e-8 if mag < 1 else 1), nh, nkv, hd, seq), want, A, seq, vmax)


def test_decode_fp8_scales_far_apart(rf, stream, kernel):
    """Rows whose scales spread over 2^-20 .. 2^20 in any order: rows far below
    the largest still count where the large ones get no weight.  A K row is off
    by at most 2^-41 of the largest K (2^-34 of the reference's scale), a V row
    likewise, which the bound below adds."""
    nh, nkv, hd, seq = 4, 1, 128, 700
    rng = np.random.default_rng(11)
    c = Cache(rf, stream, rng, HEAD, nkv, seq, seq, hd, True)
    codes, ks = (c.dev[i].to_host(None, np.uint8, stream) for i in (0, 1))
    vs = c.dev[3].to_host(None, np.uint8, stream)
    step = rng.integers(-20, 1, seq)
    ks2 = (ks.astype(int) + step).astype(np.uint8)
    vs2 = (vs.astype(int) + rng.integers(-20, 21, seq)).astype(np.uint8)
    c.dev[1], c.dev[3] = _dev(rf, ks2, stream), _dev(rf, vs2, stream)
    c.val[0] = kv8.decode(codes.reshape(seq, 1, hd), ks2.reshape(seq, 1))
    c.val[1] = kv8.decode(c.dev[2].to_host(None, np.uint8, stream).reshape(seq, 1, hd), vs2.reshape(seq, 1))
    q = rng.standard_normal((nh, hd)).astype(np.float32)
    want, A, vmax = decode_want(c, q, nh, seq)
    check(run_decode(rf, stream, c, q, nh, nkv, hd, seq), want, A, seq, vmax)


@pytest.mark.parametrize("hd", [64, 128])
def test_q_next_to_a_tie_of_its_first_term(rf, stream, kernel, hd):
    """q whose product with the softmax factor rounds to another fp16 value
    than the product rounded to f32 does: its two terms must belong together.
    K is a multiple of the identity, so each score shows one element of q, and
    one step of its first term off (2^-11) is 60 times the bound and more."""
    rng = np.random.default_rng(hd)
    f = np.float64(np.float32(4) * (np.float32(1.4426950408889634) * (np.float32(1) / np.sqrt(np.float32(hd)))))
    x = rng.uniform(1, 2, 8000000).astype(np.float32)
    x = x[(x * f).astype(np.float16) != (x * f).astype(np.float32).astype(np.float16)]
    batch = min(len(x), 32) // 2
    assert batch >= 8
    q = np.stack([np.roll(np.resize(x, hd), b) for b in range(2 * batch)]).reshape(batch, 2, hd).astype(np.float32)
    c = Cache(rf, stream, rng, HEAD, 1, hd, hd, hd, True)
    k, ks = kv8.encode(32 * np.eye(hd, dtype=np.float32)[:, None])
    c.val[0] = kv8.decode(k, ks)
    c.dev[:2] = [_dev(rf, lay(k, HEAD), stream), _dev(rf, ks.T, stream)]
    want, A, vmax = prefix_want(c, None, q, 1, hd, None)
    check(run_prefix(rf, stream, c, None, q, 2, 1, hd, hd, 0, None), want, A, hd, vmax)


# ------------------------------------------------------------------ causal rows
def run_prefill(rf, stream, c, q, nh, nkv, hd, pos0, rows):
    rs = nh * hd + 4
    qb = np.zeros((rows, rs), np.float32)
    qb[:, :nh * hd] = q.reshape(rows, -1)
    size = rf.attn_prefill_fp8_workspace(nh, nkv, hd, pos0, rows)
    ws = work(rf, stream, size)
    out = _dev(rf, np.full((rows + 1, rs), 5, np.float32), stream)
    rf.attn_prefill_fp8(stream, nh, nkv, hd, pos0, rows, _dev(rf, qb, stream), rs, *c.dev, c.ts, c.hs, ws, size, out, rs)
    got = out.to_host((rows + 1) * rs, np.float32, stream).reshape(rows + 1, rs)
    assert (got[rows] == 5).all() and (got[:, nh * hd:] == 5).all()
    guard(ws, size, stream)
    return got[:rows, :nh * hd].reshape(rows, nh, hd)


def prefill_want(c, q, group, pos0):
    rows, nh, hd = q.shape
    want, A = np.zeros(q.shape), 0.0
    for h in range(nh):
        k, v = c.val[0][:, h // group], c.val[1][:, h // group]
        s = q[:, h].astype(np.float64) @ k[:pos0 + rows].T / np.sqrt(hd)
        A = max(A, float((np.abs(q[:, h]) @ np.abs(k[:pos0 + rows]).T / np.sqrt(hd)).max()))
        s[np.arange(pos0 + rows)[None] > pos0 + np.arange(rows)[:, None]] = -np.inf
        p = np.exp(s - s.max(-1, keepdims=True))
        want[:, h] = p @ v[:pos0 + rows] / p.sum(-1, keepdims=True)
    return want, A, np.abs(c.val[1][:pos0 + rows]).max()


@pytest.mark.parametrize("pos0,rows", [(0, 1), (0, 2), (0, 16), (0, 17), (0, 33), (0, 130), (31, 1), (33, 5), (95, 33), (250, 70), (4000, 3), (3001, 64), (0, 515)])
@pytest.mark.parametrize("nh,nkv,hd,layout", [(8, 2, 128, HEAD), (8, 1, 64, TOKEN), (3, 3, 64, HEAD), (6, 2, 128, TOKEN), (7, 1, 128, HEAD)])
def test_prefill_fp8(rf, stream, kernel, nh, nkv, hd, layout, pos0, rows):
    rng = np.random.default_rng(pos0 * 31 + rows + nh)
    c = Cache(rf, stream, rng, layout, nkv, pos0 + rows, pos0 + rows + 37, hd, True)
    q = rng.standard_normal((rows, nh, hd)).astype(np.float32)
    want, A, vmax = prefill_want(c, q, nh // nkv, pos0)
    check(run_prefill(rf, stream, c, q, nh, nkv, hd, pos0, rows), want, A, pos0 + rows, vmax)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("which", [1, 3])
def test_prefill_fp8_nan_rows(rf, stream, kernel, hd, which):
    """A K or V row with scale byte 255 at position t: every row from t on is NaN, the rows before it are as if it were not there."""
    nh, nkv, pos0, rows, t = 4, 1, 20, 100, 77
    rng = np.random.default_rng(hd + which)
    c = Cache(rf, stream, rng, HEAD, nkv, pos0 + rows, pos0 + rows, hd, True)
    q = rng.standard_normal((rows, nh, hd)).astype(np.float32)
    want, A, vmax = prefill_want(c, q, nh, pos0)
    sc = c.dev[which].to_host(None, np.uint8, stream)
    sc[t] = 255
    c.dev[which] = _dev(rf, sc, stream)
    got = run_prefill(rf, stream, c, q, nh, nkv, hd, pos0, rows)
    check(got[:t - pos0], want[:t - pos0], A, pos0 + rows, vmax)
    assert np.isnan(got[t - pos0:]).all()


def test_prefill_fp8_growing_scores(rf, stream, kernel):
    """Scores tens apart, so that most blocks raise a row's maximum."""
    nh, nkv, hd, pos0, rows = 4, 1, 128, 40, 150
    rng = np.random.default_rng(5)
    c = Cache(rf, stream, rng, HEAD, nkv, pos0 + rows, pos0 + rows, hd, True, kscale=4.0)
    q = (12 * rng.standard_normal((rows, nh, hd))).astype(np.float32)
    want, A, vmax = prefill_want(c, q, nh, pos0)
    check(run_prefill(rf, stream, c, q, nh, nkv, hd, pos0, rows), want, A, pos0 + rows, vmax)


@pytest.mark.parametrize("rows", [1, 40])
def test_offsets_past_32_bits(rf, stream, kernel, rows):
    """A token stride of 2^24 elements and more: the last of 301 tokens lies past 5 GB."""
    nh, nkv, hd, seq, ts = 4, 2, 64, 301, (1 << 24) + 64
    rng = np.random.default_rng(rows)
    x = [rng.standard_normal((seq, nkv, hd)).astype(np.float32) for _ in range(2)]
    q = rng.standard_normal((rows, nh, hd)).astype(np.float32)
    n = (seq - 1) * ts + nkv * hd
    c = Cache(rf, stream, rng, TOKEN, nkv, 1, 1, hd, True)
    c.dev, c.ts, c.hs = [rf.DeviceBuffer(n), rf.DeviceBuffer(n // hd), rf.DeviceBuffer(n), rf.DeviceBuffer(n // hd)], ts, hd
    rf.kv_append_rows_fp8(stream, seq, nkv, hd, 0, None, _dev(rf, x[0], stream), nkv * hd, _dev(rf, x[1], stream), nkv * hd, *c.dev, 0, ts, hd, seq)
    c.val = [kv8.decode(*kv8.encode(t)) for t in x]
    want, A, vmax = prefill_want(c, q, 2, seq - rows)
    got = run_prefill(rf, stream, c, q, nh, nkv, hd, seq - rows, rows)
    for b in c.dev:
        b.free()
    check(got, want, A, seq, vmax)


# ------------------------------------------------------------------ a batch with a shared prefix
def run_prefix(rf, stream, p, s, q, nh, nkv, hd, prefix, cap, lens, ws=None):
    batch, rs = len(q), nh * hd + 4
    qb = np.zeros((batch, rs), np.float32)
    qb[:, :nh * hd] = q.reshape(batch, -1)
    size = rf.attn_decode_prefix_workspace(batch, nh, nkv, hd, prefix, cap)
    ws = work(rf, stream, size)
    out = _dev(rf, np.full((batch + 1, rs), 5, np.float32), stream)
    call = rf.attn_decode_prefix_fp8 if (p or s).fp8 else rf.attn_decode_prefix_f16
    none = [None] * (4 if (p or s).fp8 else 2)
    call(stream, batch, nh, nkv, hd, _dev(rf, qb, stream), rs, prefix, *(p.dev if p else none), p.ts if p else 0, p.hs if p else 0, cap,
         _dev(rf, lens, stream) if s else None, *(s.dev if s else none), s.ss if s else 0, s.ts if s else 0, s.hs if s else 0, ws, size, out, rs)
    got = out.to_host((batch + 1) * rs, np.float32, stream).reshape(batch + 1, rs)
    assert (got[batch] == 5).all() and (got[:, nh * hd:] == 5).all()
    guard(ws, size, stream)
    return got[:batch, :nh * hd].reshape(batch, nh, hd)


def prefix_want(p, s, q, nkv, prefix, lens):
    batch, nh, hd = q.shape
    want, A, vmax = np.zeros(q.shape), 0.0, 0.0
    for b in range(batch):
        for h in range(nh):
            parts = [[c[:prefix, h * nkv // nh] for c in p.val]] if p else []
            parts += [[c[b, :lens[b], h * nkv // nh] for c in s.val]] if s else []
            k, v = (np.concatenate([x[i] for x in parts]) for i in range(2))
            want[b, h:h + 1], a = kv8.attend(q[b, h:h + 1], k, v)
            A, vmax = max(A, a), max(vmax, np.abs(v).max() if len(v) else 0.0)
    return want, A, vmax


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("batch,prefix,cap", [(1, 0, 1), (1, 1, 0), (1, 300, 5), (2, 0, 40), (3, 33, 0), (3, 517, 33), (5, 1000, 130), (9, 64, 700), (17, 257, 1), (40, 129, 9)])
@pytest.mark.parametrize("nh,nkv,hd,layout", [(8, 2, 128, HEAD), (8, 1, 64, TOKEN), (3, 3, 64, HEAD), (10, 2, 128, TOKEN)])
def test_prefix(rf, stream, kernel, fp8, nh, nkv, hd, layout, batch, prefix, cap):
    rng = np.random.default_rng(batch * 7 + prefix + cap + nh)
    p = Cache(rf, stream, rng, layout, nkv, prefix, prefix + 3, hd, fp8) if prefix else None
    s = Cache(rf, stream, rng, layout, nkv, cap, cap, hd, fp8, lead=(batch,)) if cap else None
    lens = rng.integers(0, cap + 1, batch).astype(np.uint32)
    if cap:
        lens[-1] = cap
        if batch > 2:
            lens[0], lens[1] = 0, min(cap, 1)
    q = rng.standard_normal((batch, nh, hd)).astype(np.float32)
    want, A, vmax = prefix_want(p, s, q, nkv, prefix, lens)
    check(run_prefix(rf, stream, p, s, q, nh, nkv, hd, prefix, cap, lens), want, A, prefix + cap, vmax)


@pytest.mark.parametrize("fp8", [True, False])
def test_prefix_empty_rows_and_long_lengths(rf, stream, kernel, fp8):
    """Rows without any token are 0; a length past max_suffix counts as max_suffix; what lies behind a row's last token is not read as a value."""
    nh, nkv, hd, cap = 4, 2, 64, 300
    rng = np.random.default_rng(1)
    s = Cache(rf, stream, rng, TOKEN, nkv, 290, cap, hd, fp8, lead=(6,))
    lens = np.array([0, 290, 1, 0, 289, 32], np.uint32)
    q = rng.standard_normal((6, nh, hd)).astype(np.float32)
    want, A, vmax = prefix_want(None, s, q, nkv, 0, lens)
    got = run_prefix(rf, stream, None, s, q, nh, nkv, hd, 0, cap, lens)
    assert not got[[0, 3]].any()
    check(got, want, A, cap, vmax)
    long = np.array([0, 0xFFFFFFFF, 1, 0, 289, 32], np.uint32)
    p = Cache(rf, stream, rng, HEAD, nkv, 40, 40, hd, fp8)
    s2 = Cache(rf, stream, rng, TOKEN, nkv, 290, 290, hd, fp8, lead=(6,))
    want, A, vmax = prefix_want(p, s2, q, nkv, 40, lens)
    check(run_prefix(rf, stream, p, s2, q, nh, nkv, hd, 40, 290, long), want, A, 330, vmax)
    got = run_prefix(rf, stream, None, s2, q, nh, nkv, hd, 0, 290, np.zeros(6, np.uint32))
    assert not got.any()


@pytest.mark.parametrize("hd", [64, 128])
def test_prefix_f16_values_that_are_not_finite(rf, stream, kernel, hd):
    """They reach the rows that read them: an infinite V its dimension, a NaN K the whole row; no other row changes."""
    nkv, cap = 2, 150
    rng = np.random.default_rng(hd)
    p = Cache(rf, stream, rng, HEAD, nkv, 70, 70, hd, False)
    s = Cache(rf, stream, rng, TOKEN, nkv, cap, cap, hd, False, lead=(5,))
    lens = np.array([150, 149, 0, 33, 150], np.uint32)
    q = rng.standard_normal((5, 4, hd)).astype(np.float32)
    want, A, vmax = prefix_want(p, s, q, nkv, 70, lens)
    for i, (b, t) in ((0, (4, 149)), (1, (1, 148)), (0, (3, 33)), (1, (3, 40))):  # the last two behind row 3's tokens
        x = s.val[i].astype(np.float16)
        x[b, t, 1, 5] = np.nan if i == 0 else np.inf
        s.val[i] = x.astype(np.float64)
        s.dev[i] = _dev(rf, lay(x, TOKEN).view(np.uint16), stream)
    got = run_prefix(rf, stream, p, s, q, 4, nkv, hd, 70, cap, lens)
    assert np.isnan(got[4, 2:]).all() and not np.isfinite(got[1, 2:, 5]).any()
    want[4, 2:], want[1, 2:, 5], got[4, 2:], got[1, 2:, 5] = 0, 0, 0, 0
    check(got, want, A, 70 + cap, vmax)


def test_prefix_without_any_keys(rf, stream):
    out = _dev(rf, np.full(3 * 128, 5, np.float32), stream)
    q = _dev(rf, np.ones(3 * 128, np.float32), stream)
    rf.attn_decode_prefix_f16(stream, 3, 2, 1, 64, q, 128, 0, None, None, 0, 0, 0, None, None, None, 0, 0, 0, None, 0, out, 128)
    assert not out.to_host(3 * 128, np.float32, stream).any()


# ------------------------------------------------------------------ together
def test_prompt_tokens_then_a_batch(rf, stream):
    """A prompt in two chunks and two tokens of one sequence, then three
    sequences that go on from it: every output against float64 on the cache's
    own values."""
    nh, nkv, hd, cap = 8, 2, 128, 120
    rng = np.random.default_rng(8)
    w = (nh + 2 * nkv) * hd  # rows q | k | v, as a fused projection leaves them
    ts, hs = strides(HEAD, nkv, cap, hd)
    c = Cache(rf, stream, rng, HEAD, nkv, 0, cap, hd, True)
    size = max(rf.attn_prefill_fp8_workspace(nh, nkv, hd, 0, cap), rf.attn_decode_prefix_workspace(3, nh, nkv, hd, cap, 4), 16)
    ws = work(rf, stream, size)
    k, v, seen = np.zeros((cap, nkv, hd)), np.zeros((cap, nkv, hd)), 0

    def split(x):
        return (x[:, a * hd:b * hd].reshape(len(x), -1, hd) for a, b in ((0, nh), (nh, nh + nkv), (nh + nkv, nh + 2 * nkv)))

    for rows in (70, 31, 1, 1):
        x = rng.standard_normal((rows, w)).astype(np.float32)
        dx = _dev(rf, x, stream)
        rf.kv_append_rows_fp8(stream, rows, nkv, hd, seen, None, dx.ptr + 4 * nh * hd, w, dx.ptr + 4 * (nh + nkv) * hd, w, *c.dev, 0, ts, hs, cap)
        out = rf.DeviceBuffer.zeroed(rows * nh * hd, np.float32, stream)
        if rows > 1:
            rf.attn_prefill_fp8(stream, nh, nkv, hd, seen, rows, dx, w, *c.dev, ts, hs, ws, size, out, nh * hd)
        else:
            rf.attn_decode_fp8(stream, nh, nkv, hd, seen + 1, dx, *c.dev, ts, hs, ws, size, out)
        q, nk, nv = split(x)
        k[seen:seen + rows], v[seen:seen + rows] = kv8.decode(*kv8.encode(nk)), kv8.decode(*kv8.encode(nv))
        c.val = [k, v]
        want, A, vmax = prefill_want(c, q, nh // nkv, seen)
        check(out.to_host(rows * nh * hd, np.float32, stream).reshape(rows, nh, hd), want, A, seen + rows, vmax)
        seen += rows
    s = Cache(rf, stream, rng, TOKEN, nkv, 0, 4, hd, True, lead=(3,))
    s.val = [np.zeros((3, 4, nkv, hd)), np.zeros((3, 4, nkv, hd))]
    lens = np.array([0, 2, 1], np.uint32)
    for b in (1, 1, 2):  # what two of the sequences hold already
        at = int(np.count_nonzero(s.val[0][b].any((-1, -2))))
        new = rng.standard_normal((2, nkv, hd)).astype(np.float32)
        pos = np.full(3, 0xFFFFFFFF, np.uint32)
        pos[b] = at
        rf.kv_append_rows_fp8(stream, 3, nkv, hd, 0, _dev(rf, pos, stream), _dev(rf, np.repeat(new[:1], 3, 0), stream), nkv * hd,
                              _dev(rf, np.repeat(new[1:], 3, 0), stream), nkv * hd, *s.dev, s.ss, s.ts, s.hs, 4)
        for i in range(2):
            s.val[i][b, at] = kv8.decode(*kv8.encode(new[i]))
    for _ in range(2):
        x = rng.standard_normal((3, w)).astype(np.float32)
        dx = _dev(rf, x, stream)
        rf.kv_append_rows_fp8(stream, 3, nkv, hd, 0, _dev(rf, lens, stream), dx.ptr + 4 * nh * hd, w, dx.ptr + 4 * (nh + nkv) * hd, w, *s.dev,
                              s.ss, s.ts, s.hs, 4)
        q, nk, nv = split(x)
        for b in range(3):
            s.val[0][b, lens[b]], s.val[1][b, lens[b]] = kv8.decode(*kv8.encode(nk[b])), kv8.decode(*kv8.encode(nv[b]))
        lens += 1
        out = rf.DeviceBuffer.zeroed(3 * nh * hd, np.float32, stream)
        rf.attn_decode_prefix_fp8(stream, 3, nh, nkv, hd, dx, w, seen, *c.dev, ts, hs, 4, _dev(rf, lens, stream), *s.dev, s.ss, s.ts, s.hs, ws,
                                  size, out, nh * hd)
        want, A, vmax = prefix_want(c, s, q, nkv, seen, lens)
        check(out.to_host(3 * nh * hd, np.float32, stream).reshape(3, nh, hd), want, A, seen + 4, vmax)


@pytest.mark.parametrize("fp8,nh,nkv,hd,batch,prefix", [(True, 8, 2, 128, 33, 24500), (False, 8, 1, 64, 40, 40000)])
@pytest.mark.parametrize("cap", [65, 700])
def test_planned_for_many_rows(rf, stream, fp8, nh, nkv, hd, batch, prefix, cap):
    """Sizes on the far side of the planner's line, with own keys in the same launch and in one of their own."""
    rng = np.random.default_rng(batch)
    p = Cache(rf, stream, rng, TOKEN, nkv, prefix, prefix, hd, fp8)
    s = Cache(rf, stream, rng, HEAD, nkv, cap, cap, hd, fp8, lead=(batch,))
    lens = rng.integers(0, cap + 1, batch).astype(np.uint32)
    q = rng.standard_normal((batch, nh, hd)).astype(np.float32)
    want, A, vmax = prefix_want(p, s, q, nkv, prefix, lens)
    check(run_prefix(rf, stream, p, s, q, nh, nkv, hd, prefix, cap, lens), want, A, prefix + cap, vmax)


def test_prefix_over_an_engines_cache(rf, stream):
    """The shared cache is an engine's; against attn_decode_f16 on the same memory."""
    cfg = rf.model_config(dim=256, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=64, ffn=512, vocab=1024, theta=10000.0, eps=1e-5, max_seq=300)
    eng = rf.Engine(cfg, 3)
    eng.prefill_kv(9, 290)
    k, v, n = rf.P(), rf.P(), rf.SZ()
    rf.check(rf.load().llama_engine_kv(eng.h, 1, C.byref(k), C.byref(v), C.byref(n)))
    hs = n.value // 2
    q = np.random.default_rng(2).standard_normal((3, 4, 64)).astype(np.float32)
    out, one = rf.DeviceBuffer.zeroed(3 * 256, np.float32, stream), rf.DeviceBuffer.zeroed(256, np.float32, stream)
    size = rf.attn_decode_prefix_workspace(3, 4, 2, 64, 277, 0)
    rf.attn_decode_prefix_f16(stream, 3, 4, 2, 64, _dev(rf, q, stream), 256, 277, k.value, v.value, 64, hs, 0, None, None, None, 0, 0, 0,
                              work(rf, stream, size), size, out, 256)
    got = out.to_host(3 * 256, np.float32, stream).reshape(3, 256)
    kc, vc = (t.view(np.float16).reshape(2, hs // 64, 64)[:, :277].astype(np.float64) for t in eng.kv_host(1))
    for b in range(3):
        rf.attn_decode_f16(stream, 4, 2, 64, 277, _dev(rf, q[b], stream), k.value, v.value, 64, hs, one)
        want = one.to_host(256, np.float32, stream)
        A = max(kv8.attend(q[b, h:h + 1], kc[h // 2], vc[h // 2])[1] for h in range(4))
        assert np.abs(got[b] - want).max() <= 2 * kv8.bound(A, 277, np.abs(vc).max())  # each is off by its own
    eng.close()


# ------------------------------------------------------------------ streams and graphs
def test_two_streams_at_once(rf, stream, kernel):
    """Calls that overlap, each with its own workspace, give what each gives alone."""
    nh, nkv, hd, seq = 8, 2, 128, 6000
    rng = np.random.default_rng(4)
    c = [Cache(rf, stream, rng, HEAD, nkv, seq, seq, hd, True) for _ in range(2)]
    q = [rng.standard_normal((nh, hd)).astype(np.float32) for _ in range(2)]
    alone = [run_decode(rf, stream, c[i], q[i], nh, nkv, hd, seq) for i in range(2)]
    streams, size = [rf.Stream(), rf.Stream()], rf.attn_decode_fp8_workspace(nh, nkv, hd, seq)
    assert size
    ws, out = [work(rf, stream, size) for _ in range(2)], [rf.DeviceBuffer.zeroed(nh * hd, np.float32, stream) for _ in range(2)]
    dq = [_dev(rf, x, stream) for x in q]
    stream.synchronize()
    for _ in range(20):
        for i in range(2):
            rf.attn_decode_fp8(streams[i], nh, nkv, hd, seq, dq[i], *c[i].dev, c[i].ts, c[i].hs, ws[i], size, out[i])
    for i in range(2):
        streams[i].synchronize()
        np.testing.assert_array_equal(out[i].to_host(nh * hd, np.float32, stream).reshape(nh, hd), alone[i])


def test_captured_and_replayed(rf, kernel):
    """An append and a batch step in a graph, replayed with new rows, positions
    and lengths in the same buffers, each replay against the calls themselves."""
    hip = C.CDLL("libamdhip64.so")
    nh, nkv, hd, prefix, cap, batch = 8, 2, 64, 700, 300, 5
    rng = np.random.default_rng(6)
    s1 = rf.Stream()
    p = Cache(rf, s1, rng, HEAD, nkv, prefix, prefix, hd, True)
    s = Cache(rf, s1, rng, TOKEN, nkv, cap, cap, hd, True, lead=(batch,))
    w = (nh + 2 * nkv) * hd
    dx, dpos, dlen = rf.DeviceBuffer.zeroed(batch * w, np.float32, s1), rf.DeviceBuffer.zeroed(batch, np.uint32, s1), rf.DeviceBuffer.zeroed(batch, np.uint32, s1)
    size = rf.attn_decode_prefix_workspace(batch, nh, nkv, hd, prefix, cap)
    ws, out = work(rf, s1, size), rf.DeviceBuffer.zeroed(batch * nh * hd, np.float32, s1)

    def calls():
        rf.kv_append_rows_fp8(s1, batch, nkv, hd, 0, dpos, dx.ptr + 4 * nh * hd, w, dx.ptr + 4 * (nh + nkv) * hd, w, *s.dev, s.ss, s.ts, s.hs, cap)
        rf.attn_decode_prefix_fp8(s1, batch, nh, nkv, hd, dx, w, prefix, *p.dev, p.ts, p.hs, cap, dlen, *s.dev, s.ss, s.ts, s.hs, ws, size, out, nh * hd)

    def ok(rc):
        assert rc == 0, rc

    graph, run = C.c_void_p(), C.c_void_p()
    s1.synchronize()
    ok(hip.hipStreamBeginCapture(C.c_void_p(s1.h), 2))  # relaxed
    calls()
    ok(hip.hipStreamEndCapture(C.c_void_p(s1.h), C.byref(graph)))
    ok(hip.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)))
    for _ in range(4):
        x = rng.standard_normal(batch * w).astype(np.float32)
        pos = rng.integers(0, cap, batch).astype(np.uint32)
        lens = rng.integers(0, cap + 1, batch).astype(np.uint32)
        for buf, host in ((dx, x), (dpos, pos), (dlen, lens)):
            rf.check(rf.load().rfp4_h2d(buf.ptr, host.ctypes.data, host.nbytes, s1.h))
        s1.synchronize()
        ok(hip.hipGraphLaunch(run, C.c_void_p(s1.h)))
        s1.synchronize()
        got = out.to_host(batch * nh * hd, np.float32, s1)
        rf.check(rf.load().rfp4_memset_zero(out.ptr, out.nbytes, s1.h))
        calls()
        np.testing.assert_array_equal(out.to_host(batch * nh * hd, np.float32, s1), got)
    ok(hip.hipGraphExecDestroy(run))
    ok(hip.hipGraphDestroy(graph))
