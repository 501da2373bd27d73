"""What kv_append_rows_*, attn_decode_fp8, attn_prefill_fp8 and
attn_decode_prefix_* refuse, on the CPU: every check comes before a device is
touched (what passes them all ends in RFP4_E_NOT_INIT)."""
import pytest

import kv8
import numpy as np
import rfp4

INVALID, SHAPE, CAPACITY, OVERFLOW, NOT_INIT, ALIGN = -1, -2, -3, -4, -5, -6
P = 0x10000  # never dereferenced


def call(fn, args, **kw):
    lib = rfp4.load()
    return getattr(lib, fn)(None, *{**args, **kw}.values())


APPEND = dict(rows=4, nkv=2, hd=64, pos0=8, positions=None, k=P, krs=128, v=P, vrs=128, kc=P, ks=P, vc=P, vs=P, ss=0, ts=64, hs=64 * 16, cap=16)
DECODE = dict(nh=8, nkv=2, hd=64, seq=33, q=P, kc=P, ks=P, vc=P, vs=P, ts=64, hs=64 * 64, ws=P, wsb=1 << 30, out=P)
PREFILL = dict(nh=8, nkv=2, hd=128, pos0=5, rows=9, q=P, qrs=1024, kc=P, ks=P, vc=P, vs=P, ts=256, hs=128, ws=P, wsb=1 << 30, out=P, ors=1024)
PREFIX = dict(batch=3, nh=8, nkv=2, hd=128, q=P, qrs=1024, prefix=40, pk=P, pks=P, pv=P, pvs=P, pts=256, phs=128, cap=7, lens=P, sk=P,
              sks=P, sv=P, svs=P, sss=256 * 7, sts=256, shs=128, ws=P, wsb=1 << 30, out=P, ors=1024)


@pytest.fixture(autouse=True)
def _no_device():
    if rfp4._inited:  # these calls would launch on made-up addresses
        pytest.skip("the library is initialised in this process")


def half(args):
    """The same call of the fp16 entry point: no scales."""
    return {k: v for k, v in args.items() if k not in ("ks", "vs", "pks", "pvs", "sks", "svs")}


def test_good_calls_reach_the_launch():
    assert call("kv_append_rows_fp8", APPEND) == NOT_INIT
    assert call("kv_append_rows_f16", half(APPEND)) == NOT_INIT
    assert call("attn_decode_fp8", DECODE) == NOT_INIT
    assert call("attn_prefill_fp8", PREFILL) == NOT_INIT
    assert call("attn_decode_prefix_fp8", PREFIX) == NOT_INIT
    assert call("attn_decode_prefix_f16", half(PREFIX)) == NOT_INIT


def test_nothing_to_do():
    assert call("kv_append_rows_fp8", APPEND, rows=0, k=None, kc=None) == 0
    assert call("attn_prefill_fp8", PREFILL, rows=0, q=None) == 0
    assert call("attn_decode_prefix_fp8", PREFIX, batch=0, q=None) == 0


@pytest.mark.parametrize("change,code", [
    (dict(hd=96), SHAPE), (dict(nkv=0), SHAPE), (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(kc=None), INVALID),
    (dict(ks=None), INVALID), (dict(vs=None), INVALID), (dict(k=P + 4), ALIGN), (dict(krs=130), ALIGN), (dict(krs=64), SHAPE),
    (dict(kc=P + 8), ALIGN), (dict(ts=96), ALIGN), (dict(hs=1000), ALIGN), (dict(pos0=13), OVERFLOW), (dict(cap=11), OVERFLOW),
    (dict(pos0=0xFFFFFFFF), OVERFLOW), (dict(ts=0), SHAPE), (dict(hs=64 * 15), SHAPE), (dict(hs=0), SHAPE),
    (dict(positions=P, ss=64 * 31), SHAPE), (dict(positions=P, ss=0), SHAPE), (dict(hs=1 << 50), SHAPE),
])
def test_append(change, code):
    assert call("kv_append_rows_fp8", APPEND, **change) == code
    assert rfp4.load().rfp4_last_error()
    if not {"ks", "vs"} & set(change):
        assert call("kv_append_rows_f16", half(APPEND), **{k: (v if k not in ("ts", "hs") or v % 64 == 0 else v + 4) for k, v in change.items()}) == code


@pytest.mark.parametrize("change", [dict(positions=P, ss=64 * 32), dict(ts=128, hs=64), dict(positions=P, ss=64, ts=64 * 8, hs=64 * 4),
                                    dict(nkv=1, hs=0), dict(rows=1, krs=0, vrs=0)])
def test_append_layouts_that_fit(change):
    assert call("kv_append_rows_fp8", APPEND, **change) == NOT_INIT


@pytest.mark.parametrize("change,code", [
    (dict(hd=32), SHAPE), (dict(nkv=0), SHAPE), (dict(nh=0), SHAPE), (dict(nh=7), SHAPE), (dict(nh=18), SHAPE), (dict(seq=0), SHAPE),
    (dict(q=None), INVALID), (dict(out=None), INVALID), (dict(kc=None), INVALID), (dict(vs=None), INVALID), (dict(q=P + 8), ALIGN),
    (dict(out=P + 4), ALIGN), (dict(vc=P + 1), ALIGN), (dict(ts=72), ALIGN), (dict(seq=0xFFFFFFFF), SHAPE),
    (dict(seq=4096, ws=None, wsb=0), INVALID), (dict(seq=4096, wsb=64), CAPACITY), (dict(seq=4096, ws=P + 4), ALIGN),
])
def test_decode(change, code):
    assert call("attn_decode_fp8", DECODE, **change) == code
    assert rfp4.load().rfp4_last_error()


@pytest.mark.parametrize("change,code", [
    (dict(hd=0), SHAPE), (dict(nh=20), SHAPE), (dict(q=None), INVALID), (dict(qrs=1020), SHAPE), (dict(ors=1023), ALIGN), (dict(ors=0), SHAPE),
    (dict(ts=64), ALIGN), (dict(pos0=0x7FFFFFFF), SHAPE), (dict(rows=0x80000000, pos0=0), SHAPE), (dict(ks=None), INVALID),
])
def test_prefill(change, code):
    assert call("attn_prefill_fp8", PREFILL, **change) == code
    assert rfp4.load().rfp4_last_error()


@pytest.mark.parametrize("change,code", [
    (dict(hd=256), SHAPE), (dict(nh=3), SHAPE), (dict(q=None), INVALID), (dict(pk=None), INVALID), (dict(sv=None), INVALID),
    (dict(lens=None), INVALID), (dict(pk=P + 2), ALIGN), (dict(sts=100), ALIGN), (dict(sss=4), ALIGN), (dict(qrs=512), SHAPE),
    (dict(out=P + 4), ALIGN), (dict(ws=None), INVALID), (dict(wsb=16), CAPACITY), (dict(prefix=0xFFFFFFFF), SHAPE),
])
def test_prefix(change, code):
    assert call("attn_decode_prefix_fp8", PREFIX, **change) == code
    assert rfp4.load().rfp4_last_error()
    assert call("attn_decode_prefix_f16", half(PREFIX), **change) == code


def test_parts_that_are_empty_are_not_looked_at():
    assert call("attn_decode_prefix_fp8", PREFIX, prefix=0, pk=None, pv=None, pks=None, pvs=None, pts=3) == NOT_INIT
    assert call("attn_decode_prefix_fp8", PREFIX, cap=0, lens=None, sk=None, sks=None, sv=None, svs=None, sss=1) == NOT_INIT
    # an 8-bit prefix without its scales is not a prefix
    assert call("attn_decode_prefix_fp8", PREFIX, pks=None) == INVALID


def test_workspace_sizes():
    """0 where nothing is split, and never less for a longer cache than one state for each split of the shorter."""
    assert rfp4.attn_decode_fp8_workspace(32, 8, 128, 0) == 0
    assert rfp4.attn_decode_fp8_workspace(32, 8, 128, 1) == 0
    assert rfp4.attn_decode_fp8_workspace(32, 5, 128, 4096) == 0  # refused by the call itself
    assert rfp4.attn_decode_fp8_workspace(32, 8, 128, 32768) >= 2 * 32 * 132 * 4
    assert rfp4.attn_decode_prefix_workspace(0, 32, 8, 128, 100, 100) == 0
    assert rfp4.attn_decode_prefix_workspace(4, 32, 8, 128, 100, 100) >= 2 * 4 * 32 * 132 * 4


@pytest.mark.parametrize("nh,nkv,rows", [(32, 8, 1), (8, 1, 1), (8, 1, 5), (32, 8, 40), (3, 3, 130), (4, 4, 33)])
def test_a_workspace_serves_every_shorter_context(nh, nkv, rows):
    lens = sorted({1, 2, 127, 128, 129, 255, 256, 1000, 4095, 4096, 4097, 8191, 12000, 16384, 16500, 33000, 70000, 300000})
    decode = [rfp4.attn_decode_fp8_workspace(nh, nkv, 128, n) for n in lens]
    prefill = [rfp4.attn_prefill_fp8_workspace(nh, nkv, 64, n, rows) for n in lens]
    prefix = [rfp4.attn_decode_prefix_workspace(rows, nh, nkv, 128, n, 700) for n in lens]
    suffix = [rfp4.attn_decode_prefix_workspace(rows, nh, nkv, 128, 5000, n) for n in lens]
    for size in (decode, prefill, prefix, suffix):
        assert size == sorted(size)
    # and the calls ask for no more than that
    for n in lens:
        ws = rfp4.attn_decode_fp8_workspace(nh, nkv, 64, max(lens))
        assert call("attn_decode_fp8", DECODE, nh=nh, nkv=nkv, seq=n, wsb=ws) == NOT_INIT
        ws = rfp4.attn_prefill_fp8_workspace(nh, nkv, 128, max(lens), rows)
        assert call("attn_prefill_fp8", PREFILL, nh=nh, nkv=nkv, pos0=n, rows=rows, wsb=ws, qrs=nh * 128, ors=nh * 128) == NOT_INIT
        ws = rfp4.attn_decode_prefix_workspace(rows, nh, nkv, 128, max(lens), max(lens))
        for m in lens:
            assert call("attn_decode_prefix_fp8", PREFIX, batch=rows, nh=nh, nkv=nkv, prefix=n, cap=m, wsb=ws, qrs=nh * 128, ors=nh * 128) == NOT_INIT


def test_the_kernel_hook():
    assert [rfp4.load().rfp4_debug_attn_rows(m) for m in (-1, 3, 2, 1, 0)] == [-1, -1, 0, 0, 0]


def test_the_oracle_format():
    """The tests' encoder: levels encode to themselves, ties go to the even code, scales as defined."""
    codes, scales = kv8.encode(np.concatenate((kv8.LEVELS, -kv8.LEVELS))[None].astype(np.float32))
    assert scales[0] == 127 and list(codes[0]) == list(range(127)) + list(range(128, 255))
    for amax, byte in ((448, 127), (np.nextafter(np.float32(448), np.float32(500)), 128), (224, 126), (1, 119), (2.0 ** -149, 0), (0, 0),
                       (3.4028234e38, 247), (np.inf, 255), (np.nan, 255)):
        assert kv8.encode(np.array([[0, amax]], np.float32))[1][0] == byte, amax
    codes, _ = kv8.encode(np.array([[448, 17, 19, 2.0 ** -10, 3 * 2.0 ** -10, -0.0]], np.float32))
    assert list(codes[0]) == [126, 88, 90, 0, 2, 128]  # 17 and 19 lie between 16, 18 and 20; 2^-10 between 0 and 2^-9
