"""Refusals of the 4-bit KV entry points, and the plain forms that the GPU
tests compare with. Every call here is refused before the context is used, so
a zeroed block stands in for one (no device needed)."""
import ctypes as C

import numpy as np
import pytest

import kv4_ref as ref

IA, SM, DT = "INVALID_ARGUMENT", "SHAPE_MISMATCH", "DTYPE_UNSUPPORTED"


@pytest.fixture(scope="module")
def fake():
    return C.create_string_buffer(8192)


def _ptr():
    return 0x10000  # 16-byte aligned, never followed


def test_page_and_workspace_bytes(gh):
    L = gh.lib()
    assert L.glacier_hip_kv4_page_bytes(28, 4, 128) == 28 * 4 * 2 * ref.tile_bytes(128)
    assert L.glacier_hip_kv4_page_bytes(24, 2, 64) == 24 * 2 * 2 * ref.tile_bytes(64)
    for bad in ((0, 4, 128), (28, 0, 128), (28, 4, 96), (28, 4, 0)):
        assert L.glacier_hip_kv4_page_bytes(*bad) == 0
    ws = L.glacier_hip_kv4_attention_workspace_bytes
    assert ws(1, 1, 14, 2, 64) > 0 and ws(1024, 1 << 20, 64, 8, 128) > 0
    for bad in ((0, 1, 14, 2, 64), (1025, 1025, 14, 2, 64), (1, 0, 14, 2, 64),
                (1, (1 << 20) + 1, 14, 2, 64), (1, 1, 15, 2, 64), (1, 1, 18, 2, 64),
                (1, 1, 14, 0, 64), (1, 1, 14, 2, 80), (1, 1, 0, 2, 64)):
        assert ws(*bad) == 0, bad


PLAN = dict(ctx=1, lens=_ptr(), new=_ptr(), lanes=4, max_rows=8, table=_ptr(), max_pages=8, free=_ptr(),
            free_count=4, taken=_ptr(), start=_ptr(), after=_ptr(), slots=_ptr(), who=_ptr(), pos=_ptr(),
            result=_ptr(), stream=None)


@pytest.mark.parametrize("change,want", [
    (dict(ctx=None), IA), (dict(lens=None), IA), (dict(new=None), IA), (dict(table=None), IA),
    (dict(free=None), IA), (dict(taken=None), IA), (dict(start=None), IA), (dict(after=None), IA),
    (dict(slots=None), IA), (dict(result=None), IA), (dict(lanes=0), SM), (dict(lanes=1025), SM),
    (dict(max_rows=0), SM), (dict(max_rows=(1 << 20) + 1), SM), (dict(max_pages=0), SM),
    (dict(max_pages=(1 << 26) + 1), SM), (dict(lanes=1024, max_pages=1 << 22), SM),
    (dict(free_count=(1 << 30) + 1), SM)])
def test_plan_refusals(gh, fake, change, want):
    a = dict(PLAN, **{"ctx": C.addressof(fake), **change})
    assert gh.lib().glacier_hip_kv_plan_rows(*a.values()) == getattr(gh, want)


def _pool(gh, **change):
    return gh.Kv4Pool(*dict(dict(pages=_ptr(), count=4, layers=2, heads=2, hd=64), **change).values())


POOL_BAD = [(dict(pages=None), IA), (dict(pages=_ptr() + 8), IA), (dict(count=0), SM), (dict(layers=1), SM),
            (dict(heads=0), SM), (dict(hd=32), SM), (dict(hd=96), SM)]


@pytest.mark.parametrize("change,want", POOL_BAD + [
    (dict(k=None), IA), (dict(v=None), IA), (dict(slots=None), IA), (dict(dtype=3), DT), (dict(dtype=-1), DT),
    (dict(k=_ptr() + 2), IA), (dict(v=_ptr() + 2), IA), (dict(ks=127), SM), (dict(vs=127), SM),
    (dict(ks=(1 << 32) + 1), SM), (dict(rows=0), SM), (dict(rows=(1 << 20) + 1), SM), (dict(layer=2), SM),
    (dict(ctx=None), IA), (dict(pool=None), IA)])
def test_append_refusals(gh, fake, change, want):
    a = dict(ctx=C.addressof(fake), pool=None, layer=1, k=_ptr(), v=_ptr(), dtype=gh.F32, ks=128, vs=128,
             slots=_ptr(), rows=3, stream=None)
    a["pool"] = _pool(gh, **{n: v for n, v in change.items() if n in ("pages", "count", "layers", "heads", "hd")})
    a.update({n: v for n, v in change.items() if n in a})
    assert gh.lib().glacier_hip_kv4_append(*a.values()) == getattr(gh, want)


@pytest.mark.parametrize("change,want", POOL_BAD + [
    (dict(k=None), IA), (dict(v=None), IA), (dict(slots=None), IA), (dict(k=_ptr() + 4), IA),
    (dict(v=_ptr() + 8), IA), (dict(rows=0), SM), (dict(rows=(1 << 20) + 1), SM), (dict(layer=2), SM),
    (dict(ctx=None), IA), (dict(pool=None), IA)])
def test_read_refusals(gh, fake, change, want):
    a = dict(ctx=C.addressof(fake), pool=None, layer=1, slots=_ptr(), rows=3, k=_ptr(), v=_ptr(), stream=None)
    a["pool"] = _pool(gh, **{n: v for n, v in change.items() if n in ("pages", "count", "layers", "heads", "hd")})
    a.update({n: v for n, v in change.items() if n in a})
    assert gh.lib().glacier_hip_kv4_read(*a.values()) == getattr(gh, want)


ATTN_BAD = POOL_BAD + [
    (dict(ctx=None), IA), (dict(pool=None), IA), (dict(q=None), IA), (dict(q=_ptr() + 4), IA),
    (dict(table=None), IA), (dict(lens=None), IA), (dict(out=None), IA), (dict(out=_ptr() + 8), IA),
    (dict(ws=None), IA), (dict(ws=_ptr() + 8), IA), (dict(ws_bytes=0), SM), (dict(Hq=15), SM),
    (dict(Hq=18), SM), (dict(Hq=0), SM), (dict(lanes=0), SM), (dict(lanes=1025), SM), (dict(max_ctx=0), SM),
    (dict(max_ctx=65), SM), (dict(layer=2), SM)]


@pytest.mark.parametrize("change,want", ATTN_BAD)
def test_decode_attention_refusals(gh, fake, change, want):
    a = dict(ctx=C.addressof(fake), pool=None, layer=1, q=_ptr(), table=_ptr(), max_pages=4, lens=_ptr(),
             lanes=3, Hq=14, max_ctx=64, out=_ptr(), ws=_ptr(), ws_bytes=1 << 40, stream=None)
    a["pool"] = _pool(gh, **{n: v for n, v in change.items() if n in ("pages", "count", "layers", "heads", "hd")})
    a.update({n: v for n, v in change.items() if n in a})
    assert gh.lib().glacier_hip_paged_attention_kv4(*a.values()) == getattr(gh, want)


@pytest.mark.parametrize("change,want", ATTN_BAD + [
    (dict(start=None), IA), (dict(rows=0), SM), (dict(rows=(1 << 20) + 1), SM)])
def test_rows_attention_refusals(gh, fake, change, want):
    a = dict(ctx=C.addressof(fake), pool=None, layer=1, q=_ptr(), table=_ptr(), max_pages=4, start=_ptr(),
             lens=_ptr(), lanes=3, rows=20, Hq=14, max_ctx=64, out=_ptr(), ws=_ptr(), ws_bytes=1 << 40,
             stream=None)
    a["pool"] = _pool(gh, **{n: v for n, v in change.items() if n in ("pages", "count", "layers", "heads", "hd")})
    a.update({n: v for n, v in change.items() if n in a})
    assert gh.lib().glacier_hip_paged_attention_kv4_rows(*a.values()) == getattr(gh, want)


def test_workspace_one_byte_short_is_refused(gh, fake):
    L = gh.lib()
    need = L.glacier_hip_kv4_attention_workspace_bytes(3, 3, 14, 2, 64)
    assert L.glacier_hip_paged_attention_kv4(
        C.addressof(fake), _pool(gh), 1, _ptr(), _ptr(), 4, _ptr(), 3, 14, 64, _ptr(), _ptr(), need - 1,
        None) == gh.SHAPE_MISMATCH


@pytest.mark.parametrize("hd", [64, 128])
def test_layout_places_every_byte_once(hd):
    code, half = ref.tables(hd)
    for w in range(2):
        nibbles = {(int(b), int(s)) for b, s in code[w].reshape(-1, 2)}
        assert nibbles == {(b, s) for b in range(8 * hd) for s in (0, 4)}
        assert sorted(half[w].reshape(-1).tolist()) == list(range(8 * hd, 10 * hd, 2))


@pytest.mark.parametrize("hd", [64, 128])
def test_stored_rows_read_back_as_their_codes(hd):
    """A stored value is the nearest of its group's 16 levels: off by at most
    half a step, plus what the rounded minimum (half an fp16 step, 2^-11 of
    it) and the rounded step (15 * 2^-11 of it) move the levels."""
    rng = np.random.default_rng(hd)
    pool = np.zeros((3, 2, 2, 2, 10 * hd), np.uint8)
    slots = rng.permutation(48)
    x = rng.standard_normal((2, 48, 2, hd)).astype(np.float32) * 3
    ref.store_rows(pool, 1, slots, x[0], x[1])
    assert not pool[:, 0].any()
    for got, want in zip(ref.values(pool, 1, slots), x):
        g = want.reshape(48, 2, hd // 32, 32).astype(np.float64)
        lo, step = g.min(-1, keepdims=True), (g.max(-1, keepdims=True) - g.min(-1, keepdims=True)) / 15
        room = step * (0.5 + 15 * 2.0 ** -11 + 2.0 ** -11) + np.abs(lo) * 2.0 ** -11 + 2.0 ** -24
        assert (np.abs(got.reshape(g.shape) - g) <= room).all()
