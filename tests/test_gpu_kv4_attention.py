"""Attention over 4-bit pages (decode rows and runs of rows) against 64-bit
sums on the stored values.

Tolerance, of the largest stored value that a row attends: 2^-24 *
(sqrt(head_dim) * S + 16), S the row's largest |score|. A score is a sum of
head_dim products whose f32 partial sums round at 2^-24 of themselves
(sqrt(head_dim) steps of a random walk, partial sums up to about S) and moves
a weight by its own error; the fp16 hi + lo pairs of queries and weights leave
2^-22 each, exponential, sums and the final quotient a few 2^-24 more."""
import numpy as np
import pytest

import kv4_ref as ref

pytestmark = pytest.mark.gpu

LAYERS, LAYER = 3, 1


def _dev(a):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


class Cache:
    """Lanes' pages with every unused byte set to `junk` (0x7E: NaN steps and minima)."""

    def __init__(self, rng, ctx, heads, hd, junk=0x7E, k_gain=1.0, v_gain=1.0, rows=None):
        self.heads, self.hd, self.ctx = heads, hd, list(ctx)
        held = [-(-max(c, 0) // 16) for c in ctx]
        pages = sum(held) + 3
        perm = rng.permutation(pages).astype(np.int32)
        self.table = np.full((len(ctx), max(max(held), 1) + 1), -9, np.int32)
        self.pool = np.full((pages, LAYERS, heads, 2, 10 * hd), junk, np.uint8)
        slots, at = [], 0
        for i, c in enumerate(ctx):
            self.table[i, :held[i]] = perm[at:at + held[i]]
            at += held[i]
            p = np.arange(max(c, 0))
            slots.append(self.table[i, p // 16].astype(np.int64) * 16 + p % 16)
        self.slots = slots
        every = np.concatenate(slots + [np.zeros(0, np.int64)])
        n = len(every)
        if rows is None:
            gain = np.exp(0.5 * rng.standard_normal((heads, hd)))
            rows = (rng.standard_normal((n, heads, hd)) * gain * k_gain, rng.standard_normal((n, heads, hd)) * v_gain)
        ref.store_rows(self.pool, LAYER, every, *(np.asarray(r, np.float32) for r in rows))

    def lane(self, i):
        return ref.values(self.pool, LAYER, self.slots[i])

    def upload(self, gh):
        self.pd, self.td = _dev(self.pool), _dev(self.table)
        self.pool_t = gh.Kv4Pool(self.pd.data_ptr(), self.pool.shape[0], LAYERS, self.heads, self.hd)


def workspace(gh, lanes, rows, Hq, heads, hd):
    import torch

    n = gh.lib().glacier_hip_kv4_attention_workspace_bytes(lanes, rows, Hq, heads, hd)
    assert n > 0
    return torch.zeros((n,), dtype=torch.uint8, device="cuda")


def decode(gh, gctx, cache, q, max_ctx=None, lens=None, ws=None, stream=None):
    import torch

    if not hasattr(cache, "pd"):
        cache.upload(gh)
    lanes, Hq, hd = q.shape
    lens = _dev(np.array(cache.ctx if lens is None else lens, np.int32))
    qd = _dev(q.astype(np.float32))
    out = torch.full((lanes + 1, Hq * hd), 5.0, device="cuda")
    ws = workspace(gh, lanes, lanes, Hq, cache.heads, hd) if ws is None else ws
    torch.cuda.synchronize()
    gh.check(gh.lib().glacier_hip_paged_attention_kv4(
        gctx.h, cache.pool_t, LAYER, qd.data_ptr(), cache.td.data_ptr(), cache.table.shape[1],
        lens.data_ptr(), lanes, Hq, max_ctx or cache.table.shape[1] * 16, out.data_ptr(), ws.data_ptr(),
        ws.numel(), stream), "decode", gctx.h)
    torch.cuda.synchronize()
    got = out.cpu().numpy()
    assert (got[lanes] == 5.0).all()
    return got[:lanes].reshape(lanes, Hq, hd)


def run_rows(gh, gctx, cache, q, new, room=None, max_ctx=None, ws=None, start=None, lens=None):
    import torch

    if not hasattr(cache, "pd"):
        cache.upload(gh)
    n, Hq, hd = q.shape
    room = room or n
    lanes = len(cache.ctx)
    start = np.cumsum([0] + list(new)) if start is None else start
    sd = _dev(np.asarray(start, np.int32))
    lens = _dev(np.array(cache.ctx if lens is None else lens, np.int32))
    qd = _dev(np.concatenate([q.astype(np.float32), np.full((room - n, Hq, hd), np.nan, np.float32)]))
    out = torch.full((room + 1, Hq * hd), 5.0, device="cuda")
    ws = workspace(gh, lanes, room, Hq, cache.heads, hd) if ws is None else ws
    torch.cuda.synchronize()
    gh.check(gh.lib().glacier_hip_paged_attention_kv4_rows(
        gctx.h, cache.pool_t, LAYER, qd.data_ptr(), cache.td.data_ptr(), cache.table.shape[1],
        sd.data_ptr(), lens.data_ptr(), lanes, room, Hq, max_ctx or cache.table.shape[1] * 16,
        out.data_ptr(), ws.data_ptr(), ws.numel(), None), "rows", gctx.h)
    torch.cuda.synchronize()
    got = out.cpu().numpy()
    assert (got[n:] == 5.0).all()
    return got[:n].reshape(n, Hq, hd)


def hold(got, q, K, V, what=None):
    want, top = ref.attention(q.astype(np.float32), K, V)
    big = np.abs(V).max() if len(V) else 0.0
    bar = 2.0 ** -24 * (np.sqrt(q.shape[-1]) * top + 16) * big
    err = np.abs(got - want).max()
    assert err <= bar, (what, err, bar)


def check_decode(gh, gctx, rng, ctx, Hq, heads, hd, **kw):
    cache = Cache(rng, ctx, heads, hd, **kw)
    q = 1.5 * rng.standard_normal((len(ctx), Hq, hd))
    got = decode(gh, gctx, cache, q)
    for i in range(len(ctx)):
        hold(got[i], q[i], *cache.lane(i), what=(i, ctx[i]))


def check_rows(gh, gctx, rng, ctx, new, Hq, heads, hd, room=0, **kw):
    cache = Cache(rng, ctx, heads, hd, **kw)
    q = 1.5 * rng.standard_normal((sum(new), Hq, hd))
    got = run_rows(gh, gctx, cache, q, new, room=sum(new) + room)
    r = 0
    for i, n in enumerate(new):
        K, V = cache.lane(i)
        for p in range(ctx[i] - n, ctx[i]):
            hold(got[r], q[r], K[:p + 1], V[:p + 1], what=(i, p))
            r += 1


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("ctx", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 255, 256, 257, 511, 513, 1000])
def test_one_lane(gh, gctx, hd, ctx):
    check_decode(gh, gctx, np.random.default_rng(ctx + hd), [ctx], 14, 2, hd)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("G", [1, 2, 3, 4, 5, 6, 7, 8])
def test_group_sizes(gh, gctx, hd, G):
    check_decode(gh, gctx, np.random.default_rng(G), [100, 1, 33, 700], 3 * G, 3, hd)


@pytest.mark.parametrize("hd,heads,Hq", [(64, 2, 14), (128, 4, 28)])
def test_ragged_lanes(gh, gctx, hd, heads, Hq):
    """Empty lanes first, last and between, contexts around the page and chunk ends."""
    ctx = [0, 37, 0, 130, 517, 16, 1030, 1999, 1, 2048, 3, 0, 640, 641, 4000, 0]
    check_decode(gh, gctx, np.random.default_rng(hd), ctx, Hq, heads, hd)


def test_all_lanes_empty(gh, gctx):
    cache = Cache(np.random.default_rng(0), [0, 0, 0], 2, 64)
    assert not decode(gh, gctx, cache, np.ones((3, 14, 64))).any()


@pytest.mark.parametrize("lanes", [65, 300, 1024])
def test_many_lanes(gh, gctx, lanes):
    rng = np.random.default_rng(lanes)
    check_decode(gh, gctx, rng, rng.integers(0, 70, lanes).tolist(), 4, 2, 64)


def test_long_context(gh, gctx):
    check_decode(gh, gctx, np.random.default_rng(1), [30000, 5], 4, 1, 128)


def test_many_kv_heads(gh, gctx):
    check_decode(gh, gctx, np.random.default_rng(2), [300, 44], 40, 40, 64)


@pytest.mark.parametrize("hd", [64, 128])
def test_the_same_call_twice_gives_the_same_bits(gh, gctx, hd):
    rng = np.random.default_rng(5)
    ctx = [700, 3000, 44, 0, 1211]
    cache = Cache(rng, ctx, 2, hd)
    q = rng.standard_normal((5, 14, hd))
    first = decode(gh, gctx, cache, q)
    ws = workspace(gh, 5, 5, 14, 2, hd)
    for _ in range(3):
        assert np.array_equal(first, decode(gh, gctx, cache, q, ws=ws))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("gain", [1e-6, 1e-3, 30.0, 4000.0])
def test_value_magnitudes(gh, gctx, hd, gain):
    """V far from one, down to fp16's subnormal steps, the tolerance in proportion."""
    check_decode(gh, gctx, np.random.default_rng(7), [333, 40], 14, 2, hd, v_gain=gain)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("gain", [1e-4, 8.0, 60.0])
def test_score_magnitudes(gh, gctx, hd, gain):
    check_decode(gh, gctx, np.random.default_rng(8), [333, 700], 14, 2, hd, k_gain=gain)


@pytest.mark.parametrize("q_gain", [1e-20, 1e-3, 1e5, 1e18])
def test_query_magnitudes(gh, gctx, q_gain):
    """Queries far outside fp16's range, with keys that keep the scores moderate
    (or the softmax flat or one-hot)."""
    rng = np.random.default_rng(9)
    cache = Cache(rng, [333, 20], 2, 64, k_gain=min(1.0, 1e3 / q_gain) if q_gain < 1e10 else 1.0)
    q = q_gain * rng.standard_normal((2, 14, 64))
    got = decode(gh, gctx, cache, q)
    for i in range(2):
        K, V = cache.lane(i)
        if q_gain < 1e10:
            hold(got[i], q[i], K, V)
            continue
        for h in range(14):  # a single key takes all the weight
            s = K[:, h // 7] @ q[i, h].astype(np.float32).astype(np.float64)
            assert np.allclose(got[i, h], V[s.argmax(), h // 7], rtol=2e-6, atol=0)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("broken", [np.nan, np.inf, -np.inf])
def test_a_broken_query_head_breaks_no_other(gh, gctx, hd, broken):
    rng = np.random.default_rng(19)
    ctx = [700, 90]
    cache = Cache(rng, ctx, 2, hd)
    q = rng.standard_normal((2, 14, hd))
    qr = rng.standard_normal((60, 14, hd))
    want, want_rows = decode(gh, gctx, cache, q), run_rows(gh, gctx, cache, qr, [20, 40])
    q[0, 9, 5] = broken
    qr[33, 3, 5] = broken
    got, got_rows = decode(gh, gctx, cache, q), run_rows(gh, gctx, cache, qr, [20, 40])
    assert np.isnan(got[0, 9]).all() and np.isnan(got_rows[33, 3]).all()
    want[0, 9], got[0, 9] = 0, 0
    want_rows[33, 3], got_rows[33, 3] = 0, 0
    assert np.array_equal(got, want) and np.array_equal(got_rows, want_rows)


@pytest.mark.parametrize("hd", [64, 128])
def test_a_peak_over_a_long_flat_tail(gh, gctx, hd):
    """One key far above 5000 others whose weights, e^-14 each, still add up to
    a part in 240 of the sum: none may be rounded away. The stored keys are
    whole numbers, so scores round once. Tolerance: n f32 additions to a running
    sum of about 1 round by 2^-24 at most each, n * 2^-24 = 3e-4, and the
    weights' own 2^-20 are far below; losing the tail costs 4e-3."""
    n, rng = 5001, np.random.default_rng(4)
    k = np.zeros((n, 1, hd), np.float32)
    k[:, 0, 0] = -15  # codes 0 and 15 of a group with step 1: exact
    k[1234, 0, 0] = 0
    v = np.concatenate([np.full((n, 1, hd // 2), 1.0), rng.standard_normal((n, 1, hd - hd // 2))], -1)
    v[1234] = -1.0
    q = np.zeros((1, 8, hd))
    q[:, :, 0] = 14.0 / 15 * np.sqrt(hd) * (1 + 0.01 * np.arange(8))
    cache = Cache(rng, [n], 1, hd, rows=(k, v))
    got = decode(gh, gctx, cache, q)
    want, _ = ref.attention(q[0].astype(np.float32), *cache.lane(0))
    err = float(np.abs(got[0] - want).max())
    assert err < n * 2.0 ** -24 * np.abs(want).max(), err
    assert np.abs(want[0, 0] + 1).min() > 0.004


@pytest.mark.parametrize("hd", [64, 128])
def test_rising_scores(gh, gctx, hd):
    """Every page raises the running maximum, by little and by much."""
    rng, n = np.random.default_rng(6), 900
    for rise in (0.01, 0.5, 6.0):
        k = 0.02 * rng.standard_normal((n, 1, hd))
        k[:, 0, 0] = np.linspace(0, rise * n / 16, n) / 8
        q = 0.1 * rng.standard_normal((1, 4, hd))
        q[:, :, 0] = 8 * np.sqrt(hd)
        cache = Cache(rng, [n], 1, hd, rows=(k, rng.standard_normal((n, 1, hd))))
        hold(decode(gh, gctx, cache, q)[0], q[0], *cache.lane(0))


def test_nan_groups_reach_their_own_lane_and_dims_alone(gh, gctx):
    """A NaN in one V group makes those 32 dims of the lanes that attend it NaN,
    one in K every output of the KV head's query heads; the rest is unmoved."""
    rng, hd = np.random.default_rng(11), 128
    ctx = [200, 300, 50]
    base = Cache(rng, ctx, 2, hd)
    q = rng.standard_normal((3, 14, hd))
    want = decode(gh, gctx, base, q)
    for which, lane, pos in ((1, 0, 130), (0, 1, 299)):
        cache = Cache(np.random.default_rng(11), ctx, 2, hd)
        slot = cache.slots[lane][pos]
        for kind in range(2):
            at = ref.half_place(kind, which, slot % 16, 1, hd)
            cache.pool[slot // 16, LAYER, 1, which, at:at + 2] = [0x00, 0x7E]
        got = decode(gh, gctx, cache, q)
        broken = np.zeros((3, 14, hd), bool)
        broken[lane, 7:, 32:64] = True
        if which == 0:
            broken[lane, 7:] = True
        assert np.isnan(got[broken]).all()
        assert np.array_equal(got[~broken], want[~broken])


@pytest.mark.parametrize("bad", [-1, 1 << 30, "count"])
def test_a_page_outside_the_pool_makes_its_lane_nan(gh, gctx, bad):
    rng = np.random.default_rng(12)
    ctx = [100, 400, 33]
    cache = Cache(rng, ctx, 2, 64)
    q = rng.standard_normal((3, 14, 64))
    want = decode(gh, gctx, cache, q)
    table = cache.table.copy()
    table[1, 24] = len(cache.pool) if bad == "count" else bad  # the lane's last page
    cache.td = _dev(table)
    got = decode(gh, gctx, cache, q)
    assert np.isnan(got[1]).all() and np.array_equal(got[[0, 2]], want[[0, 2]])
    n = 60
    qr = rng.standard_normal((n + 2, 14, 64))
    got = run_rows(gh, gctx, cache, qr, [1, n, 1])
    # rows of the lane that end before the bad page may be whole; those on it are NaN
    assert np.isnan(got[1 + n - 16:1 + n]).all() and np.isfinite(got[[0, n + 1]]).all()


def test_lengths_that_do_not_hold_make_their_lane_nan(gh, gctx):
    rng = np.random.default_rng(13)
    cache = Cache(rng, [100, 40, 33], 2, 64)
    q = rng.standard_normal((3, 14, 64))
    want = decode(gh, gctx, cache, q)
    for lens in ([100, -1, 33], [100, 113, 33], [100, 2 ** 31 - 1, 33], [100, -2 ** 31, 33]):
        got = decode(gh, gctx, cache, q, max_ctx=112, lens=lens)
        assert np.isnan(got[1]).all() and np.array_equal(got[[0, 2]], want[[0, 2]])
    # more rows than positions
    got = run_rows(gh, gctx, cache, rng.standard_normal((52, 14, 64)), [1, 50, 1])
    assert np.isnan(got[1:51]).all() and np.isfinite(got[[0, 51]]).all()


# ---- runs of rows ---------------------------------------------------------------------
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("pos0", [0, 1, 15, 16, 33, 47])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 33, 64, 97])
def test_chunk_edges(gh, gctx, hd, pos0, n):
    check_rows(gh, gctx, np.random.default_rng(n + 100 * pos0), [pos0 + n], [n], 14, 2, hd)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("G", [1, 2, 3, 4, 5, 6, 8])
def test_rows_group_sizes(gh, gctx, hd, G):
    check_rows(gh, gctx, np.random.default_rng(G), [171, 30], [150, 3], 2 * G, 2, hd)


@pytest.mark.parametrize("hd,heads,Hq", [(64, 2, 14), (128, 4, 28)])
def test_mixed_lanes(gh, gctx, hd, heads, Hq):
    """Single tokens, drafts, prompt chunks, idle and empty lanes, and unused
    rows behind the last."""
    ctx = [700, 0, 130, 64, 1500, 9, 257, 1, 900, 0]
    new = [1, 0, 5, 64, 1, 0, 100, 1, 37, 0]
    check_rows(gh, gctx, np.random.default_rng(hd), ctx, new, Hq, heads, hd, room=19)


@pytest.mark.parametrize("hd", [64, 128])
def test_few_rows_over_a_long_context(gh, gctx, hd):
    check_rows(gh, gctx, np.random.default_rng(3), [9000, 5000], [4, 1], 14, 2, hd)


def test_many_lanes_of_rows(gh, gctx):
    rng = np.random.default_rng(21)
    ctx = rng.integers(0, 80, 700)
    new = np.minimum(ctx, rng.integers(0, 4, 700))
    check_rows(gh, gctx, rng, ctx.tolist(), new.tolist(), 4, 2, 64)


def test_no_rows_at_all(gh, gctx):
    cache = Cache(np.random.default_rng(0), [40, 3], 2, 64)
    run_rows(gh, gctx, cache, np.zeros((0, 14, 64)), [0, 0], room=9)


def test_more_tiles_than_workgroups(gh, gctx):
    check_rows(gh, gctx, np.random.default_rng(5), [1100], [1095], 40, 8, 64)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("gain", [1e-6, 1e-3, 4000.0])
def test_rows_value_magnitudes(gh, gctx, hd, gain):
    check_rows(gh, gctx, np.random.default_rng(7), [133, 40], [100, 1], 14, 2, hd, v_gain=gain)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("gain", [1e-4, 8.0, 60.0])
def test_rows_score_magnitudes(gh, gctx, hd, gain):
    check_rows(gh, gctx, np.random.default_rng(8), [133, 140], [100, 2], 14, 2, hd, k_gain=gain)


@pytest.mark.parametrize("hd", [64, 128])
def test_a_nan_value_stays_out_of_earlier_rows(gh, gctx, hd):
    """A NaN V group at a position reaches no row before it, whatever tile they share."""
    rng = np.random.default_rng(14)
    n = 130
    q = rng.standard_normal((n, 14, hd))
    base = Cache(np.random.default_rng(15), [n], 2, hd)
    want = run_rows(gh, gctx, base, q, [n])
    for bad in (20, 50, 77):
        cache = Cache(np.random.default_rng(15), [n], 2, hd)
        slot = cache.slots[0][bad]
        for kind in range(2):
            at = ref.half_place(kind, 1, slot % 16, 0, hd)
            cache.pool[slot // 16, LAYER, 0, 1, at:at + 2] = [0x00, 0x7E]
        got = run_rows(gh, gctx, cache, q, [n])
        assert np.array_equal(got[:bad], want[:bad])
        assert np.isnan(got[bad:, :7, :32]).all()
        assert np.array_equal(got[:, 7:], want[:, 7:]) and np.isfinite(got[:, :7, 32:]).all()


def test_runs_that_do_not_lie_in_the_rows_leave_them(gh, gctx):
    """Overlapping runs (together more rows than there are) write nothing, a run
    outside the rows has none; the workspace needs no first value."""
    import torch

    rng = np.random.default_rng(16)
    cache = Cache(rng, [3000, 2900, 40], 2, 64)
    q = rng.standard_normal((50, 14, 64))
    ws = workspace(gh, 3, 50, 14, 2, 64)
    ws.fill_(255)
    want = run_rows(gh, gctx, cache, q, [20, 29, 1], ws=ws)
    for start, untouched in (([0, 40, 10, 50], slice(0, 50)), ([0, 50, 0, 50], slice(0, 50)),
                             ([-9, 20, 49, 50], slice(0, 20)), ([0, 20, 49, 51], slice(49, 50)),
                             ([0, 2 ** 31 - 1, -2 ** 31, 50], slice(0, 50)), ([-2 ** 31, 2 ** 31 - 1, 0, 0], slice(0, 50))):
        sd = _dev(np.array(start, np.int32))
        lens = _dev(np.array(cache.ctx, np.int32))
        qd, out = _dev(q.astype(np.float32)), torch.full((50, 14 * 64), 5.0, device="cuda")
        torch.cuda.synchronize()
        gh.check(gh.lib().glacier_hip_paged_attention_kv4_rows(
            gctx.h, cache.pool_t, LAYER, qd.data_ptr(), cache.td.data_ptr(), cache.table.shape[1], sd.data_ptr(),
            lens.data_ptr(), 3, 50, 14, cache.table.shape[1] * 16, out.data_ptr(), ws.data_ptr(), ws.numel(), None),
            "rows", gctx.h)
        torch.cuda.synchronize()
        got = out.cpu().numpy().reshape(50, 14, 64)
        assert (got[untouched] == 5.0).all()
    assert np.array_equal(run_rows(gh, gctx, cache, q, [20, 29, 1], ws=ws), want)


# ---- together --------------------------------------------------------------------------
def _serve(gh, gctx, seed, stream=None):
    """Three lanes through a prompt step and decode steps: plan, append, attend,
    lengths and free list carried on the device; returns (outputs, steps' rows)."""
    import torch

    rng = np.random.default_rng(seed)
    heads, Hq, hd, lanes, width, pages = 2, 14, 64, 3, 20, 60
    L, steps = gh.lib(), [[33, 5, 0]] + [[1, 1, 1]] * 6 + [[1, 0, 40]] + [[1, 4, 1]] * 3
    room = 64
    i32 = lambda *n, fill=0: torch.full(n, fill, dtype=torch.int32, device="cuda")  # noqa: E731
    pool = torch.full((pages, LAYERS, heads, 2, 10 * hd), 0x7E, dtype=torch.uint8, device="cuda")
    view = gh.Kv4Pool(pool.data_ptr(), pages, LAYERS, heads, hd)
    free = _dev(rng.permutation(pages).astype(np.int32))
    ctx, table, result = i32(lanes), i32(lanes, width, fill=-1), i32(4)
    start, slots = i32(lanes + 1), torch.zeros((room,), dtype=torch.int64, device="cuda")
    ws = workspace(gh, lanes, room, Hq, heads, hd)
    qkv = [_dev(rng.standard_normal((room, (Hq + 2 * heads) * hd)).astype(np.float32)) for _ in steps]
    outs = [torch.full((room, Hq * hd), 5.0, device="cuda") for _ in steps]
    news = [_dev(np.array(n, np.int32)) for n in steps]
    qs = [x[:, :Hq * hd].contiguous() for x in qkv]
    torch.cuda.synchronize()
    p = lambda t: t.data_ptr()  # noqa: E731
    for new, x, q, out in zip(news, qkv, qs, outs):
        gh.check(L.glacier_hip_kv_plan_rows(
            gctx.h, p(ctx), p(new), lanes, room, p(table), width, p(free), pages, p(result) + 12, p(start),
            p(ctx), p(slots), None, None, p(result), stream), "plan", gctx.h)
        gh.check(L.glacier_hip_kv4_append(
            gctx.h, view, LAYER, p(x) + Hq * hd * 4, p(x) + (Hq + heads) * hd * 4, gh.F32, x.stride(0),
            x.stride(0), p(slots), room, stream), "append", gctx.h)
        gh.check(L.glacier_hip_paged_attention_kv4_rows(
            gctx.h, view, LAYER, p(q), p(table), width, p(start), p(ctx), lanes, room, Hq, width * 16, p(out),
            p(ws), ws.numel(), stream), "rows", gctx.h)
    torch.cuda.synchronize()
    return steps, [x.cpu().numpy() for x in qkv], [o.cpu().numpy() for o in outs], (heads, Hq, hd)


def _hold_served(steps, qkv, outs, shape):
    heads, Hq, hd = shape
    K, V = [np.zeros((0, heads, hd))] * 3, [np.zeros((0, heads, hd))] * 3
    for new, x, out in zip(steps, qkv, outs):
        r = 0
        for i, n in enumerate(new):
            for _ in range(n):
                row = x[r].reshape(-1, hd)
                page = np.zeros((1, 1, heads, 2, 10 * hd), np.uint8)
                ref.store_rows(page, 0, np.array([3]), row[None, Hq:Hq + heads], row[None, Hq + heads:])
                k, v = ref.values(page, 0, np.array([3]))
                K[i], V[i] = np.concatenate([K[i], k]), np.concatenate([V[i], v])
                hold(out[r].reshape(Hq, hd), row[:Hq], K[i], V[i], what=(new, i))
                r += 1
        assert (out[r:] == 5.0).all()


def test_serving_steps(gh, gctx):
    _hold_served(*_serve(gh, gctx, 1))


def test_serving_steps_on_a_caller_stream(gh, gctx):
    import torch

    _hold_served(*_serve(gh, gctx, 2, stream=torch.cuda.Stream().cuda_stream))


def test_captured_step_replays(gh, gctx):
    """A decode step (plan, append, attention of one row a lane) captured once
    and replayed: every replay takes the device's lengths and pages on, eager
    work in between, each equal to the same steps run eagerly."""
    import torch

    heads, Hq, hd, lanes, width, pages, steps = 2, 14, 128, 4, 24, 96, 40
    L, rng = gh.lib(), np.random.default_rng(31)
    feed = rng.standard_normal((steps, lanes, (Hq + 2 * heads) * hd)).astype(np.float32)
    free = rng.permutation(pages).astype(np.int32)

    def serve(graph):
        i32 = lambda *n, fill=0: torch.full(n, fill, dtype=torch.int32, device="cuda")  # noqa: E731
        pool = torch.full((pages, LAYERS, heads, 2, 10 * hd), 0x7E, dtype=torch.uint8, device="cuda")
        view = gh.Kv4Pool(pool.data_ptr(), pages, LAYERS, heads, hd)
        fr, table, result = _dev(free), i32(lanes, width, fill=-1), i32(4)
        ctx, new, start = i32(lanes), i32(lanes, fill=1), i32(lanes + 1)
        slots = torch.zeros((lanes,), dtype=torch.int64, device="cuda")
        x = torch.zeros((lanes, (Hq + 2 * heads) * hd), device="cuda")
        q, out = torch.zeros((lanes, Hq * hd), device="cuda"), torch.zeros((lanes, Hq * hd), device="cuda")
        ws = workspace(gh, lanes, lanes, Hq, heads, hd)
        p = lambda t: t.data_ptr()  # noqa: E731
        torch.cuda.synchronize()

        def step(stream):
            gh.check(L.glacier_hip_kv_plan_rows(
                gctx.h, p(ctx), p(new), lanes, lanes, p(table), width, p(fr), pages, p(result) + 12, p(start),
                p(ctx), p(slots), None, None, p(result), stream), "plan", gctx.h)
            gh.check(L.glacier_hip_kv4_append(
                gctx.h, view, LAYER, p(x) + Hq * hd * 4, p(x) + (Hq + heads) * hd * 4, gh.F32, x.stride(0),
                x.stride(0), p(slots), lanes, stream), "append", gctx.h)
            gh.check(L.glacier_hip_paged_attention_kv4(
                gctx.h, view, LAYER, p(q), p(table), width, p(ctx), lanes, Hq, width * 16, p(out), p(ws),
                ws.numel(), stream), "decode", gctx.h)

        s = torch.cuda.Stream()
        g = None
        if graph:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                step(s.cuda_stream)
            torch.cuda.synchronize()
        got = []
        for t in range(steps):
            x.copy_(torch.from_numpy(feed[t]))
            q.copy_(x[:, :Hq * hd])
            torch.cuda.synchronize()
            if g is not None:
                g.replay()
            else:
                step(s.cuda_stream)
            torch.cuda.synchronize()
            got.append(out.cpu().numpy())
        return got, ctx.cpu().numpy(), table.cpu().numpy(), result.cpu().numpy()

    eager, replayed = serve(False), serve(True)
    for a, b in zip(eager[0], replayed[0]):
        assert np.array_equal(a, b)
    for a, b in zip(eager[1:], replayed[1:]):
        assert np.array_equal(a, b)
    assert (eager[1] == steps).all() and eager[3][0] == 0


def test_two_streams_with_a_workspace_each(gh, gctx):
    import torch

    rng = np.random.default_rng(41)
    caches = [Cache(rng, [3000, 700], 2, 128), Cache(rng, [1500, 2500], 2, 128)]
    qs = [rng.standard_normal((2, 14, 128)) for _ in range(2)]
    alone = [decode(gh, gctx, c, q) for c, q in zip(caches, qs)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    held = []
    for i in range(2):
        held.append((_dev(qs[i].astype(np.float32)), _dev(np.array(caches[i].ctx, np.int32)),
                     workspace(gh, 2, 2, 14, 2, 128), [torch.empty((2, 14 * 128), device="cuda") for _ in range(6)]))
    torch.cuda.synchronize()
    for r in range(6):
        for i in range(2):
            q, lens, ws, outs = held[i]
            gh.check(gh.lib().glacier_hip_paged_attention_kv4(
                gctx.h, caches[i].pool_t, LAYER, q.data_ptr(), caches[i].td.data_ptr(), caches[i].table.shape[1],
                lens.data_ptr(), 2, 14, caches[i].table.shape[1] * 16, outs[r].data_ptr(), ws.data_ptr(),
                ws.numel(), streams[i].cuda_stream), "decode", gctx.h)
    torch.cuda.synchronize()
    for i in range(2):
        for r in range(6):
            assert np.array_equal(held[i][3][r].cpu().numpy().reshape(2, 14, 128), alone[i])


def test_attention_in_pages_past_4_gib(gh, gctx):
    """Lanes whose pages lie in the last pages of an 11.5 GB pool."""
    import torch

    rng = np.random.default_rng(51)
    heads, hd, pages = 4, 128, 40000
    cache = Cache(rng, [300, 77], heads, hd)
    n = len(cache.pool)
    big = torch.zeros((pages, 28, heads, 2, 10 * hd), dtype=torch.uint8, device="cuda")
    big[-n:, LAYER] = _dev(cache.pool[:, LAYER])
    q = rng.standard_normal((2, 28, hd))
    want = decode(gh, gctx, cache, q)
    cache.pd, cache.td = big, _dev(np.where(cache.table < 0, cache.table, cache.table + pages - n))
    cache.pool_t = gh.Kv4Pool(big.data_ptr(), pages, 28, heads, hd)
    assert np.array_equal(decode(gh, gctx, cache, q), want)
    qr = rng.standard_normal((40, 28, hd))
    got = run_rows(gh, gctx, cache, qr, [37, 3])
    for r, (lane, end) in enumerate([(0, 264 + i) for i in range(37)] + [(1, 75 + i) for i in range(3)]):
        K, V = cache.lane(lane)
        hold(got[r], qr[r], K[:end], V[:end])
