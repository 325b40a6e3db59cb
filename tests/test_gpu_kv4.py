"""Plans, appends and reads of the 4-bit paged KV cache against their plain
forms. Plans, page bytes and read values are compared exactly: the quantiser's
roundings are all defined, and code * step + minimum takes one f32 rounding
(code * step has 15 bits)."""
import numpy as np
import pytest

import kv4_ref as ref

pytestmark = pytest.mark.gpu


def _dev(a):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


class _Plan:
    def __init__(self, ctx, new, max_rows, table, free, taken):
        import torch

        self.lanes, self.max_rows, self.width = len(ctx), max_rows, table.shape[1]
        self.ctx, self.new = _dev(np.array(ctx, np.int32)), _dev(np.array(new, np.int32))
        self.table, self.free = _dev(table), _dev(np.array(list(free) or [0], np.int32))
        self.count = len(free)
        self.result = torch.tensor([9, 9, 9, taken], dtype=torch.int32, device="cuda")
        i32 = lambda n: torch.full((n,), 77, dtype=torch.int32, device="cuda")  # noqa: E731
        self.start, self.after = i32(self.lanes + 1), i32(self.lanes)
        self.who, self.pos = i32(max_rows), i32(max_rows)
        self.slots = torch.full((max_rows,), 77, dtype=torch.int64, device="cuda")
        torch.cuda.synchronize()

    def run(self, gh, gctx, in_place=False, brief=False, stream=None):
        p = lambda t: t.data_ptr()  # noqa: E731
        gh.check(gh.lib().glacier_hip_kv_plan_rows(
            gctx.h, p(self.ctx), p(self.new), self.lanes, self.max_rows, p(self.table), self.width,
            p(self.free) if self.count else None, self.count, p(self.result) + 12, p(self.start),
            p(self.ctx) if in_place else p(self.after), p(self.slots), None if brief else p(self.who),
            None if brief else p(self.pos), p(self.result), stream), "plan", gctx.h)
        if stream is None:
            gctx.sync()
        return [t.cpu().numpy() for t in (self.table, self.start, self.ctx if in_place else self.after,
                                          self.slots, self.who, self.pos, self.result)]


def _table(rng, ctx, width, pool):
    table = np.full((len(ctx), width), -5, np.int32)
    perm = rng.permutation(pool).astype(np.int32)
    at = 0
    for i, c in enumerate(ctx):
        n = min(width, max(0, -(-c // 16)))
        table[i, :n] = perm[at:at + n]
        at += n
    return table, perm[at:]


PLANS = {
    "one token": ([5], [1], 1),
    "a new page": ([16], [1], 3),
    "from nothing": ([0], [17], 17),
    "idle lanes": ([0, 33, 0], [0, 0, 0], 4),
    "page ends": ([15, 16, 17, 31, 32, 0], [1, 1, 1, 2, 16, 32], 60),
    "a long prompt": ([3, 0, 700], [1, 5000, 1], 5100),
    "odd": ([40, 1, 999], [0, 300, 7], 307),
}


@pytest.mark.parametrize("name", PLANS)
@pytest.mark.parametrize("in_place", [False, True])
def test_plan(gh, gctx, name, in_place):
    ctx, new, room = PLANS[name]
    table, free = _table(np.random.default_rng(len(name)), ctx, 400, 1000)
    want = ref.plan(ctx, new, room, table, free, 2)
    got = _Plan(ctx, new, room, table, free, 2).run(gh, gctx, in_place)
    for w, g in zip(want, got):
        assert np.array_equal(w, g)


@pytest.mark.parametrize("lanes", [63, 64, 65, 512, 1024])
def test_plan_of_many_lanes(gh, gctx, lanes):
    rng = np.random.default_rng(lanes)
    ctx = rng.integers(0, 900, lanes).tolist()
    new = np.where(rng.random(lanes) < 0.1, rng.integers(0, 200, lanes), rng.integers(0, 2, lanes)).tolist()
    table, free = _table(rng, ctx, 80, 100000)
    want = ref.plan(ctx, new, sum(new) + 300, table, free, 11)
    got = _Plan(ctx, new, sum(new) + 300, table, free, 11).run(gh, gctx)
    for w, g in zip(want, got):
        assert np.array_equal(w, g)


def test_plan_without_lanes_and_positions_of_rows(gh, gctx):
    table, free = _table(np.random.default_rng(1), [9, 16], 4, 20)
    want = ref.plan([9, 16], [8, 2], 12, table, free, 0)
    got = _Plan([9, 16], [8, 2], 12, table, free, 0).run(gh, gctx, brief=True)
    for i in (0, 1, 2, 3, 6):
        assert np.array_equal(want[i], got[i])
    assert (got[4] == 77).all() and (got[5] == 77).all()


@pytest.mark.parametrize("ctx,new,room,width,free,taken,status", [
    ([5, -1], [1, 1], 4, 4, 9, 0, 1), ([5, 3], [1, -2], 4, 4, 9, 0, 1), ([5, 3], [3, 2], 4, 4, 9, 0, 1),
    ([5, 3], [2 ** 31 - 1, 2 ** 31 - 1], 4, 4, 9, 0, 1), ([60, 3], [5, 1], 9, 4, 9, 0, 8),
    ([2 ** 31 - 1, 3], [1, 1], 9, 4, 9, 0, 8), ([16, 32], [1, 1], 4, 4, 1, 0, 8), ([16, 32], [1, 1], 4, 4, 9, 8, 8),
    ([16, 32], [1, 1], 4, 4, 9, -1, 8), ([16], [1], 4, 4, 0, 0, 8), ([16, 32], [1, 1], 4, 4, 9, 2 ** 31 - 1, 8)])
def test_plan_that_does_not_hold_takes_nothing(gh, gctx, ctx, new, room, width, free, taken, status):
    table = np.arange(len(ctx) * width, dtype=np.int32).reshape(-1, width)
    pages = np.arange(100, 100 + free, dtype=np.int32)
    want = ref.plan(ctx, new, room, table, pages, taken)
    assert want[6][0] == status
    got = _Plan(ctx, new, room, table, pages, taken).run(gh, gctx)
    for w, g in zip(want, got):
        assert np.array_equal(w, g)


def test_plan_just_fits(gh, gctx):
    """The last table entry, the last free page and the last row."""
    table = np.full((2, 4), -1, np.int32)
    table[0, :3], table[1, :1] = [4, 9, 2], [7]
    want = ref.plan([48, 16], [16, 48], 64, table, [11, 12, 13, 14], 0)
    got = _Plan([48, 16], [16, 48], 64, table, [11, 12, 13, 14], 0).run(gh, gctx)
    assert want[6][0] == 0
    for w, g in zip(want, got):
        assert np.array_equal(w, g)


def test_plan_with_an_unset_page_gives_its_rows_no_slot(gh, gctx):
    table = np.full((2, 4), -1, np.int32)
    table[1, 0] = 3
    want = ref.plan([5, 5], [20, 2], 30, table, [8, 9], 0)
    got = _Plan([5, 5], [20, 2], 30, table, [8, 9], 0).run(gh, gctx)
    assert (want[3][:11] == -1).all()
    for w, g in zip(want, got):
        assert np.array_equal(w, g)


# ---- append and read ------------------------------------------------------------------
def _append(gh, gctx, pool, layer, k, v, kind, ks, vs, slots, rows, stream=None):
    pages, layers, heads, _, tile = pool.shape
    gh.check(gh.lib().glacier_hip_kv4_append(
        gctx.h, gh.Kv4Pool(pool.data_ptr(), pages, layers, heads, tile // 10), layer, k, v, kind, ks, vs,
        slots.data_ptr(), rows, stream), "append", gctx.h)
    if stream is None:
        gctx.sync()


def _read(gh, gctx, pool, layer, slots, rows, fill=5.0, stream=None):
    import torch

    pages, layers, heads, _, tile = pool.shape
    out = torch.full((2, rows, heads, tile // 10), fill, device="cuda")
    torch.cuda.synchronize()
    gh.check(gh.lib().glacier_hip_kv4_read(
        gctx.h, gh.Kv4Pool(pool.data_ptr(), pages, layers, heads, tile // 10), layer, slots.data_ptr(), rows,
        out[0].data_ptr(), out[1].data_ptr(), stream), "read", gctx.h)
    gctx.sync()
    return out.cpu().numpy()


def _rows(rng, n, width, kind):
    """f32 values that the kind holds exactly, as numpy and as the kind's tensor."""
    import torch

    x = torch.from_numpy(rng.standard_normal((n, width)).astype(np.float32) * 2.5)
    t = x.to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[kind])
    return t.float().numpy(), t


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,hd", [(1, 64), (2, 64), (3, 128), (4, 128)])
@pytest.mark.parametrize("rows,left,right", [(1, 0, 0), (7, 0, 0), (16, 64, 0), (37, 3, 5), (65, 8, 8), (200, 0, 1)])
def test_append_and_read(gh, gctx, kind, heads, hd, rows, left, right):
    """Bytes of every page and values of every slot, K and V as columns of one
    matrix with `left` columns before them and `right` after, a third of the
    rows without a slot or with one past the pool."""
    import torch

    rng = np.random.default_rng(rows * heads + hd + left)
    width, pages, layers = heads * hd, rows // 8 + 3, 3
    x, t = _rows(rng, rows, left + 2 * width + right, kind)
    t = t.cuda()
    slots = rng.permutation(pages * 16)[:rows].astype(np.int64)
    skip = rng.random(rows) < 0.33
    slots[skip] = rng.choice([-1, -16, pages * 16, 1 << 40], skip.sum())
    before = rng.integers(0, 256, (pages, layers, heads, 2, 10 * hd)).astype(np.uint8)
    want = before.copy()
    k, v = x[:, left:left + width].reshape(rows, heads, hd), x[:, left + width:left + 2 * width].reshape(rows, heads, hd)
    live = ~skip
    ref.store_rows(want, 1, slots[live], k[live], v[live])
    pool, sd = _dev(before), _dev(slots)
    torch.cuda.synchronize()
    at = t.data_ptr() + left * t.element_size()
    _append(gh, gctx, pool, 1, at, at + width * t.element_size(),
            {"f32": gh.F32, "f16": gh.F16, "bf16": gh.BF16}[kind], t.stride(0), t.stride(0), sd, rows)
    assert np.array_equal(pool.cpu().numpy(), want)
    got = _read(gh, gctx, pool, 1, sd, rows)
    assert (got[:, skip] == 5.0).all()
    for g, w in zip(got, ref.values(want, 1, slots[live])):
        assert np.array_equal(g[live], w.astype(np.float32))


@pytest.mark.parametrize("hd", [64, 128])
def test_append_a_prompt(gh, gctx, hd):
    """Whole pages in row order, as a prompt's rows come, from the middle of a page on."""
    import torch

    rng, heads, rows, first = np.random.default_rng(hd), 2, 1234, 11
    x, t = _rows(rng, rows, 2 * heads * hd, "f32")
    table = rng.permutation(90)[:79]
    pos = first + np.arange(rows)
    slots = (table[pos // 16] * 16 + pos % 16).astype(np.int64)
    want = np.full((90, 1, heads, 2, 10 * hd), 0x5A, np.uint8)
    pool = _dev(want)
    ref.store_rows(want, 0, slots, x[:, :heads * hd].reshape(rows, heads, hd), x[:, heads * hd:].reshape(rows, heads, hd))
    t, sd = t.cuda(), _dev(slots)
    torch.cuda.synchronize()
    _append(gh, gctx, pool, 0, t.data_ptr(), t.data_ptr() + heads * hd * 4, gh.F32, t.stride(0), t.stride(0), sd, rows)
    assert np.array_equal(pool.cpu().numpy(), want)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_append_at_rounding_borders(gh, gctx, kind):
    """Groups whose quotients sit on, just above and just below k + 1/2: ties
    go to the even code, neighbours to their own side."""
    import torch

    hd, rows = 64, 96
    rng = np.random.default_rng(3)
    step = np.float32(2.0) ** rng.integers(-8, 5, (rows, 1)).astype(np.float32)
    low = -step * rng.integers(0, 8, (rows, 1)).astype(np.float32)
    lv = rng.integers(0, 15, (rows, hd)).astype(np.float32) + 0.5
    x = (low + lv * step).astype(np.float32)
    nudge = rng.integers(-1, 2, x.shape)
    x = np.where(nudge == 0, x, np.nextafter(x, np.where(nudge > 0, np.inf, -np.inf).astype(np.float32)))
    x[:, 0::32], x[:, 1::32] = low, low + 15 * step  # the group's minimum and maximum
    t = torch.from_numpy(x).to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[kind]).cuda()
    x = t.float().cpu().numpy()
    want = np.zeros((6, 1, 1, 2, 10 * hd), np.uint8)
    slots = np.arange(rows, dtype=np.int64)
    ref.store_rows(want, 0, slots, x.reshape(rows, 1, hd), -x.reshape(rows, 1, hd))
    pool, neg, sd = torch.zeros(want.shape, dtype=torch.uint8, device="cuda"), -t, _dev(slots)
    torch.cuda.synchronize()
    _append(gh, gctx, pool, 0, t.data_ptr(), neg.data_ptr(), {"f32": gh.F32, "f16": gh.F16, "bf16": gh.BF16}[kind],
            hd, hd, sd, rows)
    assert np.array_equal(pool.cpu().numpy(), want)


def test_append_of_flat_tiny_huge_and_broken_groups(gh, gctx):
    """Constant groups, steps that fp16 rounds to zero, the largest magnitude
    that is stored, and groups with a NaN, an infinity or more than 32768."""
    import torch

    hd, cases = 64, []
    base = np.linspace(-1, 1, 32, dtype=np.float32)
    for g in (base * 0, base * 0 + 3.1415927, base * 1e-7, base * 1e-30, 1000 + base * 1e-3, base * 32768, -base * 0 - 32768):
        cases.append(g)
    for odd in (np.nan, np.inf, -np.inf, 32768.004, -40000.0, 3e38):
        g = base.copy()
        g[7] = odd
        cases.append(g)
    rows = len(cases)
    x = np.stack([np.concatenate([c, base]) for c in cases]).astype(np.float32)
    want = np.zeros((2, 1, 1, 2, 10 * hd), np.uint8)
    slots = np.arange(rows, dtype=np.int64)
    ref.store_rows(want, 0, slots, x.reshape(rows, 1, hd), x[:, ::-1].reshape(rows, 1, hd))
    t, u, sd = _dev(x), _dev(x[:, ::-1]), _dev(slots)
    pool = torch.zeros(want.shape, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    _append(gh, gctx, pool, 0, t.data_ptr(), u.data_ptr(), gh.F32, hd, hd, sd, rows)
    got = _read(gh, gctx, pool, 0, sd, rows)
    for g, w in zip(got, ref.values(want, 0, slots)):
        assert np.array_equal(g, w.astype(np.float32), equal_nan=True)
    assert np.isnan(got[0, 7:, 0, :32]).all() and np.isfinite(got[0, :, 0, 32:]).all()


def test_pages_past_4_gib(gh, gctx):
    """A pool of 40000 pages of 28 layers (11.5 GB), rows in its last page."""
    import torch

    heads, hd, layers, pages = 4, 128, 28, 40000
    pool = torch.zeros((pages, layers, heads, 2, 10 * hd), dtype=torch.uint8, device="cuda")
    rng = np.random.default_rng(0)
    x, t = _rows(rng, 16, 2 * heads * hd, "f32")
    slots = (pages - 1) * 16 + np.arange(16, dtype=np.int64)
    t, sd = t.cuda(), _dev(slots)
    torch.cuda.synchronize()
    _append(gh, gctx, pool, 27, t.data_ptr(), t.data_ptr() + heads * hd * 4, gh.F32, t.stride(0), t.stride(0), sd, 16)
    want = np.zeros((1, 1, heads, 2, 10 * hd), np.uint8)
    k, v = x[:, :heads * hd].reshape(16, heads, hd), x[:, heads * hd:].reshape(16, heads, hd)
    ref.store_rows(want, 0, np.arange(16), k, v)
    assert np.array_equal(pool[-1, 27].cpu().numpy(), want[0, 0])
    assert not pool[:-1, 27].any().item() and not pool[-1, :27].any().item()
    got = _read(gh, gctx, pool, 27, sd, 16)
    for g, w in zip(got, ref.values(want, 0, np.arange(16))):
        assert np.array_equal(g, w.astype(np.float32))
