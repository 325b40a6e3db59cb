"""Plain forms of the 4-bit paged KV operators in numpy: the quantiser and the
page layout of glacier_hip.h byte by byte, the plan, and attention in 64 bits."""
import numpy as np

PAGE = 16


def quantise(x):
    """x [..., 32] f32 -> codes (uint8), step, minimum (fp16)."""
    x = np.asarray(x, dtype=np.float32)
    with np.errstate(all="ignore"):
        bad = ~(np.abs(x) <= np.float32(32768.0)).all(-1)
        lo, hi = x.min(-1), x.max(-1)
        step = ((hi - lo) / np.float32(15.0)).astype(np.float16)
        low = lo.astype(np.float16)
        step[bad], low[bad] = np.nan, np.nan
        d = step.astype(np.float64)[..., None]
        t = x.astype(np.float64) - low.astype(np.float64)[..., None]
        code = np.where(d > 0, np.clip(np.rint(t / np.where(d > 0, d, 1.0)), 0, 15), 0)
    return np.nan_to_num(code).astype(np.uint8), step, low


def tile_bytes(hd):
    return 10 * hd


def code_place(which, P, d, hd):
    """(byte, shift) of dim d of position P in a K (0) or V (1) tile's codes."""
    ng, nh = hd // 32, hd // 64
    if which == 0:
        g, c, b, high = d // 32, d % 32 // 8, d % 8 // 2, d % 2
        return P * hd // 2 + (c * ng + g) * 4 + b, 4 * high
    j, block = d % 16, d // 16
    h, b, high = block // 4, block % 4 // 2, block % 2
    return (((P // 4 * 16 + j) * 2 + P // 2 % 2) * nh + h) * 4 + P % 2 * 2 + b, 4 * high


def half_place(kind, which, P, g, hd):
    """Byte of the step (kind 0) or minimum (kind 1) of group g of position P."""
    ng = hd // 32
    if kind == 1 and which == 0:
        return 9 * hd + 2 * (P * ng + g)
    return (8 + kind) * hd + 2 * (P // 4 * ng * 4 + g * 4 + P % 4)


_tables = {}


def tables(hd):
    if hd not in _tables:
        code = np.zeros((2, PAGE, hd, 2), np.int64)
        half = np.zeros((2, PAGE, 2, hd // 32), np.int64)
        for w in range(2):
            for P in range(PAGE):
                for d in range(hd):
                    code[w, P, d] = code_place(w, P, d, hd)
                for kind in range(2):
                    for g in range(hd // 32):
                        half[w, P, kind, g] = half_place(kind, w, P, g, hd)
        _tables[hd] = code, half
    return _tables[hd]


def store_rows(pool, layer, slots, k, v):
    """Write rows (k, v [n][heads][hd] f32) into pool [pages][layers][heads][2][10 hd] u8."""
    n, heads, hd = k.shape
    code, half = tables(hd)
    P, flat = slots % PAGE, pool.reshape(-1)
    assert np.shares_memory(flat, pool)
    for w, x in ((0, k), (1, v)):
        c, step, low = quantise(x.reshape(n, heads, hd // 32, 32))
        c = c.reshape(n, heads, hd)
        base = ((slots[:, None] // PAGE * pool.shape[1] + layer) * heads + np.arange(heads)) * 2 + w
        base = base[..., None] * (10 * hd)
        at = code[w][P][:, None]  # [n][1][hd][byte, shift]
        for shift in (0, 4):
            d = np.nonzero(code[w, 0, :, 1] == shift)[0]
            place = base + at[:, :, d, 0]
            flat[place] = c[:, :, d] if shift == 0 else flat[place] | c[:, :, d] << 4
        for kind, m in ((0, step), (1, low)):
            raw = np.ascontiguousarray(m).view(np.uint8).reshape(n, heads, hd // 32, 2)
            place = base + half[w][P][:, None, kind]
            flat[place], flat[place + 1] = raw[..., 0], raw[..., 1]


def values(pool, layer, slots):
    """K, V [slots][heads][hd] f64 stored at slots."""
    hd = pool.shape[-1] // 10
    code, half = tables(hd)
    out = []
    for w in range(2):
        t = pool[slots // PAGE, layer, :, w]  # [n][heads][10 hd]
        P = slots % PAGE
        at, half_at = code[w][P][:, None], half[w][P]
        c = np.take_along_axis(t, np.broadcast_to(at[..., 0], t.shape[:2] + at.shape[2:3]), -1)
        c = c >> at[..., 1].astype(np.uint8) & 15
        m = []
        for kind in range(2):
            b = np.broadcast_to(half_at[:, None, kind], t.shape[:2] + half_at.shape[2:3])
            raw = np.stack([np.take_along_axis(t, b, -1), np.take_along_axis(t, b + 1, -1)], -1)
            m.append(np.repeat(np.ascontiguousarray(raw).view(np.float16)[..., 0].astype(np.float64), 32, -1))
        out.append(c * m[0] + m[1])
    return out


def plan(ctx, new, max_rows, table, free, taken):
    """kv_plan_rows: (table, row_start, ctx_after, slots, lanes, positions, result)."""
    table = table.copy()
    lanes = len(ctx)
    slots = np.full(max_rows, -1, np.int64)
    who, pos = np.full(max_rows, -1, np.int32), np.full(max_rows, -1, np.int32)
    pages = [-(-(c + n) // PAGE) - -(-c // PAGE) for c, n in zip(ctx, new)]
    status = 0
    if min(ctx) < 0 or min(new) < 0 or sum(new) > max_rows:
        status = 1
    elif any(c + n > table.shape[1] * PAGE for c, n in zip(ctx, new)) or taken < 0 or \
            taken + sum(pages) > len(free):
        status = 8
    if status:
        return table, np.zeros(lanes + 1, np.int32), np.array(ctx, np.int32), slots, who, pos, \
            np.array([status, 0, 0, taken], np.int32)
    start, at = [0], taken
    for i in range(lanes):
        held = -(-ctx[i] // PAGE)
        table[i, held:held + pages[i]] = free[at:at + pages[i]]
        at += pages[i]
        for k in range(new[i]):
            r, p = start[-1] + k, ctx[i] + k
            who[r], pos[r] = i, p
            if table[i, p // PAGE] >= 0:
                slots[r] = int(table[i, p // PAGE]) * PAGE + p % PAGE
        start.append(start[-1] + new[i])
    return table, np.array(start, np.int32), np.array(ctx, np.int32) + np.array(new, np.int32), slots, \
        who, pos, np.array([0, start[-1], sum(pages), at], np.int32)


def attention(q, K, V):
    """One row: q [Hq][hd] f32 against K, V [n][heads][hd] f64; also the largest |score|."""
    Hq, hd = q.shape
    G = Hq // K.shape[1]
    out, top = np.zeros((Hq, hd)), 0.0
    if len(K) == 0:
        return out, top
    for h in range(Hq):
        s = K[:, h // G] @ q[h].astype(np.float64) / np.sqrt(hd)
        top = max(top, float(np.abs(s).max()))
        w = np.exp(s - s.max())
        out[h] = w @ V[:, h // G] / w.sum()
    return out, top
