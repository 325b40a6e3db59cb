"""Timed cases of the 4-bit paged KV cache: planning a step's pages and slots, storing rows, attention over the pages.

A case is a dict of plain values; its "kind" says which operators a pass runs:

* "plan": page tables, slots and row descriptors of one step from the lanes'
  lengths, glacier_hip_kv_plan_rows;
* "store": K and V rows quantised into their slots and read back as the values
  the pages now hold, glacier_hip_kv4_append and glacier_hip_kv4_read;
* "decode": one query row a lane, glacier_hip_paged_attention_kv4;
* "rows": runs of query rows of several lanes (prompt chunks, drafted tokens,
  single tokens side by side), causal, glacier_hip_paged_attention_kv4_rows.

Pages hold 16 positions of every layer, [layer][KV head][K, V][10 * head_dim
bytes]. In a tile (P position, NG = head_dim / 32 groups, NH = head_dim / 64):

* K codes: byte P * head_dim / 2 + (c * NG + g) * 4 + b holds dims
  32 g + 8 c + 2 b (low nibble) and + 1 of position P;
* V codes: byte ((((P / 4) * 16 + j) * 2 + P / 2 % 2) * NH + h) * 4 +
  P % 2 * 2 + b holds dims 16 (4 h + 2 b) + j (low nibble) and
  16 (4 h + 2 b + 1) + j;
* from byte 8 * head_dim on fp16 steps [P / 4][g][P % 4] of both; from byte
  9 * head_dim on fp16 minima, [P][g] in K tiles and [P / 4][g][P % 4] in V
  tiles.

A value is code * step + minimum of its position's group of 32 dims.
"""
import functools
import math
import os
import sys

import numpy as np
import torch

own = False

PAGE = 16
LAYERS = 28        # layers a page holds; the last one is stored and read
MAX_TABLE = 4352   # positions of a lane's page table where no context is longer


# ---- cases ----------------------------------------------------------------------------
def _geometry(name):
    """Query heads, KV heads and head_dim."""
    return {"7b": (28, 4, 128), "05b": (14, 2, 64), "mha": (4, 4, 128), "pairs": (4, 2, 64),
            "wide": (40, 8, 64), "eights": (32, 4, 128)}[name]


def _ints(text):
    return [int(v) for v in text.split(",")]


def listed():
    return [
        # one decode step of a small batch: a new row a lane, two of them on a new page
        dict(name="plan_8_lanes", kind="plan", ctx="37,130,512,1030,1999,2048,4000,5", new="1,1,1,1,1,1,1,1",
             room=8),
        # a step of continuous batching at full size: most lanes decode, some bring prompt
        # chunks, some are idle; a quarter of the row buffers stays unused
        dict(name="plan_512_lanes_mixed", kind="plan", ctx=",".join(str((i * 977) % 4001) for i in range(512)),
             new=",".join(str(0 if i % 7 == 3 else 251 if i % 16 == 5 else 1) for i in range(512)), room=11000),
        # the row of a batch-1 token of the small model
        dict(name="store_05b_1_row", kind="store", geometry="05b", rows=1, x="f32", pad=0, skip=0),
        # the rows of 32 decode lanes, each on a page of its own, taken out of a fused QKV output
        dict(name="store_7b_32_rows", kind="store", geometry="7b", rows=32, x="f32", pad=3584, skip=0),
        # a prompt chunk of odd length in bf16, its padding rows without a slot
        dict(name="store_7b_1999_rows_bf16", kind="store", geometry="7b", rows=2048, x="bf16", pad=0, skip=49),
        # a whole step of prompts
        dict(name="store_7b_16384_rows", kind="store", geometry="7b", rows=16384, x="f16", pad=0, skip=0),
        # one user's token of the small model at a short context
        dict(name="decode_05b_1_lane", kind="decode", geometry="05b", ctx="200"),
        # four users of very different contexts
        dict(name="decode_7b_4_lanes", kind="decode", geometry="7b", ctx="512,2048,4096,8192"),
        # a full batch of long, ragged contexts
        dict(name="decode_7b_32_lanes", kind="decode", geometry="7b",
             ctx=",".join(str(1 + (i * 5953 + 611) % 8192) for i in range(32))),
        # drafted tokens of six lanes verified in one step
        dict(name="rows_05b_6_lanes_draft", kind="rows", geometry="05b", ctx="37,130,517,1030,1999,4096",
             new="5,5,3,5,1,5"),
        # a mixed step: single tokens, a draft and two prompt chunks
        dict(name="rows_7b_8_lanes_mixed", kind="rows", geometry="7b", ctx="700,3001,64,1500,4096,257,909,2100",
             new="1,1,64,1,4,257,1,300"),
        # a fresh prompt in one chunk
        dict(name="rows_7b_prompt_2048", kind="rows", geometry="7b", ctx="2048", new="2048"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _text(values):
    return ",".join(str(v) for v in values)


def draw(rng):
    kind = rng.choice(["plan", "store", "store", "decode", "decode", "decode", "rows", "rows", "rows"])
    if kind == "plan":
        lanes = _log(rng, 1, 512)
        ctx = [rng.choice([0, _log(rng, 1, 4000)]) for _ in range(lanes)]
        new = [rng.choice([0, 1, 1, 1, 1, _log(rng, 2, 300)]) for _ in range(lanes)]
        while sum(new) > 10000:
            new[new.index(max(new))] = 1
        return dict(kind=kind, ctx=_text(ctx), new=_text(new), room=sum(new) + rng.choice([0, 1, 300]) or 1)
    if kind == "store":
        geometry, rows = rng.choice(["7b", "05b", "mha", "pairs", "wide"]), _log(rng, 1, 8000)
        return dict(kind=kind, geometry=geometry, rows=rows, x=rng.choice(["f32", "f16", "bf16"]),
                    pad=rng.choice([0, 0, 8, 896]), skip=rng.choice([0, 0, min(rows // 3, 40)]))
    geometry = rng.choice(["7b", "7b", "05b", "05b", "mha", "pairs", "wide", "eights"])
    if kind == "decode":
        while True:
            longest = _log(rng, 16, 20000)
            ctx = [rng.choice([0, 1, 16]) if rng.random() < 0.06 else _log(rng, 2, longest)
                   for _ in range(_log(rng, 1, 200))]
            # (the plain form pads every lane to the longest context)
            if 0 < len(ctx) * max(ctx) <= 200000:
                return dict(kind=kind, geometry=geometry, ctx=_text(ctx))
    while True:
        ctx, new = [], []
        for _ in range(_log(rng, 1, 24)):
            c = _log(rng, 1, 6000)
            ctx.append(c)
            new.append(min(c, rng.choice([0, 1, 1, 1, rng.randint(2, 8), rng.randint(2, 40), _log(rng, 16, 1200)])))
        # (the plain form pads every lane to the longest run and context)
        if 0 < len(ctx) * max(new) * max(ctx) <= 4000000:
            return dict(kind=kind, geometry=geometry, ctx=_text(ctx), new=_text(new))


# ---- the pages' layout ------------------------------------------------------------------
@functools.lru_cache(maxsize=None)
def _places(hd):
    """Byte places of a position in a K and a V tile, [2][16][hd / 2 + hd / 8] (codes in
    the order of _join, then steps and minima), on the GPU."""
    ng, nh = hd // 32, hd // 64
    at = np.zeros((2, 16, hd // 2 + hd // 8), dtype=np.int64)
    p = np.arange(16)[:, None]
    at[0, :, :hd // 2] = p * (hd // 2) + np.arange(hd // 2)
    j, h, b = (v.reshape(1, -1) for v in np.meshgrid(np.arange(16), np.arange(nh), np.arange(2), indexing="ij"))
    at[1, :, :hd // 2] = ((((p // 4) * 16 + j) * 2 + p // 2 % 2) * nh + h) * 4 + p % 2 * 2 + b
    g, b = (v.reshape(1, -1) for v in np.meshgrid(np.arange(ng), np.arange(2), indexing="ij"))
    quads = 2 * ((p // 4) * ng * 4 + g * 4 + p % 4) + b
    at[:, :, hd // 2:hd // 2 + 2 * ng] = 8 * hd + quads
    at[0, :, hd // 2 + 2 * ng:] = 9 * hd + 2 * (p * ng + g) + b
    at[1, :, hd // 2 + 2 * ng:] = 9 * hd + quads
    return torch.from_numpy(at).cuda()


def _quantise(x):
    """Codes [..., hd], steps and minima [..., hd / 32] (fp16) of f32 rows [..., hd]."""
    v = x.unflatten(-1, (-1, 32))
    lo, hi = v.amin(-1), v.amax(-1)
    step = ((hi - lo).double() / 15).float().half()
    low = lo.half()
    # a quotient next to a rounding border needs more than 32 bits
    d, w = step.double().unsqueeze(-1), v.double() - low.double().unsqueeze(-1)
    code = torch.where(d > 0, torch.round(w / torch.where(d > 0, d, 1.0)), 0.0).clamp(0, 15)
    return code.to(torch.uint8).flatten(-2), step, low


def _join(k, v):
    """Bytes [..., 2, hd / 2 + hd / 8] of quantised K and V rows (each codes, steps, minima)."""
    hd = k[0].shape[-1]
    kc = k[0].unflatten(-1, (hd // 32, 4, 4, 2)).transpose(-3, -4).flatten(-4, -2)  # [.., c g b, nibble]
    vc = v[0].unflatten(-1, (hd // 64, 2, 2, 16)).movedim(-1, -4).flatten(-4, -2)   # [.., j h b, nibble]
    rows = [torch.cat((c[..., 0] | (c[..., 1] << 4), s.contiguous().view(torch.uint8), m.contiguous().view(torch.uint8)), -1)
            for c, s, m in ((kc, k[1], k[2]), (vc, v[1], v[2]))]
    return torch.stack(rows, -2)


def _values(rows):
    """K and V values [..., hd] (f32) of bytes [..., 2, hd / 2 + hd / 8]."""
    hd = rows.shape[-1] * 8 // 5
    ng = hd // 32
    code = torch.stack((rows[..., :hd // 2] & 15, rows[..., :hd // 2] >> 4), -1).float()
    meta = rows[..., hd // 2:].contiguous().view(torch.float16).float()
    k = code[..., 0, :, :].unflatten(-2, (4, ng, 4)).transpose(-3, -4).flatten(-4)
    v = code[..., 1, :, :].unflatten(-2, (16, hd // 64, 2)).movedim(-4, -1).flatten(-4)
    step, low = meta[..., :ng].repeat_interleave(32, -1), meta[..., ng:].repeat_interleave(32, -1)
    return k * step[..., 0, :] + low[..., 0, :], v * step[..., 1, :] + low[..., 1, :]


def _slot_bytes(pool, slots):
    """Flat byte places [rows][KV heads][2][hd / 2 + hd / 8] of slots in the last layer."""
    pages, layers, heads, _, tile = pool.shape
    at = _places(tile // 10)[:, slots % PAGE].transpose(0, 1).unsqueeze(1)
    base = ((slots // PAGE * layers + layers - 1).unsqueeze(-1) * heads +
            torch.arange(heads, device="cuda")) * (2 * tile)
    return base[..., None, None] + torch.tensor([0, tile], device="cuda")[:, None] + at


def _lane_values(pool, table):
    """K and V [lanes][KV heads][positions][hd] (f32) of whole page tables."""
    tiles = pool[table.long(), -1]  # [lanes][pages][heads][2][tile]
    tile = tiles.shape[-1]
    at = _places(tile // 10).reshape(2, -1)
    rows = torch.stack((tiles[..., 0, :][..., at[0]], tiles[..., 1, :][..., at[1]]), -2)
    rows = rows.unflatten(-1, (PAGE, -1)).transpose(-2, -3)  # [lanes][pages][heads][16][2][bytes]
    k, v = _values(rows)
    return tuple(x.transpose(1, 2).flatten(2, 3) for x in (k, v))


# ---- inputs -----------------------------------------------------------------------------
def _gen(seed, what):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * int(seed) + what)
    return g


def _kv_rows(g, rows, heads, hd):
    """K rows with the uneven channels that rotary keys have, Gaussian V rows."""
    gain = torch.exp(0.6 * torch.randn((heads, hd), generator=g, device="cuda"))
    shift = torch.randn((heads, hd), generator=g, device="cuda")
    k = torch.randn((rows, heads, hd), generator=g, device="cuda") * gain + shift
    return k, torch.randn((rows, heads, hd), generator=g, device="cuda")


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _plan_inputs(case, seed):
    ctx, new = _ints(case["ctx"]), _ints(case["new"])
    g = _gen(seed, 1)
    width = -(-max([MAX_TABLE] + [c + n for c, n in zip(ctx, new)]) // PAGE)
    held = [-(-c // PAGE) for c in ctx]
    need = sum(-(-(c + n) // PAGE) for c, n in zip(ctx, new)) - sum(held)
    pages = torch.randperm(sum(held) + need + 50, generator=g, device="cuda").to(torch.int32)
    column = torch.arange(width, device="cuda")
    first = _int32(np.cumsum([0] + held)[:-1].tolist())
    table = torch.where(column < _int32(held)[:, None], pages[(first[:, None] + column).clamp(max=pages.numel() - 1)], -1)
    return dict(ctx=_int32(ctx), new=_int32(new), table=table.to(torch.int32).contiguous(),
                free=pages[sum(held):].contiguous(), taken=_int32([7]), room=case["room"])


def _store_inputs(case, seed):
    heads, hd = _geometry(case["geometry"])[1:]
    g, rows = _gen(seed, 2), case["rows"]
    k, v = _kv_rows(g, rows, heads, hd)
    dtype = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[case["x"]]
    # K and V as columns of one projection's output, `pad` columns of queries before them
    x = torch.zeros((rows, case["pad"] + 2 * heads * hd), dtype=dtype, device="cuda")
    k_rows, v_rows = x[:, case["pad"]:].split(heads * hd, 1)
    k_rows.copy_(k.view(rows, -1))
    v_rows.copy_(v.view(rows, -1))
    slots = torch.randperm(-(-rows // PAGE), generator=g, device="cuda")[:, None] * PAGE + torch.arange(PAGE, device="cuda")
    slots = slots.flatten()[:rows].contiguous()
    if rows <= 64:  # single tokens of as many lanes: a page each
        slots = torch.randperm(rows, generator=g, device="cuda") * PAGE + torch.randint(0, PAGE, (rows,), generator=g, device="cuda")
    pages = int(slots.amax()) // PAGE + 1
    if case["skip"]:
        slots[-case["skip"]:] = -1
    pool = torch.zeros((pages, LAYERS, heads, 2, 10 * hd), dtype=torch.uint8, device="cuda")
    return dict(k=k_rows, v=v_rows, slots=slots, pool=pool, heads=heads, hd=hd, kept=rows - case["skip"])


def _attention_inputs(case, seed):
    q_heads, heads, hd = _geometry(case["geometry"])
    ctx = _ints(case["ctx"])
    new = _ints(case["new"]) if case["kind"] == "rows" else [1] * len(ctx)
    g = _gen(seed, 3)
    held = [-(-c // PAGE) for c in ctx]
    total = max(1, sum(held))
    perm = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    width = max(1, max(held))
    first = _int32(np.cumsum([0] + held)[:-1].tolist())
    column = torch.arange(width, device="cuda")
    table = torch.where(column < _int32(held)[:, None], perm[(first[:, None] + column).clamp(max=total - 1)], 0)
    pool = torch.zeros((total, LAYERS, heads, 2, 10 * hd), dtype=torch.uint8, device="cuda")
    k, v = _kv_rows(g, total * PAGE, heads, hd)
    every = torch.arange(total * PAGE, device="cuda")
    pool.view(-1)[_slot_bytes(pool, every)] = _join(_quantise(k), _quantise(v))
    starts = np.cumsum([0] + new)
    q = 1.5 * torch.randn((int(starts[-1]), q_heads * hd), generator=g, device="cuda")
    return dict(q=q, pool=pool, table=table.to(torch.int32).contiguous(), ctx=_int32(ctx), new=_int32(new),
                starts=_int32(starts.tolist()), most=max(1, max(ctx)), longest=max(new), heads=heads, q_heads=q_heads,
                hd=hd)


def prepare(case, seed):
    make = {"plan": _plan_inputs, "store": _store_inputs}.get(case["kind"], _attention_inputs)
    return dict(make(case, seed), kind=case["kind"])


# ---- the plain forms --------------------------------------------------------------------
def _plain_plan(s):
    ctx, new, table, taken = s["ctx"].long(), s["new"].long(), s["table"], s["taken"].long()
    held, after = (ctx + PAGE - 1) // PAGE, (ctx + new + PAGE - 1) // PAGE
    need = after - held
    page_end, row_end = need.cumsum(0), new.cumsum(0)
    status = torch.where((ctx < 0).any() | (new < 0).any() | (row_end[-1] > s["room"]), 1,
                         torch.where((after > table.shape[1]).any() | (taken[0] + page_end[-1] > s["free"].numel()), 8, 0))
    good = status == 0
    column = torch.arange(table.shape[1], device="cuda")
    fresh = good & (column >= held[:, None]) & (column < after[:, None])
    source = taken + (page_end - need)[:, None] + column - held[:, None]
    table = torch.where(fresh, s["free"][source.clamp(0, s["free"].numel() - 1)], table)
    row = torch.arange(s["room"], device="cuda")
    lane = torch.searchsorted(row_end, row, right=True)
    live = good & (lane < ctx.numel())
    lane = lane.clamp(max=ctx.numel() - 1)
    position = ctx[lane] + row - (row_end - new)[lane]
    page = table[lane, (position // PAGE).clamp(0, table.shape[1] - 1)].long()
    starts = torch.where(good, torch.cat((torch.zeros_like(row_end[:1]), row_end)), 0)
    result = torch.stack((status, torch.where(good, row_end[-1], 0), torch.where(good, page_end[-1], 0),
                          taken[0] + torch.where(good, page_end[-1], 0)))
    return dict(table=table, starts=starts.int(), ctx=torch.where(good, ctx + new, ctx).int(),
                slots=torch.where(live & (page >= 0), page * PAGE + position % PAGE, -1),
                lanes=torch.where(live, lane, -1).int(), positions=torch.where(live, position, -1).int(),
                result=result.int())


def _plain_store(s):
    rows = s["slots"].numel()
    k, v = (_quantise(s[n].float().view(rows, s["heads"], s["hd"])) for n in ("k", "v"))
    at = _slot_bytes(s["pool"], s["slots"][:s["kept"]])
    s["pool"].view(-1)[at] = _join(k, v)[:s["kept"]]
    k, v = _values(s["pool"].view(-1)[at])
    return k.flatten(1), v.flatten(1)


def _plain_softmax(scores):
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(torch.isinf(top), 0.0, top))
    total = weights.sum(-1, keepdim=True)
    return weights / torch.where(total == 0, 1.0, total)


def _plain_attention(s):
    group, lanes = s["q_heads"] // s["heads"], s["ctx"].numel()
    k, v = _lane_values(s["pool"], s["table"])  # [lanes][heads][positions][hd]
    row = torch.arange(s["longest"], device="cuda")
    source = (s["starts"][:-1, None] + row).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][source].view(lanes, s["longest"], s["heads"], group, s["hd"])
    q = q.permute(0, 2, 3, 1, 4).reshape(lanes, s["heads"], group * s["longest"], s["hd"])
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(s["hd"])
    seen = s["ctx"][:, None] - s["new"][:, None] + row + 1  # positions that each row attends
    hidden = torch.arange(k.shape[2], device="cuda") >= seen[..., None]
    scores = scores.unflatten(2, (group, -1)).masked_fill_(hidden[:, None, None], -math.inf)
    out = torch.matmul(_plain_softmax(scores).flatten(2, 3), v)
    out = out.view(lanes, s["heads"], group, s["longest"], s["hd"]).permute(0, 3, 1, 2, 4).reshape(lanes, s["longest"], -1)
    at = torch.arange(s["q"].shape[0], device="cuda")
    lane = torch.searchsorted(s["starts"][1:].contiguous(), at, right=True)
    return out[lane, at - s["starts"][lane]]


# ---- the framework's calls --------------------------------------------------------------
@functools.lru_cache(maxsize=None)
def _framework():
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "glacier-engine_amd"))
    import glacier_hip as gh

    return gh, gh.Context(0)


@functools.lru_cache(maxsize=None)
def _workspace(size):
    """One zero-filled workspace a size, as a server keeps it for its steps."""
    return torch.zeros((max(1, size),), dtype=torch.uint8, device="cuda")


def _pool_of(gh, s):
    pages, layers, heads, _, tile = s["pool"].shape
    return gh.Kv4Pool(s["pool"].data_ptr(), pages, layers, heads, tile // 10)


def _calls(s):
    """The entry points of a pass with their arguments, and its outputs."""
    gh, ctx = _framework()
    lib, p = gh.lib(), lambda t: t.data_ptr()  # noqa: E731
    if s["kind"] == "plan":
        lanes, room = s["ctx"].numel(), s["room"]
        whole = lambda n, t=torch.int32: torch.empty((n,), dtype=t, device="cuda")  # noqa: E731
        out = dict(table=s["table"], starts=whole(lanes + 1), ctx=whole(lanes), slots=whole(room, torch.int64),
                   lanes=whole(room), positions=whole(room), result=whole(4))
        return [(lib.glacier_hip_kv_plan_rows, (
            ctx.h, p(s["ctx"]), p(s["new"]), lanes, room, p(s["table"]), s["table"].shape[1], p(s["free"]),
            s["free"].numel(), p(s["taken"]), p(out["starts"]), p(out["ctx"]), p(out["slots"]), p(out["lanes"]),
            p(out["positions"]), p(out["result"]), None))], out
    pool = _pool_of(gh, s)
    layer = s["pool"].shape[1] - 1
    if s["kind"] == "store":
        kind = {torch.float32: gh.F32, torch.float16: gh.F16, torch.bfloat16: gh.BF16}[s["k"].dtype]
        out = tuple(torch.empty((s["kept"], s["heads"] * s["hd"]), device="cuda") for _ in range(2))
        return [(lib.glacier_hip_kv4_append, (ctx.h, pool, layer, p(s["k"]), p(s["v"]), kind, s["k"].stride(0),
                                              s["v"].stride(0), p(s["slots"]), s["slots"].numel(), None)),
                (lib.glacier_hip_kv4_read, (ctx.h, pool, layer, p(s["slots"]), s["kept"], p(out[0]), p(out[1]),
                                            None))], out
    lanes, rows = s["ctx"].numel(), s["q"].shape[0]
    out = torch.empty_like(s["q"])
    space = _workspace(lib.glacier_hip_kv4_attention_workspace_bytes(lanes, rows, s["q_heads"], s["heads"], s["hd"]))
    head = (ctx.h, pool, layer, p(s["q"]), p(s["table"]), s["table"].shape[1])
    tail = (s["q_heads"], s["most"], p(out), p(space), space.numel(), None)
    if s["kind"] == "decode":
        return [(lib.glacier_hip_paged_attention_kv4, head + (p(s["ctx"]), lanes) + tail)], out
    return [(lib.glacier_hip_paged_attention_kv4_rows, head + (p(s["starts"]), p(s["ctx"]), lanes, rows) + tail)], out


def _framework_run(s):
    if "calls" not in s:
        s["calls"] = _calls(s)
    calls, out = s["calls"]
    for entry, args in calls:
        rc = entry(*args)
        if rc:
            gh, ctx = _framework()
            gh.check(rc, "perf case", ctx.h)
    return out


def run(state):
    if own:
        return _framework_run(state)
    if state["kind"] == "plan":
        return _plain_plan(state)
    if state["kind"] == "store":
        return _plain_store(state)
    return _plain_attention(state)


# ---- what a pass cannot do without --------------------------------------------------------
def work(case):
    if case["kind"] == "plan":
        ctx, new = _ints(case["ctx"]), _ints(case["new"])
        pages = sum(-(-(c + n) // PAGE) - -(-c // PAGE) for c, n in zip(ctx, new))
        return dict(bytes=16 * len(ctx) + 8 * pages + 16 * case["room"] + 24, flops=0)
    q_heads, heads, hd = _geometry(case["geometry"])
    if case["kind"] == "store":
        size, kept = 4 if case["x"] == "f32" else 2, case["rows"] - case["skip"]
        # rows in, pages out, pages in, values out
        return dict(bytes=int(kept * 2 * heads * hd * (size + 2 * 0.625 + 4)) + 16 * case["rows"], flops=0)
    ctx = _ints(case["ctx"])
    new = _ints(case["new"]) if case["kind"] == "rows" else [min(1, c) for c in ctx]
    attended = sum(n * (c - n) + n * (n + 1) // 2 for c, n in zip(ctx, new))
    read = sum(c for c, n in zip(ctx, new) if n)
    rows = sum(new) if case["kind"] == "rows" else len(ctx)
    return dict(bytes=int(2 * read * heads * hd * 0.625) + sum(-(-c // PAGE) * 4 for c in ctx) + 8 * rows * q_heads * hd,
                flops=4 * attended * q_heads * hd)


# ---- the definitions in 64 bits -----------------------------------------------------------
def exact(case, seed):
    def store():
        s = _store_inputs(case, seed)
        out = []
        for x in (s["k"], s["v"]):
            x = x[:s["kept"]].double().reshape(s["kept"], -1, 32)
            low = x.min(2, keepdim=True).values
            step = ((x.max(2, keepdim=True).values - low).float() / torch.tensor(15.0, device="cuda")).half().double()
            low = low.half().double()
            code = torch.floor((x - low) / step)
            for _ in range(2):  # up to the nearest, a tie to the even code
                rest = x - low - (code + 0.5) * step
                code = code + ((rest > 0) | ((rest == 0) & (code % 2 == 1))).double()
            out.append((low + step * code.clamp(0, 15)).view(s["kept"], -1))
        return tuple(out)

    def attention():
        s = _attention_inputs(case, seed)
        hd, group = s["hd"], s["q_heads"] // s["heads"]
        ng, nh = hd // 32, hd // 64
        q, out = s["q"].double().view(-1, s["q_heads"], hd), torch.zeros((s["q"].shape[0], s["q_heads"], hd), dtype=torch.float64, device="cuda")
        d, pos = torch.arange(hd, device="cuda"), torch.arange(PAGE, device="cuda")[:, None]
        at_k = pos * (hd // 2) + ((d % 32) // 8 * ng + d // 32) * 4 + d % 8 // 2
        block = d // 16
        at_v = ((((pos // 4) * 16 + d % 16) * 2 + pos // 2 % 2) * nh + block // 4) * 4 + pos % 2 * 2 + block % 4 // 2
        quad = (pos // 4) * ng * 4 + d // 32 * 4 + pos % 4
        flat = pos * ng + d // 32
        starts = s["starts"].tolist()
        for lane, c in enumerate(s["ctx"].tolist()):
            n = starts[lane + 1] - starts[lane]
            if c == 0 or n == 0:
                continue
            tiles = s["pool"][s["table"][lane, :-(-c // PAGE)].long(), LAYERS - 1]
            seen = torch.arange(c, device="cuda") <= torch.arange(c - n, c, device="cuda")[:, None]
            for h in range(s["heads"]):
                kv = []
                for which, at, shift, low_at in ((0, at_k, d % 2 * 4, flat), (1, at_v, block % 2 * 4, quad)):
                    t = tiles[:, h, which].contiguous()
                    code = (t[:, at].int() >> shift.int()) & 15
                    half = t[:, 8 * hd:].contiguous().view(torch.float16).double()
                    kv.append((code.double() * half[:, quad] + half[:, hd // 2 + low_at]).reshape(-1, hd)[:c])
                for j in range(h * group, (h + 1) * group):
                    scores = q[starts[lane]:starts[lane + 1], j] @ kv[0].t() * hd ** -0.5
                    weights = torch.softmax(torch.where(seen, scores, -math.inf), -1)
                    out[starts[lane]:starts[lane + 1], j] = weights @ kv[1]
        return out.view(-1, s["q_heads"] * hd)

    if case["kind"] == "plan":
        return None  # whole numbers only
    return store() if case["kind"] == "store" else attention()
