"""Performance cases of the 8-bit K/V cache: appending rows, attending over them, evicting blocks, in a caller's buffers.

The cache keeps, for each sequence and KV head, blocks of 32 positions as 8-bit codes (code - 128) * scale, one scale
for a block's K and one for its V, and the last len % 32 rows in fp16 (the tail). Blocks lie in slots; the table gives
the slot of each block in order. `mass` holds, by slot, the attention weight that a block has had.

Kinds of a case
  append  n rows of each sequence after `ctx` cached ones, and the same rows read back as attention sees them
  step    one decoding step of every sequence: its new row is appended, its query heads attend; with `track`, the
          weights that the blocks get are added to their mass
  chunk   n rows appended and n positions attending, each to its own row and those before it: a prompt's next part,
          or a few tokens to be verified at once
  evict   the blocks with the least mass leave, those at both ends stay

Types are the rows' and the outputs': f32 as the engine's activations, f16 as its cache. A pass begins from the same
state each time: the small arrays that a call changes (lengths, masses, tail, table) are copied back into place first,
as a program does that goes back to a position. Lengths are ragged where there are several sequences.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

B = 32  # positions of a block
F = {"f32": torch.float32, "f16": torch.float16}


def listed():
    return [
        # one token of a chat at its start: latency only
        dict(name="step_short", kind="step", dtype="f32", seqs=1, kv_heads=8, group=2, dim=64, ctx=100, max_len=512,
             track=False, evicted=False),
        # decode after 4096 positions, the shape and context of the package's benchmark, weights kept for eviction; the
        # new row closes its block
        dict(name="step_4127_track", kind="step", dtype="f32", seqs=1, kv_heads=8, group=3, dim=64, ctx=4127,
             max_len=4608, track=True, evicted=True),
        # one long document
        dict(name="step_long", kind="step", dtype="f16", seqs=1, kv_heads=8, group=3, dim=64, ctx=131000,
             max_len=131072, track=False, evicted=False),
        # eight long sequences decoding together: the cache is far larger than the last-level cache
        dict(name="step_batch_long", kind="step", dtype="f16", seqs=8, kv_heads=8, group=3, dim=64, ctx=100003,
             max_len=102400, track=True, evicted=True),
        # sixteen sequences, wider heads, f32
        dict(name="step_batch_wide", kind="step", dtype="f32", seqs=16, kv_heads=4, group=8, dim=128, ctx=6001,
             max_len=8192, track=False, evicted=False),
        # five drafted tokens verified for each of four sequences
        dict(name="chunk_verify", kind="chunk", dtype="f32", seqs=4, kv_heads=8, group=2, dim=64, ctx=2020, n=5,
             max_len=4096, track=False, evicted=False),
        # a page of text after a chat
        dict(name="chunk_page", kind="chunk", dtype="f32", seqs=1, kv_heads=8, group=3, dim=64, ctx=1000, n=300,
             max_len=2048, track=True, evicted=False),
        # part of a long document, fp16, the weights of its rows kept
        dict(name="chunk_document", kind="chunk", dtype="f16", seqs=1, kv_heads=8, group=3, dim=64, ctx=16001, n=1000,
             max_len=20480, track=True, evicted=False),
        # a short prompt's rows
        dict(name="append_short", kind="append", dtype="f32", seqs=1, kv_heads=8, group=1, dim=64, ctx=96, n=37,
             max_len=512, evicted=False),
        # a document's rows, read from a model's fp16 cache
        dict(name="append_document", kind="append", dtype="f16", seqs=2, kv_heads=8, group=1, dim=64, ctx=0, n=16391,
             max_len=32768, evicted=False),
        # a chat that has grown past its budget of half its blocks
        dict(name="evict_chat", kind="evict", seqs=1, kv_heads=8, group=3, dim=64, ctx=4500, max_len=4608, keep=64,
             first=1, last=8, evicted=True),
        # sixteen long sequences cut to a quarter
        dict(name="evict_long", kind="evict", seqs=16, kv_heads=8, group=3, dim=64, ctx=130000, max_len=131072,
             keep=1024, first=2, last=32, evicted=False),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["step", "step", "step", "chunk", "chunk", "append", "evict"])
    c = dict(kind=kind, seqs=_log(rng, 1, 16), kv_heads=rng.choice([1, 2, 4, 8]), group=rng.choice([1, 2, 3, 4, 6, 8]),
             dim=rng.choice([64, 64, 128]), evicted=rng.random() < 0.5)
    if kind == "evict":
        ctx = _log(rng, 32, 131072)
        nb = ctx // B
        keep = rng.randint(0, nb)
        first = rng.randint(0, min(2, keep))
        c.update(ctx=ctx, keep=keep, first=first, last=rng.randint(0, min(16, keep - first)))
        new = 0
    else:
        c["dtype"] = rng.choice(["f32", "f16"])
        row = c["seqs"] * c["kv_heads"] * c["dim"]
        if kind == "append":
            c.update(ctx=B * rng.randint(0, 64), n=_log(rng, 1, max(1, min(16384, (1 << 24) // row))))
        elif kind == "step":
            c.update(ctx=_log(rng, 1, max(64, min(131072, (1 << 28) // row))), n=1, track=rng.random() < 0.5)
        else:
            n = _log(rng, 2, 512)
            c.update(ctx=_log(rng, 1, max(64, min(16384, (1 << 27) // (row * c["group"] * n // 64)))), n=n,
                     track=rng.random() < 0.5)
        new = c["n"]
    c["max_len"] = B * (-(-(c["ctx"] + new) // B) + rng.randint(0, 64))
    return c


# ---- inputs ----------------------------------------------------------------------------------------------------
def _lengths(case):
    """Cached rows of each sequence: ctx, and down to 3/8 of it for the others; whole blocks before an append."""
    step = 1 if case["kind"] != "append" else B
    return [max(0, case["ctx"] - case["ctx"] * 5 * s // (8 * case["seqs"]) // step * step) for s in range(case["seqs"])]


def _shared(shapes, device):
    """Tensors over one buffer, each at a multiple of 256 bytes: one copy puts all of them back."""
    at, size = {}, 0
    for name, (shape, dtype) in shapes.items():
        at[name] = size
        size += -(-math.prod(shape) * dtype.itemsize // 256) * 256
    whole = torch.zeros(size, dtype=torch.uint8, device=device)
    return whole, {name: whole[at[name]:at[name] + math.prod(shape) * dtype.itemsize].view(dtype).view(shape)
                   for name, (shape, dtype) in shapes.items()}


def _inputs(case, seed):
    """The cache's arrays, and the rows and queries of a call."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    S, H, D, slots = case["seqs"], case["kv_heads"], case["dim"], case["max_len"] // B

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    small = dict(state=((S, 4), torch.int32), tail_bad=((S, H), torch.int32))
    if case.get("track") or case["kind"] == "evict":
        small["mass"] = ((S, H, slots), torch.float32)
    if case["kind"] == "evict":
        small["table"] = ((S, H, slots), torch.int32)
    else:
        small.update(k_tail=((S, H, B, D), torch.float16), v_tail=((S, H, B, D), torch.float16))
    whole, c = _shared(small, "cuda")
    lens = _lengths(case)
    c["state"][:, 0] = torch.tensor(lens, dtype=torch.int32)
    # a new cache's blocks lie in order; after evictions any slot may hold any block
    order = torch.argsort(uniform(S, H, slots), dim=2) if case["evicted"] else \
        torch.arange(slots, device="cuda").expand(S, H, slots)
    if "table" in c:
        c["table"].copy_(order)
    else:
        c["table"] = order.to(torch.int32).contiguous()
    if "mass" in c:
        # most blocks have little weight, a few have much; slots not in use have none
        used = torch.tensor([-(-n // B) for n in lens], device="cuda")[:, None, None]
        m = torch.exp(1.5 * normal(S, H, slots)) * (torch.arange(slots, device="cuda") < used)
        c["mass"].scatter_(2, c["table"].long(), m)
    else:
        c["mass"] = torch.zeros(S, H, slots, device="cuda")
    if case["kind"] == "evict":
        for name, shape, dtype in (("k_codes", (S, H, 1, B, D), torch.uint8), ("v_codes", (S, H, 1, B, D), torch.uint8),
                                   ("k_scale", (S, H, 1), torch.float32), ("v_scale", (S, H, 1), torch.float32),
                                   ("k_tail", (S, H, B, D), torch.float16), ("v_tail", (S, H, B, D), torch.float16)):
            c[name] = torch.zeros(shape, dtype=dtype, device="cuda")  # not read by an eviction
        return dict(case=case, whole=whole, first=whole.clone(), c=c)
    for name in ("k", "v"):
        codes = torch.empty(S, H, slots, B, D, dtype=torch.uint8, device="cuda")
        for s in range(S):
            codes[s] = (36.0 * normal(H, slots, B, D, dtype=torch.float16)).round().clamp(-127, 127) + 128.0
        c[name + "_codes"] = codes
        c[name + "_scale"] = (0.5 + uniform(S, H, slots)) / 36.0
        c[name + "_tail"].copy_(normal(S, H, B, D))
    n, dt = case.get("n", 1), F[case["dtype"]]
    state = dict(case=case, whole=whole, first=whole.clone(), c=c,
                 k=normal(S, n, H, D).to(dt), v=normal(S, n, H, D).to(dt))
    if case["kind"] == "append":
        state.update(k_out=torch.empty(S, n, H, D, dtype=dt, device="cuda"),
                     v_out=torch.empty(S, n, H, D, dtype=dt, device="cuda"))
    else:
        state["q"] = (2.0 * normal(S, n, H * case["group"], D)).to(dt)
        state["out"] = torch.empty_like(state["q"])
    return state


def prepare(case, seed):
    state = _inputs(case, seed)
    if own:
        at = os.path.join(os.getcwd(), "lastro-rust_amd")
        if at not in sys.path:
            sys.path.insert(0, at)
        import moert
        cache = moert.Kv8(case["seqs"], case["kv_heads"], case["dim"], case["max_len"],
                          {name: t.data_ptr() for name, t in state["c"].items()})
        state.update(cache=cache, rows=moert.F32 if case.get("dtype") == "f32" else moert.F16)
        if "q" in state:
            size = cache.workspace(case["kv_heads"] * case["group"], case.get("n", 1), track=case["track"])
            state.update(ws=torch.empty(size, dtype=torch.uint8, device="cuda"), ws_bytes=size)
    return state


# ---- one pass ---------------------------------------------------------------------------------------------------
def run(state):
    case, c = state["case"], state["c"]
    kind = case["kind"]
    state["whole"].copy_(state["first"])
    if own:
        cache = state["cache"]
        stream = torch.cuda.current_stream().cuda_stream
        n = case.get("n", 1)
        if kind == "evict":
            cache.evict(case["keep"], first=case["first"], last=case["last"], stream=stream)
        else:
            cache.append(state["k"].data_ptr(), state["v"].data_ptr(), n, dtype=state["rows"], stream=stream)
        if kind == "append":
            # the last n rows of each sequence
            cache.read(state["k_out"].data_ptr(), state["v_out"].data_ptr(), -n, n, dtype=state["rows"], stream=stream)
        elif kind != "evict":
            cache.attend(state["q"].data_ptr(), state["out"].data_ptr(), case["kv_heads"] * case["group"], n,
                         case["dim"] ** -0.5, state["ws"].data_ptr(), state["ws_bytes"], dtype=state["rows"],
                         mass_decay=1.0 if case["track"] else None, stream=stream)
    elif kind == "evict":
        _evict(case, c)
    else:
        _append(case, c, state["k"], state["v"])
        if kind == "append":
            _read(case, c, state["k_out"], state["v_out"])
        else:
            _attend(case, c, state["q"], state["out"])
    if kind == "evict":
        return dict(table=c["table"], mass=c["mass"], state=c["state"])
    if kind == "append":
        return dict(k=state["k_out"], v=state["v_out"], state=c["state"])
    out = dict(out=state["out"], k_scale=c["k_scale"], v_scale=c["v_scale"], k_tail=c["k_tail"], v_tail=c["v_tail"],
               state=c["state"])
    if case["track"]:
        out["mass"] = c["mass"]
    return out


def _where_v(D):
    """Position in a block of V of (position t, element e): a lane's 8 positions of an element side by side."""
    U = D // 16
    t, e = torch.meshgrid(torch.arange(B, device="cuda"), torch.arange(D, device="cuda"), indexing="ij")
    return (((e // U * 4 + t % 16 // 4) * U + e % U) * 8 + t % 4 + 4 * (t // 16)).reshape(-1)


def _rows_of_v(blocks):
    """Blocks of V [.., B, D], as the cache lays them out, as rows."""
    D = blocks.shape[-1]
    U = D // 16
    x = blocks.reshape(*blocks.shape[:-2], 16, 4, U, 2, 4)  # element / U, group, element % U, half, position in group
    k = x.dim() - 5
    return x.permute(*range(k), k + 3, k + 1, k + 4, k, k + 2).reshape(blocks.shape)


def _blocks_of_v(rows):
    """Rows [.., B, D] as a block of V."""
    D = rows.shape[-1]
    x = rows.reshape(*rows.shape[:-2], 2, 4, 4, 16, D // 16)  # half, group, position in group, element / U, element % U
    k = x.dim() - 5
    return x.permute(*range(k), k + 3, k + 1, k + 4, k, k + 2).reshape(rows.shape)


def _append(case, c, k, v):
    S, H, D, n = case["seqs"], case["kv_heads"], case["dim"], k.shape[1]
    length = c["state"][:, 0].long()
    old, tail = length // B, length % B
    whole = (tail + n) // B  # blocks that are full now
    most = (B - 1 + n) // B
    span = torch.arange(B + n, device="cuda")
    from_tail = span[None, :] < tail[:, None]
    new = (span[None, :] - tail[:, None]).clamp(0, n - 1)[:, None, :, None].expand(S, H, B + n, D)
    s_at, b_at = torch.nonzero(torch.arange(most, device="cuda")[None, :] < whole[:, None], as_tuple=True)
    slot = c["table"].long()[s_at, :, old[s_at] + b_at]  # [blocks, H]
    t = torch.arange(B, device="cuda")[None, :]
    left = (tail + n) % B
    wrote = torch.where(whole[:, None] > 0, t < left[:, None], (t >= tail[:, None]) & (t < (tail + n)[:, None]))
    at = (whole[:, None] * B + t).clamp(max=B + n - 1)[:, None, :, None].expand(S, H, B, D)
    heads = torch.arange(H, device="cuda")[None, :]
    for name, rows in (("k", k), ("v", v)):
        held = c[name + "_tail"] if name == "k" else _rows_of_v(c["v_tail"])
        rows = torch.cat([rows.half().transpose(1, 2), held], 2)  # [S, H, n + B, D]
        rows = torch.gather(rows, 2, torch.where(from_tail[:, None, :, None], n + span[None, None, :, None], new))
        full = rows[:, :, :most * B].reshape(S, H, most, B, D)[s_at, :, b_at].double()  # [blocks, H, B, D]
        scale = (full.abs().amax((2, 3)) / 127.0).float()
        scale = torch.where(scale == 0, torch.ones_like(scale), scale)
        codes = (torch.round(full / scale.double()[:, :, None, None]) + 128.0).to(torch.uint8)
        c[name + "_codes"][s_at[:, None], heads, slot] = codes if name == "k" else _blocks_of_v(codes)
        c[name + "_scale"][s_at[:, None], heads, slot] = scale
        held = torch.where(wrote[:, None, :, None], torch.gather(rows, 2, at), held)
        c[name + "_tail"].copy_(held if name == "k" else _blocks_of_v(held))
    c["state"][:, 0] += n


def _unpack(case, c, blocks):
    """K and V [S, H, blocks * B, D] of the first blocks of every sequence in f32, the tail among them."""
    S, H, D = case["seqs"], case["kv_heads"], case["dim"]
    slot = c["table"][:, :, :blocks].long()
    s_at, h_at = torch.arange(S, device="cuda")[:, None, None], torch.arange(H, device="cuda")[None, :, None]
    length = c["state"][:, 0].long()
    has_tail = torch.nonzero(length % B, as_tuple=True)[0]
    got = []
    for name in ("k", "v"):
        x = (c[name + "_codes"][s_at, h_at, slot].float() - 128.0) * c[name + "_scale"][s_at, h_at, slot][..., None, None]
        x[has_tail, :, length[has_tail] // B] = c[name + "_tail"][has_tail].float()
        got.append((x if name == "k" else _rows_of_v(x)).reshape(S, H, blocks * B, D))
    return got


def _read(case, c, k_out, v_out):
    n = k_out.shape[1]
    length = c["state"][:, 0].long()
    k, v = _unpack(case, c, -(-(case["ctx"] + n) // B))
    at = (length[:, None] - n + torch.arange(n, device="cuda"))[:, None, :, None].expand(-1, k.shape[1], -1, k.shape[3])
    k_out.copy_(torch.gather(k, 2, at).transpose(1, 2))
    v_out.copy_(torch.gather(v, 2, at).transpose(1, 2))


def _attend(case, c, q, out):
    S, H, G, D, n = case["seqs"], case["kv_heads"], case["group"], case["dim"], q.shape[1]
    blocks = -(-(case["ctx"] + n) // B)
    k, v = _unpack(case, c, blocks)
    length = c["state"][:, 0].long()
    x = q.float().reshape(S, n, H, G, D).permute(0, 2, 1, 3, 4).reshape(S, H, n * G, D) * case["dim"] ** -0.5
    sees = length[:, None] - n + 1 + torch.arange(n, device="cuda").repeat_interleave(G)[None, :]  # rows of each query
    s = torch.matmul(x, k.transpose(2, 3).contiguous())
    s.masked_fill_(torch.arange(blocks * B, device="cuda")[None, None, None, :] >= sees[:, None, :, None], -math.inf)
    p = torch.exp(s - s.amax(3, keepdim=True))
    # sums over the positions block by block first: one long f32 chain loses what the type holds
    wide = torch.float64 if case["dtype"] == "f32" and blocks * B > 2048 else torch.float32
    total = p.reshape(S, H, n * G, blocks, B).sum(4)
    share = 1.0 / total.sum(3, keepdim=True)
    o = torch.matmul(p.to(wide), v.to(wide)).float() * share
    out.copy_(o.reshape(S, H, n, G, D).permute(0, 2, 1, 3, 4).reshape(S, n, H * G, D))
    if case["track"]:
        w = (total * share).sum(2)  # [S, H, blocks], 0 behind a sequence's rows
        c["mass"].scatter_add_(2, c["table"][:, :, :blocks].long(), w)


def _evict(case, c):
    S, H, slots = c["table"].shape
    keep, first, last = case["keep"], case["first"], case["last"]
    table = c["table"].long()
    whole = (c["state"][:, 0].long() // B)[:, None, None]
    at = torch.arange(slots, device="cuda")[None, None, :]
    m = torch.gather(c["mass"], 2, table)
    free = (at >= first) & (at < whole - last)
    # rank among the blocks that may leave: by mass, the lower index first among equals
    order = torch.argsort(torch.where(free, m, torch.full_like(m, -1.0)), dim=2, descending=True, stable=True)
    rank = torch.empty_like(order).scatter_(2, order, at.expand(S, H, slots).contiguous())
    leaves = free & (rank >= keep - first - last) & (whole > keep)
    tail = (at == whole) & ((c["state"][:, 0].long() % B)[:, None, None] > 0)
    # kept blocks in order, the tail's slot, those that left, those not in use
    kind = torch.where(leaves, 2, torch.where(at < whole, 0, torch.where(tail, 1, 3)))
    moved = torch.argsort(kind, dim=2, stable=True)
    c["mass"].scatter_(2, table, torch.where(leaves, torch.zeros_like(m), m))
    c["table"].copy_(torch.gather(table, 2, moved))
    c["state"][:, 0] -= (B * (whole[:, 0, 0] - keep).clamp(min=0)).to(torch.int32)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------
def work(case):
    S, H, G, D, n = case["seqs"], case["kv_heads"], case["group"], case["dim"], case.get("n", 1)
    lens = _lengths(case)
    if case["kind"] == "evict":
        # a mass and a table entry of each block read, the entry and what leaves written
        nb = sum(x // B for x in lens)
        return dict(bytes=H * (12 * nb + 4 * max(0, nb - S * case["keep"])) + 8 * S, flops=0)
    size = 4 if case["dtype"] == "f32" else 2
    rows = 2 * S * n * H * D
    if case["kind"] == "append":
        return dict(bytes=rows * (2 * size + 2), flops=4 * rows)  # read, coded, the codes read, written
    cached = 2 * H * D * sum(lens) + 8 * H * sum(-(-x // B) for x in lens)  # codes and scales; new rows come as inputs
    seen = sum(x + i + 1 for x in lens for i in range(n))
    mass = 8 * H * sum(-(-(x + n) // B) for x in lens) if case["track"] else 0
    return dict(bytes=rows * (size + 1) + cached + mass + 2 * S * n * H * G * D * size, flops=4 * H * G * D * seen)


# ---- the same in 64 bits -------------------------------------------------------------------------------------------
def exact(case, seed):
    """From the definition, one sequence after the other."""
    st = _inputs(case, seed)
    c, lens = st["c"], _lengths(case)
    if case["kind"] == "evict":
        mass, table = (c[name].cpu().numpy().astype(np.float64) for name in ("mass", "table"))
        for s, L in enumerate(lens):
            leave = max(0, L // B - case["keep"])
            for h in range(case["kv_heads"] if leave else 0):
                slots = table[s, h, case["first"]:L // B - case["last"]].astype(np.int64)
                # the least first, of equals the later one
                mass[s, h, slots[np.lexsort((-np.arange(slots.size), mass[s, h, slots]))[:leave]]] = 0.0
        return dict(table=None, mass=mass, state=None)
    S, H, G, D, n = case["seqs"], case["kv_heads"], case["group"], case["dim"], case.get("n", 1)
    if case["kind"] != "append" and 4.0 * n * H * G * D * sum(lens) > 2e12:
        return None
    place = _where_v(D)
    got = dict(k=[], v=[]) if case["kind"] == "append" else dict(out=[])
    scales = {name: c[name + "_scale"].double() for name in "kv"}
    mass = c["mass"].double()
    for s in range(S):
        L = lens[s]
        old = L // B
        slots = c["table"][s].long()
        heads = torch.arange(H, device="cuda")[:, None]
        rows = {}
        for name in "kv":
            def plain(x):
                return x if name == "k" else x.flatten(-2)[..., place].reshape(x.shape)
            cached = (plain(c[name + "_codes"][s][heads, slots[:, :old]]).double() - 128) * \
                scales[name][s][heads, slots[:, :old]][..., None, None]
            fresh = torch.cat([plain(c[name + "_tail"][s])[:, :L % B], st[name][s].half().transpose(0, 1)], 1).double()
            for b in range(fresh.shape[1] // B):
                x = fresh[:, b * B:(b + 1) * B]
                amax = x.abs().amax((1, 2))
                one = torch.where(amax > 0, (amax / 127).float().double(), torch.ones_like(amax))
                scales[name][s][heads[:, 0], slots[:, old + b]] = one
                fresh[:, b * B:(b + 1) * B] = torch.round(x / one[:, None, None]) * one[:, None, None]
            rows[name] = torch.cat([cached.reshape(H, old * B, D), fresh], 1)
        if case["kind"] == "append":
            for name in "kv":
                got[name].append(rows[name][:, L:].transpose(0, 1))
            continue
        out = torch.empty(n, H, G, D, dtype=torch.float64, device="cuda")
        weight = torch.zeros(H, old + (L % B + n + B - 1) // B, dtype=torch.float64, device="cuda")
        hide = torch.arange(L + n, device="cuda")[None, :] > L + torch.arange(n, device="cuda")[:, None]
        for h in range(H):
            for j in range(G):
                a = (st["q"][s, :, h * G + j].double() * D ** -0.5) @ rows["k"][h].T.contiguous()
                a = torch.softmax(a.masked_fill(hide, -math.inf), 1)
                out[:, h, j] = a @ rows["v"][h]
                w = torch.nn.functional.pad(a.sum(0), (0, weight.shape[1] * B - (L + n)))
                weight[h] += w.reshape(-1, B).sum(1)
        got["out"].append(out.reshape(n, H * G, D))
        mass[s][heads, slots[:, :weight.shape[1]]] += weight
    got = {name: torch.stack(x).cpu().numpy() for name, x in got.items()}
    if case["kind"] == "append":
        return dict(**got, state=None)
    got.update(k_scale=scales["k"].cpu().numpy(), v_scale=scales["v"].cpu().numpy(), k_tail=None, v_tail=None, state=None)
    if case["track"]:
        got["mass"] = mass.cpu().numpy()
    return {name: None if x is None else np.asarray(x) for name, x in got.items()}
