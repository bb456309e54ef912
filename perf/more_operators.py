"""Performance cases of a paged K/V cache in 16 bits that many sequences share: planning a step's pages, appending rows,
attention of one new position, attention of whole prompts, all over a caller's buffers.

The pool holds pages of `page` positions; the table names the pages of each sequence in order. Within a page each KV head
has blocks of 32 positions. K: position t, element e of a block at ((e / 8) * 32 + t) * 8 + e % 8. V: at
((t / 16 * 2 + t % 8 / 4) * dim + e) * 8 + t % 4 + 4 * (t % 16 / 8). Rows of a batch are packed: sequence s has rows
[starts[s], starts[s + 1]), in no page yet before an append, the last ones of its length after it.

Kinds of a case
  plan    the lengths of a step's requests: pages of those that ended go back on the free list, the others get the pages
          that they lack; the slot of each new row and its position
  append  packed rows into their slots
  step    one new position of every sequence (`idle`: of two in three) over all rows of its own
  prompt  the new rows of each sequence, each over its own row and those before it; `ctx` rows were there before

Types are the rows' and the outputs': f32 and f16 over a cache in fp16, bf16 over one in bf16. A plan begins from the same
state each time: the arrays that it changes are copied back into place first, as a program does that goes back a step.
"""
import math
import os
import sys

import torch

own = False

B = 32  # positions of a block
F = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # a decoding step of a full batch: one row each
        dict(name="plan_step", kind="plan", seqs=64, page=64, max_pages=64, rows=2500, fresh=0, ended=0, pad=0,
             short=0),
        # a busy server's batch: most decode, some have ended, new prompts come in
        dict(name="plan_batch", kind="plan", seqs=1000, page=32, max_pages=256, rows=3000, fresh=120, ended=70, pad=55,
             short=0),
        # the rows of a decoding step, as a model makes them
        dict(name="append_step", kind="append", dtype="f32", seqs=64, kv_heads=8, dim=64, page=64, ctx=2500, n=1, pad=0),
        # prompts of different lengths, one behind the other
        dict(name="append_prompts", kind="append", dtype="bf16", seqs=12, kv_heads=8, dim=128, page=64, ctx=0, n=3001,
             pad=19),
        # one token of a chat at its start: latency only
        dict(name="step_chat", kind="step", dtype="f32", seqs=1, kv_heads=8, group=2, dim=64, page=32, ctx=100,
             max_pages=16, idle=False),
        # decode after 4096 positions, the shape and context of the package's benchmark
        dict(name="step_4097", kind="step", dtype="f32", seqs=1, kv_heads=8, group=3, dim=64, page=64, ctx=4097,
             max_pages=72, idle=False),
        # one long document
        dict(name="step_document", kind="step", dtype="f16", seqs=1, kv_heads=8, group=3, dim=64, page=256, ctx=131000,
             max_pages=512, idle=False),
        # a server's batch of ragged sequences, wide heads: the cache is far larger than the last-level cache
        dict(name="step_batch", kind="step", dtype="bf16", seqs=64, kv_heads=8, group=4, dim=128, page=64, ctx=8003,
             max_pages=128, idle=True),
        # a short prompt
        dict(name="prompt_chat", kind="prompt", dtype="f32", seqs=1, kv_heads=8, group=2, dim=64, page=32, ctx=0, n=37,
             max_pages=16, pad=0),
        # pages of text after chats, the engine's activations
        dict(name="prompt_after_chat", kind="prompt", dtype="f32", seqs=3, kv_heads=8, group=3, dim=64, page=64, ctx=1000,
             n=300, max_pages=32, pad=0),
        # prompts of different lengths in one batch, wide heads
        dict(name="prompt_batch", kind="prompt", dtype="bf16", seqs=12, kv_heads=4, group=8, dim=128, page=128, ctx=0,
             n=2500, max_pages=32, pad=27),
        # a whole document at once
        dict(name="prompt_document", kind="prompt", dtype="f16", seqs=1, kv_heads=8, group=3, dim=64, page=256, ctx=0,
             n=16384, max_pages=64, pad=0),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["plan", "append", "step", "step", "prompt", "prompt"])
    c = dict(kind=kind, page=rng.choice([32, 64, 128, 256]))
    if kind == "plan":
        c.update(seqs=_log(rng, 1, 1000), rows=_log(rng, 1, 8000))
        c.update(fresh=rng.randint(0, c["seqs"] // 4), ended=rng.randint(0, c["seqs"] // 4), pad=rng.randint(0, 64),
                 max_pages=-(-(c["rows"] + 1) // c["page"]) + rng.randint(0, 16),
                 short=rng.choice([0, 0, 0, rng.randint(1, 64)]))  # pages that the pool lacks for all of them
        return c
    c.update(dtype=rng.choice(["f32", "f16", "bf16"]), kv_heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 128]),
             seqs=_log(rng, 1, 64))
    row = c["seqs"] * c["kv_heads"] * c["dim"]
    if kind == "append":
        c.update(ctx=_log(rng, 1, 4000) - 1, n=_log(rng, 1, max(1, min(16384, (1 << 24) // row))), pad=rng.randint(0, 64))
        return c
    c["group"] = rng.choice([1, 2, 3, 4, 6, 8])
    if kind == "step":
        c.update(ctx=_log(rng, 1, max(64, min(131072, (1 << 28) // row))), idle=rng.random() < 0.3)
    else:
        n = _log(rng, 1, 8192)
        most = max(1, (1 << 35) // (row * c["group"] * n))  # rows that a query may see
        c.update(n=min(n, max(1, most)), pad=rng.randint(0, 64))
        c["ctx"] = 0 if rng.random() < 0.5 else _log(rng, 1, max(1, min(16384, most)))
    c["max_pages"] = -(-(c["ctx"] + c.get("n", 0)) // c["page"]) + rng.randint(0, 16)
    return c


# ---- inputs ----------------------------------------------------------------------------------------------------
def _new(case):
    """New rows of each sequence: n, and down to 1/4 of it for the others."""
    n = case.get("n", 1)
    if case["kind"] == "step":
        return [0 if case["idle"] and s % 3 == 1 else 1 for s in range(case["seqs"])]
    return [max(1, n - n * 3 * s // (4 * case["seqs"])) for s in range(case["seqs"])]


def _lengths(case):
    """Rows of each sequence before an append or a plan, and with the new ones otherwise."""
    ctx, S = case["ctx"], case["seqs"]
    before = [ctx - ctx * 5 * s // (8 * S) for s in range(S)]
    if case["kind"] == "prompt":
        return [a + b for a, b in zip(before, _new(case))]
    return before


def _shared(shapes):
    """Tensors over one buffer, each at a multiple of 256 bytes: one copy puts all of them back."""
    at, size = {}, 0
    for name, shape in shapes.items():
        at[name] = size
        size += -(-math.prod(shape) // 64) * 64
    whole = torch.zeros(size, dtype=torch.int32, device="cuda")
    return whole, {name: whole[at[name]:at[name] + math.prod(shape)].view(shape) for name, shape in shapes.items()}


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _plan_sizes(case):
    """Lengths before, new rows, pages of the pool; of running sequences first, then of new prompts."""
    S, P, fresh = case["seqs"], case["page"], case["fresh"]
    most = max(1, min(case["rows"], case["max_pages"] * P - 1))

    def spread(n):  # most are short
        return [max(1, int(most * ((i + 0.5) / n) ** 2)) for i in range(n)]

    rows, new = spread(S - fresh) + [0] * fresh, [1] * (S - fresh) + spread(fresh)
    pages = sum(-(-(a + b) // P) for a, b in zip(rows, new)) + 5 - case["short"]
    return rows, new, max(pages, sum(-(-a // P) for a in rows))


def _plan_inputs(case, seed):
    g = torch.Generator().manual_seed(seed)
    S, P, M = case["seqs"], case["page"], case["max_pages"]
    rows, new, pages = _plan_sizes(case)
    # the sequences in any order; some of those that run have ended
    mixed = torch.randperm(S, generator=g)
    new = torch.tensor(new)
    new[torch.randperm(S - case["fresh"], generator=g)[:case["ended"]]] = -1
    rows, new = torch.tensor(rows)[mixed], new[mixed]
    held = (rows + P - 1) // P
    whole, c = _shared(dict(state=(S, 4), table=(S, M), free=(pages + 1,)))
    order = torch.randperm(pages, generator=g)
    table = torch.zeros(S, M, dtype=torch.int32)
    at = 0
    for s, h in enumerate(held.tolist()):
        table[s, :h] = order[at:at + h]
        at += h
    c["table"].copy_(table)
    c["free"][0] = pages - at
    c["free"][1:1 + pages - at] = order[at:].to(torch.int32)
    c["state"][:, 0] = rows.to(torch.int32)
    c["state"][:, 2] = (rows - 1).clamp(min=0).to(torch.int32)
    tokens = int(new.clamp(min=0).sum()) + case["pad"]
    return dict(case=case, c=c, whole=whole, first=whole.clone(), pages=pages, tokens=tokens, new=_ints(new.tolist()),
                starts=torch.zeros(S + 1, dtype=torch.int32, device="cuda"),
                slots=torch.zeros(max(tokens, 1), dtype=torch.int32, device="cuda"),
                positions=torch.zeros(max(tokens, 1), dtype=torch.int32, device="cuda"))


def _inputs(case, seed):
    if case["kind"] == "plan":
        return _plan_inputs(case, seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    S, H, D, P = case["seqs"], case["kv_heads"], case["dim"], case["page"]
    dt = F[case["dtype"]]
    held = torch.bfloat16 if case["dtype"] == "bf16" else torch.float16
    kind, lens, new = case["kind"], _lengths(case), _new(case)
    after = [a + b for a, b in zip(lens, new)] if kind == "append" else lens
    used = [-(-x // P) for x in after]
    pages, M = sum(used) + 3, case.get("max_pages", max(used) + 1)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    # a pool that has been in use: its pages lie in any order, and hold old rows behind the lengths
    c = {name: normal(pages, H, P // B, B * D, dtype=held) for name in "kv"}
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    c["table"] = torch.zeros(S, M, dtype=torch.int32, device="cuda")
    at = 0
    for s in range(S):
        c["table"][s, :used[s]] = order[at:at + used[s]]
        at += used[s]
    c["state"] = torch.zeros(S, 4, dtype=torch.int32, device="cuda")
    c["state"][:, 0] = _ints(after if kind != "append" else [a + b for a, b in zip(lens, new)])
    c["state"][:, 2] = _ints([a - b if kind != "append" else x for a, b, x in zip(after, new, lens)]).clamp(min=0)
    c["free"] = torch.zeros(pages + 1, dtype=torch.int32, device="cuda")
    real = sum(new)
    tokens = real + case.get("pad", 0)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    state = dict(case=case, c=c, pages=pages, max_pages=M, tokens=tokens, real=real, at=starts, lens=after,
                 starts=_ints(starts))
    if kind == "append":
        slots = torch.full((tokens,), -1, dtype=torch.int32, device="cuda")
        for s in range(S):
            p = torch.arange(lens[s], lens[s] + new[s], device="cuda")
            slots[starts[s]:starts[s + 1]] = c["table"][s].long()[p // P].mul(P).add(p % P).to(torch.int32)
        state.update(slots=slots, k=normal(tokens, H, D).to(dt), v=normal(tokens, H, D).to(dt))
    else:
        state["groups"] = _groups(lens, new)
        state["q"] = (2.0 * normal(max(tokens, 1), H * case["group"], D)).to(dt)
        state["out"] = torch.zeros_like(state["q"])
    return state


def _groups(lens, new):
    """Sequences with new rows, those with about as many scores together: (which, most new rows, most rows)."""
    groups = []
    for s in sorted((s for s, n in enumerate(new) if n), key=lambda s: lens[s] * new[s]):
        if groups and len(groups[-1]) < 64 and lens[s] * new[s] <= 4 * lens[groups[-1][0]] * new[groups[-1][0]]:
            groups[-1].append(s)
        else:
            groups.append([s])
    return [(torch.tensor(x, device="cuda"), max(new[s] for s in x), max(lens[s] for s in x)) for x in groups]


def prepare(case, seed):
    state = _inputs(case, seed)
    if own:
        at = os.path.join(os.getcwd(), "lastro-rust_amd")
        if at not in sys.path:
            sys.path.insert(0, at)
        import moert
        kind, dtype = case["kind"], case.get("dtype", "f16")
        cache = moert.Pages(case["seqs"], case.get("kv_heads", 8), case.get("dim", 64), case["page"], state["pages"],
                            case["max_pages"] if kind != "append" else state["max_pages"],
                            {name: t.data_ptr() for name, t in state["c"].items()},
                            dtype=moert.BF16 if dtype == "bf16" else moert.F16)
        state.update(cache=cache, rows={"f32": moert.F32, "f16": moert.F16, "bf16": moert.BF16}[dtype])
        if kind in ("step", "prompt"):
            size = cache.workspace(case["kv_heads"] * case["group"], state["tokens"] if kind == "prompt" else 0)
            state.update(ws=torch.empty(size, dtype=torch.uint8, device="cuda"), ws_bytes=size)
    return state


# ---- one pass ---------------------------------------------------------------------------------------------------
def run(state):
    case, c = state["case"], state["c"]
    kind = case["kind"]
    if kind == "plan":
        state["whole"].copy_(state["first"])
    if own:
        cache = state["cache"]
        stream = torch.cuda.current_stream().cuda_stream
        if kind == "plan":
            cache.plan(state["new"].data_ptr(), state["tokens"], state["starts"].data_ptr(), state["slots"].data_ptr(),
                       state["positions"].data_ptr(), stream=stream)
        elif kind == "append":
            cache.append(state["k"].data_ptr(), state["v"].data_ptr(), state["slots"].data_ptr(), state["tokens"],
                         dtype=state["rows"], stream=stream)
        elif kind == "step":
            cache.attend(state["q"].data_ptr(), state["out"].data_ptr(), case["kv_heads"] * case["group"],
                         case["dim"] ** -0.5, state["ws"].data_ptr(), state["ws_bytes"],
                         starts=state["starts"].data_ptr() if case["idle"] else 0, tokens=state["tokens"],
                         dtype=state["rows"], stream=stream)
        else:
            cache.prompt(state["q"].data_ptr(), state["out"].data_ptr(), case["kv_heads"] * case["group"],
                         case["dim"] ** -0.5, state["starts"].data_ptr(), state["tokens"], state["ws"].data_ptr(),
                         state["ws_bytes"], dtype=state["rows"], stream=stream)
    elif kind == "plan":
        _plan(case, c, state)
    elif kind == "append":
        _append(case, c, state)
    else:
        for group in state["groups"]:
            _attend(case, c, state, *group)
    if kind == "plan":
        return dict(state=c["state"], table=c["table"], free=c["free"], starts=state["starts"], slots=state["slots"],
                    positions=state["positions"])
    if kind == "append":
        return dict(k=c["k"], v=c["v"])
    return dict(out=state["out"])


def _plan(case, c, st):
    P, M, T = case["page"], case["max_pages"], st["tokens"]
    new, rows = st["new"].long(), c["state"][:, 0].long()
    free, table = c["free"].long(), c["table"].long()
    count, col = free[0], torch.arange(M, device="cuda")[None, :]
    held = (rows + P - 1) // P
    # what has ended gives its pages back, in order
    ended = new < 0
    back = torch.where(ended, held, 0)
    gone = ended[:, None] & (col < held[:, None])
    to = torch.where(gone, 1 + count + (torch.cumsum(back, 0) - back)[:, None] + col, free.numel())
    free = torch.cat([free, free[:1]]).scatter(0, to.reshape(-1), table.reshape(-1))[:-1]
    count = count + back.sum()
    rows, held = torch.where(ended, 0, rows), torch.where(ended, 0, held)
    # the others, in order, while there are pages
    n = new.clamp(min=0)
    end = torch.cumsum(n, 0)
    ok = (n == 0) | (end <= T) & (rows + n <= M * P)
    need = torch.where(ok, (rows + n + P - 1) // P - held, 0)
    upto = torch.cumsum(need, 0)
    ok = ok & ((need == 0) | (upto <= count))
    gets = ok[:, None] & (col >= held[:, None]) & (col < (held + need)[:, None])
    which = (count - (upto - need)[:, None] - (col - held[:, None])).clamp(0, free.numel() - 1)
    table = torch.where(gets, free[which], table)
    free[0] = count - torch.where(ok, need, 0).sum()
    starts = torch.cat([end[:1] * 0, end]).clamp(max=T)
    tok = torch.arange(max(T, 1), device="cuda")
    s = torch.searchsorted(starts[1:].contiguous(), tok, right=True).clamp(max=case["seqs"] - 1)
    there = (tok < starts[-1]) & ok[s]
    pos = rows[s] + tok - starts[s]
    slot = table[s, (pos // P).clamp(0, M - 1)] * P + pos % P
    if T:
        st["slots"].copy_(torch.where(there, slot, -1))
        st["positions"].copy_(torch.where(there, pos, -1))
    st["starts"].copy_(starts)
    c["table"].copy_(table)
    c["free"].copy_(free)
    c["state"][:, 1] = torch.where(ended, 0, c["state"][:, 1] + torch.where(ok, 0, n))
    c["state"][:, 0] = torch.where(ok, rows + n, rows)
    c["state"][:, 2] = torch.where(ok, rows, -1)


def _append(case, c, st):
    H, D, P, real = case["kv_heads"], case["dim"], case["page"], st["real"]
    slot = st["slots"][:real].long()
    page, block, t = slot // P, slot % P // B, slot % B
    shape = (-1, H, P // B, D // 8, B, 8)
    c["k"].view(shape)[page, :, block, :, t] = st["k"][:real].to(c["k"].dtype).view(real, H, D // 8, 8)
    c["v"].view(-1, H, P // B, 4, D, 8)[page, :, block, t // 16 * 2 + t % 8 // 4, :, t % 4 + t % 16 // 8 * 4] = \
        st["v"][:real].to(c["v"].dtype)


def _unpack(case, c, seqs, pages):
    """K and V [sequences, H, rows, D] in f32, of the first pages of some sequences."""
    H, D, P = case["kv_heads"], case["dim"], case["page"]
    at, n = c["table"][seqs, :pages].long(), len(seqs)
    k = c["k"][at].float().view(n, pages, H, P // B, D // 8, B, 8).permute(0, 2, 1, 3, 5, 4, 6).reshape(n, H, -1, D)
    # of V: half of a block, quarter, element, eight of a half, position
    v = c["v"][at].float().view(n, pages, H, P // B, 2, 2, D, 2, 4).permute(0, 2, 1, 3, 4, 7, 5, 8, 6)
    return k, v.reshape(n, H, -1, D)


def _attend(case, c, st, seqs, n, length):
    """The new rows of some sequences, padded to n of them and `length` rows that they see."""
    H, G, D = case["kv_heads"], case["group"], case["dim"]
    k, v = _unpack(case, c, seqs, -(-length // case["page"]))
    length = k.shape[2]
    lens, lo = c["state"][seqs, 0].long(), st["starts"][seqs].long()
    new = st["starts"][seqs + 1] - lo
    i = torch.arange(n, device="cuda")
    rows = (lo[:, None] + torch.minimum(i, new[:, None] - 1))  # a padded one is the last one again
    sees = (lens - new)[:, None] + torch.minimum(i, new[:, None] - 1) + 1
    hide = torch.arange(length, device="cuda") >= sees[:, :, None]
    wide = torch.float64 if case["dtype"] == "f32" and length > 2048 else torch.float32
    # all KV heads at once, or one after the other where their scores would be many
    step = H if len(seqs) * H * G * n * length <= 1 << 30 else 1
    for h in range(0, H, step):
        heads = slice(h * G, (h + step) * G)
        q = st["q"][:, heads][rows].float().view(len(seqs), n, step, G, D).permute(0, 2, 3, 1, 4) * D ** -0.5
        a = torch.matmul(q.reshape(len(seqs), step, G * n, D), k[:, h:h + step].transpose(2, 3).contiguous())
        a.view(len(seqs), step, G, n, length).masked_fill_(hide[:, None, None], -math.inf)
        p = a.sub_(a.amax(3, keepdim=True)).exp_()
        o = torch.matmul(p.to(wide), v[:, h:h + step].to(wide)) / p.sum(3, keepdim=True, dtype=wide)
        st["out"][:, heads][rows] = o.view(len(seqs), step * G, n, D).transpose(1, 2).to(st["out"].dtype)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------
def work(case):
    kind, P = case["kind"], case["page"]
    if kind == "plan":
        # new lengths, states, starts; a table entry and one of the free list for each page that is given or comes back;
        # slots and positions. Which sequences have ended is drawn: their mean
        rows, new, _ = _plan_sizes(case)
        S, runs = case["seqs"], case["seqs"] - case["fresh"]
        on = 1 - case["ended"] / runs
        given = sum((-(-(a + b) // P) - -(-a // P)) * (on if a else 1) for a, b in zip(rows, new))
        back = sum(-(-a // P) for a in rows) * (1 - on)
        return dict(bytes=int(S * (4 + 16 + 16 + 4) + 8 * (given + back) + 8 * (sum(new) - case["ended"])), flops=0)
    H, D, G = case["kv_heads"], case["dim"], case.get("group", 1)
    size, lens, new = 4 if case["dtype"] == "f32" else 2, _lengths(case), _new(case)
    if kind == "append":
        return dict(bytes=sum(new) * (2 * H * D * (size + 2) + 4), flops=0)
    on = [x if n else 0 for x, n in zip(lens, new)]
    seen = sum(n * x - n * (n - 1) // 2 for x, n in zip(lens, new))
    return dict(bytes=4 * H * D * sum(on) + 4 * sum(-(-x // P) for x in on) + 2 * size * H * G * D * sum(new),
                flops=4 * H * G * D * seen)


# ---- the same in 64 bits -------------------------------------------------------------------------------------------
def _place(kind, t, e, dim):
    if kind == "k":
        return ((e // 8) * 32 + t) * 8 + e % 8
    return ((t // 16 * 2 + t % 8 // 4) * dim + e) * 8 + t % 4 + 4 * (t % 16 // 8)


def _plan_by_steps(case, st):
    """One sequence after the other, one page after the other."""
    P, T, new = case["page"], st["tokens"], st["new"].tolist()
    state, table, free = (st["c"][name].tolist() for name in ("state", "table", "free"))
    for s, n in enumerate(new):
        if n < 0:
            for page in table[s][:-(-state[s][0] // P)]:
                free[0] += 1
                free[free[0]] = page
            state[s][:3] = [0, 0, 0]
    starts, slots, positions, out_of_pages = [0], [], [], False
    for s, n in enumerate(max(x, 0) for x in new):
        rows = state[s][0]
        held, need = -(-rows // P), -(-(rows + n) // P) - -(-rows // P)
        fits = n == 0 or len(slots) + n <= T and rows + n <= case["max_pages"] * P
        if fits and need and (out_of_pages or need > free[0]):
            fits, out_of_pages = False, True
        if fits:
            for i in range(need):
                table[s][held + i] = free[free[0]]
                free[0] -= 1
        place = [table[s][p // P] * P + p % P if fits else -1 for p in range(rows, rows + n)]
        slots, positions = slots + place, positions + [p if fits else -1 for p in range(rows, rows + n)]
        starts.append(min(T, len(slots)))
        state[s][:3] = [rows + n, state[s][1], rows] if fits else [rows, state[s][1] + n, -1]
    got = dict(state=state, table=table, free=free, starts=starts)
    got.update((name, (x + [-1] * T)[:max(T, 1)]) for name, x in (("slots", slots), ("positions", positions)))
    return {name: torch.tensor(x).numpy() for name, x in got.items()}


def exact(case, seed):
    """From the definition: every element by its place in the pool, softmax in 64 bits."""
    st = _inputs(case, seed)
    if case["kind"] == "plan":
        return _plan_by_steps(case, st)
    c, H, D, P = st["c"], case["kv_heads"], case["dim"], case["page"]
    e = torch.arange(D, device="cuda")[None, :]
    if case["kind"] == "append":
        got = {}
        slot = st["slots"][:st["real"]].long()
        for kind in "kv":
            held = c[kind].double().flatten()
            for h in range(H):
                head = (slot // P * H + h) * (P * D) + slot % P // B * (B * D)
                at = head[:, None] + _place(kind, slot[:, None] % B, e, D)
                held[at.flatten()] = st[kind][:st["real"], h].to(c[kind].dtype).double().flatten()
            got[kind] = held.view(c[kind].shape).cpu().numpy()
        return got
    G = case["group"]
    if 4.0 * H * G * D * sum((b - a) * x for a, b, x in zip(st["at"], st["at"][1:], st["lens"])) > 4e12:
        return None
    out = torch.zeros(st["out"].shape, dtype=torch.float64, device="cuda")
    for s, length in enumerate(st["lens"]):
        lo, hi = st["at"][s], st["at"][s + 1]
        if lo == hi:
            continue
        pos = torch.arange(length, device="cuda")
        page = c["table"][s].long()[pos // P]
        for h in range(H):
            head = (page * H + h) * (P * D) + pos % P // B * (B * D)
            k, v = (c[kind].flatten()[head[:, None] + _place(kind, pos[:, None] % B, e, D)].double() for kind in "kv")
            kt = k.T.contiguous()
            for g in range(G):
                for i in range(lo, hi, 4096):
                    j = min(hi, i + 4096)
                    last = length - (hi - lo) + torch.arange(i - lo, j - lo, device="cuda")
                    a = (st["q"][i:j, h * G + g].double() @ kt) / math.sqrt(D)
                    a = a.masked_fill(pos[None, :] > last[:, None], -math.inf)
                    out[i:j, h * G + g] = torch.softmax(a, 1) @ v
    return dict(out=out.cpu().numpy())
