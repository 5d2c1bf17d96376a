"""The operators of the 8-bit paged key/value cache: block tables and slot maps from the sequences' lengths, the append of
new tokens, the attention of single tokens over the pages. Each in a plain form (elementary torch operations) and as the
calls a program makes of the framework.

A cache is what such a program allocates once: codes [2 (keys, values), blocks, kv heads, tokens of a block, head size] and one
binary32 scale per token and head. Sequences own scattered blocks; places that no token has been written to hold NaN scales."""
import math

import torch

own = False


def listed():
    return [
        # one decode step of a small server: a token for each of eight sequences, latency only
        {"name": "map 8 decode", "op": "map", "sequences": 8, "kind": "decode", "tokens": 8, "block": 16, "context": 512, "short": 0},
        # a step that mixes decoding with prompt chunks, and runs out of free blocks before its last sequences
        {"name": "map 201 mixed", "op": "map", "sequences": 201, "kind": "mixed", "tokens": 4100, "block": 16, "context": 2048, "short": 1},
        # a queue of prompts admitted at once
        {"name": "map 4096 prompts", "op": "map", "sequences": 4096, "kind": "prompts", "tokens": 1000000, "block": 32, "context": 4096, "short": 0},
        # the new token of a single sequence
        {"name": "append 1 token", "op": "append", "tokens": 1, "padded": 0, "kv_heads": 8, "head": 128, "block": 16, "type": "f32", "rope": True},
        # a decode batch: the widest that the model benchmark decodes
        {"name": "append 64 tokens", "op": "append", "tokens": 64, "padded": 0, "kv_heads": 8, "head": 128, "block": 16, "type": "f32", "rope": True},
        # a prompt chunk in binary16, with rows behind the last token
        {"name": "append 471 of 512 f16", "op": "append", "tokens": 471, "padded": 41, "kv_heads": 8, "head": 64, "block": 16, "type": "f16", "rope": True},
        # a long prompt whose keys are rotated already
        {"name": "append 8191 tokens", "op": "append", "tokens": 8191, "padded": 0, "kv_heads": 8, "head": 128, "block": 16, "type": "f32", "rope": False},
        # one sequence of the small model: latency only
        {"name": "attend tiny at 57", "op": "attend", "rows": 1, "idle": 0, "heads": 8, "kv_heads": 2, "head": 64, "context": 57, "block": 16, "window": 0, "type": "f32", "rope": True},
        # one sequence with a long history
        {"name": "attend 8b at 3901", "op": "attend", "rows": 1, "idle": 0, "heads": 32, "kv_heads": 8, "head": 128, "context": 3901, "block": 16, "window": 0, "type": "f32", "rope": True},
        # a server batch, sequences of different lengths, some rows free
        {"name": "attend 8b 32 rows at 512", "op": "attend", "rows": 32, "idle": 3, "heads": 32, "kv_heads": 8, "head": 128, "context": 512, "block": 16, "window": 0, "type": "f32", "rope": True},
        # the widest batch in binary16 with a sliding window
        {"name": "attend 1b 64 rows window", "op": "attend", "rows": 64, "idle": 0, "heads": 32, "kv_heads": 8, "head": 64, "context": 2048, "block": 32, "window": 1000, "type": "f16", "rope": False},
        # long documents: what the 8-bit pages are for
        {"name": "attend 8b 16 rows at 32000", "op": "attend", "rows": 16, "idle": 0, "heads": 32, "kv_heads": 8, "head": 128, "context": 32000, "block": 16, "window": 0, "type": "f32", "rope": True},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["map", "append", "append", "attend", "attend", "attend"])
    block = rng.choice([16, 16, 16, 32, 64, 24, 5, 1])
    if op == "map":
        kind = rng.choice(["decode", "mixed", "prompts"])
        n = _log_int(rng, 1, 4096)
        context = _log_int(rng, 16, 4096)
        tokens = n if kind == "decode" else min(n * context, _log_int(rng, n, 1000000)) if kind == "prompts" else n + _log_int(rng, 16, 8192)
        return {"op": op, "sequences": n, "kind": kind, "tokens": tokens, "block": block, "context": context, "short": rng.choice([0, 0, 1])}
    head = rng.choice([64, 128, 128, 96, 192, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 3])
    if op == "append":
        tokens = _log_int(rng, 1, min(8191, 8191 * 8 * 128 // (kv_heads * head)))
        return {"op": op, "tokens": tokens, "padded": rng.choice([0, rng.randrange(1, 65)]), "kv_heads": kv_heads, "head": head, "block": block,
                "type": rng.choice(["f32", "f32", "f16"]), "rope": rng.choice([True, False])}
    rows = rng.choice([1, _log_int(rng, 2, 128)])
    group = rng.choice([1, 2, 4, 4, 8, 3, 16])
    # the largest listed case: 16 rows x 32000 tokens of 8 heads of 128, four query heads to each
    most = 16 * 32000 * 8 * 128 // (kv_heads * head * rows) * 4 // max(4, group)
    context = _log_int(rng, 1, min(100000, most * 2 // 3))
    return {"op": op, "rows": rows, "idle": rng.randrange(0, 1 + rows // 4), "heads": kv_heads * group, "kv_heads": kv_heads, "head": head, "context": context,
            "block": block, "window": rng.choice([0, 0, _log_int(rng, 1, 4096)]), "type": rng.choice(["f32", "f32", "f16"]), "rope": rng.choice([True, False])}


class _State:
    pass


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rope_tables(rows, head):
    """cos and sin, [rows][head / 2] in binary32, of angles in 64 bits."""
    freq = 500000.0 ** (-torch.arange(0, head, 2, device="cuda", dtype=torch.float64) / head)
    angle = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * freq[None, :]
    return angle.cos().float(), angle.sin().float()


def _lengths(case):
    """Tokens that the rows of an attention attend to before a window cuts them: half to one and a half times the context, the idle ones none."""
    rows, n = case["rows"], case["context"]
    got = [n] if rows == 1 else [max(1, int(n * (0.5 + i / (rows - 1)))) for i in range(rows)]
    return got[:rows - case["idle"]] + [0] * case["idle"]


def _random_codes(shape, g):
    """Codes as quantised rows hold them: near normal, their largest at 127."""
    out = torch.empty(shape, dtype=torch.int8, device="cuda")
    flat = out.view(-1)
    for at in range(0, flat.numel(), 1 << 28):
        part = flat[at:at + (1 << 28)]
        part.copy_(torch.randn(part.numel(), device="cuda", generator=g).mul_(45).round_().clamp_(-127, 127))
    return out


def _added(case, g):
    """Tokens held and added, sequence by sequence."""
    n, kind = case["sequences"], case["kind"]
    u = torch.rand(n, device="cuda", generator=g, dtype=torch.float64)
    held = (u * case["context"]).long() + 1
    if kind == "decode":
        return held, torch.ones(n, device="cuda", dtype=torch.int64)
    w = torch.rand(n, device="cuda", generator=g, dtype=torch.float64) + 0.05
    if kind == "prompts":
        held.zero_()
        w = w * w
        more = (w / w.sum() * max(0, case["tokens"] - n)).long()
        return held, (more + 1).clamp_(max=case["context"] * 8)
    # mixed: an eighth of the sequences gets a chunk of its prompt, some wait, the others one token
    chunk = torch.rand(n, device="cuda", generator=g) < 0.125
    wait = torch.rand(n, device="cuda", generator=g) < 0.05
    w = torch.where(chunk, w, torch.zeros_like(w))
    more = (w / w.sum().clamp(min=1e-9) * max(0, case["tokens"] - n)).long()
    return held, torch.where(wait, torch.zeros_like(more), (more + 1).clamp(max=case["context"] * 8))


def prepare(case, seed):
    s = _State()
    s.case, s.call = case, None
    g = _generator(seed)
    bs = case["block"]
    if case["op"] == "map":
        n = case["sequences"]
        held, added = _added(case, g)
        s.per = -(-case["context"] * 9 // bs) + 1
        have, want = -(-held // bs), -(-(held + added) // bs)
        used, need = int(have.sum()), int((want - have).sum())
        s.cursor = torch.tensor([7], dtype=torch.int32, device="cuda")
        s.free_count = 7 + (need - need // 8 if case["short"] else need + 64)
        ids = torch.randperm(used + s.free_count, device="cuda", generator=g).int()
        s.free = ids[used:].contiguous()
        column = torch.arange(s.per, device="cuda")
        first = (torch.cumsum(have, 0) - have)[:, None] + column[None, :]
        s.table = torch.where(column[None, :] < have[:, None], ids[first.clamp_(max=ids.numel() - 1)], torch.full((), -1, dtype=torch.int32, device="cuda")).contiguous()
        s.held, s.added = held.int(), added.int()
        s.capacity = max(case["tokens"], n) + 8
        s.lengths = torch.zeros(n, dtype=torch.int32, device="cuda")
        s.offsets = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
        s.token_slot = torch.full((s.capacity,), -9, dtype=torch.int32, device="cuda")
        s.positions = torch.full((s.capacity,), -9, dtype=torch.int32, device="cuda")
        s.slot_map = torch.full((s.capacity,), -9, dtype=torch.int64, device="cuda")
        s.cursor_out = torch.zeros(1, dtype=torch.int32, device="cuda")
        s.result = torch.zeros(4, dtype=torch.int32, device="cuda")
        return s
    h, d = case["kv_heads"], case["head"]
    dtype = {"f32": torch.float32, "f16": torch.float16}[case["type"]]
    if case["op"] == "append":
        t, rows = case["tokens"], case["tokens"] + case["padded"]
        s.blocks = -(-t // bs) + 2
        s.codes = _random_codes((2, s.blocks, h, bs, d), g)
        s.scales = torch.rand((2, s.blocks, h, bs), device="cuda", generator=g) * 0.02 + 0.01
        # queries, keys and values of a token are one row of a joint projection; keys and values of few heads stand out
        s.row = torch.randn((rows, (4 * h + 2 * h) * d), device="cuda", generator=g)
        s.row *= torch.exp(torch.randn((1, (4 * h + 2 * h) * d), device="cuda", generator=g) * 0.5)
        s.row = s.row.to(dtype)
        s.key, s.value = s.row[:, 4 * h * d:5 * h * d], s.row[:, 5 * h * d:]
        # one sequence behind 37 tokens that are there, its blocks scattered
        start = 37
        order = torch.randperm(s.blocks - 1, device="cuda", generator=g)
        at = torch.arange(rows, device="cuda")
        place = at + start % bs
        s.slot_map = torch.where(at < t, order[(place // bs).clamp_(max=s.blocks - 2)] * bs + place % bs, torch.full_like(at, -1))
        s.positions = (at + start).int()
        s.count = torch.tensor([t], dtype=torch.int32, device="cuda")
        s.rope_rows = start + rows
        s.cos, s.sin = _rope_tables(s.rope_rows, d) if case["rope"] else (None, None)
        return s
    rows, heads = case["rows"], case["heads"]
    lengths = _lengths(case)
    s.per = -(-max(lengths) // bs) + 1
    held = torch.tensor(lengths, device="cuda")
    have = -(-held // bs)
    used = int(have.sum())
    s.blocks = used + 3
    ids = torch.randperm(s.blocks, device="cuda", generator=g)[:used].int()
    # rows belong to the slots of a table in another order
    order = torch.randperm(rows, device="cuda", generator=g)
    column = torch.arange(s.per, device="cuda")
    first = (torch.cumsum(have, 0) - have)[:, None] + column[None, :]
    table = torch.where(column[None, :] < have[:, None], ids[first.clamp_(max=used - 1)], torch.full((), -1, dtype=torch.int32, device="cuda"))
    s.table = torch.empty_like(table)
    s.table[order] = table
    s.kv_slots = order.int()
    s.positions = (held - 1).int()
    s.codes = _random_codes((2, s.blocks, h, bs, d), g)
    scales = torch.exp(torch.randn((2, s.blocks, h, bs), device="cuda", generator=g) * 0.3) * (1.0 / 45)
    # places behind a sequence's last token have never been written
    last = ids[(torch.cumsum(have, 0) - 1).clamp_(min=0)].long()[held > 0]
    unwritten = torch.arange(bs, device="cuda")[None, :] > ((held - 1) % bs)[held > 0][:, None]
    scales[:, last] = torch.where(unwritten[None, :, None, :], torch.full((), math.nan, device="cuda"), scales[:, last])
    s.scales = scales
    s.query = (torch.randn((rows, heads * d), device="cuda", generator=g) * 1.5).to(dtype)
    s.out = torch.empty((rows, heads, d), dtype=dtype, device="cuda")
    s.lse = torch.empty((rows, heads), dtype=torch.float32, device="cuda")
    s.rope_rows = max(lengths) + 1
    s.cos, s.sin = _rope_tables(s.rope_rows, d) if case["rope"] else (None, None)
    return s


# ------------------------------------------------------------------------------------------------ plain forms

def _rotate(x, cos, sin):
    """Pairs (2i, 2i + 1) of the last axis; cos and sin with an axis of heads."""
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)


def _plain_map(s):
    bs, n = s.case["block"], s.case["sequences"]
    held, added = s.held.long(), s.added.long()
    count = added.clamp(min=0)
    ends = torch.cumsum(count, 0)
    starts = ends - count
    bad = (held < 0) | (added < 0) | (held + added > s.per * bs) | (ends > s.capacity)
    have = (held + bs - 1) // bs
    need = torch.where(bad, torch.zeros_like(held), (held + added + bs - 1) // bs - have)
    block_ends = torch.cumsum(need, 0)
    cursor = s.cursor.long()
    served = ~bad & ((need == 0) | (block_ends <= s.free_count - cursor))
    taken = torch.where(served & (need > 0), block_ends, torch.zeros_like(held)).max()
    # new blocks, in the order of the sequences
    b = torch.arange(s.free_count, device="cuda")
    r = torch.searchsorted(block_ends, b, right=True).clamp(max=n - 1)
    good = (b < block_ends[-1]) & served[r]
    to = torch.where(good, r * s.per + have[r] + b - (block_ends - need)[r], torch.full_like(b, n * s.per))
    flat = torch.cat((s.table.view(-1), s.table.new_zeros(1)))
    flat[to] = s.free[(cursor + b).clamp(max=s.free_count - 1)]
    s.table.copy_(flat[:-1].view(n, s.per))
    # new tokens
    t = torch.arange(s.capacity, device="cuda")
    r = torch.searchsorted(ends, t, right=True).clamp(max=n - 1)
    there = t < ends[-1]
    position = torch.where(served[r], held[r] + t - starts[r], torch.full_like(t, -1))
    block = s.table[r, (position.clamp(min=0) // bs).clamp(max=s.per - 1)].long()
    place = torch.where((position >= 0) & (block >= 0), block * bs + position % bs, torch.full_like(t, -1))
    s.token_slot.copy_(torch.where(there, r, s.token_slot.long()))
    s.positions.copy_(torch.where(there, position, s.positions.long()))
    s.slot_map.copy_(torch.where(there, place, s.slot_map))
    s.lengths.copy_(torch.where(served, held + added, held))
    s.offsets.copy_(torch.cat((starts, ends[-1:])))
    s.cursor_out.copy_(cursor + taken)
    s.result.copy_(torch.stack((ends[-1].clamp(max=s.capacity), taken, (~served).sum(), block_ends[-1])))


def _plain_append(s):
    case = s.case
    h, d, bs = case["kv_heads"], case["head"], case["block"]
    t = torch.arange(s.key.shape[0], device="cuda")
    # in 64 bits: of millions of values some lie next to the border of two codes
    key, value = s.key.double().view(-1, h, d), s.value.double().view(-1, h, d)
    if case["rope"]:
        at = s.positions.long()
        key = _rotate(key, s.cos[at].double()[:, None], s.sin[at].double()[:, None])
    x = torch.stack((key, value))
    most = x.abs().amax(-1)
    some = most >= 2.0 ** -100
    scale = torch.where(some, most / 127, torch.zeros_like(most)).float()
    code = torch.where(some[..., None], torch.round(x * 127 / most[..., None]), torch.zeros_like(x))
    # rows that are stored; the others go to a block of their own that is dropped
    stored = (t < s.count) & (s.slot_map >= 0) & (s.slot_map < s.blocks * bs)
    place = torch.where(stored, s.slot_map, torch.full_like(t, s.blocks * bs))
    codes = torch.cat((s.codes, s.codes.new_zeros((2, 1, h, bs, d))), 1)
    scales = torch.cat((s.scales, s.scales.new_zeros((2, 1, h, bs))), 1)
    codes[:, place // bs, :, place % bs] = code.transpose(0, 1).to(torch.int8)
    scales[:, place // bs, :, place % bs] = scale.transpose(0, 1)
    s.codes.copy_(codes[:, :-1])
    s.scales.copy_(scales[:, :-1])


def _plain_attend(s):
    case = s.case
    rows, heads, h, d, bs = case["rows"], case["heads"], case["kv_heads"], case["head"], case["block"]
    q = s.query.float().view(rows, heads, d)
    if case["rope"]:
        at = s.positions.long().clamp(min=0)
        q = _rotate(q, s.cos[at][:, None], s.sin[at][:, None])
    q = q.view(rows, h, heads // h, d)
    blocks = s.table[s.kv_slots.long()].long()
    k_codes, v_codes = s.codes
    k_scales, v_scales = s.scales
    length = s.positions.long() + 1
    first = (length - case["window"]).clamp(min=0) if case["window"] else torch.zeros_like(length)
    j = torch.arange(s.per * bs, device="cuda")
    seen = (j[None, :] >= first[:, None]) & (j[None, :] < length[:, None]) & (blocks >= 0).repeat_interleave(bs, 1)
    where = blocks.clamp(min=0)

    def gathered(codes, scales):
        x = codes[where].float() * scales[where][..., None]                       # rows, pages, heads, tokens, size
        x = x.transpose(1, 2).reshape(rows, h, s.per * bs, d)
        return torch.where(seen[:, None, :, None], x, torch.zeros((), device="cuda"))

    score = torch.matmul(q, gathered(k_codes, k_scales).transpose(2, 3)) * (1 / math.sqrt(d))
    score = torch.where(seen[:, None, None, :], score, torch.full((), -math.inf, device="cuda"))
    most = score.amax(-1, keepdim=True)
    base = torch.where(most == -math.inf, torch.zeros_like(most), most)
    weight = torch.exp(score - base)
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight, gathered(v_codes, v_scales)) / torch.where(total > 0, total, torch.ones_like(total))
    s.out.copy_(out.view(rows, heads, d))
    s.lse.copy_((base + torch.log(total)).view(rows, heads))


# ------------------------------------------------------------------------------------------------ the framework's calls

_device = None
_workspace = None


def _calls(s):
    """What a program makes once and launches at every step: the call with its buffers."""
    global _device, _workspace
    import jitllm_b200 as jl
    if _device is None:
        _device = jl.Device(0)
        _workspace = jl.Kv8Workspace(_device)
    case = s.case
    if case["op"] == "map":
        return jl.Kv8Map(_workspace, held=s.held.data_ptr(), added=s.added.data_ptr(), sequences=case["sequences"],
                         blockTable=s.table.data_ptr(), blocksPerSlot=s.per, blockSizeTokens=case["block"],
                         freeBlocks=s.free.data_ptr(), freeCount=s.free_count, cursor=s.cursor.data_ptr(), cursorOut=s.cursor_out.data_ptr(),
                         lengths=s.lengths.data_ptr(), offsets=s.offsets.data_ptr(), tokenSlots=s.token_slot.data_ptr(),
                         positions=s.positions.data_ptr(), slotMap=s.slot_map.data_ptr(), capacity=s.capacity, result=s.result.data_ptr())
    kind = jl.GGMLType.F32 if case["type"] == "f32" else jl.GGMLType.F16
    pages = jl.Kv8Pages(_device, s.codes[0].data_ptr(), s.codes[1].data_ptr(), s.scales[0].data_ptr(), s.scales[1].data_ptr(),
                        blocks=s.blocks, blockSizeTokens=case["block"], kvHeads=case["kv_heads"], headSize=case["head"])
    rope = dict(ropeCos=s.cos.data_ptr(), ropeSin=s.sin.data_ptr(), ropeRows=s.rope_rows) if case["rope"] else {}
    if case["op"] == "append":
        return jl.Kv8Append(pages, s.key.data_ptr(), s.value.data_ptr(), kind, tokens=s.key.shape[0], keyStride=s.key.stride(0), valueStride=s.value.stride(0),
                            slotMap=s.slot_map.data_ptr(), positions=s.positions.data_ptr(), tokenCount=s.count.data_ptr(), **rope)
    return jl.Kv8Attention(pages, _workspace, s.query.data_ptr(), s.out.data_ptr(), kind, rows=case["rows"], heads=case["heads"], lse=s.lse.data_ptr(),
                           blockTable=s.table.data_ptr(), slots=case["rows"], blocksPerSlot=s.per, kvSlots=s.kv_slots.data_ptr(),
                           positions=s.positions.data_ptr(), window=case["window"], scale=1 / math.sqrt(case["head"]), **rope)


_PLAIN = {"map": _plain_map, "append": _plain_append, "attend": _plain_attend}


def run(s):
    if own:
        if s.call is None:
            s.call = _calls(s)
        s.call.launch(torch.cuda.current_stream().cuda_stream)
    else:
        _PLAIN[s.case["op"]](s)
    if s.case["op"] == "map":
        return {"table": s.table, "lengths": s.lengths, "offsets": s.offsets, "token_slot": s.token_slot, "positions": s.positions,
                "slot_map": s.slot_map, "cursor": s.cursor_out, "result": s.result}
    if s.case["op"] == "append":
        return {"pages": s.codes * s.scales[..., None]}  # the values that the codes stand for
    return {"out": s.out, "lse": s.lse}


# ------------------------------------------------------------------------------------------------ accounting

def work(case):
    h, bs = case.get("kv_heads", 0), case["block"]
    if case["op"] == "map":
        n, t = case["sequences"], case["tokens"]
        # lengths in and out, offsets; sequence, position and place of each token; the new blocks' ids read and written
        return {"bytes": 8 * n + 8 * n + 16 * t + 8 * (t // bs), "flops": 4 * t}
    d, es = case["head"], 4 if case["type"] == "f32" else 2
    if case["op"] == "append":
        t = case["tokens"]
        rope = 4 * d * t if case["rope"] else 0
        # keys and values, codes and scales, places and positions, one row of either rotation table per token; then the values that
        # the whole pages stand for: codes and scales read, binary32 written
        pages = 2 * (-(-t // bs) + 2) * bs * h
        return {"bytes": 2 * t * h * (d * es + d + 4) + 12 * t + rope + pages * (5 * d + 4), "flops": 2 * t * h * d * 6 + pages * d}
    rows, heads = case["rows"], case["heads"]
    seen = sum(min(n, case["window"]) if case["window"] else n for n in _lengths(case))
    return {"bytes": seen * h * 2 * (d + 4) + 2 * rows * heads * d * es + 4 * rows * heads + 4 * seen // bs,
            "flops": 4 * seen * heads * d}


# ------------------------------------------------------------------------------------------------ 64 bits

def _exact_append(s):
    case = s.case
    h, d, bs = case["kv_heads"], case["head"], case["block"]
    pages = s.codes.double() * s.scales.double()[..., None]
    t = case["tokens"]
    for which, x in enumerate((s.key, s.value)):
        x = x[:t].double().reshape(t, h, d)
        if which == 0 and case["rope"]:
            turn = torch.complex(s.cos.double(), s.sin.double())[s.positions[:t].long()]
            x = torch.view_as_real(torch.view_as_complex(x.reshape(t, h, d // 2, 2).contiguous()) * turn[:, None]).reshape(t, h, d)
        most = x.abs().max(dim=-1, keepdim=True).values
        x = torch.round(x * 127 / most) * (most / 127)
        at = s.slot_map[:t]
        pages[which][at.div(bs, rounding_mode="floor"), :, at.remainder(bs)] = x
    return {"pages": pages}


def _exact_attend(s):
    case = s.case
    rows, heads, h, d, bs = case["rows"], case["heads"], case["kv_heads"], case["head"], case["block"]
    out = torch.zeros((rows, heads, d), dtype=torch.float64, device="cuda")
    lse = torch.full((rows, heads), -math.inf, dtype=torch.float64, device="cuda")
    for r, n in enumerate(_lengths(case)):
        if n == 0:
            continue
        low = max(0, n - case["window"]) if case["window"] else 0
        j = torch.arange(low, n, device="cuda")
        block = s.table[s.kv_slots[r].long()].long()[j // bs]
        q = s.query[r].double().view(heads, d)
        if case["rope"]:
            turn = torch.complex(s.cos[n - 1].double(), s.sin[n - 1].double())
            q = torch.view_as_real(torch.view_as_complex(q.view(heads, d // 2, 2)) * turn).reshape(heads, d)
        for kv in range(h):
            mine = slice(kv * (heads // h), (kv + 1) * (heads // h))
            k, v = (s.codes[w, block, kv, j % bs].double() * s.scales[w, block, kv, j % bs].double()[:, None] for w in (0, 1))
            score = q[mine] @ k.T / math.sqrt(d)
            lse[r, mine] = torch.logsumexp(score, -1)
            out[r, mine] = torch.softmax(score, -1) @ v
    return {"out": out, "lse": lse}


def exact(case, seed):
    if case["op"] == "map":
        return None  # whole numbers
    s = prepare(case, seed)
    return _exact_append(s) if case["op"] == "append" else _exact_attend(s)
