"""Timed cases of the block KV cache: its tables, its writes and read-back, and the attention that reads it.

A server keeps many requests' keys and values in one pool of blocks: k_cache and v_cache I8
[n_blocks, kv_heads, block, dim] with one F32 scale per (block, kv head), and for each request a row of block ids.
A step has 1 to thousands of new rows (tokens) per request: their tables are built, k and v are written, q attends.

Kinds of case:
  tables  block tables, slots and positions of a step from the requests' lengths before and after it
  append  k and v of the step's rows written to their slots, and what their blocks then hold read back
  attend  causal attention of each request's new rows over its whole cache

Head shapes are those of a Qwen2-1.5B decoder (12 q / 2 kv heads of 128), of Llama-style 8B sizes (32 / 8 of 128),
and one head of 64 or 80 per kv head.  Lengths come from the case alone; contents and block ids from the seed.
With `own` false run() is elementary torch in 32 bits; with it true, the library's calls.
"""
import math
import random

import torch

own = False

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
GPU = "cuda"
#: the most that a drawn attend case costs
MOST_FLOPS, MOST_BYTES = 1.2e11, 4e8


def _attend(name, **kw):
    case = {"name": name, "kind": "attend", "requests": 1, "new_lo": 1, "new_hi": 1, "past_lo": 0, "past_hi": 0, "decodes": 0, "pad": 0,
            "heads": 12, "kv_heads": 2, "dim": 128, "block": 64, "dtype": "bf16", "lens": 1}
    return {**case, **kw}


def listed():
    return [
        # one generated token for each of 8 requests: the tables of the smallest step
        {"name": "tables decode 8", "kind": "tables", "requests": 8, "new_lo": 1, "new_hi": 1, "past_lo": 50, "past_hi": 2000, "ended": 0,
         "pad": 0, "block": 64, "lens": 1},
        # a step of a large server: prompts and tokens together, a quarter of the requests ended and give their blocks back
        {"name": "tables mixed 512", "kind": "tables", "requests": 512, "new_lo": 1, "new_hi": 2048, "past_lo": 1, "past_hi": 8192,
         "ended": 128, "pad": 1000, "block": 16, "lens": 2},
        # one token's k and v for each of 64 requests, at any offset of their last blocks: the write of every decode step
        {"name": "append decode 64 bf16", "kind": "append", "requests": 64, "new_lo": 1, "new_hi": 1, "past_lo": 1, "past_hi": 4096, "pad": 0,
         "heads": 12, "kv_heads": 2, "dim": 128, "block": 64, "dtype": "bf16", "lens": 3},
        # a few prompts at once, from their first token
        {"name": "append prompts 8k bf16", "kind": "append", "requests": 6, "new_lo": 1100, "new_hi": 2000, "past_lo": 0, "past_hi": 0, "pad": 17,
         "heads": 32, "kv_heads": 8, "dim": 128, "block": 64, "dtype": "bf16", "lens": 4},
        # chunks that begin and end inside small blocks, f32 as checkpoints load by default, a head size between the usual ones
        {"name": "append chunks f32 d80", "kind": "append", "requests": 9, "new_lo": 3, "new_hi": 300, "past_lo": 5, "past_hi": 900, "pad": 5,
         "heads": 10, "kv_heads": 10, "dim": 80, "block": 16, "dtype": "f32", "lens": 5},
        # one token of one request over a short cache: the call whose latency a single user feels
        _attend("attend decode 1x200 bf16", past_lo=199, past_hi=199),
        # one token over a very long cache
        _attend("attend decode 1x131072 bf16", past_lo=131071, past_hi=131071),
        # a server's decode step: 64 requests of very different lengths
        _attend("attend decode 64 ragged bf16", requests=64, past_lo=100, past_hi=8192, heads=32, kv_heads=8, lens=6),
        # a few tokens of 16 requests checked at once (speculative decoding), small blocks and heads, rows behind the last
        _attend("attend verify 16x5 f16 d64", requests=16, new_lo=5, new_hi=5, past_lo=60, past_hi=3000, heads=16, kv_heads=16, dim=64, block=16,
                dtype="f16", pad=3, lens=7),
        # a chunk of a long prompt next to 24 requests that decode: a step that mixes both
        _attend("attend chunk 512 + 24 bf16", new_lo=512, new_hi=512, past_lo=300, past_hi=3500, decodes=24, heads=32, kv_heads=8, lens=8),
        # a short prompt's chunk in f32
        _attend("attend chunk 96 f32", requests=2, new_lo=40, new_hi=96, past_lo=100, past_hi=500, block=32, dtype="f32", lens=9),
        # long prompts in one pass: the bulk of a server's attention arithmetic
        _attend("attend prompts 8k bf16", requests=3, new_lo=2000, new_hi=3800, heads=32, kv_heads=8, lens=10),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    if lo <= 0:
        return 0 if hi <= 0 or rng.random() < 0.1 else _log(rng, 1, hi)
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["tables", "append", "attend", "attend", "attend"])
    lens, block = rng.randrange(1 << 30), rng.choice([16, 32, 64, 64, 128, 256])
    if kind == "tables":
        n = _log(rng, 1, 512)
        return {"kind": kind, "requests": n, "new_lo": 1, "new_hi": _log(rng, 1, 2048), "past_lo": 1, "past_hi": _log(rng, 16, 8192),
                "ended": rng.randrange(n), "pad": rng.choice([0, rng.randrange(1, 100)]), "block": block, "lens": lens}
    heads, kv_heads, dim = rng.choice([(12, 2, 128), (12, 2, 128), (32, 8, 128), (32, 8, 128), (16, 16, 64), (10, 10, 80)])
    dt = rng.choice(["bf16", "bf16", "bf16", "f16", "f32"])
    c = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "block": block, "dtype": dt, "lens": lens,
         "pad": rng.choice([0, rng.randrange(1, 100)])}
    if kind == "append":
        n = _log(rng, 1, 64)
        hi = _log(rng, 1, max(1, 8192 // n))
        return {**c, "requests": n, "new_lo": max(1, hi // 4), "new_hi": hi, "past_lo": 0, "past_hi": _log(rng, 1, 4096)}
    while True:
        n = _log(rng, 1, 64)
        form = rng.choice(["decode", "decode", "verify", "prompt", "chunk"])
        new = 1 if form == "decode" else rng.randrange(2, 9) if form == "verify" else _log(rng, 9, 4096)
        past = 0 if form == "prompt" else _log(rng, 16, 131072 if n < 4 else 8192)
        one = {**c, "requests": n, "new_lo": max(1, new // 2), "new_hi": new, "past_lo": past // 20, "past_hi": past,
               "decodes": rng.choice([0, _log(rng, 1, 32)]) if form == "chunk" else 0}
        w = work(one)
        old, total = _lengths(one)
        # the plain form holds every request's scores side by side
        wide = len(old) * heads * max(t - o for o, t in zip(old, total)) * max(total)
        if w["flops"] * (16 if dt == "f32" else 4 if dt == "f16" else 1) <= MOST_FLOPS and w["bytes"] <= MOST_BYTES and wide < 2e9:
            return one


def _lengths(case):
    """Each request's cached tokens before and after the step."""
    rng = random.Random(case["lens"])
    old = [_log(rng, case["past_lo"], case["past_hi"]) for _ in range(case["requests"])]
    new = [_log(rng, case["new_lo"], case["new_hi"]) for _ in range(case["requests"])]
    for _ in range(case.get("decodes", 0)):
        old.append(_log(rng, case["past_lo"], case["past_hi"]))
        new.append(1)
    total = [o + n for o, n in zip(old, new)]
    for r in rng.sample(range(len(old)), case.get("ended", 0)):
        total[r] = 0
    return old, total


def _blocks(n, block):
    return -(-n // block)


def work(case):
    old, total = _lengths(case)
    block = case["block"]
    rows = sum(max(0, t - o) for o, t in zip(old, total))
    if case["kind"] == "tables":
        moved = sum(abs(_blocks(t, block) - _blocks(o, block)) for o, t in zip(old, total))
        return {"bytes": 12 * len(old) + 16 * (rows + case["pad"]) + 8 * moved, "flops": 4 * rows}
    es, width = BYTES[case["dtype"]], case["kv_heads"] * case["dim"]
    if case["kind"] == "append":
        read = sum(t - o // block * block for o, t in zip(old, total))
        held = sum(_blocks(t, block) - o // block for o, t in zip(old, total))
        # k and v in, codes and scales out, and the codes in and the values out of the read-back
        return {"bytes": 2 * rows * width * (es + 1) + 2 * read * width * (es + 1) + 16 * held * case["kv_heads"] + 8 * (rows + read),
                "flops": 8 * rows * width + 2 * read * width}
    q = case["heads"] * case["dim"]
    seen = sum((t - o) * o + (t - o) * (t - o + 1) // 2 for o, t in zip(old, total))
    held = sum(_blocks(t, block) for t in total)
    return {"bytes": 2 * rows * q * es + 2 * sum(total) * width + held * (8 * case["kv_heads"] + 4) + 8 * len(old),
            "flops": 4 * q * seen}


# ---- what a program has in hand -------------------------------------------------------------


class _Memory:
    """A library tensor's device memory as torch's array protocol wants it."""

    def __init__(self, tensor, shape, kind):
        self.tensor = tensor
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": kind, "data": (tensor.data_ptr(), False), "version": 2,
                                         "strides": None}


class Buf:
    """One tensor on the GPU: `v` in torch and, for the library's calls, `t`, the library's tensor of the same memory."""

    KINDS = {torch.float32: ("F32", "<f4"), torch.float16: ("F16", "<f2"), torch.bfloat16: ("BF16", "<i2"), torch.int8: ("I8", "|i1"),
             torch.int32: ("I32", "<i4"), torch.int64: ("I64", "<i8")}

    def __init__(self, values):
        if not own:
            self.v = values.contiguous()
            return
        import llaisys_amd as L

        name, kind = self.KINDS[values.dtype]
        self.t = L.Tensor(tuple(values.shape), getattr(L.DataType, name), L.DeviceType.AMD, 0)
        self.v = torch.as_tensor(_Memory(self.t, values.shape, kind), device=GPU)
        if values.dtype == torch.bfloat16:
            self.v = self.v.view(torch.bfloat16)
        self.v.copy_(values)


class State:
    pass


def _ints(values, dt=torch.int32):
    return torch.tensor(values, dtype=dt, device=GPU)


def _inputs(case, seed):
    """Every input of the case by name, as torch tensors on the GPU."""
    g = torch.Generator(device=GPU)
    g.manual_seed(int(seed))
    old, total = _lengths(case)
    block, n = case["block"], len(old)
    rows = [max(0, t - o) for o, t in zip(old, total)]
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    most = max(max(old), max(total))
    x = {"old": _ints(old), "total": _ints(total), "starts": _ints(starts)}
    # the pool: what the requests need before and after, a few spare blocks, all in an order of the seed's
    width = _blocks(most, block) + 2
    held = [max(_blocks(o, block), _blocks(t, block) if case["kind"] != "tables" else 0) for o, t in zip(old, total)]
    taken = sum(max(0, _blocks(t, block) - _blocks(o, block)) for o, t in zip(old, total)) if case["kind"] == "tables" else 0
    pool = sum(held) + taken + 3
    ids = torch.randperm(pool, generator=g, device=GPU).to(torch.int32)
    table = torch.full((n, width), -1, dtype=torch.int32, device=GPU)
    first = _ints([sum(held[:r]) for r in range(n)])
    col = torch.arange(width, device=GPU)[None, :]
    here = col < _ints(held)[:, None]
    table[here] = ids[(first[:, None] + col)[here]]
    x["table"] = table
    if case["kind"] == "tables":
        ring = torch.full((pool,), -1, dtype=torch.int32, device=GPU)
        # the ring's head stands anywhere, also near its end
        head = int(torch.randint(0, 3 * pool, (1,), generator=g, device=GPU))
        free = ids[sum(held):]
        ring[(head + torch.arange(free.numel(), device=GPU)) % pool] = free
        x["ring"], x["ring_in"] = ring, _ints([head, head + free.numel()], torch.int64)
        return x
    h, d, dt = case["kv_heads"], case["dim"], TORCH[case["dtype"]]
    rows_padded = starts[-1] + case["pad"]
    # a few channels of k and v are much larger than the others, as in trained models
    gain = torch.where(torch.rand(2, h, 1, d, generator=g, device=GPU) < 0.03, 8.0, 1.0)
    for i, name in enumerate(("k", "v")):
        scale = (0.8 + 0.4 * torch.rand(pool, h, generator=g, device=GPU)) * (28.0 / 127)
        codes = torch.randn(pool, h, block, d, generator=g, device=GPU).mul_(gain[i]).div_(scale[:, :, None, None])
        x[name + "_codes"], x[name + "_scale"] = codes.round_().clamp_(-127, 127).to(torch.int8), scale
        del codes
        if case["kind"] == "append":
            x[name] = torch.randn(rows_padded, h, d, generator=g, device=GPU).mul_(gain[i][:, 0]).to(dt)
    pos, slots, read = [], [], []
    if case["kind"] == "append":
        for r in range(n):
            at = torch.arange(old[r] // block * block, total[r], device=GPU)
            s = table[r].long()[at // block] * block + at % block
            read.append(s)
            slots.append(s[old[r] % block:])
        slots.append(torch.full((case["pad"],), -1, dtype=torch.int64, device=GPU))
        x["slots"], x["read"] = torch.cat(slots), torch.cat(read)
    else:
        x["q"] = torch.randn(rows_padded, case["heads"], d, generator=g, device=GPU).to(dt)
    return x


def prepare(case, seed):
    s, x, kind = State(), _inputs(case, seed), case["kind"]
    old, total = _lengths(case)
    s.case, s.scale = case, 1.0 / math.sqrt(case.get("dim", 1))
    for name, v in x.items():
        setattr(s, name, Buf(v))
    if kind == "tables":
        rows = sum(max(0, t - o) for o, t in zip(old, total)) + case["pad"]
        s.slots, s.pos = Buf(torch.zeros(rows, dtype=torch.int64, device=GPU)), Buf(torch.zeros(rows, dtype=torch.int64, device=GPU))
        s.ring_out = Buf(torch.zeros(2, dtype=torch.int64, device=GPU))
    elif kind == "append":
        shape, dt = (s.read.v.numel(), case["kv_heads"], case["dim"]), TORCH[case["dtype"]]
        s.k_back, s.v_back = Buf(torch.zeros(shape, dtype=dt, device=GPU)), Buf(torch.zeros(shape, dtype=dt, device=GPU))
    else:
        s.most_rows, s.most_keys = max(t - o for o, t in zip(old, total)), max(total)
        s.out = Buf(torch.zeros_like(s.q.v))
    torch.cuda.synchronize()
    return s


# ---- the plain forms -------------------------------------------------------------------------


def _plain_tables(s):
    block, old, total, table, ring = s.case["block"], s.old.v.long(), s.total.v.long(), s.table.v, s.ring.v
    n, f = old.numel(), ring.numel()
    b_old, b_new = (old + block - 1) // block, (total + block - 1) // block
    back, more, rows = (b_old - b_new).clamp(min=0), (b_new - b_old).clamp(min=0), (total - old).clamp(min=0)
    starts = torch.cat([rows.new_zeros(1), rows.cumsum(0)])
    head, tail = s.ring_in.v[0], s.ring_in.v[1]
    col = torch.arange(table.shape[1], device=GPU)[None, :]
    given = (col >= b_new[:, None]) & (col < b_old[:, None])
    at = (tail + (back.cumsum(0) - back)[:, None] + col - b_new[:, None]) % f
    ring[at[given]] = table[given]
    taken = (col >= b_old[:, None]) & (col < b_new[:, None])
    at = (head + (more.cumsum(0) - more)[:, None] + col - b_old[:, None]) % f
    table[taken] = ring[at[taken]]
    t = torch.arange(s.slots.v.numel(), device=GPU)
    r = torch.searchsorted(starts[1:], t, right=True).clamp(max=n - 1)
    live = t < starts[-1]
    pos = torch.where(live, old[r] + t - starts[r], 0)
    slots = torch.where(live, table[r, pos // block].long() * block + pos % block, -1)
    return table, slots, pos, starts.to(torch.int32), ring, torch.stack([head + more.sum(), tail + back.sum()])


def _plain_append(s):
    block, slots = s.case["block"], s.slots.v
    live = slots >= 0
    touched, at = torch.unique(slots[live] // block, return_inverse=True)
    # a code is the whole number next to an exact quotient: in 64 bits, which tell values next to a half apart
    off = slots[live] % block
    first = torch.full_like(touched, block).scatter_reduce_(0, at, off, "amin")
    back = []
    for x, codes, scale in ((s.k.v, s.k_codes.v, s.k_scale.v), (s.v.v, s.v_codes.v, s.v_scale.v)):
        x = x[live].float()
        was = torch.where((first == 0)[:, None], 0.0, scale[touched])
        amax = torch.zeros_like(was).scatter_reduce_(0, at[:, None].expand(-1, was.shape[1]), x.abs().amax(-1), "amax")
        now = torch.maximum(was, amax / torch.full_like(amax, 127))
        kept = codes[touched].double()
        less = torch.nan_to_num(kept * was.double()[:, :, None, None] / now.double()[:, :, None, None], nan=0.0).round()
        kept = torch.where(torch.arange(block, device=GPU)[None, None, :, None] < first[:, None, None, None], less, kept)
        q = torch.nan_to_num(x.double() / now[at].double()[:, :, None], nan=0.0).round().clamp(-127, 127)
        kept[at, :, off] = q
        codes[touched] = kept.to(torch.int8)
        scale[touched] = now
        b, o = s.read.v // block, s.read.v % block
        back.append((codes[b, :, o].float() * scale[b][:, :, None]).to(TORCH[s.case["dtype"]]))
    return back[0], back[1], s.k_scale.v, s.v_scale.v


def _plain_attend(s):
    case, q, block = s.case, s.q.v, s.case["block"]
    h, d, g = case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"]
    n, starts, total = s.total.v.numel(), s.starts.v.long(), s.total.v.long()
    key = torch.arange(s.most_keys, device=GPU)
    b, o = s.table.v.long()[:, key // block].clamp(min=0), (key % block)[None, :].expand(n, -1)
    k = (s.k_codes.v[b, :, o].float() * s.k_scale.v[b][..., None]).permute(0, 2, 3, 1).contiguous()  # [n, h, d, keys]
    v = (s.v_codes.v[b, :, o].float() * s.v_scale.v[b][..., None]).permute(0, 2, 1, 3).contiguous()  # [n, h, keys, d]
    i = torch.arange(s.most_rows, device=GPU)
    rows = starts[1:] - starts[:-1]
    at = (starts[:-1, None] + i).clamp(max=q.shape[0] - 1)
    x = q[at].float().view(n, s.most_rows, h, g, d).permute(0, 2, 3, 1, 4).reshape(n, h, g * s.most_rows, d)
    p = (x @ k).mul_(s.scale).view(n, h, g, s.most_rows, s.most_keys)
    hidden = key[None, None, :] > (total - rows)[:, None, None] + i[None, :, None]
    p.masked_fill_(hidden[:, None, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    p.div_(p.sum(-1, keepdim=True).clamp(min=1e-38))
    y = (p.view(n, h, g * s.most_rows, s.most_keys) @ v).view(n, h, g, s.most_rows, d).permute(0, 3, 1, 2, 4)
    live = i[None, :] < rows[:, None]
    s.out.v[at[live]] = y.reshape(n, s.most_rows, h * g, d)[live].to(q.dtype)
    return s.out.v


# ---- one pass --------------------------------------------------------------------------------


def run(s):
    kind = s.case["kind"]
    if not own:
        return {"tables": _plain_tables, "append": _plain_append, "attend": _plain_attend}[kind](s)
    from llaisys_amd import Ops

    if kind == "tables":
        Ops.paged_tables(s.table.t, s.slots.t, s.pos.t, s.starts.t, s.ring_out.t, s.old.t, s.total.t, s.ring.t, s.ring_in.t, s.case["block"])
        return s.table.v, s.slots.v, s.pos.v, s.starts.v, s.ring.v, s.ring_out.v
    if kind == "append":
        Ops.paged_kv_append_int8(s.k_codes.t, s.k_scale.t, s.v_codes.t, s.v_scale.t, s.k.t, s.v.t, s.slots.t)
        Ops.paged_kv_read_int8(s.k_back.t, s.v_back.t, s.k_codes.t, s.k_scale.t, s.v_codes.t, s.v_scale.t, s.read.t)
        return s.k_back.v, s.v_back.v, s.k_scale.v, s.v_scale.v
    Ops.paged_attention_int8kv(s.out.t, s.q.t, s.k_codes.t, s.k_scale.t, s.v_codes.t, s.v_scale.t, s.table.t, s.starts.t, s.total.t, s.scale)
    return s.out.v


# ---- the definition in 64 bits ---------------------------------------------------------------


def exact(case, seed):
    if case["kind"] == "tables":
        return None  # whole numbers
    x = _inputs(case, seed)
    old, total = _lengths(case)
    block, table = case["block"], x["table"].long()
    if case["kind"] == "append":
        out, scales, row = {"k": [], "v": []}, {n: x[n + "_scale"].double() for n in "kv"}, 0
        for r, (o, t) in enumerate(zip(old, total)):
            for b in range(o // block, _blocks(t, block)):
                lo, hi, blk = max(o, b * block), min(t, (b + 1) * block), int(table[r, b])
                for n in "kv":
                    new = x[n][row:row + hi - lo].double()  # [rows, h, d]
                    amax = (new.abs().amax(dim=(0, 2)) / 127).float().double()  # a scale is what 32 bits hold
                    was = scales[n][blk]
                    now = torch.maximum(was, amax) if lo > b * block else amax
                    before = x[n + "_codes"][blk, :, :lo - b * block].double()
                    before = torch.round(before * was[:, None, None] / now[:, None, None]) * now[:, None, None]
                    after = torch.round(new / now[:, None]).clamp(-127, 127) * now[:, None]
                    out[n] += [before.transpose(0, 1), after]
                    scales[n][blk] = now
                row += hi - lo
        return torch.cat(out["k"]), torch.cat(out["v"]), scales["k"], scales["v"]
    q, heads, g = x["q"].double(), case["heads"], case["heads"] // case["kv_heads"]
    out, row = torch.zeros_like(q), 0
    for r, (o, t) in enumerate(zip(old, total)):
        ids = table[r, :_blocks(t, block)]
        kv = []
        for n in "kv":
            values = x[n + "_codes"][ids].double() * x[n + "_scale"][ids].double()[:, :, None, None]
            kv.append(values.transpose(0, 1).reshape(case["kv_heads"], -1, case["dim"])[:, :t])
        last = torch.arange(o, t, device=GPU)[:, None]
        for i in range(heads):
            k, v = kv[0][i // g], kv[1][i // g]
            w = torch.mm(q[row:row + t - o, i].contiguous(), k.t().contiguous()) / math.sqrt(case["dim"])
            w = torch.softmax(w.masked_fill(torch.arange(t, device=GPU)[None, :] > last, -math.inf), dim=-1)
            out[row:row + t - o, i] = torch.mm(w, v.contiguous())
        row += t - o
    return out
