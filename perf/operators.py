"""Performance cases of serving from the 8-bit paged cache: block tables, append, and attention of new tokens over cached ones.

A cache of one layer is four tensors: codes ``k``, ``v`` (float8 e4m3, [pages, kv heads, tokens of a page, row], row = 32, 64 or 128) and a
float32 scale per page and head.  A request's tokens lie in the pages that its row of the block table names, in order.  The fields of a case:

  op           'blocks', 'append' or 'attend'
  dtype        'bf16', 'f16', 'f32': type of q, k, v and results (not for 'blocks')
  heads, kv, dim   query heads, key/value heads, head dim
  page         tokens of a page
  requests     requests in the batch
  shortest, longest   tokens of a request before the call ('append', 'blocks') or with its new ones ('attend'), spread over their logarithm
  new          new tokens of a request: 1 ... new, spread likewise (all of them `new` where `even`)
  even         every request has the same number of new tokens
  current      attend_current: a query also sees its own key
  sum          'attend': out = o + rem * v is asked for, with the new tokens' own values
  leave        'blocks': every `leave`-th request gives tokens back in place of taking new ones (0: none)
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
TOP, LOWEST = 448.0, -118  # largest e4m3 value, smallest exponent of a scale


def _attend(dtype, heads, kv, dim, page, requests, shortest, longest, new=1, even=True, current=False, sum=False):
    return dict(op="attend", dtype=dtype, heads=heads, kv=kv, dim=dim, page=page, requests=requests, shortest=shortest, longest=longest,
                new=new, even=even, current=current, sum=sum)


def _append(dtype, kv, dim, page, requests, shortest, longest, new, even):
    return dict(op="append", dtype=dtype, kv=kv, dim=dim, page=page, requests=requests, shortest=shortest, longest=longest, new=new, even=even)


def _blocks(page, requests, shortest, longest, new, even, leave):
    return dict(op="blocks", page=page, requests=requests, shortest=shortest, longest=longest, new=new, even=even, leave=leave)


def listed():
    return [
        # the smallest call: one user, a short conversation, one layer of a small model
        dict(_attend("bf16", 4, 4, 64, 16, 1, 700, 700), name="token-small"),
        # one user of a larger model with a long document: 8 heads over 65536 tokens
        dict(_attend("bf16", 8, 8, 128, 64, 1, 65536, 65536, sum=True), name="token-long"),
        # the ordinary serving step: 64 users, four query heads share each key/value head
        dict(_attend("bf16", 32, 8, 128, 64, 64, 100, 4000, sum=True), name="token-batch-shared"),
        # many users of a model with a key/value head per query head, contexts up to 12000 tokens: bound by the cache's bytes
        dict(_attend("bf16", 32, 32, 128, 64, 32, 1000, 12000), name="token-batch-large"),
        # odd sizes in float32: head dim 50, 7 requests down to a single token, small pages
        dict(_attend("f32", 6, 3, 50, 16, 7, 1, 1111, current=True), name="token-f32-d50"),
        # a draft of up to 8 tokens per request is verified at once
        dict(_attend("f16", 16, 8, 64, 32, 16, 500, 3000, new=8, even=False), name="draft-8"),
        # the next turn of conversations, or a prompt in pieces: hundreds of new tokens over a cached context
        dict(_attend("bf16", 32, 8, 128, 64, 4, 2000, 5000, new=512, sum=True), name="turn-512"),
        # the new token of 64 users goes into the cache
        dict(_append("bf16", 8, 128, 64, 64, 100, 4000, 1, True), name="append-token"),
        # prompts of a few thousand tokens, ragged, go into the cache, some behind an earlier turn
        dict(_append("bf16", 32, 128, 64, 7, 0, 1000, 3700, False), name="append-prompts"),
        # the same at an odd head dim in float32
        dict(_append("f32", 6, 50, 16, 20, 3, 300, 200, False), name="append-f32-d50"),
        # block tables of a serving step: 256 users take one token each, every 16th takes tokens back
        dict(_blocks(64, 256, 100, 4000, 1, True, 16), name="blocks-token"),
        # block tables when prompts come in: 48 requests of up to 8192 new tokens, every fifth one ends
        dict(_blocks(16, 48, 1, 4000, 8192, False, 5), name="blocks-prompts"),
    ]


def _spread(rng, low, high):
    """A whole number between the two, even over the logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low + 1), math.log(high + 1))) - 1)))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "blocks"])
    page = rng.choice([16, 32, 64, 128])
    if op == "blocks":
        return _blocks(page, _spread(rng, 1, 256), rng.randint(0, 60), _spread(rng, 64, 6000), _spread(rng, 1, 4096), rng.random() < 0.5, rng.choice([0, 0, 3, 7]))
    dtype, dim = rng.choice(["bf16", "bf16", "f16", "f32"]), rng.choice([32, 64, 128, 128, rng.randint(17, 127)])
    kv = _spread(rng, 1, 32)
    if op == "append":
        return _append(dtype, kv, dim, page, _spread(rng, 1, 64), rng.randint(0, 30), _spread(rng, 40, 2000), _spread(rng, 1, 900), rng.random() < 0.3)
    shared = rng.choice([1, 1, 2, 4, 5, 8])
    new = _spread(rng, 1, 300) if rng.random() < 0.4 else 1
    requests = _spread(rng, 1, 64 if new <= 16 else 4)
    most = min(65536, 4_000_000 // (requests * kv), 200_000_000 // (requests * kv * shared * new))  # no more bytes or products than the largest listed
    longest = _spread(rng, min(300, most), max(600, most))
    return _attend(dtype, kv * shared, kv, dim, page, requests, rng.randint(new, new + 100), max(longest, new + 200), new, rng.random() < 0.5, rng.random() < 0.3, rng.random() < 0.4)


def sizes(case):
    """(tokens, new tokens) of every request: part of the case, whatever the seed."""
    rng = random.Random("%(requests)d %(shortest)d %(longest)d %(new)d" % case)
    lengths = [_spread(rng, case["shortest"], case["longest"]) for _ in range(case["requests"])]
    new = [case["new"] if case["even"] else _spread(rng, 1, case["new"]) for _ in lengths]
    if case["op"] == "attend":
        lengths[0] = case["longest"]
        new = [min(n, t) for n, t in zip(new, lengths)]
    if case["op"] == "blocks" and case["leave"]:
        for i in range(case["leave"] - 1, len(new), case["leave"]):  # the request ends, or gives up a part of its last tokens
            new[i] = -(lengths[i] if i % 2 else min(lengths[i], 5))
    return lengths, new


def _row(dim):
    return 32 if dim <= 32 else 64 if dim <= 64 else 128


def _up(a, b):
    return -(-a // b)


def _pieces_bound(requests, tokens, page):
    m = min(requests, tokens)
    return m + min(m, tokens - m) + max(0, tokens - 2 * m) // page


def work(case):
    lengths, new = sizes(case)
    page, n = case["page"], sum(max(x, 0) for x in new)
    if case["op"] == "blocks":
        pages = sum(abs(_up(t + x, page) - _up(t, page)) for t, x in zip(lengths, new))  # written to the table or to the stack, read from the other
        return {"bytes": 4 * (4 * len(lengths) + 2 * pages + n) + 16 * _pieces_bound(len(lengths), n, page), "flops": n}
    size, kv, dim = BYTES[case["dtype"]], case["kv"], case["dim"]
    if case["op"] == "append":
        return {"bytes": 2 * kv * (n * dim * (size + 1) + 4 * sum(_up(x, page) for x in new)), "flops": 4 * kv * n * dim}
    heads, see = case["heads"], 1 if case["current"] else 0
    keys = sum(max(0, t - 1 + see) for t in lengths)  # the last token's visible keys: each code is read once
    pairs = sum(x * (t - x + see) + x * (x - 1) // 2 for t, x in zip(lengths, new))
    rows = heads * n * (2 * dim + 1) * size + (kv * n * dim * size if case["sum"] else 0)
    return {"bytes": 2 * kv * (keys * dim + 4 * _up(keys, page)) + 4 * _up(keys, page) + rows, "flops": 4 * dim * heads * pairs}


# ---------------------------------------------------------------------------------------------------------------- inputs
def _quantise(x):
    """Codes and power-of-two scales of [pages, heads, tokens, row]: the largest value of a page and head fits the type."""
    a = x.abs().amax(dim=(2, 3))
    s = torch.exp2(torch.ceil(torch.log2(a.double() / TOP).clamp(min=LOWEST))).float()
    s = torch.where(a > s * TOP, 2 * s, s)
    return (x / s[:, :, None, None]).to(torch.float8_e4m3fn), s


def _tables(lengths, page, width, pages, gen):
    """A table whose pages lie in random order, and the pages that are left."""
    order = torch.randperm(pages, generator=gen, device="cuda").int()
    held = torch.tensor([_up(t, page) for t in lengths], device="cuda")
    first = torch.cumsum(held, 0) - held
    at = torch.arange(width, device="cuda")[None, :]
    table = torch.where(at < held[:, None], order[(first[:, None] + at).clamp(max=pages - 1)], -1)
    return table.int(), order[int(held.sum()):]


def prepare(case, seed):
    lengths, new = sizes(case)
    page, count = case["page"], len(lengths)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    after = [t + x for t, x in zip(lengths, new)] if case["op"] != "attend" else lengths
    width = max(1, max(_up(max(a, t), page) for a, t in zip(after, lengths)))
    n = sum(max(x, 0) for x in new)
    if case["op"] == "blocks":
        before = sum(_up(t, page) for t in lengths)
        pages = before + sum(_up(max(x, 0), page) + 1 for x in new)
        table, left = _tables(lengths, page, width, pages, gen)
        free = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
        free[:left.numel()] = left
        return dict(case=case, page=page, tokens=n, lengths=ints(lengths), new=ints(new), tables=table, free=free, count=ints([left.numel()]))
    dtype, kv, dim = DTYPES[case["dtype"]], case["kv"], case["dim"]
    row = _row(dim)
    pages = sum(_up(a, page) for a in after) + 3
    table, _ = _tables(after, page, width, pages - 3, gen)
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda")  # noqa: E731
    # half of the heads look near, half break their stick over the whole context, as trained heads do: the mean of the logits is -ln(reach)
    reach = torch.tensor([3.0 if g % 2 else max(3.0, case["longest"] / 3) for g in range(kv)], device="cuda")
    lean = ((torch.log(reach) + 0.5) / math.sqrt(dim)).sqrt()
    codes, scales = [], []
    for value in (False, True):
        x = normal(pages, kv, page, row)
        if value:
            x *= torch.exp(0.5 * normal(pages, kv, page, 1))  # tokens of different weight
        else:
            x -= lean[None, :, None, None]
        x[..., dim:] = 0
        c, s = _quantise(x)
        codes.append(c)
        scales.append(s)
        del x
    state = dict(case=case, page=page, tables=table, k=codes[0], v=codes[1], ks=scales[0], vs=scales[1], lengths=ints(after))
    if case["op"] == "append":
        # the pieces of pages that the new tokens go to: (page, first row, tokens there before, new tokens)
        pieces, row_at, host = [], 0, table.cpu()
        for r, (t, x) in enumerate(zip(lengths, new)):
            for b in range(t // page, _up(t + x, page)):
                old, end = max(0, min(page, t - b * page)), min(page, t + x - b * page)
                pieces.append((int(host[r, b]), row_at + max(0, b * page - t), old, end - old))
            row_at += x
        pieces += [(-1, 0, 0, 0)] * (_pieces_bound(count, n, page) - len(pieces))
        louder = torch.exp(0.7 * normal(1, n, 1))  # some new tokens are larger than all that their page holds
        state.update(pieces=ints(pieces).reshape(-1, 4), new_k=(normal(kv, n, dim) * louder).to(dtype), new_v=(normal(kv, n, dim) * louder).to(dtype))
        return state
    shared = case["heads"] // kv
    q = normal(case["heads"], n, dim) + lean.repeat_interleave(shared)[:, None, None]
    ends = ints([sum(new[:i + 1]) for i in range(count)])
    state.update(q=q.to(dtype), ends=ends, most=max(new), own_v=normal(kv, n, dim).to(dtype) if case["sum"] else None, one=case["new"] == 1 and case["even"])
    return state


# ------------------------------------------------------------------------------------------------------------ plain forms
def _plain_blocks(s):
    page, T = s["page"], s["tokens"]
    before, new = s["lengths"].long(), s["new"].long()
    after = before + new
    had, has = (before + page - 1) // page, (after + page - 1) // page
    back, need = (had - has).clamp(min=0), (has - had).clamp(min=0)
    width, R = s["tables"].shape[1], before.numel()
    at = torch.arange(width, device="cuda")[None, :]
    # pages that come back go onto the stack, request by request
    given = (at >= has[:, None]) & (at < had[:, None])
    place = s["count"].long() + (torch.cumsum(back, 0) - back)[:, None] + at - has[:, None]
    size = s["free"].numel()
    stack = torch.cat([s["free"], s["free"].new_zeros(1)]).scatter(0, torch.where(given, place, size).reshape(-1), s["tables"].reshape(-1))[:size]
    # and the needed ones come off it
    top = s["count"].long() + back.sum() - 1
    taken = (at >= had[:, None]) & (at < has[:, None])
    place = top - (torch.cumsum(need, 0) - need)[:, None] - (at - had[:, None])
    s["tables"].copy_(torch.where(taken, stack[place.clamp(0, size - 1)], s["tables"]))
    count = s["count"] + (back.sum() - need.sum()).int()
    keep = torch.arange(size, device="cuda")
    s["free"].copy_(torch.where((keep >= s["count"]) & (keep < count), stack, s["free"]))
    # rows, slots and pieces of the new tokens
    grow = new.clamp(min=0)
    ends = torch.cumsum(grow, 0)
    t = torch.arange(T, device="cuda")
    r = torch.searchsorted(ends, t, right=True).clamp(max=R - 1)
    pos = before[r] + t - (ends - grow)[r]
    slots = s["tables"][r, pos // page].long() * page + pos % page
    parts = torch.where(grow > 0, (after + page - 1) // page - before // page, 0)
    last = torch.cumsum(parts, 0)
    i = torch.arange(_pieces_bound(R, T, page), device="cuda")
    r = torch.searchsorted(last, i, right=True).clamp(max=R - 1)
    b = before[r] // page + i - (last - parts)[r]
    old = (before[r] - b * page).clamp(0, page)
    stop = (after[r] - b * page).clamp(0, page)
    first = (ends - grow)[r] + (b * page - before[r]).clamp(min=0)
    pieces = torch.stack([s["tables"][r, b.clamp(0, width - 1)].long(), first, old, stop - old], 1)
    none = torch.tensor([-1, 0, 0, 0], device="cuda")
    pieces = torch.where((i < last[-1])[:, None], pieces, none)
    return [after.int(), count, ends.int(), slots.int(), pieces.int(), s["tables"], s["free"]]


def _plain_append_one(x, codes, scales, pieces, page):
    """One of keys and values: x [heads, tokens, dim] into codes and scales, in place."""
    live = pieces[:, 0] >= 0
    p = torch.where(live, pieces[:, 0], 0).long()
    at = torch.arange(page, device="cuda")[None, :]
    old, new = pieces[:, 2:3], pieces[:, 3:4]
    is_new = (at >= old) & (at < old + new)
    rows = (pieces[:, 1:2] + at - old).clamp(0, x.shape[1] - 1).long()
    fresh = x.float()[:, rows].permute(1, 0, 2, 3)  # [pieces, heads, page, dim]
    fresh = torch.nn.functional.pad(fresh, (0, codes.shape[-1] - x.shape[-1]))
    mask = is_new[:, None, :, None]
    a = torch.where(mask & fresh.isfinite(), fresh.abs(), 0).amax(dim=(2, 3))
    m, e = torch.frexp(a / TOP)  # a / 448 = m 2^e with 1/2 <= m < 1, rounded: put right below
    e = torch.where(m == 0.5, e - 1, e).clamp(LOWEST, 127)
    s = torch.ldexp(torch.ones_like(a), e)
    s = torch.where(a > s * TOP, 2 * s, s)
    s = torch.where((a <= s * 0.5 * TOP) & (s > 2.0 ** LOWEST), 0.5 * s, s)
    had = scales[p]
    s = torch.where(old > 0, torch.maximum(had, s), s)
    before = codes.view(torch.uint8)[p].view(torch.float8_e4m3fn).float() * (had / s)[..., None, None]
    value = torch.where(mask, fresh / s[..., None, None], before)
    coded = torch.where(value.isfinite(), value, float("nan")).to(torch.float8_e4m3fn).view(torch.uint8)
    coded = torch.where((at < old + new)[:, None, :, None], coded, codes.view(torch.uint8)[p])
    spare = codes.shape[0] - 1  # pieces without a page write the spare page's own bytes back to it
    to = torch.where(live, p, spare)
    keep = live[:, None]
    codes.view(torch.uint8).index_copy_(0, to, torch.where(keep[..., None, None], coded, codes.view(torch.uint8)[spare]))
    scales.index_copy_(0, to, torch.where(keep, s, scales[spare]))


def _plain_attend(s):
    case, page = s["case"], s["page"]
    kv, dim, dtype = case["kv"], case["dim"], s["q"].dtype
    lengths, ends, most = s["lengths"].long(), s["ends"].long(), s["most"]
    new = torch.diff(ends, prepend=ends.new_zeros(1))
    R, shared, width = lengths.numel(), case["heads"] // kv, s["tables"].shape[1]
    pages = s["tables"].long().clamp(min=0)
    gather = lambda c: c.view(torch.uint8)[pages].view(torch.float8_e4m3fn).permute(0, 2, 1, 3, 4).reshape(R, kv, width * page, -1)[..., :dim].float()  # noqa: E731
    scale = lambda x: x[pages].transpose(1, 2).repeat_interleave(page, 2)[:, :, None]  # noqa: E731
    rows = ((ends - new)[:, None] + torch.arange(most, device="cuda")).clamp(max=s["q"].shape[1] - 1)
    q = s["q"].float()[:, rows].reshape(kv, shared, R, most, dim).permute(2, 0, 1, 3, 4).reshape(R, kv, shared * most, dim)
    x = (q @ gather(s["k"]).transpose(2, 3)) * scale(s["ks"]) * (1.0 / math.sqrt(dim))
    x = x.view(R, kv, shared, most, -1)
    key = torch.arange(width * page, device="cuda")
    position = (lengths - new)[:, None] + torch.arange(most, device="cuda") + (1 if case["current"] else 0)
    sees = (key[None, None, :] < torch.minimum(position, lengths[:, None])[..., None])[:, None, None]
    soft = torch.where(sees, x.clamp(min=0) + torch.log1p(torch.exp(-x.abs())), 0.0).double()
    total = soft.sum(-1, keepdim=True)
    right = total - torch.cumsum(soft, -1)  # what the keys to the right of each take off the stick, in logarithms
    a = torch.where(sees, torch.exp(-right).float() / (1 + torch.exp(-x)), 0.0) * scale(s["vs"])[:, :, :, None]
    o = (a.view(R, kv, shared * most, -1) @ gather(s["v"])).view(R, kv * shared, most, dim)
    rem = torch.exp(-total[..., 0]).float().view(R, kv * shared, most)
    t = torch.arange(s["q"].shape[1], device="cuda")
    r = torch.searchsorted(ends, t, right=True)
    i = t - (ends - new)[r]
    o, rem = o[r, :, i].transpose(0, 1), rem[r, :, i].transpose(0, 1)
    if case["sum"]:
        o = o + rem.to(dtype).float()[..., None] * s["own_v"].float().repeat_interleave(shared, 0)
    return [o.to(dtype), rem.to(dtype)]


def run(s):
    case = s["case"]
    if case["op"] == "blocks":
        if own:
            from stickbreaking_attention_b200 import sb_cache_blocks
            b = sb_cache_blocks(s["lengths"], s["new"], s["tables"], s["free"], s["count"], s["page"], s["tokens"])
            return [b.lengths, b.free_count, b.ends, b.slots, b.pieces, s["tables"], s["free"]]
        return _plain_blocks(s)
    if case["op"] == "append":
        if own:
            from stickbreaking_attention_b200 import SbCache, sb_cache_append
            sb_cache_append(s["new_k"], s["new_v"], SbCache(s["k"], s["v"], s["ks"], s["vs"]), s["pieces"])
        else:
            _plain_append_one(s["new_k"], s["k"], s["ks"], s["pieces"], s["page"])
            _plain_append_one(s["new_v"], s["v"], s["vs"], s["pieces"], s["page"])
        return [s["k"], s["v"], s["ks"], s["vs"]]
    if own:
        from stickbreaking_attention_b200 import SbCache, sb_attn_cached
        return list(sb_attn_cached(s["q"], SbCache(s["k"], s["v"], s["ks"], s["vs"]), s["tables"], s["lengths"], None if s["one"] else s["ends"],
                                   attend_current=case["current"], v=s["own_v"]))
    return _plain_attend(s)


# ------------------------------------------------------------------------------------------------------- 64-bit definition
def _e4m3(x):
    """The nearest e4m3 values of float64 numbers (ties to even) that do not exceed 448."""
    _, e = torch.frexp(x)
    step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
    return torch.round(x / step) * step


def exact(case, seed):
    if case["op"] == "blocks":
        return None
    s = prepare(case, seed)
    if case["op"] == "append":
        out = []
        for x, codes, scales in ((s["new_k"].double(), s["k"], s["ks"]), (s["new_v"].double(), s["v"], s["vs"])):
            dim = x.shape[-1]
            values, scales = codes.float().double(), scales.double().clone()
            for p, first, old, new in s["pieces"].tolist():
                if p < 0:
                    continue
                part = x[:, first:first + new]
                a = part.abs().amax(dim=(1, 2))
                m, e = torch.frexp(a / TOP)
                scale = torch.where(m == 0.5, e - 1, e).clamp(min=LOWEST).double().exp2()
                if old:
                    scale = torch.maximum(scale, scales[p])
                    values[p, :, :old] = _e4m3(values[p, :, :old] * (scales[p] / scale)[:, None, None])
                values[p, :, old:old + new, :dim] = _e4m3(part / scale[:, None, None])
                values[p, :, old:old + new, dim:] = 0
                scales[p] = scale
            out += [values, scales]
        return [out[0], out[2], out[1], out[3]]
    kv, dim, page, heads = case["kv"], case["dim"], s["page"], case["heads"]
    shared = heads // kv
    lengths, new = sizes(case)
    outs, rems, at = [], [], 0
    for r, (length, n) in enumerate(zip(lengths, new)):
        p = s["tables"][r, :_up(length, page)].long()
        k, v = ((c[p].float().double() * z[p].double()[..., None, None]).transpose(0, 1).reshape(kv, -1, c.shape[-1])[:, :length, :dim]
                for c, z in ((s["k"], s["ks"]), (s["v"], s["vs"])))
        o, rem = [], []
        for h in range(heads):
            q = s["q"][h, at:at + n].double()
            beta = torch.sigmoid(q @ k[h // shared].T / math.sqrt(dim))
            i = torch.arange(length - n, length, device="cuda")[:, None] + (1 if case["current"] else 0)
            beta = torch.where(torch.arange(length, device="cuda")[None] < i, beta, 0.0)
            stick = torch.cumprod(torch.cat([torch.ones_like(beta[:, :1]), 1 - beta.flip(1)], 1), 1)  # what is left of it, from the right
            o.append((beta * stick[:, :-1].flip(1)) @ v[h // shared])
            rem.append(stick[:, -1])
        outs.append(torch.stack(o))
        rems.append(torch.stack(rem))
        at += n
    o, rem = torch.cat(outs, 1), torch.cat(rems, 1)
    if case["sum"]:
        o = o + rem[..., None] * s["own_v"].double().repeat_interleave(shared, 0)
    return [o, rem]
