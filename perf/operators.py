"""Attention over packed prompts and over a cache held in 8 bits, as cases that
can be timed and checked: each in its plain form (elementary torch operations
in 32 bits) and through the library's entry points.

``kind`` says what one pass is:

* ``prompt``: attention of packed prompts of different lengths over their own
  keys (and, where ``cached`` is not zero, that many earlier ones), grouped
  heads, causal or not, with or without a sliding window.
* ``write``: the keys and values of new tokens quantised into the cache after
  ``cached`` earlier ones, and what the touched blocks then hold read back.
* ``attend``: attention of the last ``tokens`` tokens of each sequence over
  the cache.

The cache holds blocks of 32 tokens.  A block has, for each head, a plane of
keys and a plane of values, ``32 P`` bytes each with P the head size rounded up
to a multiple of 32, and a 32-bit scale for each plane; a byte u stands for
(u - 128) scale.  With c = d // 32, element (token t, d) of a key plane is byte
(c, (d % 32) // 8, t % 16, t // 16, d % 8) of an array [P / 32, 4, 16, 2, 8], of
a value plane byte (c, (t % 16) // 4, d % 16, (d % 32) // 16, 4 (t // 16) + t % 4)
of one of the same shape.
"""

import math
import random

import torch

own = False  # whether run() calls the library

BLOCK = 32  # tokens


def _prompt(name, sequences, tokens, ragged, heads, kv_heads, head_dim, cached=0, causal=True, window=0):
    return {"name": name, "kind": "prompt", "sequences": sequences, "tokens": tokens, "ragged": ragged,
            "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "cached": cached, "causal": causal,
            "window": window}


def _write(name, sequences, tokens, ragged, kv_heads, head_dim, cached=0):
    return {"name": name, "kind": "write", "sequences": sequences, "tokens": tokens, "ragged": ragged,
            "kv_heads": kv_heads, "head_dim": head_dim, "cached": cached}


def _attend(name, sequences, tokens, context, ragged, heads, kv_heads, head_dim, window=0):
    return {"name": name, "kind": "attend", "sequences": sequences, "tokens": tokens, "context": context,
            "ragged": ragged, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "window": window}


def listed():
    return [
        # a short question: the latency of one call
        _prompt("prompt_short", 1, 45, 0, 32, 8, 128),
        # two dozen prompts of different lengths in one batch
        _prompt("prompt_packed", 24, 1000, 1, 32, 8, 128),
        # one long document
        _prompt("prompt_long", 1, 8192, 0, 32, 8, 128),
        # small heads in groups of seven, each token seeing the last 512
        _prompt("prompt_window", 4, 4000, 2, 28, 4, 64, window=512),
        # the ragged last chunk of a long prompt: few rows, many keys
        _prompt("prompt_chunk", 1, 333, 0, 32, 8, 128, cached=7000),
        # one new token in each of 64 sequences
        _write("write_step", 64, 1, 3, 8, 128, cached=5000),
        # whole prompts into an empty cache
        _write("write_prompts", 8, 2000, 4, 8, 128),
        # one conversation, one token: the latency of one call
        _attend("decode_one", 1, 1, 600, 0, 32, 8, 128),
        # 64 conversations of different lengths, one token each
        _attend("decode_batch", 64, 1, 8192, 5, 32, 8, 128),
        # one token after a very long document
        _attend("decode_long", 1, 1, 131000, 0, 32, 8, 128),
        # five drafted tokens checked at once in each of 16 sequences, groups of
        # five heads
        _attend("decode_drafts", 16, 5, 4096, 6, 40, 8, 64),
        # a chunk of a prompt whose earlier tokens are in the cache
        _attend("chunk_cached", 1, 512, 8192, 0, 32, 8, 128),
    ]


# --- ranges ---------------------------------------------------------------


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


# A drawn case's limits: no more work than the largest listed one, and scores
# in the plain form that fit the card with room to spare.
_MOST_FLOPS = 5.5e11
_MOST_BYTES = 9e8
_MOST_SCORES = 1 << 31


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        if w["flops"] > _MOST_FLOPS or w["bytes"] > _MOST_BYTES or _scores(case) > _MOST_SCORES:
            continue
        if 3072 not in case.values() and case.get("heads", 0) * case["head_dim"] != 3072:
            return case


def _draw(rng):
    kind = rng.choice(["prompt", "prompt", "write", "attend", "attend"])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 16])
    group = rng.choice([1, 2, 3, 4, 4, 5, 7, 8])
    head_dim = rng.choice([64, 80, 96, 128, 128, 128, 256])
    ragged = rng.choice([0, rng.randrange(1, 1 << 20)])
    sequences = rng.choice([1, _log_int(rng, 2, 64)])
    heads = kv_heads * group
    if kind == "prompt":
        return _unnamed(_prompt("", sequences, _log_int(rng, 1, 8192), ragged, heads, kv_heads, head_dim,
                                cached=rng.choice([0, 0, _log_int(rng, 1, 8192)]), **_mask(rng)))
    if kind == "write":
        tokens = rng.choice([1, _log_int(rng, 1, 8192)])
        return _unnamed(_write("", sequences, tokens, ragged, kv_heads, head_dim,
                               cached=rng.choice([0, _log_int(rng, 1, 16384)])))
    tokens = rng.choice([1, 1, _log_int(rng, 2, 8), _log_int(rng, 16, 1024)])
    context = max(tokens, _log_int(rng, 1, 131072))
    window = rng.choice([0, 0, 0, _log_int(rng, 16, 4096)])
    return _unnamed(_attend("", sequences, tokens, context, ragged, heads, kv_heads, head_dim, window=window))


def _mask(rng):
    if rng.random() < 0.15:
        return {"causal": False}
    return {"window": rng.choice([0, 0, 0, _log_int(rng, 16, 4096)])}


def _unnamed(case):
    del case["name"]
    return case


def _lengths(case):
    """New tokens of each sequence, and tokens of each sequence after them."""
    n = case["sequences"]
    rng = random.Random(case["ragged"])

    def spread(least, most):
        if not case["ragged"]:
            return [most] * n
        return [most] + [rng.randint(least, most) for _ in range(n - 1)]

    if case["kind"] == "attend":
        return [case["tokens"]] * n, spread(case["tokens"], case["context"])
    new = spread(1, case["tokens"])
    cached = spread(0, case["cached"]) if case["cached"] else [0] * n
    return new, [a + b for a, b in zip(new, cached)]


def _scores(case):
    if case["kind"] == "write":
        return 0
    new, total = _lengths(case)
    return case["sequences"] * case["heads"] * max(new) * max(total)


# --- inputs ---------------------------------------------------------------


def _normal(g, *shape, std=1.0):
    return torch.randn(*shape, device="cuda", generator=g).mul_(std).to(torch.float16)


def _keys(g, tokens, heads, head_dim):
    """Keys whose channels differ in size, as a trained projection's do."""
    gain = torch.randn(heads, head_dim, device="cuda", generator=g).mul_(0.4).exp_()
    return (torch.randn(tokens, heads, head_dim, device="cuda", generator=g) * gain).to(torch.float16)


def _offsets(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _blocks(n):
    return -(-n // BLOCK)


def _padded(head_dim):
    return -(-head_dim // 32) * 32


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    new, total = _lengths(case)
    d, kv_heads = case["head_dim"], case["kv_heads"]
    s = {"case": dict(case), "tokens": sum(new), "most_new": max(new), "most_total": max(total)}
    s["new_at"], s["lengths"] = _offsets(new), _ints(total)
    s["positions"] = _ints([t - n for n, t in zip(new, total)])
    if case["kind"] != "write":
        s["q"] = _normal(g, s["tokens"], case["heads"], d, std=1.5)
        s["out"] = torch.empty_like(s["q"])
    if case["kind"] == "prompt":
        s["keys"] = sum(total)
        s["key_at"] = _offsets(total)
        s["k"] = _keys(g, s["keys"], kv_heads, d)
        s["v"] = _normal(g, s["keys"], kv_heads, d)
        return s
    # a cache whose blocks were given out in no order, some unused
    p = _padded(d)
    table_blocks = _blocks(max(total))
    used = case["sequences"] * table_blocks
    s["cache_blocks"], s["table_blocks"] = used + 3, table_blocks
    order = torch.randperm(used + 3, device="cuda", generator=g)[:used].to(torch.int32)
    s["table"] = order.view(case["sequences"], table_blocks)
    planes = (s["cache_blocks"], kv_heads, 2, BLOCK * p)
    s["cache"] = torch.randint(1, 256, planes, dtype=torch.uint8, device="cuda", generator=g)
    s["scales"] = torch.rand(planes[:3], device="cuda", generator=g).mul_(0.01).add_(0.01)
    if case["kind"] == "write":
        s["k"] = _keys(g, s["tokens"], kv_heads, d)
        s["v"] = _normal(g, s["tokens"], kv_heads, d)
        # what is read back: the touched blocks, from each one's first token
        first = [(t - n) // BLOCK * BLOCK for n, t in zip(new, total)]
        held = [t - f for f, t in zip(first, total)]
        s["held"], s["held_at"], s["first"] = sum(held), _offsets(held), _ints(first)
        s["k_held"] = torch.empty(s["held"], kv_heads, d, dtype=torch.float16, device="cuda")
        s["v_held"] = torch.empty_like(s["k_held"])
    return s


# --- one pass -------------------------------------------------------------


def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"prompt": _own_prompt, "write": _own_write, "attend": _own_attend}[kind](s, s["case"])
    return {"prompt": _plain_prompt, "write": _plain_write, "attend": _plain_attend}[kind](s, s["case"])


_kept = {}


def _library(workspace_bytes=0):
    """What a program keeps: the library's entry points, a stream, a workspace
    for the largest call so far."""
    if not _kept:
        from mote_amd import ops
        from mote_amd.device import Stream

        _kept.update(ops=ops, stream=Stream(), workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    if _kept["workspace"].numel() < workspace_bytes:
        _kept["workspace"] = torch.empty(workspace_bytes, dtype=torch.uint8, device="cuda")
    return _kept["ops"], _kept["stream"], _kept["workspace"]


def _own_prompt(s, case):
    ops, stream, work_area = _library()
    shape = (case["sequences"], s["tokens"], s["keys"], s["most_total"], case["heads"], case["kv_heads"],
             case["head_dim"])
    need = ops.prompt_attention_workspace(*shape)
    if need > work_area.numel():
        work_area = _library(need)[2]
    ops.prompt_attention_f16(
        s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["out"].data_ptr(), s["new_at"].data_ptr(),
        s["key_at"].data_ptr(), *shape, case["head_dim"] ** -0.5, work_area.data_ptr(), work_area.numel(), stream,
        causal=case["causal"], window=case["window"])
    return s["out"]


def _own_write(s, case):
    ops, stream, _ = _library()
    heads = (case["kv_heads"], case["head_dim"], s["table_blocks"], s["cache_blocks"])
    ops.kv_cache_append_q8(
        s["k"].data_ptr(), s["v"].data_ptr(), s["new_at"].data_ptr(), s["positions"].data_ptr(),
        s["table"].data_ptr(), s["cache"].data_ptr(), s["scales"].data_ptr(), case["sequences"], s["tokens"],
        *heads, stream)
    ops.kv_cache_read_q8_f16(
        s["cache"].data_ptr(), s["scales"].data_ptr(), s["held_at"].data_ptr(), s["first"].data_ptr(),
        s["table"].data_ptr(), s["k_held"].data_ptr(), s["v_held"].data_ptr(), case["sequences"], s["held"],
        *heads, stream)
    return {"k": s["k_held"], "v": s["v_held"]}


def _own_attend(s, case):
    ops, stream, work_area = _library()
    shape = (case["sequences"], s["tokens"], case["tokens"], s["most_total"], case["heads"], case["kv_heads"],
             case["head_dim"])
    need = ops.cache_attention_workspace(*shape)
    if need > work_area.numel():
        work_area = _library(need)[2]
    ops.cache_attention_q8_f16(
        s["q"].data_ptr(), s["cache"].data_ptr(), s["scales"].data_ptr(), s["new_at"].data_ptr(),
        s["lengths"].data_ptr(), s["table"].data_ptr(), s["out"].data_ptr(), *shape, s["table_blocks"],
        s["cache_blocks"], case["head_dim"] ** -0.5, work_area.data_ptr(), work_area.numel(), stream,
        window=case["window"])
    return s["out"]


# --- the plain forms ------------------------------------------------------


def _rows(at, most):
    """Packed row of (sequence, token), [n, most], and whether there is one."""
    i = torch.arange(most, device="cuda")
    there = i < (at[1:] - at[:-1])[:, None]
    return torch.where(there, at[:-1, None] + i, 0), there


def _attention(q, k, v, new, total, causal, window):
    """q [n, most_new, heads, d], k and v [n, most_total, kv_heads, d] in 32
    bits, new and total the lengths in use; a row that sees nothing is zero."""
    n, rows, heads, d = q.shape
    keys, kv_heads = k.shape[1:3]
    group = heads // kv_heads
    q = q.view(n, rows, kv_heads, group, d).permute(0, 2, 3, 1, 4).reshape(n * kv_heads, group * rows, d)
    k = k.permute(0, 2, 3, 1).reshape(n * kv_heads, d, keys)
    v = v.transpose(1, 2).reshape(n * kv_heads, keys, d)
    scores = torch.bmm(q, k).mul_(d ** -0.5).view(n, kv_heads * group, rows, keys)
    j = torch.arange(keys, device="cuda")[None, None, :]
    at = (total - new)[:, None, None] + torch.arange(rows, device="cuda")[None, :, None]
    sees = (j < total[:, None, None]).expand(n, rows, keys)
    if causal:
        sees = sees & (j <= at)
    if window:
        sees = sees & (j > at - window)
    scores.masked_fill_(~sees[:, None], float("-inf"))
    most = scores.amax(3, keepdim=True)
    most = torch.where(most == float("-inf"), 0.0, most)
    p = scores.sub_(most).exp_()
    p /= p.sum(3, keepdim=True).clamp_min_(1e-30)
    o = torch.bmm(p.view(n * kv_heads, group * rows, keys), v)
    return o.view(n, kv_heads, group, rows, d).permute(0, 3, 1, 2, 4).reshape(n, rows, heads, d)


def _plain_prompt(s, case):
    new_rows, there = _rows(s["new_at"], s["most_new"])
    key_rows, _ = _rows(s["key_at"], s["most_total"])
    new = s["new_at"][1:] - s["new_at"][:-1]
    o = _attention(s["q"].float()[new_rows], s["k"].float()[key_rows], s["v"].float()[key_rows], new, s["lengths"],
                   case["causal"], case["window"])
    return o[there].to(torch.float16)


def _plane_values(planes, which, p):
    """The tokens' bytes [..., 32, P] of key (0) or value (1) planes."""
    lead, c = planes.shape[:-1], p // 32
    if which == 0:  # c, g, m, half, j -> half m, c g j
        x = planes.view(*lead, c, 4, 16, 2, 8).movedim((-2, -3, -5, -4, -1), (-5, -4, -3, -2, -1))
    else:  # c, g, m, dd, (half, r) -> half g r, c dd m
        x = planes.view(*lead, c, 4, 16, 2, 2, 4).movedim((-2, -5, -1, -6, -3, -4), (-6, -5, -4, -3, -2, -1))
    return x.reshape(*lead, BLOCK, p)


def _cached(s, case, which, table):
    """Keys or values of the blocks in `table` [n, b], [n, 32 b, kv_heads, d]
    in 32 bits."""
    n, b = table.shape
    planes = s["cache"][:, :, which][table.long()]  # n, b, heads, bytes
    x = _plane_values(planes, which, _padded(case["head_dim"]))[..., : case["head_dim"]]
    x = (x.float() - 128.0) * s["scales"][:, :, which][table.long()][..., None, None]
    return x.transpose(2, 3).reshape(n, b * BLOCK, case["kv_heads"], case["head_dim"])


def _plain_attend(s, case):
    k, v = (_cached(s, case, which, s["table"]) for which in (0, 1))
    n, rows = case["sequences"], case["tokens"]
    new = s["new_at"][1:] - s["new_at"][:-1]
    q = s["q"].float().view(n, rows, case["heads"], case["head_dim"])
    return _attention(q, k, v, new, s["lengths"], True, case["window"]).to(torch.float16).reshape(s["q"].shape)


def _plain_write(s, case):
    d, kv_heads = case["head_dim"], case["kv_heads"]
    # the touched blocks of every sequence: their tokens' rows, old and new
    most = s["most_new"] + BLOCK - 1
    b = _blocks(most + 1)
    slot = s["first"][:, None] // BLOCK + torch.arange(b, device="cuda")
    table = torch.gather(s["table"], 1, slot.clamp_max(s["table_blocks"] - 1).long())
    at = s["first"][:, None] + torch.arange(b * BLOCK, device="cuda")
    old = at < s["positions"][:, None]
    is_new = ~old & (at < s["lengths"][:, None])
    row = torch.where(is_new, s["new_at"][:-1, None] + at - s["positions"][:, None], 0)
    held = {}
    for name, which in (("k", 0), ("v", 1)):
        x = s[name].float()[row] * is_new[..., None, None]
        x = x.view(-1, b, BLOCK, kv_heads, d)
        of = s["scales"][:, :, which][table.long()]  # n, b, heads
        has_old = (old.view(-1, b, BLOCK).any(2))[..., None]
        of = torch.where(has_old, of, 0.0)
        scale = torch.maximum(of, x.abs().amax((2, 4)) / 127.0)
        inverse = torch.where(scale > 0, 1.0 / scale, 0.0)[:, :, None, :, None]
        planes = s["cache"][:, :, which][table.long()]
        q = _plane_values(planes, which, _padded(d))[..., :d].transpose(2, 3).float() - 128.0
        # what is there is kept, or rounded again to a scale that has grown
        again = torch.round(q * (of[:, :, None, :, None] * inverse)).clamp_(-127.0, 127.0)
        grown = (scale > of)[:, :, None, :, None]
        fresh = torch.round(x * inverse).clamp_(-127.0, 127.0)
        q = torch.where(old.view(-1, b, BLOCK, 1, 1), torch.where(grown, again, q), fresh)
        y = (q * scale[:, :, None, :, None]).reshape(-1, b * BLOCK, kv_heads, d)
        held[name] = y[at < s["lengths"][:, None]].to(torch.float16)
    return held


# --- what a pass cannot do without ----------------------------------------


def _pairs(case):
    """(query, key) pairs that see each other, and keys that any query sees."""
    new, total = _lengths(case)
    window = case["window"]
    pairs = seen = 0
    for n, t in zip(new, total):
        if not case.get("causal", True):
            pairs, seen = pairs + n * t, seen + t
            continue
        least = t - n + 1  # keys of the first query
        if not window:
            pairs, seen = pairs + n * (least + t) // 2, seen + t
            continue
        whole = min(n, max(0, window - least))  # queries that see less than the window
        pairs += whole * least + whole * (whole - 1) // 2 + (n - whole) * window
        seen += min(t, window + n - 1)
    return pairs, seen


def work(case):
    new, total = _lengths(case)
    d, kv_heads = case["head_dim"], case["kv_heads"]
    plane = 2 * kv_heads * d  # elements of a token's keys and values
    if case["kind"] == "write":
        held = sum(t - (t - n) // BLOCK * BLOCK for n, t in zip(new, total))
        # new tokens read, their bytes written, the touched blocks read back;
        # a product and a rounding for each value on each way
        return {"bytes": plane * (3 * sum(new) + 3 * held), "flops": 2 * plane * (sum(new) + held)}
    pairs, seen = _pairs(case)
    q = 2 * 2 * case["heads"] * d * sum(new)  # queries read, outputs written
    per_token = plane * 2 if case["kind"] == "prompt" else plane + 8 * kv_heads / BLOCK
    return {"bytes": int(q + seen * per_token), "flops": 4 * d * case["heads"] * pairs}


# --- the same in 64 bits ---------------------------------------------------


def _byte_of(which, t, d):
    """Byte of element (t, d) in a plane, as the layout is defined."""
    c, x = d // 32, d % 32
    if which == 0:
        return (((c * 4 + x // 8) * 16 + t % 16) * 2 + t // 16) * 8 + d % 8
    return (((c * 4 + t % 16 // 4) * 16 + d % 16) * 2 + x // 16) * 8 + 4 * (t // 16) + t % 4


def _held64(s, case, which, sequence, first, last):
    """What the cache holds of tokens [first, last), [heads, last - first, d]."""
    t = torch.arange(first, last, device="cuda")
    d = torch.arange(case["head_dim"], device="cuda")
    block = s["table"][sequence].long()[t // BLOCK]
    at = _byte_of(which, (t % BLOCK)[:, None], d[None, :])
    byte = s["cache"][block, :, which].gather(2, at[:, None].expand(-1, case["kv_heads"], -1))
    return ((byte.double() - 128) * s["scales"][block, :, which].double()[..., None]).transpose(0, 1)


def _softmax64(q, k, v, case, first):
    """Queries [rows, d] at positions first, first + 1, ... over keys [t, d]."""
    scores = (q @ k.t()) / math.sqrt(case["head_dim"])
    j = torch.arange(k.shape[0], device="cuda")[None]
    i = first + torch.arange(q.shape[0], device="cuda")[:, None]
    if case.get("causal", True):
        scores[j > i] = float("-inf")
    if case["window"]:
        scores[j <= i - case["window"]] = float("-inf")
    return torch.softmax(scores, 1) @ v


def exact(case, seed):
    s = prepare(case, seed)
    new, total = _lengths(case)
    if case["kind"] == "write":
        return {"k": _exact_write(s, case, 0, new, total), "v": _exact_write(s, case, 1, new, total)}
    if case["sequences"] * case["heads"] > 8000:
        return None  # too many small products to be quick
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    group = case["heads"] // case["kv_heads"]
    row = key = 0
    for i, (n, t) in enumerate(zip(new, total)):
        if case["kind"] == "prompt":
            k, v = (s[x][key:key + t].double().transpose(0, 1) for x in ("k", "v"))
        else:
            k, v = (_held64(s, case, which, i, 0, t) for which in (0, 1))
        for h in range(case["heads"]):
            q = s["q"][row:row + n, h].double()
            out[row:row + n, h] = _softmax64(q, k[h // group], v[h // group], case, t - n)
        row, key = row + n, key + t
    return out


def _exact_write(s, case, which, new, total):
    """The touched blocks' values: the scale of a block is the largest of its
    old one (where it holds earlier tokens) and of the new tokens' largest
    magnitude over 127."""
    given = (s["k"] if which == 0 else s["v"]).double()
    out = []
    row = 0
    for i, (n, t) in enumerate(zip(new, total)):
        at = t - n
        x = given[row:row + n].transpose(0, 1)  # heads, n, d
        row += n
        head = min(n, -at % BLOCK) if at % BLOCK else 0  # tokens that join a block begun earlier
        if at % BLOCK:
            block = s["table"][i].long()[at // BLOCK]
            old = _held64(s, case, which, i, at // BLOCK * BLOCK, at)
            of = s["scales"][block, :, which].double()
            scale = torch.maximum(of, x[:, :head].abs().amax((1, 2)) / 127)[:, None, None]
            both = torch.cat([old, x[:, :head]], 1)
            out.append((torch.round(both / scale) * scale).transpose(0, 1))
        x = torch.nn.functional.pad(x[:, head:], (0, 0, 0, -(n - head) % BLOCK))
        x = x.reshape(case["kv_heads"], -1, BLOCK, case["head_dim"])
        scale = x.abs().amax((2, 3), keepdim=True) / 127
        y = torch.where(scale > 0, torch.round(x / scale) * scale, x).flatten(1, 2)[:, : n - head]
        out.append(y.transpose(0, 1))
    return torch.cat(out)
