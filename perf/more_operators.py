"""The MLP of a mixture of experts, and the microscaled formats it multiplies in,
as cases that can be timed and checked: each in its plain form (elementary torch
operations) and through the library's entry points.

``kind`` says what one pass is:

* ``route``: the experts of each token from the router's logits (softmax or
  sigmoid scores, a bias for the choice, groups of experts, the best ``top`` and
  their weights), and the plan of the products: the (token, choice) pairs in the
  order of their experts.  The last ``padded`` tokens have no expert.
* ``quantize``: rows to microscaled ``bits`` and back to their own type.
* ``linear``: y = x W^T, W in microscaled 4 bits, x in 4 or 6.
* ``gate_up``: for every pair, silu(x Wg^T) (x Wu^T) with its expert's weights;
  rows in the plan's order.
* ``down``: for every token the weighted sum of its pairs' products with their
  experts' weights.

The microscaled formats: blocks of 32 elements along a row, each with a scale
byte b that stands for 2^(b - 127).  4 bits: sign, 2 bits of exponent, 1 of
mantissa (0, 0.5, 1, 1.5, 2, 3, 4, 6), element 2 i of a block in the low half of
its byte i.  6 bits: sign, 2, 3 (0 to 2 in eighths, to 4 in quarters, to 7.5 in
halves), element i in bits 6 i to 6 i + 5 of 24 bytes; the first 16 bytes of all
of a row's blocks lie before the last 8 of all.  Rows are padded with zero bytes
to a multiple of four blocks, values and scales.
"""

import functools
import math
import random

import numpy as np
import torch

own = False  # whether run() calls the library

BLOCK = 32  # elements of a scale
PADDED = 128  # a row's elements are stored in multiples of these


def _route(name, tokens, experts, top, score, type, bias=False, groups=1, top_groups=1, best=1, renormalize=True,
           scale=1.0, padded=0):
    return {"name": name, "kind": "route", "tokens": tokens, "experts": experts, "top": top, "score": score,
            "type": type, "bias": bias, "groups": groups, "top_groups": top_groups, "best": best,
            "renormalize": renormalize, "scale": scale, "padded": padded}


def _quantize(name, rows, features, bits, type):
    return {"name": name, "kind": "quantize", "rows": rows, "features": features, "bits": bits, "type": type}


def _linear(name, rows, outputs, features, bits, type):
    return {"name": name, "kind": "linear", "rows": rows, "outputs": outputs, "features": features, "bits": bits,
            "type": type}


def _experts(name, kind, tokens, top, experts, hidden, inner, bits, ragged, skew=0.7, padded=0):
    return {"name": name, "kind": kind, "tokens": tokens, "top": top, "experts": experts, "hidden": hidden,
            "inner": inner, "bits": bits, "ragged": ragged, "skew": skew, "padded": padded}


def listed():
    return [
        # one generated token: the latency of a choice and its plan
        _route("route_one", 1, 128, 8, "softmax", "f16"),
        # a chunk of prompts, experts in groups, balanced by a bias, its end padded
        _route("route_prompt", 4096, 256, 8, "sigmoid", "f32", bias=True, groups=8, top_groups=4, best=2, scale=2.5,
               padded=60),
        # the activations of 64 sequences' tokens before a product
        _quantize("quantize_batch", 64, 4096, 4, "f16"),
        # a prompt's activations before a down projection
        _quantize("quantize_prompt", 4000, 14336, 6, "f16"),
        # one token through an up projection: the latency of a weight-streaming call
        _linear("linear_one", 1, 14336, 4096, 6, "f16"),
        # 48 sequences through a down projection
        _linear("linear_batch", 48, 4096, 14336, 4, "f32"),
        # a chunk of prompts through an up projection (the most operations)
        _linear("linear_prompt", 4096, 14336, 4096, 4, "f16"),
        # one token's eight experts, small ones
        _experts("gate_up_one", "gate_up", 1, 8, 128, 2048, 768, 6, 1),
        # 64 sequences over 32 experts, widths that are not multiples of 128
        _experts("gate_up_batch", "gate_up", 64, 4, 32, 2880, 2880, 6, 2),
        # a chunk of prompts over many small experts, its end padded
        _experts("gate_up_prompt", "gate_up", 4096, 8, 128, 2048, 768, 4, 3, padded=60),
        # 48 sequences, the weighted sum of six experts each
        _experts("down_batch", "down", 48, 6, 64, 4096, 1408, 4, 4),
        # a chunk of prompts over few experts of unequal use
        _experts("down_prompt", "down", 5000, 4, 32, 2880, 2880, 6, 5, skew=1.0),
    ]


# --- ranges ---------------------------------------------------------------


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """A row's elements: whole blocks, often a multiple of 128 or more."""
    step = rng.choice([32, 64, 128, 256, 512])
    return max(step, _log_int(rng, low, high) // step * step)


# A drawn case's limits: no more work than the largest listed ones.
_MOST_FLOPS = 4.8e11
_MOST_BYTES = 3.5e8
_MOST_ELEMENTS = 4000 * 14336
_MOST_WEIGHTS = 1 << 30  # of all experts, used or not


def draw(rng):
    while True:
        case = _draw(rng)
        if case["kind"] in ("gate_up", "down"):
            if case["experts"] * case["hidden"] * case["inner"] > _MOST_WEIGHTS:
                continue
        if case["kind"] == "quantize":
            if case["rows"] * case["features"] <= _MOST_ELEMENTS:
                return case
            continue
        w = work(case)
        if w["flops"] <= _MOST_FLOPS and w["bytes"] <= _MOST_BYTES:
            return case


def _draw(rng):
    kind = rng.choice(["route", "quantize", "linear", "linear", "gate_up", "gate_up", "down", "down"])
    tokens = rng.choice([1, _log_int(rng, 1, 8), _log_int(rng, 2, 64), _log_int(rng, 16, 8192), _log_int(rng, 64, 8192)])
    bits = rng.choice([4, 6])
    type = rng.choice(["f16", "f32"])
    if kind == "quantize":
        return _unnamed(_quantize("", tokens, _width(rng, 64, 32768), bits, type))
    if kind == "linear":
        return _unnamed(_linear("", tokens, rng.choice([_log_int(rng, 16, 16384), _width(rng, 256, 16384)]),
                                _width(rng, 64, 16384), bits, type))
    experts = rng.choice([8, 16, 32, 60, 64, 128, 160, 256])
    top = rng.choice([1, 2, 4, 6, 8])
    padded = rng.choice([0, 0, rng.randrange(tokens)])
    if kind == "route":
        divisors = [g for g in range(1, experts // max(top, 2) + 1) if experts % g == 0]
        groups = rng.choice([1, rng.choice(divisors)])
        top_groups = rng.randint(-(-top * groups // experts), groups)
        return _unnamed(_route("", tokens, experts, top, rng.choice(["softmax", "sigmoid"]), type,
                               bias=rng.random() < 0.5, groups=groups, top_groups=top_groups, best=rng.choice([1, 2]),
                               renormalize=rng.random() < 0.7, scale=rng.choice([1.0, 2.5]), padded=padded))
    return _unnamed(_experts("", kind, tokens, top, experts, _width(rng, 256, 8192), _width(rng, 128, 8192), bits,
                             rng.randrange(1 << 20), skew=rng.choice([0.3, 0.7, 1.2]), padded=padded))


def _unnamed(case):
    del case["name"]
    return case


# --- inputs ---------------------------------------------------------------


@functools.lru_cache(maxsize=64)
def _choices(tokens, top, experts, ragged, skew):
    """The experts of each token, [tokens, top], some experts liked more."""
    rng = np.random.default_rng(ragged)
    liked = rng.standard_normal(experts) * skew
    return np.argsort(-(rng.gumbel(size=(tokens, experts)) + liked), axis=1)[:, :top].astype(np.int32)


def _case_choices(case):
    """The same with no expert for the padded tokens."""
    ids = _choices(case["tokens"], case["top"], case["experts"], case["ragged"], case["skew"]).copy()
    if case["padded"]:
        ids[-case["padded"]:] = -1
    return ids


def _in_experts_order(ids, experts):
    """offsets [experts + 1] and the pairs in their experts' order, on the host."""
    flat = ids.reshape(-1)
    order = np.argsort(np.where(flat < 0, experts, flat), kind="stable")
    offsets = np.zeros(experts + 1, np.int64)
    offsets[1:] = np.cumsum(np.bincount(flat[flat >= 0], minlength=experts))
    rows = order.astype(np.int32)
    rows[offsets[-1]:] = -1
    return offsets, rows


def _padded(features):
    return -(-features // PADDED) * PADDED


def _bytes(g, *shape):
    return torch.randint(0, 256, shape, dtype=torch.uint8, device="cuda", generator=g)


def _weights(g, experts, outputs, features):
    """Values and scales whose products of unit inputs are about one."""
    middle = 127 - int(round(math.log2(2.5 * math.sqrt(features))))
    width = _padded(features)
    scales = torch.randint(middle - 1, middle + 2, (experts, outputs, width // BLOCK), dtype=torch.uint8,
                           device="cuda", generator=g)
    scales[..., features // BLOCK:] = 0
    values = _bytes(g, experts, outputs, width // 2)
    values[..., features // 2:] = 0
    return values, scales


def _activations(g, rows, features):
    """Unit rows, some channels larger, as a norm leaves them."""
    gain = torch.randn(features, device="cuda", generator=g).mul_(0.5).exp_()
    return torch.randn(rows, features, device="cuda", generator=g).mul_(gain)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": dict(case)}
    if case["kind"] == "route":
        return _prepare_route(s, case, g)
    if case["kind"] == "quantize":
        dtype = {"f16": torch.float16, "f32": torch.float32}[case["type"]]
        s["x"] = _activations(g, case["rows"], case["features"]).to(dtype)
        _quantized_room(s, case["rows"], case["features"], case["bits"])
        s["back"] = torch.empty_like(s["x"])
        return s
    if case["kind"] == "linear":
        s["w"], s["ws"] = _weights(g, 1, case["outputs"], case["features"])
        s["x"], s["xs"] = _plain_quantize(_activations(g, case["rows"], case["features"]), case["bits"])
        dtype = {"f16": torch.float16, "f32": torch.float32}[case["type"]]
        s["y"] = torch.empty(case["rows"], case["outputs"], dtype=dtype, device="cuda")
        return s
    # another seed: other tokens for other experts, as many to each as before
    rng = np.random.default_rng(seed)
    ids = _case_choices(case)
    real = case["tokens"] - case["padded"]
    ids[:real] = rng.permutation(case["experts"]).astype(np.int32)[ids[:real]][rng.permutation(real)]
    offsets, rows = _in_experts_order(ids, case["experts"])
    s["starts"] = offsets.tolist()
    s["ids"], s["rows"] = torch.from_numpy(ids).cuda(), torch.from_numpy(rows).cuda()
    s["offsets"] = torch.from_numpy(offsets.astype(np.int32)).cuda()
    pairs, hidden, inner = case["tokens"] * case["top"], case["hidden"], case["inner"]
    if case["kind"] == "gate_up":
        s["w"], s["ws"] = _weights(g, case["experts"], 2 * inner, hidden)
        s["x"], s["xs"] = _plain_quantize(_activations(g, case["tokens"], hidden), case["bits"])
        s["h"] = torch.zeros(pairs, inner, dtype=torch.float16, device="cuda")
        return s
    s["w"], s["ws"] = _weights(g, case["experts"], hidden, inner)
    s["x"], s["xs"] = _plain_quantize(_activations(g, pairs, inner), case["bits"])
    weights = torch.rand(case["tokens"], case["top"], device="cuda", generator=g).add_(0.1)
    s["weights"] = (weights / weights.sum(1, keepdim=True)) * (s["ids"] >= 0)
    s["y"] = torch.empty(case["tokens"], hidden, dtype=torch.float16, device="cuda")
    return s


def _prepare_route(s, case, g):
    tokens, experts, top = case["tokens"], case["experts"], case["top"]
    x = torch.randn(tokens, experts, device="cuda", generator=g).mul_(1.5)
    x += torch.randn(experts, device="cuda", generator=g).mul_(0.5)
    if case["padded"]:
        x[-case["padded"]:] = float("-inf")
    s["logits"] = x.to({"f16": torch.float16, "f32": torch.float32}[case["type"]])
    s["bias"] = torch.randn(experts, device="cuda", generator=g).mul_(0.05) if case["bias"] else None
    s["ids"] = torch.empty(tokens, top, dtype=torch.int32, device="cuda")
    s["weights"] = torch.empty(tokens, top, device="cuda")
    s["offsets"] = torch.empty(experts + 1, dtype=torch.int32, device="cuda")
    s["rows"] = torch.empty(tokens * top, dtype=torch.int32, device="cuda")
    return s


def _quantized_room(s, rows, features, bits):
    width = _padded(features)
    s["values"] = torch.empty(rows, width * bits // 8, dtype=torch.uint8, device="cuda")
    s["scales"] = torch.empty(rows, width // BLOCK, dtype=torch.uint8, device="cuda")


# --- one pass -------------------------------------------------------------


def run(s):
    kind = s["case"]["kind"]
    return (_OWN if own else _PLAIN)[kind](s, s["case"])


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


def _own_route(s, case):
    ops, stream, _ = _library()
    route = {"f16": ops.route_experts_f16, "f32": ops.route_experts_f32}[case["type"]]
    route(s["logits"].data_ptr(), None if s["bias"] is None else s["bias"].data_ptr(), s["ids"].data_ptr(),
          s["weights"].data_ptr(), case["tokens"], case["experts"], case["top"], stream,
          score={"softmax": ops.SOFTMAX, "sigmoid": ops.SIGMOID}[case["score"]], groups=case["groups"],
          top_groups=case["top_groups"], group_best=case["best"], renormalize=case["renormalize"],
          scale=case["scale"])
    ops.plan_experts(s["ids"].data_ptr(), s["offsets"].data_ptr(), s["rows"].data_ptr(), case["tokens"], case["top"],
                     case["experts"], stream)
    return {"ids": s["ids"], "weights": s["weights"], "offsets": s["offsets"], "rows": s["rows"]}


def _own_quantize(s, case):
    ops, stream, _ = _library()
    there, back = {"f16": (ops.mx_quantize_f16, ops.mx_dequantize_f16),
                   "f32": (ops.mx_quantize_f32, ops.mx_dequantize_f32)}[case["type"]]
    shape = (case["rows"], case["features"], case["bits"])
    there(s["x"].data_ptr(), s["values"].data_ptr(), s["scales"].data_ptr(), *shape, stream)
    back(s["values"].data_ptr(), s["scales"].data_ptr(), s["back"].data_ptr(), *shape, stream)
    return s["back"]


def _own_linear(s, case):
    ops, stream, _ = _library()
    linear = {"f16": ops.mx_linear_f16, "f32": ops.mx_linear_f32}[case["type"]]
    linear(s["x"].data_ptr(), s["xs"].data_ptr(), s["w"].data_ptr(), s["ws"].data_ptr(), s["y"].data_ptr(),
           case["rows"], case["outputs"], case["features"], case["bits"], stream)
    return s["y"]


def _own_gate_up(s, case):
    ops, stream, _ = _library()
    ops.experts_gate_up_silu_mx_f16(
        s["x"].data_ptr(), s["xs"].data_ptr(), s["w"].data_ptr(), s["ws"].data_ptr(), s["offsets"].data_ptr(),
        s["rows"].data_ptr(), s["h"].data_ptr(), case["tokens"], case["top"], case["experts"], case["hidden"],
        case["inner"], case["bits"], stream)
    return s["h"]


def _own_down(s, case):
    ops, stream, work_area = _library()
    shape = (case["tokens"], case["top"], case["experts"], case["hidden"], case["inner"])
    need = ops.experts_down_workspace(*shape)
    if need > work_area.numel():
        work_area = _library(need)[2]
    ops.experts_down_mx_f16(
        s["x"].data_ptr(), s["xs"].data_ptr(), s["w"].data_ptr(), s["ws"].data_ptr(), s["ids"].data_ptr(),
        s["offsets"].data_ptr(), s["rows"].data_ptr(), s["weights"].data_ptr(), s["y"].data_ptr(), *shape,
        case["bits"], work_area.data_ptr(), work_area.numel(), stream)
    return s["y"]


_OWN = {"route": _own_route, "quantize": _own_quantize, "linear": _own_linear, "gate_up": _own_gate_up,
        "down": _own_down}


# --- the plain forms ------------------------------------------------------


def _plain_route(s, case):
    tokens, experts, top = case["tokens"], case["experts"], case["top"]
    x = s["logits"].double()  # 64 bits: scores that 32 would round to the same are told apart
    there = torch.isfinite(x)
    if case["score"] == "softmax":
        most = torch.where(there, x, -1e300).amax(1, keepdim=True)
        e = torch.where(there, torch.exp(x - most), 0.0)
        score = e / e.sum(1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-x))
    choice = score if s["bias"] is None else score + s["bias"].double()
    choice = torch.where(there, choice, -torch.inf)
    groups = case["groups"]
    if case["top_groups"] < groups:
        best = torch.sort(choice.view(tokens, groups, -1), 2, descending=True)[0][:, :, :case["best"]]
        none = best[:, :, 0] == -torch.inf
        of = torch.where(best == -torch.inf, 0.0, best).sum(2).masked_fill(none, -torch.inf)
        kept = torch.sort(of, dim=1, descending=True, stable=True)[1][:, :case["top_groups"]]
        out = torch.ones(tokens, groups, dtype=torch.bool, device="cuda").scatter_(1, kept, False)
        choice = choice.view(tokens, groups, -1).masked_fill(out[:, :, None], -torch.inf).view(tokens, experts)
    choice, ids = torch.sort(choice, dim=1, descending=True, stable=True)
    choice, ids = choice[:, :top], ids[:, :top]
    none = choice == -torch.inf
    weights = torch.gather(score, 1, ids).masked_fill(none, 0.0)
    if case["renormalize"]:
        total = weights.sum(1, keepdim=True)
        weights = torch.where(total > 0, weights / total, 0.0)
    ids = ids.masked_fill(none, -1).to(torch.int32)
    offsets, rows = _plain_plan(ids, experts)
    return {"ids": ids, "weights": (weights * case["scale"]).float(), "offsets": offsets, "rows": rows}


def _plain_plan(ids, experts):
    flat = ids.reshape(-1)
    none = flat < 0
    expert, rows = torch.sort(torch.where(none, experts, flat), stable=True)
    of = torch.arange(experts + 1, dtype=torch.int32, device="cuda")
    offsets = torch.searchsorted(expert, of).to(torch.int32)
    return offsets, torch.where(expert == experts, -1, rows).to(torch.int32)


_SIZE = {4: (2, 6.0, 1), 6: (2, 7.5, 3)}  # exponent of the largest element, it, bits of mantissa


def _powers(device):
    """2^(b - 127) of every scale byte; 255 is not a number."""
    return torch.tensor([2.0 ** (b - 127) for b in range(255)] + [math.nan], dtype=torch.float32, device=device)


def _to_element(y, bits):
    """y to the nearest element, halves to the even one."""
    _, most, mantissa = _SIZE[bits]
    y = y.clamp(-most, most)
    exponent = (torch.frexp(y)[1] - 1).clamp_min(0)
    step = torch.exp2((exponent - mantissa).float())
    return torch.round(y / step) * step


def _plain_values(x, bits):
    """Each element as the multiple of its scale that it becomes, and the
    exponents of the scales."""
    x = x.float().view(x.shape[0], -1, BLOCK)
    most = x.abs().amax(2, keepdim=True)
    shared = torch.where(most > 0, torch.frexp(most)[1] - 1 - _SIZE[bits][0], -127).clamp_min(-127)
    # in two steps: 2^-shared alone can pass what 32 bits hold
    half = torch.div(shared, 2, rounding_mode="floor")
    y = x * torch.exp2(-half.float()) * torch.exp2((half - shared).float())
    return _to_element(y, bits), shared


def _elements(bits, device):
    """What each code stands for."""
    mantissa = _SIZE[bits][2]
    code = torch.arange(1 << (bits - 1), device=device)
    exponent, part = code >> mantissa, (code & ((1 << mantissa) - 1)).float() / (1 << mantissa)
    size = torch.where(exponent > 0, (1 + part) * torch.exp2((exponent - 1).float()), part)
    return torch.cat([size, -size])


def _plain_quantize(x, bits):
    """The bytes that stand for x: values [rows, padded features bits / 8] and scales."""
    rows, features = x.shape
    y, shared = _plain_values(x, bits)
    more = (0, 0, 0, (_padded(features) - features) // BLOCK)
    scales = torch.nn.functional.pad((shared + 127).to(torch.uint8), more).squeeze(2)
    y = torch.nn.functional.pad(y, more)
    size = _elements(bits, x.device)[:1 << (bits - 1)]
    code = torch.bucketize(y.abs(), size).to(torch.uint8) | (y < 0).to(torch.uint8) << (bits - 1)
    if bits == 4:
        return (code[..., ::2] | code[..., 1::2] << 4).view(rows, -1), scales
    a, b, c, d = (code[..., i::4] for i in range(4))
    block = torch.stack([a | b << 6, b >> 2 | c << 4, c >> 4 | d << 2], -1).view(rows, -1, 24)
    return torch.cat([block[..., :16].reshape(rows, -1), block[..., 16:].reshape(rows, -1)], 1), scales


def _plain_read(values, scales, bits):
    """What values [..., padded features bits / 8] and scales [..., padded
    features / 32] stand for, in 32 bits."""
    if bits == 4:
        code = torch.stack([values & 15, values >> 4], -1).flatten(-2)
    else:
        at = values.shape[-1] // 24 * 16
        block = torch.cat([values[..., :at].unflatten(-1, (-1, 16)), values[..., at:].unflatten(-1, (-1, 8))], -1)
        p, q, r = (block[..., i::3] for i in range(3))
        code = torch.stack([p & 63, p >> 6 | (q & 15) << 2, q >> 4 | (r & 3) << 4, r >> 2], -1).flatten(-3)
    of = _powers(values.device)[scales.int()]
    return (_elements(bits, values.device)[code.int()].unflatten(-1, (-1, BLOCK)) * of[..., None]).flatten(-2)


def _plain_quantize_pass(s, case):
    y, shared = _plain_values(s["x"], case["bits"])
    return (y * torch.exp2(shared.float())).view(s["x"].shape).to(s["x"].dtype)


def _plain_linear(s, case):
    x = _plain_read(s["x"], s["xs"], case["bits"])
    return (x @ _plain_read(s["w"][0], s["ws"][0], 4).t()).to(s["y"].dtype)


def _used(s):
    """Experts with pairs, and their rows in the plan."""
    starts = s["starts"]
    return [(e, a, b) for e, (a, b) in enumerate(zip(starts, starts[1:])) if b > a]


def _plain_gate_up(s, case):
    x = _plain_read(s["x"], s["xs"], case["bits"])
    h = torch.zeros(s["h"].shape, device="cuda")
    inner = case["inner"]
    token = s["rows"] // case["top"]
    for e, a, b in _used(s):
        y = x[token[a:b].long()] @ _plain_read(s["w"][e], s["ws"][e], 4).t()
        gate, up = y[:, :inner], y[:, inner:]
        h[a:b] = gate / (1 + torch.exp(-gate)) * up
    return h.to(torch.float16)


def _plain_down(s, case):
    x = _plain_read(s["x"], s["xs"], case["bits"])
    tokens, top = case["tokens"], case["top"]
    products = torch.zeros(tokens * top, case["hidden"], device="cuda")
    for e, a, b in _used(s):
        products[s["rows"][a:b].long()] = x[a:b] @ _plain_read(s["w"][e], s["ws"][e], 4).t()
    products = products.view(tokens, top, -1)
    y = torch.zeros(tokens, case["hidden"], device="cuda")
    for j in range(top):
        y += s["weights"][:, j, None] * products[:, j]
    return y.to(torch.float16)


_PLAIN = {"route": _plain_route, "quantize": _plain_quantize_pass, "linear": _plain_linear,
          "gate_up": _plain_gate_up, "down": _plain_down}


# --- what a pass cannot do without ----------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "route":
        element = 2 if case["type"] == "f16" else 4
        scores, pairs = case["tokens"] * case["experts"], case["tokens"] * case["top"]
        return {"bytes": scores * element + 4 * (3 * pairs + 2 * case["experts"] + 1), "flops": 4 * scores}
    if kind == "quantize":
        n = case["rows"] * case["features"]
        # there: read, largest, division and rounding, written; back: a product
        element = 2 if case["type"] == "f16" else 4
        return {"bytes": 2 * n * element + 2 * _held(n, case["bits"]), "flops": 4 * n}
    if kind == "linear":
        m, n, k = case["rows"], case["outputs"], case["features"]
        element = 2 if case["type"] == "f16" else 4
        return {"bytes": _held(m * k, case["bits"]) + _held(n * k, 4) + m * n * element, "flops": 2 * m * n * k}
    ids = _case_choices(case)
    pairs = int((ids >= 0).sum())
    used = np.unique(ids[ids >= 0]).size
    size = case["hidden"] * case["inner"]
    tokens = case["tokens"] - case["padded"]
    if kind == "gate_up":
        moved = _held(2 * used * size, 4) + _held(tokens * case["hidden"], case["bits"]) + 2 * pairs * case["inner"]
        return {"bytes": moved, "flops": 4 * pairs * size}
    moved = _held(used * size, 4) + _held(pairs * case["inner"], case["bits"]) + 2 * case["tokens"] * case["hidden"]
    return {"bytes": moved, "flops": 2 * pairs * size}


def _held(elements, bits):
    return elements * bits // 8 + elements // BLOCK


# --- the same in 64 bits ---------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"route": _exact_route, "quantize": _exact_quantize, "linear": _exact_linear, "gate_up": _exact_gate_up,
            "down": _exact_down}[case["kind"]](s, case)


def _exact_route(s, case):
    """The best experts one after the other, each the first of the largest."""
    x = s["logits"].double().cpu().numpy()
    bias = np.zeros(case["experts"]) if s["bias"] is None else s["bias"].double().cpu().numpy()
    ids = np.full((case["tokens"], case["top"]), -1, np.int32)
    weights = np.zeros((case["tokens"], case["top"]))
    of = np.arange(case["experts"]) // (case["experts"] // case["groups"])
    for t, row in enumerate(x):
        allowed = np.isfinite(row)
        if not allowed.any():
            continue
        if case["score"] == "softmax":
            score = np.where(allowed, np.exp(row - row[allowed].max()), 0)
            score /= math.fsum(score)
        else:
            score = 1 / (1 + np.exp(-row))
        choice = score + bias
        worth = [sum(sorted(choice[allowed & (of == g)])[-case["best"]:]) if (allowed & (of == g)).any() else -np.inf
                 for g in range(case["groups"])]
        kept = sorted(range(case["groups"]), key=lambda g: -worth[g])[:case["top_groups"]]
        left = np.where(allowed & np.isin(of, kept), choice, -np.inf)
        for j in range(case["top"]):
            best = int(left.argmax())
            if left[best] == -np.inf:
                break
            ids[t, j], weights[t, j] = best, score[best]
            left[best] = -np.inf
        if case["renormalize"] and weights[t].sum() > 0:
            weights[t] /= weights[t].sum()
    offsets, rows = _in_experts_order(ids, case["experts"])
    return {"ids": torch.from_numpy(ids).cuda(), "weights": torch.from_numpy(weights * case["scale"]).cuda(),
            "offsets": torch.from_numpy(offsets.astype(np.int32)).cuda(), "rows": torch.from_numpy(rows).cuda()}


def _elements64(bits):
    """Every value that an element's code can stand for, by its code."""
    if bits == 4:
        up = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    else:
        up = [i / 8 for i in range(16)] + [2 + i / 4 for i in range(8)] + [4 + i / 2 for i in range(8)]
    return torch.tensor(up + [-v for v in up], dtype=torch.float64, device="cuda")


def _exact_quantize(s, case):
    """The nearest of all elements, of two as near the one with the even code."""
    bits = case["bits"]
    elements = _elements64(bits)
    up = elements[:len(elements) // 2]
    x = s["x"].double().view(case["rows"], -1, BLOCK)
    out = torch.empty_like(x)
    for a in range(0, case["rows"], 512):  # a part at a time: 64 bits of everything is much
        part = x[a:a + 512]
        most = part.abs().amax(2, keepdim=True)
        shared = torch.where(most > 0, torch.floor(torch.log2(most)) - _SIZE[bits][0], -127.0).clamp_min(-127.0)
        y = part.abs() / 2.0 ** shared
        above = torch.searchsorted(up, y).clamp(1, len(up) - 1)
        low, high = up[above - 1], up[above]
        up_is_nearer = (high - y < y - low) | ((high - y == y - low) & (above % 2 == 0))
        out[a:a + 512] = torch.where(up_is_nearer, high, low) * 2.0 ** shared * part.sign()
    return out.view(s["x"].shape)


def _read64(values, scales, bits):
    blocks = scales.shape[-1]
    if bits == 4:
        stream = values.view(*scales.shape, 16)
    else:
        stream = torch.cat([values[..., :16 * blocks].view(*scales.shape, 16),
                            values[..., 16 * blocks:].view(*scales.shape, 8)], -1)
    out = torch.empty(*scales.shape, BLOCK, dtype=torch.float64, device="cuda")
    elements = _elements64(bits)
    for i in range(BLOCK):  # the bits of element i, in one byte or two
        byte, shift = bits * i // 8, bits * i % 8
        word = stream[..., byte].long()
        if shift + bits > 8:
            word = word + 256 * stream[..., byte + 1].long()
        out[..., i] = elements[torch.div(word, 1 << shift, rounding_mode="floor") % (1 << bits)]
    return (out * torch.exp2(scales.double() - 127)[..., None]).flatten(-2)


def _exact_linear(s, case):
    x = _read64(s["x"], s["xs"], case["bits"])
    step = max(1, (1 << 26) // case["features"])  # outputs at a time
    parts = [x @ _read64(s["w"][0, a:a + step], s["ws"][0, a:a + step], 4).t()
             for a in range(0, case["outputs"], step)]
    return torch.cat(parts, 1)


def _pairs_of(s):
    """(expert, its rows of the plan) of the experts in use."""
    for e, a, b in _used(s):
        yield e, torch.arange(a, b, device="cuda")


def _exact_gate_up(s, case):
    x = _read64(s["x"], s["xs"], case["bits"])
    h = torch.zeros(s["h"].shape, dtype=torch.float64, device="cuda")
    for e, at in _pairs_of(s):
        rows = x[torch.div(s["rows"][at], case["top"], rounding_mode="floor").long()]
        w = _read64(s["w"][e], s["ws"][e], 4)
        gate = rows @ w[:case["inner"]].t()
        h[at] = gate * torch.sigmoid(gate) * (rows @ w[case["inner"]:].t())
    return h


def _exact_down(s, case):
    x = _read64(s["x"], s["xs"], case["bits"])
    y = torch.zeros(s["y"].shape, dtype=torch.float64, device="cuda")
    weights = s["weights"].double().view(-1)
    for e, at in _pairs_of(s):
        pairs = s["rows"][at].long()
        token = torch.div(pairs, case["top"], rounding_mode="floor")
        # an expert is chosen once by a token: no row is added to twice
        y[token] += weights[pairs, None] * (x[at] @ _read64(s["w"][e], s["ws"][e], 4).t())
    return y
