"""The work the operators of generation are measured on.

Three operators stand between a network's projections and its attention once
it answers token by token, and each case is one pass through one of them:

- ``rotate``       the norm of every head of the queries and keys and the
                   rotation by position, from one projection's output;
- ``rotate back``  its gradients: of queries and keys and of both weights;
- ``cache``        keys and values of new tokens written into the pages of a
                   cache, in 8 bits or as they are, and read back from it;
- ``attend``       attention of new tokens over the cache of their sequences,
                   which may begin with a prefix that all of them share.

``run`` computes them in elementary torch operations, or where ``own`` is set
by the entry points of ``libtchip``, called as a binding calls them: operands,
outputs and layout structs are laid out once, and a pass is the calls alone.
``exact`` gives the same results in 64 bits.
"""

import math
import random

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPSILON = 1e-6
BASE = 10000.0
STEPS = 127  # of an 8-bit entry on either side of zero
NO_PAGE = -1  # as 32 unsigned bits: past every pool


def listed():
    return [
        # One step of generation for a few requests far into their answers.
        {"name": "rotate bf16 16 tokens", "kind": "rotate", "dtype": "bf16", "weight": "bf16", "tokens": 16,
         "heads": 32, "key heads": 8, "size": 128, "rotary": 128, "pairs": "halves", "norm": True, "far": 131072},
        # A training step's tokens: past the caches.
        {"name": "rotate bf16 large", "kind": "rotate", "dtype": "bf16", "weight": "f32", "tokens": 16384,
         "heads": 32, "key heads": 8, "size": 128, "rotary": 128, "pairs": "halves", "norm": True, "far": 16384},
        # The gradients, with heads that are no power of two, rotated in part
        # and by neighbours.
        {"name": "rotate back f16 odd", "kind": "rotate back", "dtype": "f16", "weight": "f32", "tokens": 7001,
         "heads": 12, "key heads": 12, "size": 80, "rotary": 40, "pairs": "neighbours", "norm": True, "far": 4000},
        # The gradients of a training step's tokens.
        {"name": "rotate back bf16 large", "kind": "rotate back", "dtype": "bf16", "weight": "bf16", "tokens": 16384,
         "heads": 32, "key heads": 4, "size": 128, "rotary": 128, "pairs": "halves", "norm": True, "far": 16384},
        # One new token of each of many requests: launches count.
        {"name": "cache int8 64 tokens", "kind": "cache", "dtype": "bf16", "format": "int8", "key heads": 8,
         "size": 128, "page": 64, "sequences": 64, "longest": 4000, "new": 1},
        # The prompts of a batch, of different lengths, on odd pages.
        {"name": "cache int8 prompts", "kind": "cache", "dtype": "f16", "format": "int8", "key heads": 8,
         "size": 128, "page": 48, "sequences": 19, "longest": 2000, "new": 2000},
        # A prompt kept as it is, its rows no whole words of memory.
        {"name": "cache f32 odd", "kind": "cache", "dtype": "f32", "format": "plain", "key heads": 3, "size": 75,
         "page": 20, "sequences": 3, "longest": 9000, "new": 9000},
        # The next token of a single request.
        {"name": "attend bf16 one", "kind": "attend", "dtype": "bf16", "format": "plain", "heads": 16,
         "key heads": 4, "size": 128, "page": 16, "sequences": 1, "longest": 1000, "new": 1, "prefix": 0},
        # The next tokens of a large batch of requests of all lengths.
        {"name": "attend bf16 batch", "kind": "attend", "dtype": "bf16", "format": "plain", "heads": 32,
         "key heads": 8, "size": 128, "page": 64, "sequences": 64, "longest": 8192, "new": 1, "prefix": 0},
        # A few very long contexts held in 8 bits.
        {"name": "attend int8 long", "kind": "attend", "dtype": "bf16", "format": "int8", "heads": 32,
         "key heads": 8, "size": 128, "page": 128, "sequences": 4, "longest": 100000, "new": 1, "prefix": 0},
        # Many requests behind one long instruction.
        {"name": "attend int8 prefix", "kind": "attend", "dtype": "f16", "format": "int8", "heads": 32,
         "key heads": 8, "size": 128, "page": 64, "sequences": 80, "longest": 500, "new": 1, "prefix": 8000},
        # Drafted tokens checked at once, heads of their own keys and no power
        # of two in size, on odd pages.
        {"name": "attend f16 drafts", "kind": "attend", "dtype": "f16", "format": "plain", "heads": 12,
         "key heads": 12, "size": 80, "page": 20, "sequences": 24, "longest": 3000, "new": 5, "prefix": 0},
    ]


def _spread(rng, low, high):
    """A size between `low` and `high`, even over its logarithm; a third of
    them are rounded down to a multiple of 64, a third to one of 8, where
    they reach it, and a third stay as they fall."""
    size = int(low * ((high + 1) / low) ** rng.random())
    step = rng.choice((1, 8, 64))
    return min(high, size // step * step if size >= max(step, low + step) else size)


def draw(rng):
    kind = rng.choice(("rotate", "rotate back", "cache", "attend", "attend"))
    dtype = rng.choice(("f32", "f16", "bf16"))
    key_heads = rng.choice((1, 2, 3, 4, 8))
    while True:
        if kind in ("rotate", "rotate back"):
            size = _spread(rng, 16, 128) // 2 * 2
            case = {"kind": kind, "dtype": dtype, "weight": rng.choice((dtype, "f32")), "tokens": _spread(rng, 1, 32768),
                    "heads": key_heads * rng.choice((1, 1, 2, 4, 7)), "key heads": key_heads, "size": size,
                    "rotary": rng.choice((size, size, 2 * rng.randint(1, size // 2))),
                    "pairs": rng.choice(("halves", "neighbours")), "norm": rng.random() < 0.7,
                    "far": _spread(rng, 100, 1000000)}
        else:
            case = {"kind": kind, "dtype": dtype, "format": rng.choice(("plain", "int8"))}
            if kind == "attend":
                case["heads"] = key_heads * rng.choice((1, 1, 2, 4, 7, 8, 16))
            longest = _spread(rng, 1, 32768)
            case |= {"key heads": key_heads, "size": _spread(rng, 16, 128), "page": _spread(rng, 1, 256),
                     "sequences": _spread(rng, 1, 200), "longest": longest,
                     "new": rng.choice((1, 1, rng.randint(1, 16)) if kind == "attend" else (1, longest))}
            if kind == "attend":
                case["prefix"] = rng.choice((0, 0, _spread(rng, 1, 16384)))
        need = work(case)
        if need["bytes"] <= 1.2e9 and need["flops"] <= 1.1e10:
            return case


# ---- operands ---------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(generator, shape, dtype, scale=1.0, shift=0.0):
    return torch.randn(shape, generator=generator, device="cuda").mul_(scale).add_(shift).to(TORCH[dtype])


def _empty(shape, dtype):
    return torch.empty(shape, device="cuda", dtype=TORCH.get(dtype, dtype))


def _rotary_inputs(case, seed):
    """Queries and keys side by side with values in one projection's output,
    at positions that packed or running sequences have."""
    g = _generator(seed)
    tokens, heads, shared, size = (case[k] for k in ("tokens", "heads", "key heads", "size"))
    q, k, _ = _normal(g, (tokens, heads + 2 * shared, size), case["dtype"], 1.5).split((heads, shared, shared), 1)
    state = {"q": q, "k": k,
             "positions": torch.randint(0, case["far"], (tokens,), generator=g, device="cuda", dtype=torch.int32),
             "frequencies": (BASE ** (-torch.arange(0, case["rotary"], 2, dtype=torch.float64) / case["rotary"])
                             ).float().cuda()}
    if case["norm"]:
        state |= {"q weight": _normal(g, (size,), case["weight"], 0.2, 1.0),
                  "k weight": _normal(g, (size,), case["weight"], 0.2, 1.0)}
    if case["kind"] == "rotate back":
        state |= {"d q out": _normal(g, (tokens, heads, size), case["dtype"], 1e-2),
                  "d k out": _normal(g, (tokens, shared, size), case["dtype"], 1e-2)}
    return state


def _row(case):
    """Elements from a cache's row to the next: whole words of 16 bytes."""
    per = 16 if case["format"] == "int8" else 16 // SIZE[case["dtype"]]
    return -(-case["size"] // per) * per


def _counts(case):
    """(cached tokens, new tokens) of each sequence, drawn from the case alone."""
    rng = random.Random(case["longest"] * 1009 + case["sequences"] * 31 + case["new"])
    lengths = [max(1, round(case["longest"] * rng.uniform(0.15, 1.0))) for _ in range(case["sequences"])]
    lengths[rng.randrange(len(lengths))] = case["longest"]
    return lengths, [min(n, case["new"]) for n in lengths]


def _pages(case, lengths):
    """Pages of the shared prefix and of each sequence."""
    page = case["page"]
    return -(-case.get("prefix", 0) // page), [-(-n // page) for n in lengths]


def _entries(g, case, shape):
    """A cache's entries and, in 8 bits, the step of each row."""
    if case["format"] == "plain":
        return _normal(g, shape, case["dtype"]), None
    entries = torch.randn(shape, generator=g, device="cuda", dtype=torch.float16).mul_(STEPS / 3)
    steps = torch.randn(shape[:-1], generator=g, device="cuda").mul_(0.3).exp_().mul_(3 / STEPS)
    return entries.round_().clamp_(-STEPS, STEPS).to(torch.int8), steps


def _cache_inputs(case, seed):
    """A pool of pages in no order and the tables of the sequences; what the
    tables do not need names no page."""
    g = _generator(seed)
    lengths, new = _counts(case)
    prefix_pages, pages = _pages(case, lengths)
    count = prefix_pages + sum(pages) + 3
    order = torch.randperm(count, generator=g, device="cuda").int()
    table = torch.full((len(pages), max(pages) + 1), NO_PAGE, dtype=torch.int32)
    filled = order.cpu()
    at = prefix_pages
    for s, n in enumerate(pages):
        table[s, :n] = filled[at:at + n]
        at += n
    shape = (count, case["key heads"], case["page"], _row(case))
    state = {"pages": table.cuda(), "prefix pages": order[:prefix_pages].clone(), "lengths": lengths, "new": new,
             "device lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"),
             "offsets": torch.tensor([0] + new, device="cuda").cumsum(0).int()}
    tokens = sum(new)
    if case["kind"] == "cache":
        kind = torch.int8 if case["format"] == "int8" else case["dtype"]
        state |= {"keys": _empty(shape, kind), "values": _empty(shape, kind)}
        if case["format"] == "int8":
            state |= {"key steps": _empty(shape[:-1], "f32"), "value steps": _empty(shape[:-1], "f32")}
        # Keys and values side by side, as one projection gives them.
        state["k"], state["v"] = _normal(g, (tokens, 2 * case["key heads"], case["size"]), case["dtype"], 1.2).split(
            case["key heads"], 1)
    else:
        (state["keys"], state["key steps"]), (state["values"], state["value steps"]) = (
            _entries(g, case, shape) for _ in range(2))
        for name in ("keys", "values"):
            state[name][..., case["size"]:] = 0
        state |= {"q": _normal(g, (tokens, case["heads"], case["size"]), case["dtype"], 1.2),
                  "scale": case["size"] ** -0.5}
    return state


def prepare(case, seed):
    """The inputs, and the storage that the results are written to."""
    dtype, size = case["dtype"], case["size"]
    if case["kind"] in ("rotate", "rotate back"):
        state = _rotary_inputs(case, seed)
        shapes = {"q": (case["tokens"], case["heads"], size), "k": (case["tokens"], case["key heads"], size)}
        if case["kind"] == "rotate":
            out = {n + " out": _empty(shape, dtype) for n, shape in shapes.items()}
        else:
            # The gradients take the place of queries and keys in a
            # projection's, whose values another operator writes.
            out = dict(zip(("d q", "d k"), _empty(
                (case["tokens"], case["heads"] + 2 * case["key heads"], size), dtype).split(
                    (case["heads"], case["key heads"], case["key heads"]), 1)))
            if case["norm"]:
                out |= {"d q weight": _empty(size, case["weight"]), "d k weight": _empty(size, case["weight"])}
    else:
        state = _cache_inputs(case, seed)
        tokens = sum(state["new"])
        if case["kind"] == "cache":
            out = {n: _empty((tokens, case["key heads"], size), dtype) for n in ("read keys", "read values")}
        else:
            out = {"out": _empty((tokens, case["heads"], size), dtype),
                   "normalizers": _empty((case["heads"], tokens), "f32")}
    state |= {"case": case, "out": out}
    # The library runs on a stream of its own: what torch queued is done
    # before it reads it.
    torch.cuda.synchronize()
    return state


# ---- one pass -----------------------------------------------------------------


def run(state):
    if not own:
        return PLAIN[state["case"]["kind"]](state)
    from tensorcrate_amd import lib

    if "calls" not in state:
        state["calls"] = CALLS[state["case"]["kind"]](lib, state)
    for name, args in state["calls"]:
        lib.call(name, *args)
    return state["out"]


def _ptr(tensor):
    return None if tensor is None else tensor.data_ptr()


def _rotary_calls(lib, s):
    code = {"f32": lib.F32, "f16": lib.F16, "bf16": lib.BF16}
    case, out = s["case"], s["out"]
    heads, shared, size = case["heads"], case["key heads"], case["size"]
    plan = lib.rotary(code[case["dtype"]], code[case["weight"]], case["tokens"], heads, shared, size, case["rotary"],
                      lib.HALVES if case["pairs"] == "halves" else lib.NEIGHBOURS, case["norm"], EPSILON,
                      _ptr(s["positions"]), _ptr(s["frequencies"]), s["q"].stride()[:2], s["k"].stride()[:2],
                      (heads * size, size), (shared * size, size))
    weights = (_ptr(s.get("q weight")), _ptr(s.get("k weight")))
    if case["kind"] == "rotate":
        return [("tc_rotary_norm", (plan, _ptr(s["q"]), _ptr(s["k"]), *weights, _ptr(out["q out"]),
                                    _ptr(out["k out"])))]
    return [("tc_rotary_norm_backward", (plan, _ptr(s["d q out"]), _ptr(s["d k out"]), _ptr(s["q"]), _ptr(s["k"]),
                                         *weights, _ptr(out["d q"]), _ptr(out["d k"]), _ptr(out.get("d q weight")),
                                         _ptr(out.get("d k weight"))))]


def _cache(lib, s):
    code = {"f32": lib.F32, "f16": lib.F16, "bf16": lib.BF16}
    case = s["case"]
    cache = lib.cache(code[case["dtype"]], lib.CACHE_INT8 if case["format"] == "int8" else lib.CACHE_PLAIN,
                      case["key heads"], case["size"], case["page"], s["keys"].shape[0], _ptr(s["keys"]),
                      _ptr(s["values"]), _ptr(s.get("key steps")), _ptr(s.get("value steps")))
    batch = lib.cache_batch(sum(s["new"]), case["sequences"], _ptr(s["offsets"]), _ptr(s["device lengths"]),
                            _ptr(s["pages"]), s["pages"].shape[1], case.get("prefix", 0),
                            _ptr(s["prefix pages"]) if case.get("prefix") else None)
    return cache, batch


def _cache_calls(lib, s):
    cache, batch = _cache(lib, s)
    operands = lambda k, v: (_ptr(k), *k.stride()[:2], _ptr(v), *v.stride()[:2])
    return [("tc_cache_write", (cache, batch, *operands(s["k"], s["v"]))),
            ("tc_cache_read", (cache, batch, *operands(s["out"]["read keys"], s["out"]["read values"])))]


def _attend_calls(lib, s):
    cache, batch = _cache(lib, s)
    out = s["out"]
    return [("tc_cache_attention", (cache, batch, s["case"]["heads"], s["scale"], _ptr(s["q"]), *s["q"].stride()[:2],
                                    _ptr(out["out"]), *out["out"].stride()[:2], _ptr(out["normalizers"])))]


CALLS = {"rotate": _rotary_calls, "rotate back": _rotary_calls, "cache": _cache_calls, "attend": _attend_calls}


# ---- the plain forms: elementary operations in 32 bits ---------------------------


def _turned(x, cos, sin, pairs):
    """The first elements of each head, in pairs, turned by their angles."""
    n = 2 * cos.shape[1]
    cos, sin = cos[:, None], sin[:, None]
    if pairs == "halves":
        a, b = x[..., :n // 2], x[..., n // 2:n]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    else:
        a, b = x[..., 0:n:2], x[..., 1:n:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((turned, x[..., n:]), -1)


def _angles(s):
    angles = s["positions"].double()[:, None] * s["frequencies"].double()
    return angles.cos().float(), angles.sin().float()


def _rotate_plain(s):
    case, out = s["case"], {}
    cos, sin = _angles(s)
    for n in "qk":
        x = s[n].float()
        if case["norm"]:
            x = x * (x.square().mean(-1, keepdim=True) + EPSILON).rsqrt() * s[n + " weight"].float()
        out[n + " out"] = _turned(x, cos, sin, case["pairs"]).to(s[n].dtype)
    return out


def _rotate_back_plain(s):
    case, out = s["case"], {}
    cos, sin = _angles(s)
    for n in "qk":
        d = _turned(s[f"d {n} out"].float(), cos, -sin, case["pairs"])
        if case["norm"]:
            x, weight = s[n].float(), s[n + " weight"]
            scale = (x.square().mean(-1, keepdim=True) + EPSILON).rsqrt()
            unit = x * scale
            out[f"d {n} weight"] = (d * unit).sum((0, 1)).to(weight.dtype)
            d = d * weight.float()
            d = scale * (d - unit * (d * unit).mean(-1, keepdim=True))
        out["d " + n] = d.to(s[n].dtype)
    return {n: out[n] for n in s["out"]}


def _places(s):
    """Page and slot in it of each new token."""
    page = s["case"]["page"]
    sequence = torch.repeat_interleave(torch.arange(len(s["new"]), device="cuda"), s["offsets"].diff().long(),
                                       output_size=sum(s["new"]))
    place = (s["device lengths"] - s["offsets"][1:])[sequence].long() + torch.arange(sum(s["new"]), device="cuda")
    return s["pages"][sequence, place // page].long(), place % page


def _cache_plain(s):
    size, out = s["case"]["size"], {}
    page, slot = _places(s)
    for n, name in (("k", "key"), ("v", "value")):
        pool, x = s[name + "s"], s[n]
        if s["case"]["format"] == "plain":
            pool[page, :, slot, :size] = x
            out[f"read {name}s"] = pool[page, :, slot, :size]
            continue
        # The step is rounded to 32 bits, and the quotients before they are
        # to whole numbers: 64 bits round those as 32 would.
        steps = (x.float().abs().amax(-1).double() / STEPS).float()
        entries = (x.double() / steps.double()[..., None]).float().round().clamp(-STEPS, STEPS)
        pool[page, :, slot, :size] = torch.where(steps[..., None] > 0, entries, 0.0).to(torch.int8)
        s[name + " steps"][page, :, slot] = steps
        read = pool[page, :, slot, :size].float() * s[name + " steps"][page, :, slot][..., None]
        out[f"read {name}s"] = read.to(x.dtype)
    return out


def _rows(s, name, pages, count):
    """[key head, token, element] of the first `count` tokens on these pages, in 32 bits."""
    pool = s[name + "s"][pages].float()
    if s["case"]["format"] == "int8":
        pool = pool * s[name + " steps"][pages][..., None]
    return pool.transpose(0, 1).flatten(1, 2)[:, :count, :s["case"]["size"]]


def _attend_plain(s):
    case = s["case"]
    heads, shared, size, prefix = (case[k] for k in ("heads", "key heads", "size", "prefix"))
    group, tokens = heads // shared, sum(s["new"])
    q = s["q"].float().view(tokens, shared, group, size).permute(1, 2, 0, 3)  # [key head, query of it, token, element]
    first = [_rows(s, name, s["prefix pages"].long(), prefix) for name in ("key", "value")]
    out, normalizers, at = [], [], 0
    for sequence, (length, new) in enumerate(zip(s["lengths"], s["new"])):
        pages = s["pages"][sequence, :-(-length // case["page"])].long()
        k, v = (torch.cat((shared_rows, _rows(s, name, pages, length)), 1)
                for shared_rows, name in zip(first, ("key", "value")))
        rows = q[:, :, at:at + new].reshape(shared, group * new, size)
        scores = torch.matmul(rows, k.transpose(1, 2).contiguous()).mul_(s["scale"]).view(shared, group, new, -1)
        if new > 1:
            place = torch.arange(prefix + length, device="cuda")
            scores.masked_fill_(place > place[prefix + length - new:, None], -math.inf)
        most = scores.amax(3, keepdim=True)
        e = scores.sub_(most).exp_()
        total = e.sum(3, keepdim=True)
        mixed = torch.matmul(e.view(shared, group * new, -1), v).view(shared, group, new, size) / total
        out.append(mixed.permute(2, 0, 1, 3).reshape(new, heads, size))
        normalizers.append((most + total.log())[..., 0].reshape(heads, new))
        at += new
    return {"out": torch.cat(out).to(s["q"].dtype), "normalizers": torch.cat(normalizers, 1)}


PLAIN = {"rotate": _rotate_plain, "rotate back": _rotate_back_plain, "cache": _cache_plain, "attend": _attend_plain}


# ---- what a pass cannot do without ----------------------------------------------


def work(case):
    element, size, shared = SIZE[case["dtype"]], case["size"], case["key heads"]
    if case["kind"] in ("rotate", "rotate back"):
        rows = case["tokens"] * (case["heads"] + shared)
        weights = 2 * size * SIZE[case["weight"]] if case["norm"] else 0
        passes, operations = 2, 7.0 if case["norm"] else 3.0
        if case["kind"] == "rotate back":
            # Without a norm the gradients do not need the queries and keys.
            passes, weights, operations = (3, 2 * weights, 15.0) if case["norm"] else (2, 0, 3.0)
        return {"bytes": passes * element * rows * size + 4 * case["tokens"] + 2 * case["rotary"] + weights,
                "flops": operations * rows * size}
    lengths, new = _counts(case)
    prefix_pages, pages = _pages(case, lengths)
    entry = 2 * size + 8 if case["format"] == "int8" else 2 * size * element  # of a key and a value of one head
    tables = 4 * (prefix_pages + sum(pages)) + 8 * len(lengths)
    if case["kind"] == "cache":
        rows = sum(new) * shared
        return {"bytes": rows * (2 * entry + 4 * size * element) + 4 * sum(new) + 8 * len(lengths),
                "flops": (8.0 if case["format"] == "int8" else 0.0) * rows * size + 2.0 * rows}
    prefix, tokens = case["prefix"], sum(new)
    pairs = sum(n * (prefix + length - n) + n * (n + 1) // 2 for length, n in zip(lengths, new)) * case["heads"]
    return {"bytes": (prefix + sum(lengths)) * shared * entry + tables + tokens * case["heads"] * (2 * size * element + 4),
            "flops": 4.0 * pairs * size}


# ---- the same in 64 bits ----------------------------------------------------------


def _rotation(s, case):
    """Both elements' places of each pair, and the cosine and sine of its angle."""
    n = case["rotary"]
    angles = s["positions"].double().unsqueeze(1) * s["frequencies"].double()
    i = torch.arange(n // 2, device="cuda")
    a, b = (i, i + n // 2) if case["pairs"] == "halves" else (2 * i, 2 * i + 1)
    return a, b, angles.cos().unsqueeze(1), angles.sin().unsqueeze(1)


def _exact_rotary(case, seed):
    s = _rotary_inputs(case, seed)
    a, b, cos, sin = _rotation(s, case)
    out = {}
    for n in ("q", "k"):
        x = s[n].double()
        scale = 1 / torch.sqrt((x * x).sum(2, keepdim=True) / case["size"] + EPSILON)
        weight = s[n + " weight"].double() if case["norm"] else None
        if case["kind"] == "rotate":
            y = x * scale * weight if case["norm"] else x
            z = y.clone()
            z[:, :, a] = cos * y[:, :, a] - sin * y[:, :, b]
            z[:, :, b] = sin * y[:, :, a] + cos * y[:, :, b]
            out[n + " out"] = z
            continue
        z = s[f"d {n} out"].double()
        y = z.clone()
        y[:, :, a] = cos * z[:, :, a] + sin * z[:, :, b]
        y[:, :, b] = cos * z[:, :, b] - sin * z[:, :, a]
        if case["norm"]:
            out[f"d {n} weight"] = torch.einsum("the,the->e", y, x * scale)
            g = y * weight
            y = scale * g - scale ** 3 * x * (g * x).sum(2, keepdim=True) / case["size"]
        out["d " + n] = y
    order = ("q out", "k out") if case["kind"] == "rotate" else ("d q", "d k", "d q weight", "d k weight")
    return {n: out[n] for n in order if n in out}


def exact(case, seed):
    if case["kind"] in ("rotate", "rotate back"):
        return _exact_rotary(case, seed)
    s = _cache_inputs(case, seed)
    if case["kind"] == "cache":
        out = {}
        for n, name in (("k", "read keys"), ("v", "read values")):
            x = s[n].double()
            if case["format"] == "int8":
                # What the 8 bits stand for goes by roundings to 32 bits on
                # the way: of the step and of the quotients.
                step = (x.abs().amax(2, keepdim=True) / STEPS).float().double()
                whole = torch.round((x / step.clamp(min=1e-300)).float().double()).clamp(-STEPS, STEPS)
                x = whole * step
            out[name] = x
        return out
    size, group, page = case["size"], case["heads"] // case["key heads"], case["page"]
    tokens = sum(s["new"])
    out = torch.empty((tokens, case["heads"], size), dtype=torch.float64, device="cuda")
    normalizers = torch.empty((case["heads"], tokens), dtype=torch.float64, device="cuda")

    def taken(name, pages, head, count):
        rows = s[name + "s"][pages, head].double()
        if case["format"] == "int8":
            rows *= s[name + " steps"][pages, head].double().unsqueeze(2)
        return rows.reshape(-1, rows.shape[2])[:count, :size]

    for head in range(case["key heads"]):
        mine = slice(head * group, (head + 1) * group)
        begin = [taken(name, s["prefix pages"].long(), head, case["prefix"]) for name in ("key", "value")]
        at = 0
        for number, (length, new) in enumerate(zip(s["lengths"], s["new"])):
            pages = s["pages"][number, :(length + page - 1) // page].long()
            k, v = (torch.cat((rows, taken(name, pages, head, length))) for rows, name in zip(begin, ("key", "value")))
            for row in range(at, at + new):
                seen = case["prefix"] + length - (at + new - 1 - row)
                log_p = s["q"][row, mine].double() @ k[:seen].T * s["scale"]
                normalizers[mine, row] = torch.logsumexp(log_p, 1)
                out[row, mine] = torch.softmax(log_p, 1) @ v[:seen]
            at += new
    return {"out": out, "normalizers": normalizers}
