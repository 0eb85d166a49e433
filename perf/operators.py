"""The work the language-model operators are measured on.

Four operators stand between a network's products and its optimizer when it is
trained to give the next token, and each case is one pass through one of them:

- ``norm``       layer norm of every row, forward;
- ``norm back``  its gradients: of the rows, of the weight and of the bias;
- ``tokens``     from a row of logits, the log probability of its token, the
                 entropy and the most probable tokens;
- ``tokens back``  the gradient of the logits, from those of the log
                 probability and of the entropy;
- ``clip``       the norm over all gradients of a model, and the gradients
                 scaled down to a largest norm;
- ``attention``  causal attention over packed sequences, with query heads that
                 share key and value heads; forward, or (``train``) forward
                 and the gradients of queries, keys and values.

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
EPSILON = 1e-5
NO_TOKEN = -1  # as 32 unsigned bits: past every vocabulary


def listed():
    return [
        # The rows of one small batch: a few microseconds, where launches count.
        {"name": "norm f32 64 rows", "kind": "norm", "dtype": "f32", "weight": "f32", "rows": 64, "cols": 1024,
         "gap": 0},
        # A training step's activations in a 16-bit type: past the caches.
        {"name": "norm bf16 large", "kind": "norm", "dtype": "bf16", "weight": "bf16", "rows": 16384, "cols": 4096,
         "gap": 0},
        # The gradients, over rows that are views of longer ones and start
        # anywhere, with the weight kept in 32 bits.
        {"name": "norm back f16 odd", "kind": "norm back", "dtype": "f16", "weight": "f32", "rows": 10007,
         "cols": 2050, "gap": 7},
        # One step of generation for a few requests, with alternatives.
        {"name": "tokens f32 16 rows", "kind": "tokens", "dtype": "f32", "rows": 16, "cols": 50001, "top": 20,
         "masked": 0},
        # Scoring a batch over a large vocabulary, its last entries unused.
        {"name": "tokens bf16 large", "kind": "tokens", "dtype": "bf16", "rows": 4096, "cols": 100000, "top": 8,
         "masked": 96},
        # The loss's gradient over an odd vocabulary.
        {"name": "tokens back bf16 odd", "kind": "tokens back", "dtype": "bf16", "rows": 4096, "cols": 50001,
         "masked": 0, "entropy": True},
        # The gradients of the dense network 1024 -> 4096 -> 4096 -> 1024.
        {"name": "clip f32 network", "kind": "clip", "dtype": "f32", "tensors": 6, "elements": 25175040,
         "limit": 1.0},
        # A model of many layers, matrices in 16 bits and vectors in 32.
        {"name": "clip mixed many", "kind": "clip", "dtype": "mixed", "tensors": 300, "elements": 300000001,
         "limit": 1.0},
        # A first small model's training step.
        {"name": "attention f32 short", "kind": "attention", "dtype": "f32", "tokens": 200, "heads": 4,
         "key heads": 2, "size": 32, "sequences": 3, "unused": 5, "packed": True, "train": True},
        # Training on one long sequence.
        {"name": "attention bf16 long", "kind": "attention", "dtype": "bf16", "tokens": 8192, "heads": 16,
         "key heads": 4, "size": 128, "sequences": 1, "unused": 0, "packed": False, "train": True},
        # Training on many sequences of different lengths behind one another,
        # over one projection's output, with a head size that is no power of two.
        {"name": "attention f16 packed", "kind": "attention", "dtype": "f16", "tokens": 7001, "heads": 12,
         "key heads": 12, "size": 80, "sequences": 19, "unused": 33, "packed": True, "train": True},
        # A long prompt before generation, all query heads on one key head.
        {"name": "attention bf16 prompt", "kind": "attention", "dtype": "bf16", "tokens": 16384, "heads": 8,
         "key heads": 1, "size": 64, "sequences": 1, "unused": 0, "packed": True, "train": False},
    ]


def _spread(rng, low, high):
    """A size between `low` and `high`, even over its logarithm; a third of
    them are rounded down to a multiple of 64, a third to one of 8, where
    they reach it, and a third stay as they fall."""
    size = int(low * ((high + 1) / low) ** rng.random())
    step = rng.choice((1, 8, 64))
    return min(high, size // step * step if size >= max(step, low + step) else size)


def draw(rng):
    kind = rng.choice(("norm", "norm back", "tokens", "tokens back", "clip", "attention", "attention"))
    dtype = rng.choice(("f32", "f16", "bf16"))
    while True:
        if kind in ("norm", "norm back"):
            case = {"kind": kind, "dtype": dtype, "weight": rng.choice((dtype, "f32")),
                    "rows": _spread(rng, 1, 32768), "cols": _spread(rng, 8, 16384),
                    "gap": rng.choice((0, 0, rng.randint(1, 64)))}
        elif kind in ("tokens", "tokens back"):
            case = {"kind": kind, "dtype": dtype, "rows": _spread(rng, 1, 8192), "cols": _spread(rng, 100, 160000),
                    "masked": rng.choice((0, rng.randint(1, 60)))}
            case |= {"top": rng.choice((0, rng.randint(1, 64)))} if kind == "tokens" else {
                "entropy": rng.random() < 0.5}
        elif kind == "clip":
            tensors = _spread(rng, 1, 500)
            case = {"kind": kind, "dtype": rng.choice((dtype, "mixed")), "tensors": tensors,
                    "elements": tensors * 4 + _spread(rng, 1000, 300000000), "limit": rng.choice((1.0, 1.0, 50.0))}
        else:
            key_heads, size, tokens = rng.choice((1, 2, 3, 4, 8)), _spread(rng, 8, 128), _spread(rng, 1, 16384)
            case = {"kind": kind, "dtype": dtype, "tokens": tokens, "heads": key_heads * rng.choice((1, 1, 2, 4, 7)),
                    "key heads": key_heads, "size": size, "sequences": _spread(rng, 1, min(tokens, 64)),
                    "unused": rng.choice((0, 0, rng.randint(0, tokens // 2))), "packed": rng.random() < 0.5,
                    "train": rng.random() < 0.6}
            scores = case["heads"] * tokens ** 2
            if scores > (1.1e9 if case["train"] else 2.2e9) or (dtype == "f32" and scores > 3e8):
                continue
        if work(case)["bytes"] <= 1.3e9:
            return case


# ---- operands ---------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(generator, shape, dtype, scale=1.0, shift=0.0):
    return torch.randn(shape, generator=generator, device="cuda").mul_(scale).add_(shift).to(TORCH[dtype])


def _empty(shape, dtype):
    return torch.empty(shape, device="cuda", dtype=TORCH.get(dtype, dtype))


def _rows(generator, case, scale, shift=0.0):
    """Rows x cols, the first columns of longer rows where the case has a gap."""
    return _normal(generator, (case["rows"], case["cols"] + case["gap"]), case["dtype"], scale, shift)[:, :case["cols"]]


def _norm_inputs(case, seed):
    g = _generator(seed)
    state = {"x": _rows(g, case, 2.0, 0.5), "weight": _normal(g, (case["cols"],), case["weight"], 0.2, 1.0),
             "bias": _normal(g, (case["cols"],), case["weight"], 0.1)}
    if case["kind"] == "norm back":
        x = state["x"].float()
        state |= {"dy": _rows(g, case, 1e-2), "means": x.mean(1),
                  "scales": (x.var(1, correction=0) + EPSILON).rsqrt()}
    return state


def _token_inputs(case, seed):
    """Logits some of which stand out, as a trained model's do; unused entries
    at the end of the vocabulary are masked, and some rows have no token."""
    g = _generator(seed)
    rows, cols = case["rows"], case["cols"]
    logits = torch.randn((rows, cols), generator=g, device="cuda").mul_(2.0)
    tokens = torch.randint(0, cols - case["masked"], (rows,), generator=g, device="cuda", dtype=torch.int32)
    likely = torch.rand((rows, 1), generator=g, device="cuda").mul_(15.0)
    logits.scatter_add_(1, tokens.long()[:, None], likely)
    logits[:, cols - case["masked"]:] = -math.inf
    tokens[torch.rand((rows,), generator=g, device="cuda") < 0.05] = NO_TOKEN
    state = {"logits": logits.to(TORCH[case["dtype"]]), "tokens": tokens}
    if case["kind"] == "tokens back":
        x = state["logits"].float()
        normalizers = torch.logsumexp(x, 1)
        p = (x - normalizers[:, None]).exp_()
        state |= {"normalizers": normalizers, "entropies": normalizers - p.mul_(x.clamp_(min=-1e30)).sum(1),
                  "d log probabilities": torch.randn((rows,), generator=g, device="cuda").sub_(0.5).div_(rows)}
        if case["entropy"]:
            state["d entropies"] = torch.randn((rows,), generator=g, device="cuda").mul_(0.1 / rows)
    return state


def _tensors(case):
    """(type, elements) of each tensor: a network's layers, or sizes spread
    over a large range, mixed ones keeping the small tensors in 32 bits."""
    count, total = case["tensors"], case["elements"]
    if case["dtype"] == "f32" and (count, total) == (6, 25175040):
        sizes = [4194304, 4096, 16777216, 4096, 4194304, 1024]
    else:
        rng = random.Random(count * 1000003 + total)
        share = [math.exp(rng.uniform(0, 8)) for _ in range(count)]
        sizes = [max(1, int((total - count) * s / sum(share))) for s in share]
        sizes[sizes.index(max(sizes))] += total - sum(sizes)
    middle = sorted(sizes)[count // 2]
    return [(case["dtype"] if case["dtype"] != "mixed" else "bf16" if s > middle else "f32", s) for s in sizes]


def _clip_inputs(case, seed):
    """The gradients of each type behind one another, their norm about 3."""
    g = _generator(seed)
    tensors = _tensors(case)
    scale = 3.0 / math.sqrt(case["elements"])
    return {"flat": {dtype: _normal(g, (sum(s for d, s in tensors if d == dtype),), dtype, scale)
                     for dtype in sorted({d for d, _ in tensors})}, "tensors": tensors}


def _lengths(case):
    """The sequences' lengths, drawn from the case alone; some may be of one token."""
    rng = random.Random(case["tokens"] * 1009 + case["sequences"])
    total = max(case["sequences"], case["tokens"] - case["unused"])
    share = [math.exp(rng.uniform(0, 3)) for _ in range(case["sequences"])]
    lengths = [1 + int((total - case["sequences"]) * s / sum(share)) for s in share]
    lengths[0] += total - sum(lengths)
    return lengths


def _attention_inputs(case, seed):
    g = _generator(seed)
    tokens, heads, shared, size, dtype = (case[k] for k in ("tokens", "heads", "key heads", "size", "dtype"))
    if case["packed"]:  # one projection gives queries, keys and values
        q, k, v = _normal(g, (tokens, heads + 2 * shared, size), dtype, 1.2).split((heads, shared, shared), 1)
    else:
        q, k, v = (_normal(g, (tokens, n, size), dtype, 1.2) for n in (heads, shared, shared))
    offsets = torch.tensor([0] + _lengths(case)).cumsum(0).to("cuda", torch.int32)
    state = {"q": q, "k": k, "v": v, "offsets": offsets, "scale": size ** -0.5}
    if case["train"]:
        state["d out"] = _normal(g, (tokens, heads, size), dtype, 1e-2)
    return state


def prepare(case, seed):
    """The inputs, and the storage that the results are written to."""
    kind = case["kind"]
    if kind in ("norm", "norm back"):
        state = _norm_inputs(case, seed)
        rows, cols = state["x"].shape
        if kind == "norm":
            out = {"y": _empty((rows, cols), case["dtype"]), "means": _empty(rows, "f32"),
                   "scales": _empty(rows, "f32")}
        else:
            out = {"dx": _empty((rows, cols), case["dtype"]), "dweight": _empty(cols, case["weight"]),
                   "dbias": _empty(cols, case["weight"])}
    elif kind == "tokens":
        state = _token_inputs(case, seed)
        rows, top = case["rows"], case["top"]
        out = {"log probabilities": _empty(rows, "f32"), "normalizers": _empty(rows, "f32"),
               "entropies": _empty(rows, "f32")}
        if top:
            out |= {"top log probabilities": _empty((rows, top), "f32"),
                    "top tokens": _empty((rows, top), torch.int32)}
    elif kind == "tokens back":
        state = _token_inputs(case, seed)
        out = {"d logits": _empty(state["logits"].shape, case["dtype"])}
    elif kind == "clip":
        state = _clip_inputs(case, seed)
        out = {"norm": _empty(1, "f32")} | {dtype: torch.empty_like(t) for dtype, t in state["flat"].items()}
    else:
        state = _attention_inputs(case, seed)
        tokens, heads, size = state["q"].shape
        out = {"out": _empty((tokens, heads, size), case["dtype"]), "normalizers": _empty((heads, tokens), "f32")}
        if case["train"] and case["packed"]:
            shared = case["key heads"]
            whole = _empty((tokens, heads + 2 * shared, size), case["dtype"])
            out["dq"], out["dk"], out["dv"] = whole.split((heads, shared, shared), 1)
        elif case["train"]:
            out |= {"d" + n: torch.empty_like(state[n]) for n in "qkv"}
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


def _norm_calls(lib, s):
    code = {"f32": lib.F32, "f16": lib.F16, "bf16": lib.BF16}
    case, x, out = s["case"], s["x"], s["out"]
    rows, cols = x.shape
    return [("tc_layer_norm", (code[case["dtype"]], code[case["weight"]], _ptr(x), x.stride(0), rows, cols,
                               _ptr(s["weight"]), _ptr(s["bias"]), EPSILON, _ptr(out["y"]), cols, _ptr(out["means"]),
                               _ptr(out["scales"])))]


def _norm_back_calls(lib, s):
    code = {"f32": lib.F32, "f16": lib.F16, "bf16": lib.BF16}
    case, x, dy, out = s["case"], s["x"], s["dy"], s["out"]
    rows, cols = x.shape
    return [("tc_layer_norm_backward", (code[case["dtype"]], code[case["weight"]], _ptr(dy), dy.stride(0), _ptr(x),
                                        x.stride(0), rows, cols, _ptr(s["weight"]), _ptr(s["means"]),
                                        _ptr(s["scales"]), _ptr(out["dx"]), cols, _ptr(out["dweight"]),
                                        _ptr(out["dbias"])))]


def _token_calls(lib, s):
    code = {"f32": lib.F32, "f16": lib.F16, "bf16": lib.BF16}
    case, out = s["case"], s["out"]
    return [("tc_log_probabilities", (code[case["dtype"]], _ptr(s["logits"]), case["cols"], case["rows"], case["cols"],
                                      _ptr(s["tokens"]), _ptr(out["log probabilities"]), _ptr(out["normalizers"]),
                                      _ptr(out["entropies"]), case["top"], _ptr(out.get("top log probabilities")),
                                      _ptr(out.get("top tokens"))))]


def _token_back_calls(lib, s):
    code = {"f32": lib.F32, "f16": lib.F16, "bf16": lib.BF16}
    case = s["case"]
    return [("tc_log_probabilities_backward",
             (code[case["dtype"]], _ptr(s["logits"]), case["cols"], case["rows"], case["cols"], _ptr(s["tokens"]),
              _ptr(s["normalizers"]), _ptr(s["entropies"]), _ptr(s["d log probabilities"]),
              _ptr(s.get("d entropies")), _ptr(s["out"]["d logits"]), case["cols"]))]


def _clip_calls(lib, s):
    code = {"f32": lib.F32, "f16": lib.F16, "bf16": lib.BF16}
    at = {dtype: 0 for dtype in s["flat"]}
    inputs, outputs = [], []
    for dtype, size in s["tensors"]:
        here, flat = at[dtype], s["flat"][dtype]
        inputs.append(flat.data_ptr() + here * flat.element_size())
        outputs.append(s["out"][dtype].data_ptr() + here * flat.element_size())
        at[dtype] += size
    count = len(inputs)
    return [("tc_clip_global_norm", (count, (lib.u32 * count)(*[code[d] for d, _ in s["tensors"]]),
                                     (lib.vp * count)(*inputs), (lib.u64 * count)(*[n for _, n in s["tensors"]]),
                                     s["case"]["limit"], (lib.vp * count)(*outputs), _ptr(s["out"]["norm"])))]


def _attention_calls(lib, s):
    code = {"f32": lib.F32, "f16": lib.F16, "bf16": lib.BF16}
    case, out = s["case"], s["out"]
    steps = [t.stride()[:2] for t in (s["q"], s["k"], s["v"], out["out"])]
    plan = lib.attention(code[case["dtype"]], case["tokens"], case["heads"], case["key heads"], case["size"],
                         s["scale"], _ptr(s["offsets"]), case["sequences"], *steps)
    calls = [("tc_attention", (plan, _ptr(s["q"]), _ptr(s["k"]), _ptr(s["v"]), _ptr(out["out"]),
                               _ptr(out["normalizers"])))]
    if case["train"]:
        calls.append(("tc_attention_backward", (plan, _ptr(s["d out"]), _ptr(s["q"]), _ptr(s["k"]), _ptr(s["v"]),
                                                _ptr(out["out"]), _ptr(out["normalizers"]), _ptr(out["dq"]),
                                                _ptr(out["dk"]), _ptr(out["dv"]))))
    return calls


CALLS = {"norm": _norm_calls, "norm back": _norm_back_calls, "tokens": _token_calls,
         "tokens back": _token_back_calls, "clip": _clip_calls, "attention": _attention_calls}


# ---- the plain forms: elementary operations in 32 bits ---------------------------


def _norm_plain(s):
    x = s["x"].float()
    means = x.mean(1)
    centred = x - means[:, None]
    scales = (centred.square().mean(1) + EPSILON).rsqrt()
    y = centred * scales[:, None] * s["weight"].float() + s["bias"].float()
    return {"y": y.to(s["x"].dtype), "means": means, "scales": scales}


def _norm_back_plain(s):
    dy, weight = s["dy"].float(), s["weight"].float()
    scales = s["scales"][:, None]
    unit = (s["x"].float() - s["means"][:, None]) * scales
    g = dy * weight
    dx = scales * (g - g.mean(1, keepdim=True) - unit * (g * unit).mean(1, keepdim=True))
    return {"dx": dx.to(s["dy"].dtype), "dweight": (dy * unit).sum(0).to(s["weight"].dtype),
            "dbias": dy.sum(0).to(s["weight"].dtype)}


def _token_plain(s):
    x, tokens, top = s["logits"].float(), s["tokens"].long(), s["case"]["top"]
    most = x.amax(1, keepdim=True)
    e = (x - most).exp()
    total = e.sum(1, keepdim=True)
    normalizers = (most + total.log())[:, 0]
    picked = x.gather(1, tokens.clamp(min=0)[:, None])[:, 0] - normalizers
    mean = (e * x.clamp(min=-1e30)).sum(1) / total[:, 0]
    out = {"log probabilities": torch.where(tokens >= 0, picked, 0.0), "normalizers": normalizers,
           "entropies": normalizers - mean}
    if top:
        # Whole numbers in the logits' order, equal logits by their index.
        bits = (x + 0.0).view(torch.int32)
        order = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF).long()
        order = order * 2 ** 32 + (2 ** 31 - torch.arange(x.shape[1], device=x.device))
        index = order.topk(top, 1).indices
        out |= {"top log probabilities": x.gather(1, index) - normalizers[:, None], "top tokens": index.int()}
    return out


def _token_back_plain(s):
    x, tokens = s["logits"].float(), s["tokens"].long()
    log_p = x - s["normalizers"][:, None]
    p = log_p.exp()
    g = torch.where(tokens >= 0, s["d log probabilities"], 0.0)
    d = -g[:, None] * p
    d.scatter_add_(1, tokens.clamp(min=0)[:, None], g[:, None])
    if "d entropies" in s:
        d -= s["d entropies"][:, None] * p * (log_p.clamp(min=-1e30) + s["entropies"][:, None])
    return {"d logits": d.to(s["logits"].dtype)}


def _clip_plain(s):
    flat = {dtype: t.float() for dtype, t in s["flat"].items()}
    norm = torch.stack([t.square().sum() for t in flat.values()]).sum().sqrt()
    factor = torch.where(norm > s["case"]["limit"], s["case"]["limit"] / norm, 1.0)
    return {"norm": norm.reshape(1)} | {dtype: (t * factor).to(s["flat"][dtype].dtype) for dtype, t in flat.items()}


def _attention_plain(s):
    dtype, shared = s["q"].dtype, s["k"].shape[1]
    heads, tokens = s["q"].shape[1], s["q"].shape[0]
    q, k, v = (t.float().transpose(0, 1).contiguous() for t in (s["q"], s["k"], s["v"]))
    k, v = (t.repeat_interleave(heads // shared, 0) for t in (k, v))
    place = torch.arange(tokens, device=q.device)
    sequence = torch.bucketize(place, s["offsets"].long(), right=True)
    inside = place < s["offsets"][-1]
    seen = (sequence[:, None] == sequence) & (place[:, None] >= place) & inside
    scores = torch.matmul(q, k.transpose(1, 2).contiguous()).mul_(s["scale"]).masked_fill_(~seen, -math.inf)
    most = scores.amax(2, keepdim=True).clamp(min=-1e30)
    e = scores.sub_(most).exp_()
    total = e.sum(2, keepdim=True)
    p = e.div_(total.clamp(min=1e-30))
    mixed = torch.matmul(p, v)
    out = {"out": mixed.transpose(0, 1).to(dtype), "normalizers": (most + total.log())[:, :, 0]}
    if "d out" in s:
        d = s["d out"].float().transpose(0, 1).contiguous()
        dv = torch.matmul(p.transpose(1, 2).contiguous(), d)
        dp = torch.matmul(d, v.transpose(1, 2).contiguous())
        ds = dp.sub_((d * mixed).sum(2, keepdim=True)).mul_(p).mul_(s["scale"])
        dq = torch.matmul(ds, k)
        dk = torch.matmul(ds.transpose(1, 2).contiguous(), q)
        dk, dv = (t.view(shared, heads // shared, tokens, -1).sum(1) for t in (dk, dv))
        out |= {n: t.transpose(0, 1).to(dtype) for n, t in (("dq", dq), ("dk", dk), ("dv", dv))}
    return out


PLAIN = {"norm": _norm_plain, "norm back": _norm_back_plain, "tokens": _token_plain,
         "tokens back": _token_back_plain, "clip": _clip_plain, "attention": _attention_plain}


# ---- what a pass cannot do without ----------------------------------------------


def work(case):
    kind = case["kind"]
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if kind in ("norm", "norm back"):
        n, row, col = case["rows"] * case["cols"], case["rows"], case["cols"]
        element, weight = size[case["dtype"]], size[case["weight"]]
        if kind == "norm":
            return {"bytes": 2 * element * n + 2 * weight * col + 8 * row, "flops": 7.0 * n}
        return {"bytes": 3 * element * n + 3 * weight * col + 8 * row, "flops": 13.0 * n}
    if kind == "tokens":
        n = case["rows"] * case["cols"]
        return {"bytes": size[case["dtype"]] * n + case["rows"] * (16 + 8 * case["top"]), "flops": 5.0 * n}
    if kind == "tokens back":
        n = case["rows"] * case["cols"]
        return {"bytes": 2 * size[case["dtype"]] * n + 20 * case["rows"], "flops": (6.0 if case["entropy"] else 4.0) * n}
    if kind == "clip":
        return {"bytes": sum(2 * size[d] * n for d, n in _tensors(case)) + 4, "flops": 3.0 * case["elements"]}
    tokens, heads, shared, width = (case[k] for k in ("tokens", "heads", "key heads", "size"))
    queries, keys = size[case["dtype"]] * tokens * heads * width, size[case["dtype"]] * tokens * shared * width
    pairs = sum(n * (n + 1) // 2 for n in _lengths(case)) * heads
    if case["train"]:
        # Read: queries, keys, values, the result's gradient; written: the
        # result and three gradients.  Two products forward and five back.
        return {"bytes": 4 * queries + 4 * keys + 4 * tokens * heads, "flops": 14.0 * pairs * width}
    return {"bytes": 2 * queries + 2 * keys + 4 * tokens * heads, "flops": 4.0 * pairs * width}


# ---- the same in 64 bits ----------------------------------------------------------


def exact(case, seed):
    kind = case["kind"]
    if kind == "norm":
        s = {k: t.double() for k, t in _norm_inputs(case, seed).items()}
        variance, mean = torch.var_mean(s["x"], 1, correction=0, keepdim=True)
        scale = 1 / (variance + EPSILON).sqrt()
        return {"y": s["weight"] * ((s["x"] - mean) * scale) + s["bias"], "means": mean[:, 0], "scales": scale[:, 0]}
    if kind == "norm back":
        # The statistics are inputs here, as the forward pass left them.
        s = {k: t.double() for k, t in _norm_inputs(case, seed).items()}
        scale, n = s["scales"][:, None], case["cols"]
        unit = s["x"].sub(s["means"][:, None]).mul(scale)
        g = s["weight"] * s["dy"]
        along, up = (g * unit).sum(1, keepdim=True) / n, g.sum(1, keepdim=True) / n
        return {"dx": (g - up - along * unit) * scale, "dweight": torch.einsum("ij,ij->j", unit, s["dy"]),
                "dbias": s["dy"].sum(0)}
    if kind == "tokens":
        s = _token_inputs(case, seed)
        x, tokens = s["logits"].double(), s["tokens"].long()
        log_p = torch.log_softmax(x, 1)
        rows = torch.arange(case["rows"], device=x.device)
        some = tokens != NO_TOKEN
        given = torch.zeros(case["rows"], dtype=torch.float64, device=x.device)
        given[some] = log_p[rows[some], tokens[some]]
        out = {"log probabilities": given, "normalizers": torch.logsumexp(x, 1),
               "entropies": torch.special.entr(log_p.exp()).sum(1)}
        if case["top"]:
            out |= {"top log probabilities": log_p.topk(case["top"], 1).values, "top tokens": None}
        return out
    if kind == "tokens back":
        s = _token_inputs(case, seed)
        x, tokens = s["logits"].double(), s["tokens"].long()
        p = (x - s["normalizers"].double()[:, None]).exp()
        some = tokens != NO_TOKEN
        g = s["d log probabilities"].double() * some
        d = -p * g[:, None]
        rows = torch.arange(case["rows"], device=x.device)
        d[rows[some], tokens[some]] += g[some]
        if case["entropy"]:
            entropies, weight = s["entropies"].double()[:, None], s["d entropies"].double()[:, None]
            d += weight * (torch.special.entr(p) - p * entropies)
        return {"d logits": d}
    if kind == "clip":
        flat = {dtype: t.double() for dtype, t in _clip_inputs(case, seed)["flat"].items()}
        norm = math.sqrt(sum(float(t.dot(t)) for t in flat.values()))
        factor = min(1.0, case["limit"] / norm)
        return {"norm": torch.tensor([norm], dtype=torch.float64)} | {d: t * factor for d, t in flat.items()}
    s = _attention_inputs(case, seed)
    q, k, v = (s[n].double() for n in "qkv")
    group, ends = case["heads"] // case["key heads"], s["offsets"].tolist()
    out = {"out": torch.zeros_like(q), "normalizers": q.new_full((case["heads"], case["tokens"]), -math.inf)}
    if case["train"]:
        d = s["d out"].double()
        out |= {"dq": torch.zeros_like(q), "dk": torch.zeros_like(k), "dv": torch.zeros_like(v)}
    for begin, end in zip(ends, ends[1:]):
        later = torch.ones((end - begin, end - begin), dtype=torch.bool, device=q.device).triu(1)
        for head in range(case["heads"]):
            a, b, c = q[begin:end, head], k[begin:end, head // group], v[begin:end, head // group]
            log_p = (a @ b.T * s["scale"]).masked_fill(later, -math.inf)
            normalizer = torch.logsumexp(log_p, 1)
            p = (log_p - normalizer[:, None]).exp()
            out["out"][begin:end, head] = p @ c
            out["normalizers"][head, begin:end] = normalizer
            if case["train"]:
                up = d[begin:end, head]
                dp = up @ c.T
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) * s["scale"]
                out["dq"][begin:end, head] = ds @ b
                out["dk"][begin:end, head // group] += ds.T @ a
                out["dv"][begin:end, head // group] += p.T @ up
    return out
