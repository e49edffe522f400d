"""What stands between the compressed projections of a training step, as cases that can be timed and compared.

Three kinds of case, each one pass through public entry points:

  gated   `gated_feed_forward`: both projections of a gated feed-forward block, the activation and the
          product.  Forward only (`train` false, as in evaluation or generation), or with the gradients
          of the input, both weights and the biases.
  rotary  `rotary`: queries and keys turned by the angles of their positions, the whole head or its first
          features, in either pairing.  Forward only or with the gradients.
  clip    `clip_gradients`: the global norm over many gradient tensors, and the clipped gradients, written
          to other buffers or in place.

Where `own` is false the same results come from elementary torch operations in 32 bits.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
ACTIVATIONS = ("silu", "gelu", "gelu_tanh", "relu", "sigmoid")
_package = None


def _stacr():
    global _package
    if _package is None:
        sys.path.insert(0, os.path.join(_ROOT, "stac-r_amd"))
        import stacr_amd

        _package = stacr_amd
    return _package


# ---------------------------------------------------------------------------------------- cases
def _gated(name, rows, d, ff, dtype="bf16", act="silu", bias=False, train=True):
    return {"name": name, "kind": "gated", "rows": rows, "d": d, "ff": ff, "dtype": dtype, "act": act, "bias": bias,
            "train": train}


def _rotary(name, batch, seq, heads, kv_heads, head, rot, dtype="bf16", layout="half", start=0, packed=False,
            train=True):
    return {"name": name, "kind": "rotary", "batch": batch, "seq": seq, "heads": heads, "kv_heads": kv_heads,
            "head": head, "rot": rot, "dtype": dtype, "layout": layout, "start": start, "packed": packed,
            "train": train}


def _clip(name, d, layers, ff, vocab, dtype="bf16", norm="2", over=True, place="out"):
    return {"name": name, "kind": "clip", "d": d, "layers": layers, "ff": ff, "vocab": vocab, "dtype": dtype,
            "norm": norm, "over": over, "place": place}


def listed():
    return [
        # generation: one token through a 1024 -> 4096 block, a read of the weights
        _gated("gated_one_token", 1, 1024, 4096, train=False),
        # a batch of twelve sequences, one new token each, through the 2048 -> 8192 block in fp16
        _gated("gated_few_tokens", 12, 2048, 8192, dtype="f16", act="gelu_tanh", train=False),
        # a training step at batch 8 x 1024 of the headline width
        _gated("gated_train", 8192, 1024, 4096),
        # a training step at 16 x 2048 tokens of the 1.4 B shape: the largest
        _gated("gated_train_wide", 32768, 2048, 8192),
        # a ragged last batch in fp16 with biases; features that no tile divides
        _gated("gated_train_ragged", 3001, 1000, 2731, dtype="f16", act="gelu", bias=True),
        # fp32 training at the narrow width
        _gated("gated_train_fp32", 4096, 768, 2048, dtype="f32"),
        # generation: one new token for each of eight sequences, a quarter of the head turned, fused q k v
        _rotary("rotary_one_token", 8, 1, 16, 16, 128, 32, start=2047, packed=True, train=False),
        # training at batch 8 x 1024, 16 heads of 64
        _rotary("rotary_train", 8, 1024, 16, 16, 64, 64),
        # one long sequence with shared key heads, neighbouring features paired
        _rotary("rotary_long", 1, 32768, 32, 8, 128, 128, layout="interleaved", start=32768),
        # the gradients of a small fp32 model, clipped: launches and host time
        _clip("clip_small", 256, 2, 1000, 999, dtype="f32"),
        # the gradients of a 24-layer model of width 1024, 16-bit matrices and 32-bit norms and biases, clipped
        _clip("clip_model", 1024, 24, 4096, 50257, dtype="mixed"),
        # the same widths in place with the norm under the limit, as in most steps of a settled run
        _clip("clip_under_limit", 1024, 12, 4096, 50257, dtype="bf16", over=False, place="in"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _features(rng, low, high):
    n = _log(rng, low, high)
    how = rng.random()
    return n if how < 0.25 else max(8, n // 8 * 8) if how < 0.5 else max(64, n // 64 * 64)


def draw(rng):
    kind = rng.choice(("gated", "gated", "rotary", "clip"))
    if kind == "gated":
        dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
        d, ff, rows = _features(rng, 128, 2048), _features(rng, 256, 8192), _log(rng, 1, 32768)
        # fp32 is trained at the small sizes
        most = 4096 * 768 * 2048 * 8 if dtype == "f32" else 32768 * 2048 * 8192
        rows = max(1, min(rows, most // (d * ff)))
        case = _gated("", rows, d, ff, dtype, rng.choice(ACTIVATIONS), rng.random() < 0.3,
                      rows >= 16 and rng.random() < 0.7)
    elif kind == "rotary":
        batch, seq = _log(rng, 1, 16), _log(rng, 1, 32768)
        kv = rng.choice((1, 2, 3, 4, 8, 12))
        heads = kv * rng.choice((1, 1, 2, 4))
        head = rng.choice((32, 64, 80, 96, 128))
        rot = rng.choice((head, head, head // 2, head // 4 // 2 * 2))
        seq = max(1, min(seq, 32768 * 40 * 128 // (batch * (heads + kv) * head)))
        case = _rotary("", batch, seq, heads, kv, head, rot, rng.choice(("bf16", "bf16", "f16", "f32")),
                       rng.choice(("half", "interleaved")), rng.choice((0, _log(rng, 1, 65536))), rng.random() < 0.4,
                       seq > 1 and rng.random() < 0.7)
    else:
        d = _features(rng, 64, 1024)
        case = _clip("", d, _log(rng, 1, 24), _features(rng, 128, 4096), _log(rng, 100, 50257),
                     rng.choice(("bf16", "f16", "f32", "mixed")), rng.choice(("2", "2", "2", "inf", "1")),
                     rng.random() < 0.6, rng.choice(("out", "out", "in")))
        # in place there is something to clip in the first pass alone
        case["over"] = case["over"] and case["place"] == "out"
        if case["dtype"] == "f32":
            case["layers"] = max(1, case["layers"] // 2)
    del case["name"]
    return case


# -------------------------------------------------------------------------------------- prepare
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(shape, g, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _prepare_gated(case, g):
    rows, d, ff, dtype = case["rows"], case["d"], case["ff"], DTYPES[case["dtype"]]
    # normalized activations with a spread over the channels
    spread = torch.exp(0.3 * torch.randn(d, generator=g, device="cuda"))
    s = {"x": (torch.randn(rows, d, generator=g, device="cuda") * spread).to(dtype),
         "w_gate": _normal((ff, d), g, dtype, d ** -0.5), "w_up": _normal((ff, d), g, dtype, d ** -0.5),
         "b_gate": None, "b_up": None}
    if case["bias"]:
        s["b_gate"], s["b_up"] = _normal((ff,), g, dtype, 0.5), _normal((ff,), g, dtype, 0.5)
    if case["train"]:
        s["dh"] = _normal((rows, ff), g, dtype)
        for name in ("x", "w_gate", "w_up", "b_gate", "b_up"):
            if s[name] is not None:
                s[name].requires_grad_(True)
    return s


def _prepare_rotary(case, g):
    b, t, head, rot, dtype = case["batch"], case["seq"], case["head"], case["rot"], DTYPES[case["dtype"]]
    hq, hk = case["heads"], case["kv_heads"]
    if case["packed"]:  # views of the fused projection's output
        qkv = _normal((b, t, hq + 2 * hk, head), g, dtype)
        q, k = qkv[:, :, :hq], qkv[:, :, hq:hq + hk]
    else:
        q, k = _normal((b, t, hq, head), g, dtype), _normal((b, t, hk, head), g, dtype)
    inv = 10000.0 ** (-torch.arange(rot // 2, device="cuda", dtype=torch.float64) * 2 / rot)
    angle = torch.arange(case["start"] + t, device="cuda", dtype=torch.float64)[:, None] * inv
    s = {"cos": angle.cos().float(), "sin": angle.sin().float()}
    # each sequence has a place of its own in its context (padding on the left)
    shift = torch.randint(0, case["start"] + 1, (b, 1), generator=g, device="cuda")
    s["positions"] = shift + torch.arange(t, device="cuda")
    s["q"], s["k"] = q, k
    if case["train"]:
        s["q"], s["k"] = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
        s["dq"], s["dk"] = _normal((b, t, hq, head), g, dtype), _normal((b, t, hk, head), g, dtype)
    return s


def _gradient_sizes(case):
    d, ff = case["d"], case["ff"]
    layer = [("m", d * d)] * 4 + [("m", ff * d)] * 3 + [("v", d)] * 2 + [("v", ff)] * 2
    return [("m", case["vocab"] * d)] + layer * case["layers"] + [("v", d)]


def _prepare_clip(case, g):
    """Gradients as views of one bucket of each type, packed without gaps."""
    matrix = torch.bfloat16 if case["dtype"] == "mixed" else DTYPES[case["dtype"]]
    vector = torch.float32 if case["dtype"] == "mixed" else matrix
    sizes = _gradient_sizes(case)
    total = {t: sum(n for k, n in sizes if (matrix if k == "m" else vector) == t) for t in {matrix, vector}}
    flat, out, at = {}, {}, {}
    for t, n in sorted(total.items(), key=str):
        flat[t] = torch.empty(n, dtype=t, device="cuda").normal_(generator=g)
        flat[t].mul_(0.01)
        out[t] = torch.empty_like(flat[t]) if case["place"] == "out" else flat[t]
        at[t] = 0
    grads, outs = [], []
    for k, n in sizes:
        t = matrix if k == "m" else vector
        grads.append(flat[t][at[t]:at[t] + n])
        outs.append(out[t][at[t]:at[t] + n])
        at[t] += n
    count = sum(total.values())
    guess = {"2": 0.01 * math.sqrt(count), "inf": 0.05, "1": 0.008 * count}[case["norm"]]
    return {"grads": grads, "outs": outs if case["place"] == "out" else None, "flat": list(out.values()),
            "max_norm": guess * (0.3 if case["over"] else 3.0), "norm": float(case["norm"])}


_PREPARE = {"gated": _prepare_gated, "rotary": _prepare_rotary, "clip": _prepare_clip}


def prepare(case, seed):
    return {"case": case, **_PREPARE[case["kind"]](case, _generator(seed))}


# ------------------------------------------------------------------------------------ plain form
def _act_and_slope(g, act):
    if act in ("silu", "sigmoid"):
        s = 1 / (1 + torch.exp(-g))
        return (s, s * (1 - s)) if act == "sigmoid" else (g * s, s * (1 + g * (1 - s)))
    if act == "relu":
        on = (g > 0).float()
        return g * on, on
    if act == "gelu":
        below = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * below, below + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    t = torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g))
    inner = math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * g * g)
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * inner


def _plain_gated(s):
    case = s["case"]
    dtype = s["x"].dtype
    x, wg, wu = (s[n].detach().float() for n in ("x", "w_gate", "w_up"))
    g, u = x @ wg.t(), x @ wu.t()
    if case["bias"]:
        g, u = g + s["b_gate"].detach().float(), u + s["b_up"].detach().float()
    a, slope = _act_and_slope(g, case["act"])
    out = {"h": (a * u).to(dtype)}
    if case["train"]:
        dh = s["dh"].float()
        dg, du = dh * u * slope, dh * a
        out["dx"] = (dg @ wg + du @ wu).to(dtype)
        out["dw_gate"], out["dw_up"] = (dg.t() @ x).to(dtype), (du.t() @ x).to(dtype)
        if case["bias"]:
            out["db_gate"], out["db_up"] = dg.sum(0).to(dtype), du.sum(0).to(dtype)
    return out


def _turn(x, c, s, layout):
    """x (batch, seq, heads, head) turned by the angles of cosine c and sine s (batch, seq, 1, rot / 2)."""
    y, half = x.float(), c.shape[-1]
    turned, rest = y[..., :2 * half], y[..., 2 * half:]
    if layout == "half":
        a, b = turned[..., :half], turned[..., half:]
        z = torch.cat((a * c - b * s, b * c + a * s, rest), -1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        z = torch.cat((torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2), rest), -1)
    return z.to(x.dtype)


def _plain_rotary(s):
    layout = s["case"]["layout"]
    c, n = s["cos"][s["positions"]][:, :, None], s["sin"][s["positions"]][:, :, None]
    out = {"q": _turn(s["q"].detach(), c, n, layout), "k": _turn(s["k"].detach(), c, n, layout)}
    if s["case"]["train"]:
        out["dq"], out["dk"] = _turn(s["dq"], c, -n, layout), _turn(s["dk"], c, -n, layout)
    return out


def _plain_clip(s):
    p = s["norm"]
    of = {2.0: lambda g: (g * g).sum(), 1.0: lambda g: g.abs().sum(), math.inf: lambda g: g.abs().amax()}[p]
    parts = torch.stack([of(g.float()) for g in s["grads"]])
    norm = parts.amax() if p == math.inf else parts.sum() if p == 1.0 else parts.sum().sqrt()
    factor = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    for g, o in zip(s["grads"], s["outs"] or s["grads"]):
        o.copy_(g.float() * factor)
    return {"norm": norm, "grads": s["flat"]}


_PLAIN = {"gated": _plain_gated, "rotary": _plain_rotary, "clip": _plain_clip}


# ------------------------------------------------------------------------------- the framework's
def _own_gated(s):
    case = s["case"]
    call = (s["x"], s["w_gate"], s["w_up"], s["b_gate"], s["b_up"])
    if not case["train"]:
        return {"h": _stacr().gated_feed_forward(*call, activation=case["act"])}
    h = _stacr().gated_feed_forward(*call, activation=case["act"])
    names = ["dx", "dw_gate", "dw_up", "db_gate", "db_up"][:5 if case["bias"] else 3]
    grads = torch.autograd.grad(h, [t for t in call if t is not None], s["dh"])
    return {"h": h, **dict(zip(names, grads))}


def _own_rotary(s):
    case = s["case"]
    q, k = _stacr().rotary(s["q"], s["k"], s["cos"], s["sin"], positions=s["positions"], layout=case["layout"])
    if not case["train"]:
        return {"q": q, "k": k}
    dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
    return {"q": q, "k": k, "dq": dq, "dk": dk}


def _own_clip(s):
    norm = _stacr().clip_gradients(s["grads"], s["max_norm"], norm_type=s["norm"], out=s["outs"])
    return {"norm": norm, "grads": s["flat"]}


_OWN = {"gated": _own_gated, "rotary": _own_rotary, "clip": _own_clip}


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["kind"]](state)


# ------------------------------------------------------------------------------------------ work
def work(case):
    if case["kind"] == "gated":
        n, d, f, size = case["rows"], case["d"], case["ff"], SIZE[case["dtype"]]
        weights = 2 * f * d + (2 * f if case["bias"] else 0)
        moved, flops = n * d + weights + n * f, 4 * n * d * f
        if case["train"]:  # dh in; dx and the parameters' gradients out
            moved, flops = moved + n * f + n * d + weights, 3 * flops
        return {"bytes": moved * size, "flops": flops}
    if case["kind"] == "rotary":
        tokens = case["batch"] * case["seq"]
        moved = 2 * tokens * (case["heads"] + case["kv_heads"]) * case["head"] * SIZE[case["dtype"]]
        turned = 3 * tokens * (case["heads"] + case["kv_heads"]) * case["rot"]
        passes = 2 if case["train"] else 1
        table = tokens * (case["rot"] * 4 + 8)
        return {"bytes": passes * moved + table, "flops": passes * turned}
    count = {"m": 0, "v": 0}
    for k, n in _gradient_sizes(case):
        count[k] += n
    size = {"mixed": (2, 4)}.get(case["dtype"]) or (SIZE[case["dtype"]],) * 2
    read = count["m"] * size[0] + count["v"] * size[1]
    # nothing changes in place where the norm is under the limit
    return {"bytes": read * (1 if case["place"] == "in" else 2), "flops": 3 * (count["m"] + count["v"])}


# ----------------------------------------------------------------------------------------- exact
def _exact_gated(s):
    """In 64 bits, the gradients by automatic differentiation."""
    case = s["case"]
    names = [n for n in ("x", "w_gate", "w_up", "b_gate", "b_up") if s[n] is not None]
    v = {n: s[n].detach().double().requires_grad_(case["train"]) for n in names}
    gate = torch.matmul(v["x"], v["w_gate"].T)
    up = torch.matmul(v["x"], v["w_up"].T)
    if case["bias"]:
        gate, up = gate + v["b_gate"], up + v["b_up"]
    act = {"silu": lambda t: t * torch.sigmoid(t), "sigmoid": torch.sigmoid, "relu": lambda t: t.clamp(min=0),
           "gelu": lambda t: t * torch.special.ndtr(t),
           "gelu_tanh": lambda t: t * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (t + 0.044715 * t ** 3))}[case["act"]]
    h = act(gate) * up
    out = {"h": h.detach()}
    if case["train"]:
        grads = torch.autograd.grad(h, [v[n] for n in names], s["dh"].double())
        out.update(zip(["d" + n for n in names], grads))
    return out


def _exact_rotary(s):
    """A pair is a complex number, the turn a product with exp(i angle) as the tables have it."""
    case = s["case"]
    at = s["positions"].reshape(-1)
    unit = torch.complex(s["cos"][at].double(), s["sin"][at].double())
    unit = unit.reshape(case["batch"], case["seq"], 1, -1)
    rot = case["rot"]

    def turn(x, by):
        y = x.detach().double().clone()
        if case["layout"] == "half":
            z = torch.complex(y[..., :rot // 2].contiguous(), y[..., rot // 2:rot].contiguous()) * by
            y[..., :rot // 2], y[..., rot // 2:rot] = z.real, z.imag
        else:
            z = torch.view_as_complex(y[..., :rot].reshape(*y.shape[:-1], rot // 2, 2).contiguous()) * by
            y[..., :rot] = torch.view_as_real(z).flatten(-2)
        return y

    out = {"q": turn(s["q"], unit), "k": turn(s["k"], unit)}
    if case["train"]:
        out["dq"], out["dk"] = turn(s["dq"], unit.conj()), turn(s["dk"], unit.conj())
    return out


def _exact_clip(s):
    if s["case"]["place"] == "in":
        sources = s["flat"]
    else:  # the buckets in the order of the outputs, from their views
        sources = [torch.cat([g for g in s["grads"] if g.dtype == o.dtype]) for o in s["flat"]]
    wide = [f.double() for f in sources]
    norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(w, s["norm"]) for w in wide]), s["norm"])
    return {"norm": norm, "grads": [w * min(1.0, s["max_norm"] / (float(norm) + 1e-6)) for w in wide]}


_EXACT = {"gated": _exact_gated, "rotary": _exact_rotary, "clip": _exact_clip}


def exact(case, seed):
    return _EXACT[case["kind"]](prepare(case, seed))
