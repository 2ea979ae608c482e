"""The operators of a decoder on an encoder's states that are timed: the linear layer on 8-bit operands
with a scale for each block of 128, rolling caches in 8 bits as they are written, read back and attended
to, and attention to an encoder's states of another length, kept in 32, 16 or 8 bits.

Sizes are those of the HTDemucs-shaped workloads of bench.py and tests/ (widths 384 and 512, heads of 48
and 64, feed-forward widths 1536 and 2048, 1344 time and 8 x 336 = 2688 frequency tokens, 4 chunks) or
generic. `draw` gives more cases of the same operators from one token up to long sequences. Where `own`
is false `run` is made of elementary torch operations in 32 bits; where it is true it calls the
framework's layers.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
TINY = 2.0 ** -100  # the smallest maximum that a scale is made from
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "bf16": 2, "e4m3": 1}


# ------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # The feed-forward's first map for five streams' new tokens: the weights are all the work.
        {"name": "linear_step", "op": "linear", "rows": 5, "fin": 512, "fout": 2048, "act": "gelu",
         "residual": False, "input": "e4m3", "out": "bf16"},
        # The feed-forward's second map over four chunks, adding the residual; its input is rounded
        # to 8 bits on the way.
        {"name": "linear_chunks", "op": "linear", "rows": 10752, "fin": 1536, "fout": 384,
         "act": "none", "residual": True, "input": "bf16", "out": "bf16"},
        # A wide model's map over a long batch: the largest product.
        {"name": "linear_wide", "op": "linear", "rows": 8192, "fin": 4096, "fout": 4096,
         "act": "swish", "residual": False, "input": "e4m3", "out": "bf16"},
        # Four chunks' keys and values into their caches, which hold fewer tokens than the chunks have:
        # what a prompt leaves behind.
        {"name": "write_chunks", "op": "write", "batch": 4, "tokens": 2688, "kv_heads": 8,
         "head_dim": 48, "sinks": 4, "slots": 2053, "dtype": "f32", "position": 0, "ragged": True},
        # A long recording's cache back to 16 bits.
        {"name": "read_long", "op": "read", "batch": 2, "tokens": 16384, "kv_heads": 8,
         "head_dim": 64, "sinks": 4, "slots": 16391, "dtype": "bf16", "position": 1000,
         "ragged": False},
        # One live stream's next token on an 8-bit cache: latency is all.
        {"name": "step_one", "op": "step", "batch": 1, "steps": 1, "heads": 8, "kv_heads": 8,
         "head_dim": 48, "left": 511, "sinks": 4, "spare": 0, "dtype": "f32", "position": 2000},
        # Sixty-four live streams with long windows, grouped heads, at unlike places.
        {"name": "step_streams", "op": "step", "batch": 64, "steps": 1, "heads": 16, "kv_heads": 4,
         "head_dim": 64, "left": 4095, "sinks": 4, "spare": 3, "dtype": "bf16", "position": 9000},
        # Eight streams that take sixteen tokens at once.
        {"name": "step_block", "op": "step", "batch": 8, "steps": 16, "heads": 8, "kv_heads": 2,
         "head_dim": 64, "left": 1023, "sinks": 4, "spare": 0, "dtype": "bf16", "position": 5000},
        # A decoder's next token on one chunk's time tokens.
        {"name": "memory_one", "op": "memory", "batch": 1, "queries": 1, "states": 1344, "heads": 8,
         "kv_heads": 8, "head_dim": 48, "dtype": "f32", "held": "f32", "ragged": False},
        # Sixty-four decoders' next tokens on the frequency tokens of a chunk each, in 8 bits.
        {"name": "memory_streams", "op": "memory", "batch": 64, "queries": 1, "states": 2688,
         "heads": 16, "kv_heads": 4, "head_dim": 64, "dtype": "bf16", "held": "e4m3",
         "ragged": True},
        # Time tokens on frequency tokens, four padded chunks, as the cross transformer has them.
        {"name": "memory_chunks", "op": "memory", "batch": 4, "queries": 1344, "states": 2688,
         "heads": 8, "kv_heads": 8, "head_dim": 48, "dtype": "f32", "held": "f32", "ragged": True},
        # A long prompt on a long recording, grouped heads: the longest sequences.
        {"name": "memory_long", "op": "memory", "batch": 1, "queries": 8192, "states": 16384,
         "heads": 8, "kv_heads": 2, "head_dim": 64, "dtype": "bf16", "held": "bf16",
         "ragged": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "write", "read", "step", "step", "memory", "memory",
                     "memory"])
    dtype = rng.choice(["f32", "bf16"])
    heads, kv_heads = rng.choice([(8, 8), (8, 8), (8, 2), (6, 3), (4, 1), (5, 5), (16, 4)])
    hd = rng.choice([32, 48, 64, 64, 72, 96, 128])
    if op == "linear":
        fin, fout = rng.choice([(384, 384), (384, 1152), (384, 1536), (1536, 384), (512, 2048),
                                (2048, 512), (512, 1536), (2048, 2048), (320, 200), (1000, 777)])
        return {"op": op, "rows": _log(rng, 1, 10752), "fin": fin, "fout": fout,
                "act": rng.choice(["none", "none", "gelu", "relu", "swish"]),
                "residual": rng.random() < 0.5,
                "input": rng.choice(["e4m3", "e4m3", "bf16", "f32"]), "out": dtype}
    if op in ("write", "read"):
        batch, tokens = rng.choice([1, 2, 4]), _log(rng, 1, 8192)
        sinks = rng.choice([0, 1, 4, 33])
        return {"op": op, "batch": batch, "tokens": tokens, "kv_heads": kv_heads, "head_dim": hd,
                "sinks": sinks,
                "slots": sinks + (_log(rng, 1, 8192) if op == "write" else tokens + 3),
                "dtype": dtype, "position": rng.choice([0, _log(rng, 1, 100000)]),
                "ragged": rng.random() < 0.5}
    if op == "step":
        return {"op": op, "batch": _log(rng, 1, 64), "steps": rng.choice([1, 1, 1, 2, 5, 16]),
                "heads": heads, "kv_heads": kv_heads, "head_dim": hd,
                "left": _log(rng, 16, 4096) - 1, "sinks": rng.choice([0, 1, 4, 33]),
                "spare": rng.choice([0, 1, 40]), "dtype": dtype,
                "position": rng.choice([0, _log(rng, 1, 100000), _log(rng, 1, 100000)])}
    short = rng.random() < 0.5  # a decoder's steps, or whole sequences
    queries = rng.choice([1, 1, 2, 5, 16, 61]) if short else _log(rng, 100, 3000)
    return {"op": op, "batch": _log(rng, 1, 64) if short else rng.choice([1, 1, 2, 4]),
            "queries": queries, "states": _log(rng, 1, 4096), "heads": heads, "kv_heads": kv_heads,
            "head_dim": hd, "dtype": dtype, "held": rng.choice([dtype, dtype, "e4m3"]),
            "ragged": rng.random() < 0.5}


# ------------------------------------------------------------------ inputs, from a seed alone
def _positions(case):
    """Tokens that each stream has had before the call: some far apart, some just begun."""
    p = case["position"]
    return [p if i % 4 != 3 else p // (3 + i) for i in range(case["batch"])]


def _counts(case):
    """Rows of each stream that are tokens: the first has all of them, the others fewer."""
    n = case["tokens"]
    return [n - (n * i) // (2 * case["batch"]) if case["ragged"] else n
            for i in range(case["batch"])]


def _query_counts(case):
    n = case["queries"]
    return [n - (n * i) // (2 * case["batch"]) if case["ragged"] else n
            for i in range(case["batch"])]


def _state_counts(case):
    """States of each sequence: the first is full, the last of four or more has none yet."""
    n, b = case["states"], case["batch"]
    if not case["ragged"]:
        return [n] * b
    return [0 if b >= 4 and i == b - 1 else n - (n * i) // (2 * b) for i in range(b)]


def _slots(case):
    if case["op"] == "step":
        return case["sinks"] + case["left"] + case["steps"] + case["spare"]
    return case["slots"]


class _Rand:
    """Seeded tensors on the GPU, drawn in a fixed order."""

    def __init__(self, case, seed):
        text = ",".join(f"{k}={v}" for k, v in sorted(case.items()) if k != "name")
        mix = sum((i + 1) * ord(c) for i, c in enumerate(text))
        self.g = torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + mix)

    def normal(self, *shape, std=1.0, dtype=torch.float32):
        return torch.randn(shape, generator=self.g, device="cuda").mul_(std).to(dtype)

    def rows(self, *shape, heads):
        """Keys or values as projections give them: rows of unlike size."""
        size = torch.exp(self.normal(*shape[:-1], heads, 1, std=0.3))
        x = self.normal(*shape[:-1], heads, shape[-1] // heads, std=1.2)
        return (x * size).reshape(shape)

    def held(self, *shape, heads):
        """Such rows as an 8-bit cache holds them: e4m3 values, and a scale for each head's."""
        x = self.rows(*shape, heads=heads)
        q, scale = _quantise(x.reshape(*shape[:-1], heads, shape[-1] // heads))
        return q.reshape(shape), scale


def _i32(values):
    return torch.tensor(values, dtype=torch.int32).to("cuda")


def prepare(case, seed):
    r, op = _Rand(case, seed), case["op"]
    s = {"case": case}
    if op == "linear":
        m, k, n = case["rows"], case["fin"], case["fout"]
        # activations with some channels a hundred times the others, as residual streams have them
        x = r.normal(m, k) * torch.exp(r.normal(m, 1, std=0.5))
        x[:, 7::97] *= 100
        if case["input"] == "e4m3":
            s["x"], s["scales"] = _quantise_blocks(x)
        else:
            s["x"], s["scales"] = x.to(DTYPES[case["input"]]), None
        w = r.normal(n, k, std=1 / math.sqrt(k))
        s["weight"], s["bias"] = w, r.normal(n, std=0.1)
        s["wq"], s["wscales"] = _quantise_tiles(w)
        s["residual"] = r.normal(m, n, dtype=DTYPES[case["out"]]) if case["residual"] else None
        if own:
            _to_framework(s)
        return s
    b, hd, kv, dt = case["batch"], case["head_dim"], case["kv_heads"], DTYPES[case["dtype"]]
    if op == "memory":
        t, n = case["queries"], case["states"]
        s["q"] = r.normal(b, t, case["heads"] * hd, std=1.3, dtype=dt)
        for name in "kv":
            if case["held"] == "e4m3":
                s[name], s[name + "_scales"] = r.held(b, n, kv * hd, heads=kv)
            else:
                s[name] = r.rows(b, n, kv * hd, heads=kv).to(dt)
                s[name + "_scales"] = None
        s["lengths"] = _i32(_state_counts(case)) if case["ragged"] else None
        s["query_lengths"] = _i32(_query_counts(case)) if case["ragged"] else None
        s["out"] = torch.zeros_like(s["q"])
    else:
        t = case["steps"] if op == "step" else case["tokens"]
        if op == "step":
            s["q"] = r.normal(b, t, case["heads"] * hd, std=1.3, dtype=dt)
            s["out"] = torch.zeros_like(s["q"])
        else:
            s["steps"] = _i32(_counts(case)) if case["ragged"] else None
        for name in "kv":
            if op == "read":
                s[name] = torch.zeros(b, t, kv * hd, dtype=dt, device="cuda")
            else:
                s[name] = r.rows(b, t, kv * hd, heads=kv).to(dt)
            s[name + "_cache"], s[name + "_scales"] = r.held(b, _slots(case), kv * hd, heads=kv)
        s["positions"] = _i32(_positions(case))
    if own:
        _to_framework(s)
    return s


def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state)
    return {"linear": _linear, "write": _write, "read": _read, "step": _step,
            "memory": _memory}[op](state)


# ------------------------------------------------------------------------------- the plain forms
def _quantise(x):
    """(e4m3 values, scale) of each row: scale = max |x| * (1 / 448), value = x * (448 * (1 / max))."""
    top = x.abs().amax(-1, keepdim=True).clamp_min(TINY)
    q = (x * (E4M3_MAX * torch.reciprocal(top))).clamp(-E4M3_MAX, E4M3_MAX)
    return q.to(torch.float8_e4m3fn), (top * (1 / E4M3_MAX)).squeeze(-1)


def _padded(x, *to):
    """x with zeros behind its last two dimensions, up to multiples of `to`."""
    rows, cols = (-x.shape[-2]) % to[0], (-x.shape[-1]) % to[1]
    return torch.nn.functional.pad(x, (0, cols, 0, rows))


def _quantise_blocks(x):
    """Rows in blocks of 128: values [m, k], scales [m, ceil(k / 128)]."""
    m, k = x.shape
    q, scale = _quantise(_padded(x, 1, BLOCK).reshape(m, -1, BLOCK))
    return q.reshape(m, -1)[:, :k].contiguous(), scale


def _quantise_tiles(w):
    """Tiles of 128 x 128: values [n, k], scales [ceil(n / 128), ceil(k / 128)]."""
    n, k = w.shape
    p = _padded(w, BLOCK, BLOCK)
    a, b = p.shape[0] // BLOCK, p.shape[1] // BLOCK
    tiles = p.reshape(a, BLOCK, b, BLOCK).transpose(1, 2).reshape(a, b, BLOCK * BLOCK)
    q, scale = _quantise(tiles)
    q = q.reshape(a, b, BLOCK, BLOCK).transpose(1, 2).reshape(p.shape)
    return q[:n, :k].contiguous(), scale


def _act(y, act):
    if act == "gelu":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    if act == "relu":
        return y.clamp_min(0)
    if act == "swish":
        return y / (1 + torch.exp(-y))
    return y


def _linear(s):
    case = s["case"]
    m, k, n = case["rows"], case["fin"], case["fout"]
    xq, xs = (s["x"], s["scales"]) if s["scales"] is not None else _quantise_blocks(s["x"].float())
    x = xq.float() * xs.repeat_interleave(BLOCK, 1)[:, :k]
    w = s["wscales"].repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    y = _act(torch.matmul(x, (s["wq"].float() * w).t()) + s["bias"], case["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(DTYPES[case["out"]])


def _heads(x, n):
    """[B, T, n * hd] -> [B, n, T, hd] in 32 bits."""
    b, t, w = x.shape
    return x.float().reshape(b, t, n, w // n).transpose(1, 2)


def _values(q, scales):
    """What an 8-bit cache stands for, in 32 bits."""
    n = scales.shape[-1]
    x = q.float().reshape(*q.shape[:-1], n, q.shape[-1] // n) * scales[..., None]
    return x.reshape(q.shape)


def _attend(q, k, v, seen):
    """Softmax attention over the keys that `seen` (broadcast to the scores) marks, in 32 bits; zeros
    for a query that sees none."""
    group = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    p = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(1 / math.sqrt(q.shape[-1]))
    if seen is not None:
        p.masked_fill_(~seen, -math.inf)
    p.sub_(p.amax(-1, keepdim=True).clamp_min(-3e38)).exp_()
    p.div_(p.sum(-1, keepdim=True).clamp_min(1e-30))
    return torch.matmul(p, v)


def _memory(s):
    case = s["case"]
    kv, n = case["kv_heads"], case["states"]
    k, v = ((_values(s[x], s[x + "_scales"]) if case["held"] == "e4m3" else s[x]) for x in "kv")
    seen = None
    if s["lengths"] is not None:
        i = torch.arange(n, device="cuda")
        seen = (i < s["lengths"][:, None])[:, None, None, :]
    o = _attend(_heads(s["q"], case["heads"]), _heads(k, kv), _heads(v, kv), seen)
    o = o.transpose(1, 2).reshape(s["q"].shape).to(s["q"].dtype)
    if s["query_lengths"] is not None:  # rows behind a sequence's queries are left as they were
        i = torch.arange(case["queries"], device="cuda")
        o = torch.where((i < s["query_lengths"][:, None])[..., None], o, s["out"])
    s["out"].copy_(o)
    return s["out"]


def _slot(case, p):
    sinks = case["sinks"]
    return torch.where(p < sinks, p, sinks + (p - sinks) % (_slots(case) - sinks))


def _taken(s):
    """(stream, row, slot) of the rows that a write leaves in the caches: of rows that share a slot,
    the last."""
    case = s["case"]
    ring = _slots(case) - case["sinks"]
    i = torch.arange(case["tokens"], device="cuda")[None]
    count = s["steps"][:, None] if s["steps"] is not None else torch.full_like(
        s["positions"][:, None], case["tokens"])
    p = s["positions"].long()[:, None] + i
    kept = (i < count) & ((p < case["sinks"]) | (i >= count - ring))
    b, t = torch.nonzero(kept, as_tuple=True)
    return b, t, _slot(case, p[b, t])


def _put(s, b, t, slot):
    """Rows of k and v to slots of the 8-bit caches."""
    kv, hd = s["case"]["kv_heads"], s["case"]["head_dim"]
    for name in "kv":
        q, scale = _quantise(s[name][b, t].float().reshape(-1, kv, hd))
        s[name + "_cache"][b, slot] = q.reshape(-1, kv * hd)
        s[name + "_scales"][b, slot] = scale


def _caches(s):
    return {n: s[n] for n in ("k_cache", "k_scales", "v_cache", "v_scales")}


def _write(s):
    _put(s, *_taken(s))
    return _caches(s)


def _read(s):
    case = s["case"]
    i = torch.arange(case["tokens"], device="cuda")[None]
    rows = torch.arange(case["batch"], device="cuda")[:, None]
    slot = _slot(case, s["positions"].long()[:, None] + i)
    for name in "kv":
        x = _values(s[name + "_cache"][rows, slot], s[name + "_scales"][rows, slot])
        x = x.to(s[name].dtype)
        if s["steps"] is not None:
            x = torch.where((i < s["steps"][:, None])[..., None], x, s[name])
        s[name].copy_(x)
    return {"k": s["k"], "v": s["v"]}


def _step(s):
    case = s["case"]
    t, sinks, slots = case["steps"], case["sinks"], _slots(case)
    pos = s["positions"].long()[:, None]
    new = pos + torch.arange(t, device="cuda")[None]
    b, i = (x.reshape(-1) for x in torch.meshgrid(
        torch.arange(case["batch"], device="cuda"), torch.arange(t, device="cuda"), indexing="ij"))
    _put(s, b, i, _slot(case, new).reshape(-1))
    # the last token of each slot once the new ones are in; below 0 (or of a sink not reached): none
    slot = torch.arange(slots, device="cuda")[None]
    end = pos + t - 1
    last = end - (end - sinks - (slot - sinks)) % (slots - sinks)
    at = torch.where(slot < sinks, torch.where(slot <= end, slot, -1),
                     torch.where(last >= sinks, last, -1))[:, None, :]
    mine = new[:, :, None]
    seen = (at >= 0) & (at <= mine) & ((at >= mine - case["left"]) | (at < sinks))
    k, v = (_values(s[n + "_cache"], s[n + "_scales"]) for n in "kv")
    n = case["kv_heads"]
    o = _attend(_heads(s["q"], case["heads"]), _heads(k, n), _heads(v, n), seen[:, None])
    s["out"].copy_(o.transpose(1, 2).reshape(s["q"].shape))
    return dict(_caches(s), out=s["out"])


# --------------------------------------------------------------------------- the framework's calls
class _Memory:
    """A framework tensor's memory as torch reads it; torch holds this object as long as a view of
    it lives, and this object the tensor."""

    def __init__(self, t, typestr):
        self.tensor = t
        self.__cuda_array_interface__ = {"shape": t.shape, "typestr": typestr, "version": 2,
                                         "data": (t.device_ptr, False), "strides": None}


_NAMES = {torch.float32: "f32", torch.bfloat16: "bf16", torch.int32: "i32",
          torch.float8_e4m3fn: "e4m3"}
_RAW = {"f32": "<f4", "bf16": "<i2", "i32": "<i4", "e4m3": "|u1"}
_TORCH = {v: k for k, v in _NAMES.items()}
_device = None


def _framework():
    global _device
    from metalaudio_amd import nn
    if _device is None:
        _device = nn.AudioDevice(0)
    return nn, _device


def _empty(shape, dtype):
    """A framework tensor and torch's view of its memory."""
    nn, dev = _framework()
    t = nn.Tensor(dev, shape, dtype=dtype)
    return t, torch.as_tensor(_Memory(t, _RAW[dtype]), device="cuda").view(_TORCH[dtype])


_INPUTS = ("x", "scales", "residual", "q", "k", "v", "k_cache", "v_cache", "k_scales", "v_scales",
           "positions", "steps", "lengths", "query_lengths", "out")


def _to_framework(s):
    """The framework's layers and tensors that a program keeps, in place of the torch ones."""
    nn, dev = _framework()
    case, op = s["case"], s["case"]["op"]
    f = s["own"] = {}
    for name in _INPUTS:
        f[name] = None
        if s.get(name) is not None:
            x = s[name]
            f[name], view = _empty(tuple(x.shape), _NAMES[x.dtype])
            view.copy_(x)
            f[name + "_view"] = view
    if op == "linear":
        f["layer"] = nn.Linear(dev, case["fin"], case["fout"], activation=case["act"],
                               precision="e4m3_block")
        f["layer"].load_weights(s["weight"].cpu().numpy(), s["bias"].cpu().numpy())
        f["out"], f["out_view"] = _empty((case["rows"], case["fout"]), case["out"])
    elif op == "step":
        f["layer"] = nn.WindowAttention(dev, case["heads"], case["head_dim"],
                                        num_kv_heads=case["kv_heads"], window_left=case["left"],
                                        sinks=case["sinks"])
    elif op == "memory":
        f["layer"] = nn.MemoryAttention(dev, case["heads"], case["head_dim"],
                                        num_kv_heads=case["kv_heads"])
    else:
        f["layer"] = nn.KVCache(dev, case["kv_heads"], case["head_dim"], sinks=case["sinks"])
    for name in (*_INPUTS, "weight", "wq"):
        s.pop(name, None)


def _own(s):
    op, f = s["case"]["op"], s["own"]
    layer = f["layer"]
    if op == "linear":
        layer.forward_scaled(f["x"], f["scales"], f["out"], residual=f["residual"])
        return f["out_view"]
    if op == "memory":
        layer.forward(f["q"], f["k"], f["v"], f["out"], lengths=f["lengths"],
                      query_lengths=f["query_lengths"], k_scales=f["k_scales"],
                      v_scales=f["v_scales"])
        return f["out_view"]
    if op == "read":
        layer.read(f["k_cache"], f["v_cache"], f["positions"], f["k"], f["v"],
                   k_scales=f["k_scales"], v_scales=f["v_scales"], steps=f["steps"])
        return {"k": f["k_view"], "v": f["v_view"]}
    got = {n: f[n + "_view"] for n in ("k_cache", "k_scales", "v_cache", "v_scales")}
    if op == "write":
        layer.write(f["k"], f["v"], f["positions"], f["k_cache"], f["v_cache"],
                    k_scales=f["k_scales"], v_scales=f["v_scales"], steps=f["steps"])
        return got
    layer.step(f["q"], f["k"], f["v"], f["positions"], f["k_cache"], f["v_cache"], f["out"],
               k_scales=f["k_scales"], v_scales=f["v_scales"])
    return dict(got, out=f["out_view"])


# ----------------------------------------------------------------------------- work, and 64 bits
def work(case):
    op = case["op"]
    if op == "linear":
        m, k, n, e = case["rows"], case["fin"], case["fout"], BYTES[case["out"]]
        kb, nb = -(-k // BLOCK), -(-n // BLOCK)
        return {"bytes": m * k * BYTES[case["input"]] + (4 * m * kb if case["input"] == "e4m3" else 0)
                + n * k + 4 * nb * kb + 4 * n + m * n * e * (2 if case["residual"] else 1),
                "flops": 2.0 * m * n * k}
    e, hd, kv = BYTES[case["dtype"]], case["head_dim"], case["kv_heads"]
    if op in ("write", "read"):
        rows = 0
        for p, n in zip(_positions(case), _counts(case)):
            if op == "write":  # rows that a later one of the call does not replace
                first = max(0, min(n, case["sinks"] - p))
                n = min(n, first + min(n - first, _slots(case) - case["sinks"]))
            rows += n
        return {"bytes": 2 * rows * kv * (hd * (e + 1) + 4), "flops": 2.0 * rows * kv * hd}
    h = case["heads"]
    if op == "memory":
        held = 4 + hd if case["held"] == "e4m3" else e * hd  # a head's row
        queries, states = _query_counts(case), _state_counts(case)
        return {"bytes": 2 * e * h * hd * sum(queries)
                + 2 * kv * held * sum(n for q, n in zip(queries, states) if q),
                "flops": 4.0 * h * hd * sum(q * n for q, n in zip(queries, states))}
    pairs = keys = 0
    for p in _positions(case):
        for t in range(p, p + case["steps"]):
            lo = max(0, t - case["left"])
            pairs += t - lo + 1 + min(lo, case["sinks"])
        lo = max(0, p - case["left"])
        keys += p - lo + min(lo, case["sinks"])
    new = case["batch"] * case["steps"]
    return {"bytes": new * hd * e * 2 * (h + kv) + 2 * kv * (hd + 4) * (new + keys),
            "flops": 4.0 * pairs * h * hd}


def _round_e4m3(x):
    """The nearest e4m3 value, ties to even, from the format's spacing: 2^(e - 3), e >= -6."""
    x = x.double()
    e = torch.frexp(x)[1].sub(1).clamp_min(-6)
    step = torch.ldexp(torch.ones_like(x), e - 3)
    return torch.round(x / step).mul(step).clamp(-E4M3_MAX, E4M3_MAX)


def _levels(x):
    """e4m3 values (as 64-bit numbers) and scales of fp32 rows, the scales fp32 as they are kept."""
    top = torch.max(x.abs(), -1).values.clamp_min(TINY)
    inv = torch.full_like(top, E4M3_MAX) * (torch.ones_like(top) / top)  # in fp32, as defined
    return _round_e4m3(x * inv[..., None]), (top.double() / E4M3_MAX).float().double()


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"linear": _exact_linear, "write": _exact_write, "read": _exact_read,
            "step": _exact_step, "memory": _exact_memory}[case["op"]](case, s)


def _exact_linear(case, s):
    """Block by block: the sum of each block's products, times its two scales."""
    m, k, n = case["rows"], case["fin"], case["fout"]
    y = torch.zeros(m, n, dtype=torch.float64, device="cuda")
    for at in range(0, k, BLOCK):
        if s["scales"] is None:
            x, xs = _levels(s["x"][:, at:at + BLOCK].float())
        else:
            x, xs = s["x"][:, at:at + BLOCK].double(), s["scales"][:, at // BLOCK].double()
        for to in range(0, n, BLOCK):
            w = s["weight"][to:to + BLOCK, at:at + BLOCK]
            q, scale = _levels(w.reshape(1, -1))
            y[:, to:to + BLOCK] += (x @ q.reshape(w.shape).T) * (xs * scale)[:, None]
    y += s["bias"].double()
    if case["act"] == "gelu":
        y = y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
    elif case["act"] == "relu":
        y = torch.where(y > 0, y, torch.zeros_like(y))
    elif case["act"] == "swish":
        y = y * torch.sigmoid(y)
    return y if s["residual"] is None else y + s["residual"].double()


def _place(case, p):
    sinks = case["sinks"]
    return p if p < sinks else sinks + (p - sinks) % (_slots(case) - sinks)


def _held(case, s, counts):
    """The caches as 64-bit numbers with each stream's first `counts` rows of k and v in them, one
    after the other, so that the last one of a slot stays: (values, scales) of k and of v."""
    kv, hd = case["kv_heads"], case["head_dim"]
    got = {}
    for name in "kv":
        q, scale = s[name + "_cache"].double(), s[name + "_scales"].double()
        for b, (p0, n) in enumerate(zip(_positions(case), counts)):
            if n == 0:
                continue
            x, xs = _levels(s[name][b, :n].float().reshape(n, kv, hd))
            last = {_place(case, p0 + i): i for i in range(n)}
            to, row = (torch.tensor(list(z), device="cuda") for z in (last.keys(), last.values()))
            q[b, to], scale[b, to] = x.reshape(n, -1)[row], xs[row]
        got[name + "_cache"], got[name + "_scales"] = q, scale
    return got


def _exact_write(case, s):
    return _held(case, s, _counts(case))


def _exact_read(case, s):
    kv, hd = case["kv_heads"], case["head_dim"]
    got = {}
    for name in "kv":
        out = got[name] = torch.zeros(s[name].shape, dtype=torch.float64, device="cuda")
        for b, (p0, n) in enumerate(zip(_positions(case), _counts(case))):
            at = torch.tensor([_place(case, p0 + i) for i in range(n)], dtype=torch.long,
                              device="cuda")
            q = s[name + "_cache"][b, at].double().reshape(n, kv, hd)
            out[b, :n] = (q * s[name + "_scales"][b, at].double()[..., None]).reshape(n, -1)
    return got


def _exact_heads(case, q, k, v, seen=None):
    """One sequence, head by head: [T, H * hd] queries on [S, KV * hd] keys and values."""
    hd, group = case["head_dim"], case["heads"] // case["kv_heads"]
    cols = []
    for h in range(case["heads"]):
        at, to = h * hd, h // group * hd
        score = q[:, at:at + hd].double() @ k[:, to:to + hd].double().T / math.sqrt(hd)
        if seen is not None:
            score = torch.where(seen, score, torch.full_like(score, -math.inf))
        cols.append(torch.softmax(score, -1) @ v[:, to:to + hd].double())
    return torch.cat(cols, -1)


def _whole(case, q, scales):
    """64-bit rows [.., KV * hd] of 8-bit values and their scales."""
    x = q.double().unflatten(-1, (case["kv_heads"], case["head_dim"]))
    return (x * scales.double()[..., None]).flatten(-2)


def _exact_memory(case, s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, (t, n) in enumerate(zip(_query_counts(case), _state_counts(case))):
        if t == 0 or n == 0:
            continue
        k, v = (_whole(case, s[x][b, :n], s[x + "_scales"][b, :n]) if case["held"] == "e4m3"
                else s[x][b, :n] for x in "kv")
        out[b, :t] = _exact_heads(case, s["q"][b, :t], k, v)
    return out


def _exact_step(case, s):
    sinks, left, t = case["sinks"], case["left"], case["steps"]
    got = _held(case, s, [t] * case["batch"])
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, p0 in enumerate(_positions(case)):
        first = max(0, p0 - left)
        told = list(range(min(sinks, first))) + list(range(first, p0 + t))
        at = torch.tensor([_place(case, p) for p in told], dtype=torch.long, device="cuda")
        k, v = (_whole(case, got[n + "_cache"][b, at], got[n + "_scales"][b, at]) for n in "kv")
        key = torch.tensor(told, device="cuda")[None, :]
        mine = torch.arange(p0, p0 + t, device="cuda")[:, None]
        seen = (key <= mine) & ((mine - key <= left) | (key < sinks))
        out[b] = _exact_heads(case, s["q"][b], k, v, seen)
    return dict(got, out=out)
