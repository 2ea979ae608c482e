"""The operators of a streaming transformer over audio tokens that are timed: a root-mean-square
norm that adds the residual and writes 8 bits, the linear layer that reads them, rotary positions
over several axes, and attention over a sliding window with a few first tokens that stay visible,
over whole sequences and step by step on a rolling cache.

Sizes are those of the HTDemucs-shaped workloads of bench.py and tests/ (widths 384 and 512, heads
of 48 and 64, feed-forward widths 1536 and 2048, 1344 time and 8 x 336 = 2688 frequency tokens, 4
chunks) or generic. `draw` gives more cases of the same operators from one token up to long
sequences. Where `own` is false `run` is made of elementary torch operations in 32 bits (64 for the
angles); where it is true it calls the framework's layers.
"""
from __future__ import annotations

import math

import torch

own = False

E4M3_MAX = 448.0
TINY = 2.0 ** -100  # the smallest row maximum that a scale is made from
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "bf16": 2, "e4m3": 1}


# ------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # One step of eight live streams through a block's norm: eight rows, the smallest call.
        {"name": "norm_step", "op": "norm", "rows": 8, "features": 512, "dtype": "f32",
         "residual": True, "out": "e4m3"},
        # The frequency tokens of four chunks, an ordinary forward.
        {"name": "norm_chunks", "op": "norm", "rows": 10752, "features": 384, "dtype": "bf16",
         "residual": True, "out": "e4m3"},
        # A long recording's tokens at the feed-forward width, an odd number of rows.
        {"name": "norm_long", "op": "norm", "rows": 65537, "features": 2048, "dtype": "bf16",
         "residual": True, "out": "e4m3"},
        # The feed-forward's first map for five streams' new tokens: the weights are all the work.
        {"name": "linear_step", "op": "linear", "rows": 5, "fin": 512, "fout": 2048, "act": "gelu",
         "residual": False, "input": "e4m3", "out": "bf16"},
        # The feed-forward's second map over four chunks, adding the residual.
        {"name": "linear_chunks", "op": "linear", "rows": 10752, "fin": 1536, "fout": 384,
         "act": "none", "residual": True, "input": "e4m3", "out": "f32"},
        # A wide model's map over a long batch: the largest product.
        {"name": "linear_wide", "op": "linear", "rows": 8192, "fin": 4096, "fout": 4096,
         "act": "swish", "residual": False, "input": "e4m3", "out": "bf16"},
        # One new token for each of eight streams, far into the recording.
        {"name": "rotary_step", "op": "rotary", "batch": 8, "seq": 1, "heads": 8, "kv_heads": 8,
         "head_dim": 64, "axes": "32,16", "interleaved": False, "dtype": "f32", "origin": 900001},
        # The spectrogram's tokens of four chunks: time frames and frequency bands as two axes.
        {"name": "rotary_grid", "op": "rotary", "batch": 4, "seq": 2688, "heads": 8, "kv_heads": 8,
         "head_dim": 48, "axes": "24,24", "interleaved": False, "dtype": "bf16", "origin": 0},
        # A chunk's time tokens and one, looking both ways, two sequences of unlike lengths.
        {"name": "window_chunk", "op": "window", "batch": 2, "seq": 1345, "heads": 8,
         "kv_heads": 8, "head_dim": 48, "left": 168, "right": 168, "sinks": 4, "ragged": True,
         "dtype": "f32"},
        # A long recording, causal, grouped heads: the longest sequence.
        {"name": "window_long", "op": "window", "batch": 1, "seq": 16384, "heads": 8,
         "kv_heads": 2, "head_dim": 64, "left": 1023, "right": 0, "sinks": 4, "ragged": False,
         "dtype": "bf16"},
        # One live stream's next token: latency is all.
        {"name": "step_one", "op": "step", "batch": 1, "steps": 1, "heads": 8, "kv_heads": 8,
         "head_dim": 48, "left": 511, "sinks": 4, "spare": 0, "dtype": "f32", "position": 2000},
        # Sixty-four live streams with long windows, grouped heads, at unlike places.
        {"name": "step_streams", "op": "step", "batch": 64, "steps": 1, "heads": 16,
         "kv_heads": 4, "head_dim": 64, "left": 2047, "sinks": 4, "spare": 3, "dtype": "bf16",
         "position": 5000},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "linear", "linear", "rotary", "window", "window", "step", "step"])
    dtype = rng.choice(["f32", "bf16"])
    heads, kv_heads = rng.choice([(8, 8), (8, 8), (8, 2), (6, 3), (4, 1), (5, 5)])
    hd = rng.choice([32, 48, 64, 64, 72, 96, 128])
    if op == "norm":
        return {"op": op, "rows": _log(rng, 1, 32768),
                "features": rng.choice([257, 384, 384, 512, 768, 1000, 1536, 2048, 4096]),
                "dtype": dtype, "residual": rng.random() < 0.7,
                "out": rng.choice(["e4m3", "e4m3", "same"])}
    if op == "linear":
        fin, fout = rng.choice([(384, 384), (384, 1152), (384, 1536), (1536, 384), (512, 2048),
                                (2048, 512), (512, 1536), (2048, 2048), (320, 200), (1000, 777)])
        kind = rng.choice(["e4m3", "e4m3", "bf16"])
        return {"op": op, "rows": _log(rng, 1, 10752), "fin": fin, "fout": fout,
                "act": rng.choice(["none", "none", "gelu", "relu", "swish"]),
                "residual": rng.random() < 0.5, "input": kind,
                "out": rng.choice(["f32", "bf16"]) if kind == "e4m3" else "bf16"}
    if op == "rotary":
        inter = rng.random() < 0.5
        axes = [2 * rng.randint(1, hd // 2 // 3) for _ in range(rng.randint(1, 3))]
        if rng.random() < 0.5:  # all of the head rotated, as most models have it
            axes = [hd] if len(axes) == 1 else [hd // 2, hd // 2 - hd // 2 % 2][:2]
            axes = [a - a % 2 for a in axes]
        return {"op": op, "batch": rng.choice([1, 2, 4]), "seq": _log(rng, 1, 8192),
                "heads": heads, "kv_heads": kv_heads, "head_dim": hd,
                "axes": ",".join(map(str, axes)), "interleaved": inter, "dtype": dtype,
                "origin": rng.choice([0, 0, _log(rng, 10, 1000000)])}
    if op == "window":
        seq = _log(rng, 1, 8192)
        batch = rng.choice([1, 1, 2, 4]) if seq < 4096 else 1
        left = _log(rng, 1, 4096) - 1
        return {"op": op, "batch": batch, "seq": seq, "heads": heads, "kv_heads": kv_heads,
                "head_dim": hd, "left": left, "right": rng.choice([0, 0, left, left // 3]),
                "sinks": rng.choice([0, 1, 4, 33]), "ragged": rng.random() < 0.5, "dtype": dtype}
    return {"op": op, "batch": _log(rng, 1, 64), "steps": rng.choice([1, 1, 1, 2, 5, 16]),
            "heads": heads, "kv_heads": kv_heads, "head_dim": hd, "left": _log(rng, 16, 4096) - 1,
            "sinks": rng.choice([0, 1, 4, 33]), "spare": rng.choice([0, 1, 40]), "dtype": dtype,
            "position": rng.choice([0, _log(rng, 1, 100000), _log(rng, 1, 100000)])}


# ------------------------------------------------------------------ inputs, from a seed alone
def _lengths(case):
    """Tokens of each padded sequence: the first is full, the others shorter."""
    n = case["seq"]
    return [n - (n * i) // (2 * case["batch"]) for i in range(case["batch"])]


def _positions(case):
    """Tokens that each stream has had before the step: some far apart, some just begun."""
    p = case["position"]
    return [p if i % 4 != 3 else p // (3 + i) for i in range(case["batch"])]


def _slots(case):
    return case["sinks"] + case["left"] + case["steps"] + case["spare"]


def _grid(case):
    """Token positions on each axis: frames, then bands of them, then a third of those."""
    n, origin = case["seq"], case["origin"]
    i = torch.arange(n)
    cols = [origin + i // 8, i % 8, (i * 5) % 37] if "," in case["axes"] else [origin + i]
    return torch.stack(cols[:len(case["axes"].split(","))], -1).to(torch.int32)


class _Rand:
    """Seeded tensors on the GPU, drawn in a fixed order."""

    def __init__(self, case, seed):
        text = ",".join(f"{k}={v}" for k, v in sorted(case.items()) if k != "name")
        mix = sum((i + 1) * ord(c) for i, c in enumerate(text))
        self.g = torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + mix)

    def normal(self, *shape, std=1.0, dtype=torch.float32):
        return torch.randn(shape, generator=self.g, device="cuda").mul_(std).to(dtype)


def prepare(case, seed):
    r, op = _Rand(case, seed), case["op"]
    s = {"case": case}
    if op == "norm":
        n, f, dt = case["rows"], case["features"], DTYPES[case["dtype"]]
        # activations of rows of unlike size, as a residual stream has them
        s["x"] = (r.normal(n, f) * torch.exp(r.normal(n, 1, std=0.7))).to(dt)
        s["residual"] = r.normal(n, f, std=2.0, dtype=dt) if case["residual"] else None
        s["weight"] = 1 + r.normal(f, std=0.2)
    elif op == "linear":
        m, k, n = case["rows"], case["fin"], case["fout"]
        x = r.normal(m, k) * torch.exp(r.normal(m, 1, std=0.5))
        if case["input"] == "e4m3":
            s["x"], s["scales"] = _quantise(x)
        else:
            s["x"], s["scales"] = x.to(torch.bfloat16), None
        w = r.normal(n, k, std=1 / math.sqrt(k))
        s["weight"], s["bias"] = w, r.normal(n, std=0.1)
        s["wq"], s["wscales"] = _quantise(w)
        s["residual"] = r.normal(m, n, dtype=DTYPES[case["out"]]) if case["residual"] else None
    elif op == "rotary":
        b, t, hd, dt = case["batch"], case["seq"], case["head_dim"], DTYPES[case["dtype"]]
        s["q"] = r.normal(b, t, case["heads"] * hd, dtype=dt)
        s["k"] = r.normal(b, t, case["kv_heads"] * hd, dtype=dt)
        s["positions"] = _grid(case).to("cuda")
    elif op == "window":
        b, t, hd, dt = case["batch"], case["seq"], case["head_dim"], DTYPES[case["dtype"]]
        # keys near their queries score higher, as learnt ones do
        s["q"] = r.normal(b, t, case["heads"] * hd, std=1.3, dtype=dt)
        s["k"] = r.normal(b, t, case["kv_heads"] * hd, std=1.3, dtype=dt)
        s["v"] = r.normal(b, t, case["kv_heads"] * hd, dtype=dt)
        s["lengths"] = (torch.tensor(_lengths(case), dtype=torch.int32).to("cuda")
                        if case["ragged"] else None)
        s["out"] = torch.zeros_like(s["q"])
    else:
        b, t, hd, dt = case["batch"], case["steps"], case["head_dim"], DTYPES[case["dtype"]]
        kvw = case["kv_heads"] * hd
        s["q"] = r.normal(b, t, case["heads"] * hd, std=1.3, dtype=dt)
        s["k"], s["v"] = r.normal(b, t, kvw, std=1.3, dtype=dt), r.normal(b, t, kvw, dtype=dt)
        s["k_cache"] = r.normal(b, _slots(case), kvw, std=1.3, dtype=dt)
        s["v_cache"] = r.normal(b, _slots(case), kvw, dtype=dt)
        s["positions"] = torch.tensor(_positions(case), dtype=torch.int32).to("cuda")
        s["out"] = torch.zeros_like(s["q"])
    if own:
        _to_framework(s)
    return s


def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state)
    return {"norm": _norm, "linear": _linear, "rotary": _rotary, "window": _window,
            "step": _step}[op](state)


# ------------------------------------------------------------------------------- the plain forms
def _row_scales(x):
    top = x.abs().amax(-1, keepdim=True).clamp_min(TINY)
    return top * (1 / E4M3_MAX), E4M3_MAX * torch.reciprocal(top)


def _quantise(x):
    """(e4m3 values, scale of each row): scale = max |x| * (1 / 448), value = x * (448 * (1 / max))."""
    scale, inv = _row_scales(x)
    q = (x * inv).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return q, scale.squeeze(-1)


def _norm(s):
    case = s["case"]
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + 1e-5) * s["weight"]
    total = h.to(s["x"].dtype)
    if case["out"] == "same":
        return {"sum": total, "out": y.to(s["x"].dtype)}
    q, scale = _quantise(y)
    return {"sum": total, "out": q, "scales": scale}


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
    xq, xs = (s["x"], s["scales"]) if s["scales"] is not None else _quantise(s["x"].float())
    y = torch.matmul(xq.float(), s["wq"].float().t())
    y = _act(y * xs[:, None] * s["wscales"] + s["bias"], case["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(DTYPES[case["out"]])


def _rotary(s):
    case = s["case"]
    hd, dims = case["head_dim"], [int(a) for a in case["axes"].split(",")]
    freq, axis, first, second = [], [], [], []
    off = 0
    for a, d in enumerate(dims):
        i = torch.arange(d // 2)
        freq.append(10000.0 ** (-2.0 * i.double() / d))
        axis.append(torch.full((d // 2,), a))
        first.append(off + (2 * i if case["interleaved"] else i))
        second.append(off + (2 * i + 1 if case["interleaved"] else i + d // 2))
        off += d
    freq, axis, first, second = (torch.cat(x).cuda() for x in (freq, axis, first, second))
    angle = s["positions"].double()[:, axis] * freq
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turn(x, heads):
        y = x.float().reshape(case["batch"], case["seq"], heads, hd)
        u, v = y[..., first], y[..., second]
        y = y.clone()
        y[..., first] = u * cos - v * sin
        y[..., second] = v * cos + u * sin
        return y.reshape(x.shape).to(x.dtype)

    return {"q": turn(s["q"], case["heads"]), "k": turn(s["k"], case["kv_heads"])}


def _heads(x, n):
    """[B, T, n * hd] -> [B, n, T, hd] in 32 bits."""
    b, t, w = x.shape
    return x.float().reshape(b, t, n, w // n).transpose(1, 2)


def _attend(q, k, v, seen):
    """Softmax attention over the keys that `seen` (broadcast to the scores) marks, in 32 bits."""
    group = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    p = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(1 / math.sqrt(q.shape[-1]))
    p.masked_fill_(~seen, -math.inf)
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    p.div_(p.sum(-1, keepdim=True))
    return torch.matmul(p, v)


def _window(s):
    case = s["case"]
    q, k, v = (_heads(s[n], case["heads" if n == "q" else "kv_heads"]) for n in "qkv")
    i = torch.arange(case["seq"], device="cuda")
    ahead = i[None, :] - i[:, None]  # key - query
    seen = (ahead <= case["right"]) & ((ahead >= -case["left"]) | (i < case["sinks"])[None, :])
    lengths = s["lengths"]
    if lengths is not None:
        seen = seen & (i < lengths[:, None])[:, None, None, :]
    o = _attend(q, k, v, seen).transpose(1, 2).reshape(s["q"].shape).to(s["q"].dtype)
    if lengths is not None:  # rows past a sequence's end are left as they were
        o = torch.where((i < lengths[:, None])[..., None], o, s["out"])
    s["out"].copy_(o)
    return s["out"]


def _step(s):
    case = s["case"]
    t, sinks, slots = case["steps"], case["sinks"], _slots(case)
    ring = slots - sinks
    pos = s["positions"].long()[:, None]
    slot = torch.arange(slots, device="cuda")[None]
    # the last token of each slot before this step; below 0 (or of a sink not reached): none
    last = pos - 1 - (pos - 1 - sinks - (slot - sinks)) % ring
    held = torch.where(slot < sinks, torch.where(slot < pos, slot, -1),
                       torch.where(last >= sinks, last, -1))
    new = pos + torch.arange(t, device="cuda")[None]
    at = torch.cat([held, new], 1)[:, None, :]
    mine = new[:, :, None]
    seen = (at >= 0) & (at <= mine) & ((at >= mine - case["left"]) | (at < sinks))
    k, v = (torch.cat([s[n + "_cache"], s[n]], 1) for n in "kv")
    n = case["kv_heads"]
    o = _attend(_heads(s["q"], case["heads"]), _heads(k, n), _heads(v, n), seen[:, None])
    s["out"].copy_(o.transpose(1, 2).reshape(s["q"].shape))
    to = torch.where(new < sinks, new, sinks + (new - sinks) % ring)
    rows = torch.arange(case["batch"], device="cuda")[:, None]
    s["k_cache"][rows, to] = s["k"]
    s["v_cache"][rows, to] = s["v"]
    return {"out": s["out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


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


def _of(x):
    t, view = _empty(tuple(x.shape), _NAMES[x.dtype])
    view.copy_(x)
    return t, view


def _to_framework(s):
    """The framework's layers and tensors that a program keeps, in place of the torch ones."""
    nn, dev = _framework()
    case, op = s["case"], s["case"]["op"]
    f = s["own"] = {}
    for name in ("x", "residual", "scales", "q", "k", "v", "positions", "lengths", "out",
                 "k_cache", "v_cache"):
        f[name] = None
        if s.get(name) is not None:
            f[name], f[name + "_view"] = _of(s[name])
    if op == "norm":
        f["layer"] = nn.RMSNorm(dev, case["features"], 1e-5)
        f["layer"].load_parameters(s["weight"].cpu().numpy())
        same = case["out"] == "same"
        shape, dt = (case["rows"], case["features"]), case["dtype"]
        f["sum"], f["sum_view"] = _empty(shape, dt)
        f["out"], f["out_view"] = _empty(shape, dt if same else "e4m3")
        if not same:
            f["scales"], f["scales_view"] = _empty((case["rows"],), "f32")
    elif op == "linear":
        f["layer"] = nn.Linear(dev, case["fin"], case["fout"], activation=case["act"],
                               precision="e4m3")
        f["layer"].load_weights(s["weight"].cpu().numpy(), s["bias"].cpu().numpy())
        f["out"], f["out_view"] = _empty((case["rows"], case["fout"]), case["out"])
    elif op == "rotary":
        f["layer"] = nn.Rotary(dev, case["head_dim"], [int(a) for a in case["axes"].split(",")],
                               interleaved=case["interleaved"])
        f["q_out"], f["q_out_view"] = _empty(tuple(s["q"].shape), case["dtype"])
        f["k_out"], f["k_out_view"] = _empty(tuple(s["k"].shape), case["dtype"])
    else:
        f["layer"] = nn.WindowAttention(dev, case["heads"], case["head_dim"],
                                        num_kv_heads=case["kv_heads"], window_left=case["left"],
                                        window_right=case.get("right", 0), sinks=case["sinks"])
    for name in ("x", "residual", "scales", "q", "k", "v", "lengths", "out", "k_cache", "v_cache",
                 "weight", "wq"):
        s.pop(name, None)


def _own(s):
    case, op, f = s["case"], s["case"]["op"], s["own"]
    layer = f["layer"]
    if op == "norm":
        layer.forward_residual(f["x"], f["residual"], f["out"], sum=f["sum"], scales=f["scales"])
        got = {"sum": f["sum_view"], "out": f["out_view"]}
        return got if case["out"] == "same" else dict(got, scales=f["scales_view"])
    if op == "linear":
        layer.forward_scaled(f["x"], f["scales"], f["out"], residual=f["residual"])
        return f["out_view"]
    if op == "rotary":
        layer.forward(f["q"], f["k"], f["positions"], f["q_out"], f["k_out"])
        return {"q": f["q_out_view"], "k": f["k_out_view"]}
    if op == "window":
        layer.forward(f["q"], f["k"], f["v"], f["out"], lengths=f["lengths"])
        return f["out_view"]
    layer.step(f["q"], f["k"], f["v"], f["positions"], f["k_cache"], f["v_cache"], f["out"])
    return {"out": f["out_view"], "k_cache": f["k_cache_view"], "v_cache": f["v_cache_view"]}


# ----------------------------------------------------------------------------- work, and 64 bits
def _pairs(case):
    """(query, key) pairs of one head that see each other, and the keys read, over the batch."""
    pairs = keys = 0
    if case["op"] == "window":
        for n in _lengths(case) if case["ragged"] else [case["seq"]] * case["batch"]:
            i = torch.arange(n)
            lo, hi = (i - case["left"]).clamp_min(0), (i + case["right"]).clamp_max(n - 1)
            sinks = torch.minimum(lo, torch.tensor(case["sinks"]))
            pairs += int((hi - lo + 1 + sinks).sum())
            keys += n
    else:
        for p in _positions(case):
            for t in range(p, p + case["steps"]):
                lo = max(0, t - case["left"])
                pairs += t - lo + 1 + min(lo, case["sinks"])
            lo = max(0, p - case["left"])
            keys += p - lo + min(lo, case["sinks"])
    return pairs, keys


def work(case):
    op = case["op"]
    if op == "norm":
        n, f, e = case["rows"], case["features"], BYTES[case["dtype"]]
        o = e if case["out"] == "same" else 1
        return {"bytes": n * f * (e * (3 if case["residual"] else 2) + o) + 4 * f
                + (0 if case["out"] == "same" else 4 * n), "flops": 6.0 * n * f}
    if op == "linear":
        m, k, n, e = case["rows"], case["fin"], case["fout"], BYTES[case["out"]]
        return {"bytes": m * k * BYTES[case["input"]] + 4 * m + n * k + 8 * n
                + m * n * e * (2 if case["residual"] else 1), "flops": 2.0 * m * n * k}
    if op == "rotary":
        rows = case["batch"] * case["seq"] * (case["heads"] + case["kv_heads"])
        axes = len(case["axes"].split(","))
        return {"bytes": 2 * rows * case["head_dim"] * BYTES[case["dtype"]]
                + 4 * case["seq"] * axes, "flops": 3.0 * rows * case["head_dim"]}
    e, hd, h, kv = BYTES[case["dtype"]], case["head_dim"], case["heads"], case["kv_heads"]
    pairs, keys = _pairs(case)
    if op == "window":
        return {"bytes": e * hd * keys * (2 * h + 2 * kv), "flops": 4.0 * pairs * h * hd}
    new = case["batch"] * case["steps"]
    return {"bytes": e * hd * (new * (2 * h + 4 * kv) + keys * 2 * kv),
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
    return _round_e4m3(x * inv[:, None]), (top.double() / E4M3_MAX).float().double()


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    op = case["op"]
    if op == "norm":
        h = s["x"].double()
        if s["residual"] is not None:
            h = h + s["residual"].double()
        size = torch.linalg.vector_norm(h, dim=-1) / math.sqrt(case["features"])
        y = h / torch.sqrt(size * size + 1e-5)[:, None] * s["weight"].double()
        if case["out"] == "same":
            return {"sum": h, "out": y}
        scale = y.abs().max(-1).values.clamp_min(TINY) / E4M3_MAX
        return {"sum": h, "out": y / scale[:, None], "scales": scale}
    if op == "linear":
        w, ws = _levels(s["weight"])
        if s["scales"] is None:
            x, xs = _levels(s["x"].float())
        else:
            x, xs = s["x"].double(), s["scales"].double()
        y = (x * xs[:, None]) @ (w * ws[:, None]).T + s["bias"].double()
        if case["act"] == "gelu":
            y = y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
        elif case["act"] == "relu":
            y = torch.where(y > 0, y, torch.zeros_like(y))
        elif case["act"] == "swish":
            y = y * torch.sigmoid(y)
        return y if s["residual"] is None else y + s["residual"].double()
    if op == "rotary":
        return {n: _turned(case, s[n], s["positions"]) for n in ("q", "k")}
    if op == "window":
        lengths = _lengths(case) if case["ragged"] else [case["seq"]] * case["batch"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for b, n in enumerate(lengths):
            one = torch.ones(n, n, dtype=torch.bool, device="cuda")
            seen = one.triu(-case["left"])
            seen[:, :case["sinks"]] = True
            seen &= one.tril(case["right"])
            out[b, :n] = _exact_heads(case, s["q"][b, :n], s["k"][b, :n], s["v"][b, :n], seen)
        return out
    return _exact_step(case, s)


def _turned(case, x, positions):
    """Rotation as a product of complex numbers, one axis after the other."""
    y = x.double().reshape(case["batch"], case["seq"], -1, case["head_dim"]).clone()
    off = 0
    for a, d in enumerate(int(n) for n in case["axes"].split(",")):
        rate = torch.tensor([10000.0 ** (-2.0 * i / d) for i in range(d // 2)],
                            dtype=torch.float64, device="cuda")
        angle = torch.outer(positions[:, a].double(), rate)
        turn = torch.polar(torch.ones_like(angle), angle)[None, :, None, :]
        part = y[..., off:off + d]
        if case["interleaved"]:
            z = torch.view_as_complex(part.reshape(*part.shape[:-1], d // 2, 2).contiguous())
            y[..., off:off + d] = torch.view_as_real(z * turn).flatten(-2)
        else:
            z = torch.complex(part[..., :d // 2].contiguous(), part[..., d // 2:].contiguous())
            y[..., off:off + d] = torch.cat([(z * turn).real, (z * turn).imag], -1)
        off += d
    return y.reshape(x.shape)


def _exact_heads(case, q, k, v, seen):
    """One sequence, head by head: [T, H * hd] queries on [S, KV * hd] keys and values."""
    hd, group = case["head_dim"], case["heads"] // case["kv_heads"]
    cols = []
    for h in range(case["heads"]):
        at, to = h * hd, h // group * hd
        score = q[:, at:at + hd].double() @ k[:, to:to + hd].double().T / math.sqrt(hd)
        score = torch.where(seen, score, torch.full_like(score, -math.inf))
        cols.append(torch.softmax(score, -1) @ v[:, to:to + hd].double())
    return torch.cat(cols, -1)


def _exact_step(case, s):
    sinks, slots, left, t = case["sinks"], _slots(case), case["left"], case["steps"]
    ring = slots - sinks

    def slot(p):
        return p if p < sinks else sinks + (p - sinks) % ring

    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, p0 in enumerate(_positions(case)):
        first = max(0, p0 - left)
        old = list(range(min(sinks, first))) + list(range(first, p0))
        at = torch.tensor([slot(p) for p in old], dtype=torch.long, device="cuda")
        k = torch.cat([s["k_cache"][b, at], s["k"][b]])
        v = torch.cat([s["v_cache"][b, at], s["v"][b]])
        key = torch.tensor(old + list(range(p0, p0 + t)), device="cuda")[None, :]
        mine = torch.arange(p0, p0 + t, device="cuda")[:, None]
        seen = (key <= mine) & ((mine - key <= left) | (key < sinks))
        out[b] = _exact_heads(case, s["q"][b], k, v, seen)
    caches = {}
    for n in "kv":
        c = caches[n] = s[n + "_cache"].double()
        for b, p0 in enumerate(_positions(case)):
            for i in range(t):
                c[b, slot(p0 + i)] = s[n][b, i].double()
    return {"out": out, "k_cache": caches["k"], "v_cache": caches["v"]}
