"""The operators of transformer layers as cases that can be timed and compared: what stands around attention and the plain
linear layers in a training step, in a prompt's pass and in a pass over single tokens.

  qkv      norms of queries and keys for each head with the rotation of positions, from the joint projection of queries, keys
           and values (jt.nn.qkv_norm_rope)
  gated    both projections of a gated feed-forward layer, its activation and the product (jt.nn.gated_linear)
  dropout  dropout from a counter-based generator, with the residual added (jt.nn.dropout)

A case is a dict: "kind" names the operator, "train" says whether the gradients belong to the pass, the other entries are
sizes, the data type and options.  Where `own` is false a pass computes the operator in elementary torch operations in 32 bits;
where it is true it goes through the front end (jittor_amd), whose results are handed out as torch tensors that look at the
Vars' device buffers (no copy, no wait).
"""
import math

import numpy as np
import torch

own = False

_TORCH = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16, "int32": torch.int32}
_TYPESTR = {"float32": "<f4", "float16": "<f2", "bfloat16": "<i2", "int32": "<i4"}
_BYTES = {"float32": 4, "float16": 2, "bfloat16": 2}


# ---- the listed cases ---------------------------------------------------------------------------------------------
def listed():
    return [
        # one new token for each of four sequences, somewhere in a long context: latency
        {"name": "qkv_tokens", "kind": "qkv", "train": False, "batch": 4, "seq": 1, "heads": 32, "kv": 8, "dim": 128, "rot": 128, "axes": 1, "paired": False, "first": True,
         "table": 32768, "dtype": "bfloat16"},
        # a prompt's pass: two sequences of 4096 tokens with grouped heads, written head by head as the attention products read them
        {"name": "qkv_prompt", "kind": "qkv", "train": False, "batch": 2, "seq": 4096, "heads": 32, "kv": 8, "dim": 128, "rot": 128, "axes": 1, "paired": False, "first": True,
         "table": 8192, "dtype": "bfloat16"},
        # a training step in the framework's default type: a small model's heads of 64, as many keys as queries
        {"name": "qkv_train_f32", "kind": "qkv", "train": True, "batch": 8, "seq": 512, "heads": 16, "kv": 16, "dim": 64, "rot": 64, "axes": 1, "paired": False, "first": False,
         "table": 512, "dtype": "float32"},
        # a training step over video: positions in time, height and width, heads of 80, an odd number of patches, adjacent pairs
        {"name": "qkv_train_axes", "kind": "qkv", "train": True, "batch": 1, "seq": 9477, "heads": 16, "kv": 4, "dim": 80, "rot": 80, "axes": 3, "paired": True, "first": True,
         "table": 128, "dtype": "bfloat16"},
        # one token through a feed-forward layer: the weights are read once and nothing else counts
        {"name": "gated_token", "kind": "gated", "train": False, "rows": 1, "k": 4096, "f": 11264, "act": "silu", "dtype": "bfloat16"},
        # one token for each of 24 sequences through a smaller one, float16
        {"name": "gated_tokens", "kind": "gated", "train": False, "rows": 24, "k": 2048, "f": 5632, "act": "gelu", "dtype": "float16"},
        # a prompt of an odd length through a layer whose sizes are no multiples of a tile
        {"name": "gated_prompt_odd", "kind": "gated", "train": False, "rows": 777, "k": 1000, "f": 2600, "act": "silu", "dtype": "bfloat16"},
        # a training step of a large layer: the forward product and both of its gradients
        {"name": "gated_train", "kind": "gated", "train": True, "rows": 8192, "k": 2048, "f": 5632, "act": "silu", "dtype": "bfloat16"},
        # a training step of a small layer in the framework's default type
        {"name": "gated_train_f32", "kind": "gated", "train": True, "rows": 1024, "k": 512, "f": 1376, "act": "silu", "dtype": "float32"},
        # dropout and its gradient in a small network, float32: latency
        {"name": "dropout_small", "kind": "dropout", "train": True, "shape": "32,256", "p": 0.5, "residual": False, "dtype": "float32"},
        # behind a block of a large layer, with the residual: 8192 tokens of 4096
        {"name": "dropout_residual", "kind": "dropout", "train": True, "shape": "4,2048,4096", "p": 0.1, "residual": True, "dtype": "bfloat16"},
        # attention weights of a short odd sequence: rows that are no whole vectors
        {"name": "dropout_odd", "kind": "dropout", "train": True, "shape": "12,317,317", "p": 0.2, "residual": False, "dtype": "float16"},
    ]


# ---- other cases of the same ranges -------------------------------------------------------------------------------
def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _extent(rng, lo, hi):
    """Half of them round numbers, as models have them, the others any."""
    n = _log(rng, lo, hi)
    return max(lo, n // 64 * 64) if n >= 64 and rng.random() < 0.6 else n


def draw(rng):
    kind = rng.choice(["qkv", "qkv", "gated", "gated", "gated", "dropout"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if kind == "qkv":
        while True:
            kv = rng.choice([1, 2, 4, 8, rng.randint(1, 16)])
            dim = rng.choice([64, 128, 128, 80, 96, 256, 2 * rng.randint(8, 128)])
            c = {"kind": kind, "train": rng.random() < 0.5, "batch": _log(rng, 1, 64), "seq": 1 if rng.random() < 0.3 else _log(rng, 1, 16384), "heads": kv * rng.choice([1, 2, 4, 8]), "kv": kv,
                 "dim": dim, "rot": dim if rng.random() < 0.7 else max(2, dim // 4 * 2), "axes": rng.choice([1, 1, 3]), "paired": rng.random() < 0.4, "first": rng.random() < 0.5, "dtype": dtype}
            c["table"] = max(c["seq"], _log(rng, 64, 32768))
            n = c["batch"] * c["seq"] * (c["heads"] + 2 * kv) * dim
            if c["rot"] >= 2 * c["axes"] and n * (3 if c["train"] else 1) <= 50000000:
                return c
    if kind == "gated":
        while True:
            c = {"kind": kind, "train": rng.random() < 0.5, "rows": _log(rng, 1, 8192), "k": _extent(rng, 32, 4096), "f": _extent(rng, 32, 11264),
                 "act": rng.choice(["silu", "silu", "gelu", "relu", "sigmoid"]), "dtype": dtype}
            flops = 4.0 * c["rows"] * c["k"] * c["f"] * (3 if c["train"] else 1)
            if flops <= (1.0e12 if dtype != "float32" else 4e10):
                return c
    while True:
        shape = [_log(rng, 1, 64), _log(rng, 1, 4096), _log(rng, 1, 8192)]
        if 256 <= shape[0] * shape[1] * shape[2] <= 33600000:
            return {"kind": kind, "train": rng.random() < 0.7, "shape": ",".join(str(s) for s in shape), "p": rng.choice([0.0, 0.1, 0.1, 0.25, 0.5, round(rng.random(), 3)]),
                    "residual": rng.random() < 0.5, "dtype": dtype}


# ---- inputs -------------------------------------------------------------------------------------------------------
def _hold(t, dtype):
    """What the user's program keeps: the tensor, or the Var with its values (bfloat16 travels as its bits)."""
    t = t.to(_TORCH[dtype]).contiguous()
    if not own:
        return t
    import jittor_amd as jt
    host = t.view(torch.int16).cpu().numpy().view("uint16") if dtype == "bfloat16" else t.cpu().numpy()
    return jt.from_storage(host, dtype)


def _sections(c):
    """Rotated pairs of each axis: one part for time, the rest shared by height and width; all of them where there is one axis."""
    pairs = c["rot"] // 2
    if c["axes"] == 1:
        return [pairs]
    t = max(1, pairs // 5)
    h = (pairs - t + 1) // 2
    return [t, h, pairs - t - h]


def _angles(c):
    """[table, pairs] in 64 bits."""
    pairs = c["rot"] // 2
    freq = 10000.0 ** (-torch.arange(pairs, dtype=torch.float64, device="cuda") / pairs)
    return torch.arange(c["table"], dtype=torch.float64, device="cuda")[:, None] * freq


def _shape(c):
    return [int(s) for s in c["shape"].split(",")]


def _made(c, seed):
    """The inputs as torch tensors, in 32 bits, and their types."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))

    def normal(*shape, scale=1.0, shift=0.0):
        return torch.randn(shape, generator=g, device="cuda") * scale + shift

    made = {}
    if c["kind"] == "qkv":
        b, s, hq, hk, d = c["batch"], c["seq"], c["heads"], c["kv"], c["dim"]
        made["x"] = normal(b, s, hq + 2 * hk, d, scale=1.3)
        made["sq"], made["sk"] = normal(d, scale=0.2, shift=1.0), normal(d, scale=0.2, shift=1.0)
        a = _angles(c)
        made["table"] = torch.stack([a.cos(), a.sin()], -1).to(torch.float32)
        if c["axes"] == 1:                                  # each sequence continues somewhere in the table
            at = torch.randint(0, c["table"] - s + 1, [b, 1], generator=g, device="cuda")
            made["positions"] = at + torch.arange(s, device="cuda")
        else:
            made["positions"] = torch.randint(0, c["table"], [c["axes"], b, s], generator=g, device="cuda")
        if c["train"]:
            for name, h in (("gq", hq), ("gk", hk), ("gv", hk)):
                made[name] = normal(*([b, h, s, d] if c["first"] else [b, s, h, d]))
    elif c["kind"] == "gated":
        made["x"] = normal(c["rows"], c["k"])
        made["w"] = normal(2 * c["f"], c["k"], scale=math.sqrt(1.0 / c["k"]))
        if c["train"]:
            made["g"] = normal(c["rows"], c["f"])
    elif c["kind"] == "dropout":
        made["x"] = normal(*_shape(c))
        if c["residual"]:
            made["res"] = normal(*_shape(c))
        if c["train"]:
            made["g"] = normal(*_shape(c))
    else:
        raise ValueError("unknown kind %r" % c["kind"])
    # the table stays in 32 bits, as programs keep it
    return {k: (t, "float32" if k == "table" else "int32" if k == "positions" else c["dtype"]) for k, t in made.items()}


def _key(seed):
    """The generator's key and the call's number: 64 bits each."""
    r = np.random.RandomState(int(seed) % (1 << 32))
    return int(r.randint(0, 1 << 62, dtype=np.int64)), int(r.randint(0, 1 << 40, dtype=np.int64))


def prepare(case, seed):
    c = dict(case)
    held = {k: _hold(t, dtype) for k, (t, dtype) in _made(c, seed).items()}
    if own:
        import jittor_amd as jt
        jt.sync(list(held.values()))                        # uploads them
    elif c["kind"] == "qkv":
        held["axis"] = torch.repeat_interleave(torch.arange(c["axes"], device="cuda"), torch.tensor(_sections(c), device="cuda"))
    return {"case": c, "in": held, "key": _key(seed)}


# ---- one pass: the framework's calls ------------------------------------------------------------------------------
class _Device:
    """A computed Var's device buffer under the array interface that torch takes; keeps the Var alive."""

    def __init__(self, v):
        self.v = v
        self.__cuda_array_interface__ = {"shape": tuple(v.shape), "typestr": _TYPESTR[v.dtype], "data": (v.raw_ptr(), False), "strides": None, "version": 2}


def _out(v):
    t = torch.as_tensor(_Device(v), device="cuda")
    return t.view(torch.bfloat16) if v.dtype == "bfloat16" else t


def _run_own(c, v, key):
    import jittor_amd as jt
    nn = jt.nn
    if c["kind"] == "qkv":
        q, k, val = nn.qkv_norm_rope(v["x"], c["heads"], c["kv"], v["sq"], v["sk"], v["table"], v["positions"], sections=_sections(c) if c["axes"] > 1 else None,
                                     interleaved=c["paired"], heads_first=c["first"])
        outs = {"q": q, "k": k, "v": val}
        if c["train"]:
            loss = (q * v["gq"]).sum() + (k * v["gk"]).sum() + (val * v["gv"]).sum()
            outs.update(zip(("dx", "dsq", "dsk"), jt.grad(loss, [v["x"], v["sq"], v["sk"]])))
    elif c["kind"] == "gated":
        outs = {"y": nn.gated_linear(v["x"], v["w"], c["act"])}
        if c["train"]:
            outs.update(zip(("dx", "dw"), jt.grad((outs["y"] * v["g"]).sum(), [v["x"], v["w"]])))
    else:
        outs = {"y": nn.dropout(v["x"], c["p"], True, seed=key[0], offset=key[1], residual=v.get("res"))}
        if c["train"]:
            outs["dx"] = jt.grad((outs["y"] * v["g"]).sum(), v["x"])
    jt.sync(list(outs.values()))
    return {k: _out(o) for k, o in outs.items()}


# ---- one pass: the plain form -------------------------------------------------------------------------------------
def _rotate(z, cos, sin, rot, paired):
    """Pairs (a, b) of the first `rot` elements turned: (a cos - b sin, a sin + b cos)."""
    half = rot // 2
    a, b = (z[..., 0:rot:2], z[..., 1:rot:2]) if paired else (z[..., :half], z[..., half:rot])
    y = torch.empty_like(z)
    y[..., rot:] = z[..., rot:]
    if paired:
        y[..., 0:rot:2], y[..., 1:rot:2] = a * cos - b * sin, a * sin + b * cos
    else:
        y[..., :half], y[..., half:rot] = a * cos - b * sin, a * sin + b * cos
    return y


def _qkv_plain(c, v):
    hq, hk, first, rot = c["heads"], c["kv"], c["first"], c["rot"]
    x = v["x"].float()
    pairs = torch.arange(rot // 2, device="cuda")
    if c["axes"] == 1:
        t = v["table"][v["positions"]]                      # [batch, seq, pairs, 2]
    else:
        t = v["table"][v["positions"].permute(1, 2, 0)[:, :, v["axis"]], pairs]
    cos, sin = t[..., 0].unsqueeze(2), t[..., 1].unsqueeze(2)

    def whole(y):
        return (y.transpose(1, 2) if first else y).to(v["x"].dtype).contiguous()

    def normed(part, scale):
        r = torch.rsqrt((part * part).mean(-1, keepdim=True) + 1e-6)
        return part * r, r, scale.float()

    nq, rq, sq = normed(x[:, :, :hq], v["sq"])
    nk, rk, sk = normed(x[:, :, hq:hq + hk], v["sk"])
    outs = {"q": whole(_rotate(nq * sq, cos, sin, rot, c["paired"])), "k": whole(_rotate(nk * sk, cos, sin, rot, c["paired"])), "v": whole(v["x"][:, :, hq + hk:])}
    if c["train"]:
        def back(g, n, r, scale):
            g = g.float()
            dz = _rotate(g.transpose(1, 2) if first else g, cos, -sin, rot, c["paired"])
            dn = dz * scale
            return (dn - n * (dn * n).mean(-1, keepdim=True)) * r, (dz * n).sum((0, 1, 2)).to(v["x"].dtype)

        dq, dsq = back(v["gq"], nq, rq, sq)
        dk, dsk = back(v["gk"], nk, rk, sk)
        dv = v["gv"].float()
        outs.update(dx=torch.cat([dq, dk, dv.transpose(1, 2) if first else dv], 2).to(v["x"].dtype), dsq=dsq, dsk=dsk)
    return outs


def _act_plain(name, g):
    """The activation and its derivative."""
    if name == "relu":
        on = (g > 0).float()
        return g * on, on
    if name == "gelu":                                      # g times the normal distribution's mass below g
        below = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * below, below + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    s = 1.0 / (1.0 + torch.exp(-g))
    return (s, s * (1.0 - s)) if name == "sigmoid" else (g * s, s * (1.0 + g * (1.0 - s)))


def _gated_plain(c, v):
    x, w, f, dtype = v["x"].float(), v["w"].float(), c["f"], v["x"].dtype
    both = x @ w.t()
    gate, up = both[:, :f], both[:, f:]
    a, da = _act_plain(c["act"], gate)
    outs = {"y": (a * up).to(dtype)}
    if c["train"]:
        dh = v["g"].float()
        d = torch.cat([dh * up * da, dh * a], 1)
        outs.update(dx=(d @ w).to(dtype), dw=(d.t() @ x).to(dtype))
    return outs


_M0, _M1, _W0, _W1, _LOW = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85, 0xFFFFFFFF


def _philox_plain(group, block, key, call):
    """Philox4x32-10 (Salmon, Moraes, Dror and Shaw, 2011) of counters (group, block, call): four words of 32 bits in int64."""
    c0, c1 = group & _LOW, (group >> 32) | (block << 31)
    c2, c3 = torch.full_like(group, call & _LOW), torch.full_like(group, call >> 32)
    k0, k1 = key & _LOW, key >> 32
    for _ in range(10):
        p0, p1 = c0 * _M0, c2 * _M1                         # products of 64 bits, wrapped into the sign
        c0, c1, c2, c3 = ((p1 >> 32) & _LOW) ^ c1 ^ k0, p1 & _LOW, ((p0 >> 32) & _LOW) ^ c3 ^ k1, p0 & _LOW
        k0, k1 = (k0 + _W0) & _LOW, (k1 + _W1) & _LOW
    return torch.stack([c0, c1, c2, c3], 1)


def _halves_plain(words):
    """The eight halves of 16 bits of each group of four words, the lower of a word first."""
    return torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)


def _dropout_plain(c, v, key):
    x = v["x"]
    n = x.numel()
    group = torch.arange((n + 7) // 8, device="cuda")
    u = _halves_plain(_philox_plain(group, 0, *key)) << 16 | _halves_plain(_philox_plain(group, 1, *key))
    keep = (u[:n] >= round(c["p"] * (1 << 32))).view(x.shape)
    scale = 1.0 / (1.0 - c["p"]) if c["p"] < 1.0 else 0.0
    zero = torch.zeros((), device="cuda")

    def kept(t):
        return torch.where(keep, t.float() * scale, zero)

    y = kept(x)
    outs = {"y": (y + v["res"].float() if c["residual"] else y).to(x.dtype)}
    if c["train"]:
        outs["dx"] = kept(v["g"]).to(x.dtype)
    return outs


def run(state):
    c, v = state["case"], state["in"]
    if own:
        return _run_own(c, v, state["key"])
    if c["kind"] == "qkv":
        return _qkv_plain(c, v)
    return _gated_plain(c, v) if c["kind"] == "gated" else _dropout_plain(c, v, state["key"])


# ---- what a pass cannot do without --------------------------------------------------------------------------------
def work(case):
    """Bytes: every operand read once and every result written once (of the table the rows in use).  Flops: multiply-adds of
    products counted twice; a handful per element for the others."""
    c = dict(case)
    e = _BYTES[c["dtype"]]
    if c["kind"] == "qkv":
        tokens, d = c["batch"] * c["seq"], c["dim"]
        n = tokens * (c["heads"] + 2 * c["kv"]) * d
        small = 4.0 * tokens * c["axes"] + 4.0 * min(tokens, c["table"]) * c["rot"] + 2 * e * d
        return {"bytes": 2.0 * e * n + small + (2.0 * e * n + 2 * e * d if c["train"] else 0.0), "flops": (30.0 if c["train"] else 10.0) * n}
    if c["kind"] == "gated":
        x, w, y = c["rows"] * c["k"], 2 * c["f"] * c["k"], c["rows"] * c["f"]
        return {"bytes": float(e * ((x + w + y) * (2 if c["train"] else 1))), "flops": 4.0 * c["rows"] * c["k"] * c["f"] * (3 if c["train"] else 1)}
    n = math.prod(_shape(c))
    return {"bytes": float(e * n * (2 + (1 if c["residual"] else 0) + (2 if c["train"] else 0))), "flops": 40.0 * n}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------
def _qkv_exact(c, m):
    """Rotations as products of complex numbers, gradients by automatic differentiation."""
    x, sq, sk = (m[k].clone().requires_grad_(c["train"]) for k in ("x", "sq", "sk"))
    hq, hk, half = c["heads"], c["kv"], c["rot"] // 2
    turn = torch.view_as_complex(m["table"])                # the table is an input: its values of 32 bits are what they are
    positions = m["positions"].long().reshape(c["axes"], c["batch"], c["seq"])
    parts, at = [], 0
    for axis, count in enumerate(_sections(c)):
        parts.append(turn[positions[axis], at:at + count])
        at += count
    turn = torch.cat(parts, -1).unsqueeze(2)

    def head(z, scale):
        z = z / (z.pow(2).sum(-1, keepdim=True) / c["dim"] + 1e-6).sqrt() * scale
        first, rest = z[..., :c["rot"]], z[..., c["rot"]:]
        pairs = first.unflatten(-1, (half, 2)) if c["paired"] else first.unflatten(-1, (2, half)).transpose(-1, -2)
        y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        return torch.cat([(y if c["paired"] else y.transpose(-1, -2)).flatten(-2), rest], -1)

    outs = {"q": head(x[:, :, :hq], sq), "k": head(x[:, :, hq:hq + hk], sk), "v": x[:, :, hq + hk:]}
    if c["first"]:
        outs = {k: o.transpose(1, 2) for k, o in outs.items()}
    if c["train"]:
        grads = torch.autograd.grad([outs[k] for k in "qkv"], [x, sq, sk], [m["g" + k] for k in "qkv"])
        outs.update(zip(("dx", "dsq", "dsk"), grads))
    return outs


def _gated_exact(c, m):
    x, w = (m[k].clone().requires_grad_(c["train"]) for k in ("x", "w"))
    act = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu, "sigmoid": torch.sigmoid}[c["act"]]
    y = act(x @ w[:c["f"]].t()) * (x @ w[c["f"]:].t())
    return dict({"y": y}, **(dict(zip(("dx", "dw"), torch.autograd.grad(y, [x, w], m["g"]))) if c["train"] else {}))


def _words_exact(n, key, call):
    """The numbers of elements 0 .. n - 1, worked out on the host in unsigned integers."""
    group = np.arange((n + 7) // 8, dtype=np.uint64)
    low, shift = np.uint64(_LOW), np.uint64(32)
    u = np.zeros(8 * group.size, np.uint64)
    for block in (0, 1):
        ctr = [group & low, (group >> shift) + np.uint64(block << 31), np.full_like(group, call & _LOW), np.full_like(group, call >> 32)]
        k = [key & _LOW, key >> 32]
        for _ in range(10):
            a, b = ctr[0] * np.uint64(_M0), ctr[2] * np.uint64(_M1)
            ctr = [(b >> shift) ^ ctr[1] ^ np.uint64(k[0]), b & low, (a >> shift) ^ ctr[3] ^ np.uint64(k[1]), a & low]
            k = [(k[0] + _W0) & _LOW, (k[1] + _W1) & _LOW]
        halves = np.stack([part for word in ctr for part in (word & np.uint64(0xFFFF), word >> np.uint64(16))], 1).reshape(-1)
        u = u * np.uint64(1 << 16) + halves
    return u[:n]


def _dropout_exact(c, m, key):
    keep = torch.from_numpy(_words_exact(math.prod(_shape(c)), *key) >= np.uint64(round(c["p"] * (1 << 32)))).cuda().view(_shape(c)).double()
    factor = keep / (1.0 - c["p"]) if c["p"] < 1.0 else keep * 0.0
    outs = {"y": m["x"] * factor + (m["res"] if c["residual"] else 0.0)}
    if c["train"]:
        outs["dx"] = m["g"] * factor
    return outs


def exact(case, seed):
    c = dict(case)
    m = {k: t.to(_TORCH[dtype]).double() for k, (t, dtype) in _made(c, seed).items()}
    outs = _qkv_exact(c, m) if c["kind"] == "qkv" else _gated_exact(c, m) if c["kind"] == "gated" else _dropout_exact(c, m, _key(seed))
    return {k: o.detach().contiguous() for k, o in outs.items()}
