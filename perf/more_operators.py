"""What a transformer's training step has between its projections and after its gradients, as cases that can be
timed and compared.

    attention    scaled dot products of heads that share keys and values, with the logarithm of each row's sum, and
                 the gradient, which makes the probabilities again from it
    rotary       positions as rotations of the heads' first dimensions, of queries and keys at once; its gradient is
                 the inverse rotation
    adamw        an optimiser's step over all tensors of a model, its states in 32 bits or in 8

With ``own`` false the operators are elementary torch operations, with ``own`` true the calls that a
program makes of ``raven_amd.nx_backend.Backend``, whose results go to tensors that the program keeps.
"""

from __future__ import annotations

import functools
import math

import numpy as np
import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
SIZES = {"bfloat16": 2, "float16": 2, "float32": 4}
BLOCK = 256  # elements of a scale of 8-bit states
BETA1, BETA2, EPS, DECAY = 0.9, 0.999, 1e-8, 0.1


# ── the cases ───────────────────────────────────────────────────────────────────────────────────

def listed():
    return [
        # The first steps of a character-level model: a short batch, eight heads that share two of keys and values.
        {"name": "attn_small", "op": "attention", "grad": False, "dtype": "float16", "batch": 2, "heads": 8, "kv_heads": 2,
         "queries": 100, "keys": 100, "dim": 32, "causal": True, "lengths": False, "mask": False},
        # GPT-2 small's attention over a training batch of 8 x 1024 tokens, forward and backward.
        {"name": "attn_batch", "op": "attention", "grad": False, "dtype": "bfloat16", "batch": 8, "heads": 12, "kv_heads": 12,
         "queries": 1024, "keys": 1024, "dim": 64, "causal": True, "lengths": False, "mask": False},
        {"name": "attn_batch_grad", "op": "attention", "grad": True, "dtype": "bfloat16", "batch": 8, "heads": 12, "kv_heads": 12,
         "queries": 1024, "keys": 1024, "dim": 64, "causal": True, "lengths": False, "mask": False},
        # One long document, four query heads to a head of keys and values.
        {"name": "attn_long", "op": "attention", "grad": False, "dtype": "bfloat16", "batch": 1, "heads": 16, "kv_heads": 4,
         "queries": 8192, "keys": 8192, "dim": 128, "causal": True, "lengths": False, "mask": False},
        {"name": "attn_long_grad", "op": "attention", "grad": True, "dtype": "bfloat16", "batch": 1, "heads": 16, "kv_heads": 4,
         "queries": 8192, "keys": 8192, "dim": 128, "causal": True, "lengths": False, "mask": False},
        # An encoder in float32 over sequences of different lengths, padded, with heads of an uncommon width.
        {"name": "attn_ragged_grad", "op": "attention", "grad": True, "dtype": "float32", "batch": 3, "heads": 6, "kv_heads": 6,
         "queries": 777, "keys": 777, "dim": 80, "causal": False, "lengths": True, "mask": True},
        # A decoding step of eight sequences at far positions.
        {"name": "rope_step", "op": "rotary", "dtype": "bfloat16", "batch": 8, "heads": 16, "kv_heads": 4, "length": 1, "dim": 128,
         "rotated": 128, "interleaved": False, "inverse": False, "scaled": 8.0, "far": 1000000},
        # Queries and keys of a training batch of 8 x 1024 tokens.
        {"name": "rope_batch", "op": "rotary", "dtype": "bfloat16", "batch": 8, "heads": 12, "kv_heads": 12, "length": 1024, "dim": 64,
         "rotated": 64, "interleaved": False, "inverse": False, "scaled": 1.0, "far": 0},
        # The gradient in float32, neighbours as pairs, a quarter of the head turned.
        {"name": "rope_partial_grad", "op": "rotary", "dtype": "float32", "batch": 3, "heads": 6, "kv_heads": 2, "length": 2777, "dim": 80,
         "rotated": 20, "interleaved": True, "inverse": True, "scaled": 1.0, "far": 0},
        # A small language model in float32: many tensors, little in each.
        {"name": "opt_small", "op": "adamw", "dtype": "float32", "masters": False, "bits": 32, "layers": 2, "width": 100, "vocab": 97, "positions": 64},
        # All 148 tensors of GPT-2 small in bfloat16, with float32 masters and states.
        {"name": "opt_model", "op": "adamw", "dtype": "bfloat16", "masters": True, "bits": 32, "layers": 12, "width": 768, "vocab": 50257, "positions": 1024},
        # The same with states of 8 bits.
        {"name": "opt_model_8bit", "op": "adamw", "dtype": "bfloat16", "masters": True, "bits": 8, "layers": 12, "width": 768, "vocab": 50257, "positions": 1024},
    ]


def _log(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "rotary", "adamw"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if op == "adamw":
        return {"op": op, "dtype": dtype, "masters": dtype != "float32" and rng.random() < 0.7, "bits": rng.choice([8, 32]),
                "layers": _log(rng, 1, 24), "width": _log(rng, 16, 768), "vocab": _log(rng, 2, 30000), "positions": _log(rng, 8, 2048)}
    dim = rng.choice([32, 40, 64, 64, 80, 96, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
    if op == "rotary":
        length = _log(rng, 1, 8192)
        return {"op": op, "dtype": dtype, "batch": _log(rng, 1, max(1, 65536 // (length * heads))), "heads": heads, "kv_heads": kv_heads,
                "length": length, "dim": dim, "rotated": rng.choice([dim, dim, dim // 2, dim // 4]), "interleaved": rng.random() < 0.5,
                "inverse": rng.random() < 0.5, "scaled": rng.choice([1.0, 4.0]), "far": rng.choice([0, 100000])}
    queries = _log(rng, 2, 4096)
    causal = rng.random() < 0.6
    keys = queries if rng.random() < 0.7 else queries + _log(rng, 1, 1000)
    batch = _log(rng, 1, max(1, min(16, (1 << 28) // (queries * keys * heads))))
    if dtype == "float32" and queries > 2048:
        dtype = "bfloat16"
    return {"op": op, "grad": rng.random() < 0.6, "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads, "queries": queries,
            "keys": keys, "dim": dim, "causal": causal, "lengths": rng.random() < 0.4, "mask": queries <= 1500 and rng.random() < 0.3}


def _shapes(c):
    """Shapes of a model's tensors: embeddings, for each layer two norms, attention and feed-forward, a last norm."""
    w = c["width"]
    layer = [(w,), (w,), (w, w), (w,), (w, w), (w,), (w, w), (w,), (w, w), (w,), (w,), (w,), (w, 4 * w), (4 * w,), (4 * w, w), (w,)]
    return [(c["vocab"], w), (c["positions"], w)] + layer * c["layers"] + [(w,), (w,)]


def work(case):
    c, e = case, SIZES[case["dtype"]]
    if c["op"] == "adamw":
        n = sum(math.prod(s) for s in _shapes(c))
        states = 16 if c["bits"] == 32 else 4 + 16 / BLOCK
        return {"bytes": n * (2 * e + (8 if c["masters"] else e) + states), "flops": 16 * n}
    if c["op"] == "rotary":
        size = c["batch"] * (c["heads"] + c["kv_heads"]) * c["length"] * c["dim"]
        return {"bytes": 2 * size * e + c["batch"] * c["length"] * 4 + c["rotated"] * 4, "flops": 3 * size * c["rotated"] // c["dim"]}
    b, h, hk, sq, sk, d = (c[k] for k in ("batch", "heads", "kv_heads", "queries", "keys", "dim"))
    seen = sk * 0.75 if c["lengths"] else sk  # (lengths lie between a half and the whole)
    pairs = sq * max(seen - sq / 2, seen / 2) if c["causal"] else sq * seen
    rows, cols = b * h * sq * d * e, b * hk * sk * d * e
    small = b * h * sq * 4 + (b * sq * sk if c["mask"] else 0)
    if c["grad"]:
        return {"bytes": 4 * rows + 4 * cols + small, "flops": int(10 * b * h * pairs * d)}
    return {"bytes": 2 * rows + 2 * cols + small, "flops": int(4 * b * h * pairs * d)}


# ── inputs ──────────────────────────────────────────────────────────────────────────────────────

class State:
    """What a program has in hand: inputs, the tensors that results go to, and the backend's handles of both."""

    def __init__(self, case, inputs, results):
        self.case, self.inputs, self.results = case, inputs, results
        self.handles = None


def _heads(c, g, heads, length, spread=1.0):
    """[batch, heads, length, dim] as a projection leaves it: the heads of a token side by side."""
    x = torch.randn(c["batch"], length, heads, c["dim"], generator=g, device="cuda") * spread
    return x.to(DTYPES[c["dtype"]]).transpose(1, 2)


def _seen(c, i):
    """Which keys each query sees, [batch or 1, 1, queries, keys] (or None for all)."""
    j = torch.arange(c["keys"], device="cuda")
    keep = None
    if c["causal"]:
        at = torch.arange(c["queries"], device="cuda")[:, None] + (c["keys"] - c["queries"])
        keep = (j <= at)[None, None]
    if c["lengths"]:
        inside = (j < i["lengths"][:, None])[:, None, None]
        keep = inside if keep is None else keep & inside
    if c["mask"]:
        keep = i["mask"][:, :1] if keep is None else keep & i["mask"][:, :1]
    return keep


def _attention_inputs(c, g):
    # queries and keys are alike enough that a row's probabilities gather on some keys
    i = {"q": _heads(c, g, c["heads"], c["queries"], 1.5), "k": _heads(c, g, c["kv_heads"], c["keys"]), "v": _heads(c, g, c["kv_heads"], c["keys"])}
    if c["lengths"]:
        i["lengths"] = torch.randint((c["keys"] + 1) // 2, c["keys"] + 1, (c["batch"],), generator=g, device="cuda").int()
    if c["mask"]:
        mask = torch.rand(c["batch"], 1, c["queries"], c["keys"], generator=g, device="cuda") < 0.9
        mask[..., 0] = True
        i["mask"] = mask.expand(-1, c["heads"], -1, -1)
    if c["grad"]:
        i["g"] = _heads(c, g, c["heads"], c["queries"])
        parts = [_plain_attention(c, {k: v[b:b + 1] for k, v in i.items()}) for b in range(c["batch"])]
        i["out"] = torch.cat([p["out"].transpose(1, 2) for p in parts]).transpose(1, 2)
        i["lse"] = torch.cat([p["lse"] for p in parts])
    return i


def _rotary_inputs(c, g):
    r = c["rotated"]
    index = torch.arange(r // 2, device="cuda", dtype=torch.float64)
    frequencies = 10000.0 ** (-2 * index / r)
    if c["scaled"] != 1.0:  # turns that a long context never completes are slowed down, fast ones stay as they are
        turns = 2048 * frequencies / (2 * math.pi)
        keep = ((turns - 1) / 31).clamp(0, 1)
        frequencies = frequencies * (keep + (1 - keep) / c["scaled"])
    i = {"q": _heads(c, g, c["heads"], c["length"]), "k": _heads(c, g, c["kv_heads"], c["length"]), "frequencies": frequencies}
    start = torch.randint(0, c["far"] + 1, (c["batch"], 1), generator=g, device="cuda")
    i["positions"] = (start + torch.arange(c["length"], device="cuda")).int()
    return i


def _adamw_inputs(c, g):
    dtype = DTYPES[c["dtype"]]
    sizes = [math.prod(s) for s in _shapes(c)]
    blocks = [-(-n // BLOCK) for n in sizes]
    flat = BLOCK * sum(blocks)
    # one block of memory for each kind of tensor; what lies between two tensors is zero and stays so
    real = torch.cat([torch.arange(BLOCK * b, device="cuda") < n for n, b in zip(sizes, blocks)])

    def noise(spread):
        return torch.where(real, torch.randn(flat, generator=g, device="cuda") * spread, 0)

    w = noise(0.02)
    # tokens differ in how often they occur, layers in how far their gradients have come
    loud = torch.exp(torch.randn(flat // BLOCK, generator=g, device="cuda") * 1.5).repeat_interleave(BLOCK)
    i = {"p": w.to(dtype), "g": (noise(1e-3) * loud).to(dtype)}
    if c["masters"]:
        i["w"] = w
    m, v = noise(3e-4) * loud, (noise(1e-3) * loud).square() + torch.where(real, (1e-4 * loud).square(), 0)
    if c["bits"] == 32:
        i["m"], i["v"] = m, v
    else:
        nearest = torch.full((flat,), 32768, device="cuda", dtype=torch.int32)  # (a half: to nearest)
        (i["m"], i["m_scales"]), (i["v"], i["v_scales"]) = _eight_bits(m, nearest, False), _eight_bits(v.sqrt(), nearest, True)
        i["key"] = torch.randint(-2**31, 2**31, (2,), generator=g, device="cuda").int()
    i["rate"] = torch.full((1,), 6e-4, device="cuda")
    i["step"] = torch.full((1,), 100, device="cuda", dtype=torch.int32)
    i["factor"] = torch.full((1,), 0.7, device="cuda")  # of the gradients: their norm is cut
    return i


def _inputs(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    return {"attention": _attention_inputs, "rotary": _rotary_inputs, "adamw": _adamw_inputs}[case["op"]](case, g)


def prepare(case, seed):
    i = _inputs(case, seed)

    def like(x):
        return torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device="cuda")

    results = {}
    if case["op"] == "attention" and case["grad"]:
        results = {"dq": like(i["q"]), "dk": like(i["k"]), "dv": like(i["v"])}
    elif case["op"] == "attention":
        results = {"out": like(i["q"]), "lse": torch.empty(i["q"].shape[:3], device="cuda")}
    elif case["op"] == "rotary":
        results = {"q_out": like(i["q"]), "k_out": like(i["k"])}
    torch.cuda.synchronize()
    return State(case, i, results)


# ── the operators in elementary operations ──────────────────────────────────────────────────────

def _shared(c, x):
    """Keys or values of each query head."""
    return x.float().repeat_interleave(c["heads"] // c["kv_heads"], 1)


def _scores(c, i):
    s = torch.matmul(i["q"].float(), _shared(c, i["k"]).transpose(2, 3)) * c["dim"] ** -0.5
    keep = _seen(c, i)
    return s if keep is None else torch.where(keep, s, -math.inf)


def _plain_attention(c, i):
    s = _scores(c, i)
    top = s.amax(3, keepdim=True)
    e = torch.exp(s - top)
    total = e.sum(3, keepdim=True)
    out = torch.matmul(e / total, _shared(c, i["v"]))
    lse = (top + torch.log(total))[..., 0]
    return {"out": out.transpose(1, 2).to(i["q"].dtype).contiguous().transpose(1, 2), "lse": lse}


def _plain_attention_grad(c, i):
    dtype, g = i["q"].dtype, i["g"].float()
    p = torch.exp(_scores(c, i) - i["lse"][..., None])
    dv = torch.matmul(p.transpose(2, 3), g)
    delta = (g * i["out"].float()).sum(3, keepdim=True)
    ds = p * (torch.matmul(g, _shared(c, i["v"]).transpose(2, 3)) - delta) * c["dim"] ** -0.5
    dq = torch.matmul(ds, _shared(c, i["k"]))
    dk = torch.matmul(ds.transpose(2, 3), i["q"].float())

    def joined(x):
        return x.unflatten(1, (c["kv_heads"], -1)).sum(2).to(dtype)

    return {"dq": dq.to(dtype), "dk": joined(dk), "dv": joined(dv)}


def _plain_rotary(c, i):
    r = c["rotated"]
    angle = i["positions"].double()[:, None, :, None] * i["frequencies"]
    cos, sin = angle.cos().float(), angle.sin().float() * (-1 if c["inverse"] else 1)

    def turned(x):
        head = x[..., :r].float()
        a, b = (head[..., 0::2], head[..., 1::2]) if c["interleaved"] else (head[..., :r // 2], head[..., r // 2:])
        a, b = a * cos - b * sin, a * sin + b * cos
        head = torch.stack((a, b), 4).flatten(3) if c["interleaved"] else torch.cat((a, b), 3)
        return torch.cat((head.to(x.dtype), x[..., r:]), 3)

    return {"q_out": turned(i["q"]), "k_out": turned(i["k"])}


_LOW = 0xFFFFFFFF
_TURNS = (13, 15, 26, 6, 17, 29, 16, 24)


def _round(words, r):
    """One of Threefry-2x32's twenty rounds on 32-bit words held in 64; the key goes in after every fourth."""
    x0, x1, ks = words
    x0 = (x0 + x1) & _LOW
    x1 = (((x1 << _TURNS[r % 8]) & _LOW) | (x1 >> (32 - _TURNS[r % 8]))) ^ x0
    if r % 4 == 3:
        s = r // 4 + 1
        x0, x1 = (x0 + ks[s % 3]) & _LOW, (x1 + ks[(s + 1) % 3] + s) & _LOW
    return x0, x1, ks


def _random_bits(key, n):
    """Sixteen bits for each of n elements: a block of the generator serves four."""
    k0, k1 = key[0].long() & _LOW, key[1].long() & _LOW
    block = torch.arange(-(-n // 4), device="cuda")
    words = ((block & _LOW) + k0) & _LOW, ((block >> 32) + k1) & _LOW, (k0, k1, 0x1BD11BDA ^ k0 ^ k1)
    x0, x1, _ = functools.reduce(_round, range(20), words)
    return torch.stack((x0 & 0xFFFF, x0 >> 16, x1 & 0xFFFF, x1 >> 16), 1).reshape(-1)[:n].int()


def _eight_bits(x, u, never_zero):
    """x in blocks, as e4m3 codes of up to 448 and a float32 scale for each block. u of 65536 decides which of its two
    neighbours an element becomes; with ``never_zero`` only zeros become zero."""
    x = x.reshape(-1, BLOCK)
    most = x.abs().amax(1, keepdim=True)
    inverse = torch.where(most >= 2.0 ** -100, 448 / most, 0)
    y = x.abs() * inverse
    low = y < 2.0 ** -6  # below there steps have one size: with 2^-6 more they are those of 2^-6
    bits = (torch.where(low, y + 2.0 ** -6, y)).view(torch.int32) + (u.reshape(-1, BLOCK) << 4)
    z = (bits & ~0xFFFFF).view(torch.float32)
    z = torch.where(low, z - 2.0 ** -6, z).clamp(max=448)
    if never_zero:
        z = torch.where(y > 0, z.clamp(min=2.0 ** -9), z)
    codes = torch.copysign(z, x).to(torch.float8_e4m3fn).reshape(-1)
    return codes, torch.where(most >= 2.0 ** -100, most * (1 / 448), 0)[:, 0]


def _plain_adamw(c, i):
    """The step over all tensors at once: between two of them everything is zero."""
    g = i["g"].float() * i["factor"]
    if c["bits"] == 32:
        m, v = i["m"], i["v"]
    else:
        m = (i["m"].float().reshape(-1, BLOCK) * i["m_scales"][:, None]).reshape(-1)
        v = (i["v"].float().reshape(-1, BLOCK) * i["v_scales"][:, None]).reshape(-1).square()
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + g * g * (1 - BETA2)
    step, rate = i["step"].double(), i["rate"].double()
    size, shrink = (rate / (1 - BETA1 ** step)).float(), (1 - rate * DECAY).float()
    root = (1 / torch.sqrt(1 - BETA2 ** step)).float()
    w = i["w"] if c["masters"] else i["p"].float()
    w = w * shrink - m / (v.sqrt() * root + EPS) * size
    i["p"].copy_(w)
    if c["masters"]:
        i["w"].copy_(w)
    if c["bits"] == 32:
        i["m"].copy_(m)
        i["v"].copy_(v)
    else:
        u = _random_bits(i["key"], g.numel())
        i["m"], i["m_scales"] = _eight_bits(m, u, False)
        i["v"], i["v_scales"] = _eight_bits(v.sqrt(), (u << 8 | u >> 8) & 0xFFFF, True)
    return {k: i[k] for k in ("p", "w", "m", "v", "m_scales", "v_scales") if k in i}


def _plain(state):
    c, i = state.case, state.inputs
    if c["op"] == "attention":
        return _plain_attention_grad(c, i) if c["grad"] else _plain_attention(c, i)
    return _plain_rotary(c, i) if c["op"] == "rotary" else _plain_adamw(c, i)


# ── the framework's calls ───────────────────────────────────────────────────────────────────────

class _Storage:
    """Device memory of a torch tensor, as the backend's handles hold it."""

    def __init__(self, x):
        self.tensor, self.ptr = x, x.data_ptr()
        self.nbytes = x.untyped_storage().nbytes() - x.storage_offset() * x.element_size()


@functools.lru_cache(maxsize=1)
def _backend():
    """A program has one context."""
    from raven_amd.nx_backend import Backend

    return Backend()


def _handle(x):
    from raven_amd import dtype as dt
    from raven_amd.nx_backend import Tensor
    from raven_amd.view import View

    name = {torch.float8_e4m3fn: "float8_e4m3"}.get(x.dtype, str(x.dtype).removeprefix("torch."))
    return Tensor(_Storage(x), View.create(x.shape, x.stride()), dt.BY_NAME[name], _backend())


def _handles(state):
    """The handles of a state's tensors: its program makes them once, no data is touched."""
    c, tensors = state.case, state.inputs | state.results
    if c["op"] != "adamw":
        return {name: _handle(x) for name, x in tensors.items()}
    made, start = {name: [] if x.numel() > 2 else _handle(x) for name, x in tensors.items()}, 0
    for shape in _shapes(c):
        n = math.prod(shape)
        blocks = -(-n // BLOCK)
        for name, x in tensors.items():
            if x.numel() > 2:
                part = x[start // BLOCK:start // BLOCK + blocks] if name.endswith("scales") else x[start:start + n].view(shape)
                made[name].append(_handle(part))
        start += blocks * BLOCK
    return made


def _run_own(state):
    if state.handles is None:
        state.handles = _handles(state)
    c, h, B = state.case, state.handles, _backend()
    if c["op"] == "attention":
        scale = c["dim"] ** -0.5
        if c["grad"]:
            B.attention_grad(h["g"], h["q"], h["k"], h["v"], h["out"], h["lse"], scale, c["causal"], h.get("lengths"), h.get("mask"),
                             out=(h["dq"], h["dk"], h["dv"]))
        else:
            B.attention_train(h["q"], h["k"], h["v"], scale, c["causal"], h.get("lengths"), h.get("mask"), out=(h["out"], h["lse"]))
        return state.results
    if c["op"] == "rotary":
        B.rotary(h["q"], h["k"], h["positions"], h["frequencies"], interleaved=c["interleaved"], inverse=c["inverse"],
                 out=(h["q_out"], h["k_out"]))
        return state.results
    B.adamw(h["p"], h["g"], h["m"], h["v"], h["rate"], h["step"], beta1=BETA1, beta2=BETA2, eps=EPS, decay=DECAY, factor=h["factor"],
            masters=h.get("w"), m_scales=h.get("m_scales"), v_scales=h.get("v_scales"), key=h.get("key"))
    return {k: state.inputs[k] for k in ("p", "w", "m", "v", "m_scales", "v_scales") if k in state.inputs}


def run(state):
    return _run_own(state) if own else _plain(state)


# ── the operators in 64 bits ────────────────────────────────────────────────────────────────────

def _exact_attention(c, i):
    """A head at a time, from the definition."""
    names = ("dq", "dk", "dv") if c["grad"] else ("out", "lse")
    like = {"dq": "q", "dk": "k", "dv": "v", "out": "q"}
    out = {n: torch.zeros(i[like[n]].shape if n in like else i["q"].shape[:3], dtype=torch.float64, device="cuda") for n in names}
    span = torch.arange(c["keys"], device="cuda")
    for b in range(c["batch"]):
        hidden = torch.zeros(c["queries"], c["keys"], dtype=torch.bool, device="cuda")
        if c["causal"]:
            hidden |= span[None] - torch.arange(c["queries"], device="cuda")[:, None] > c["keys"] - c["queries"]
        if c["lengths"]:
            hidden |= span >= i["lengths"][b]
        if c["mask"]:
            hidden |= ~i["mask"][b, 0]
        for h in range(c["heads"]):
            kv = h * c["kv_heads"] // c["heads"]
            q, k, v = i["q"][b, h].double(), i["k"][b, kv].double(), i["v"][b, kv].double()
            s = (q @ k.T).div_(math.sqrt(c["dim"])).masked_fill_(hidden, -math.inf)
            if not c["grad"]:
                out["lse"][b, h] = torch.logsumexp(s, 1)
                out["out"][b, h] = torch.softmax(s, 1) @ v
                continue
            g = i["g"][b, h].double()
            p = s.sub_(i["lse"][b, h].double()[:, None]).exp_()
            out["dv"][b, kv] += p.T @ g
            p *= (g @ v.T).sub_((g * i["out"][b, h].double()).sum(1, keepdim=True))
            p /= math.sqrt(c["dim"])
            out["dq"][b, h] = p @ k
            out["dk"][b, kv] += p.T @ q
    return out


def _exact_rotary(c, i):
    """Pairs as complex numbers, which are multiplied by one of length 1."""
    r = c["rotated"]
    angle = torch.outer(i["positions"].reshape(-1).double(), i["frequencies"]).reshape(c["batch"], 1, c["length"], r // 2)
    turn = torch.polar(torch.ones_like(angle), -angle if c["inverse"] else angle)
    out = {}
    for name in ("q", "k"):
        y = i[name].double().contiguous()
        if c["interleaved"]:
            pairs = torch.view_as_complex(y[..., :r].unflatten(3, (r // 2, 2)).contiguous()) * turn
            y[..., 0:r:2], y[..., 1:r:2] = pairs.real, pairs.imag
        else:
            pairs = torch.complex(y[..., :r // 2], y[..., r // 2:r]) * turn
            y[..., :r // 2], y[..., r // 2:r] = pairs.real, pairs.imag
        out[name + "_out"] = y
    return out


def _exact_adamw(c, i):
    g = i["g"].double() * i["factor"].double()
    if c["bits"] == 32:
        m, v = i["m"].double(), i["v"].double()
    else:
        m = i["m"].double() * i["m_scales"].double().repeat_interleave(BLOCK)
        v = (i["v"].double() * i["v_scales"].double().repeat_interleave(BLOCK)) ** 2
    m = torch.lerp(g, m, BETA1)
    v = torch.lerp(g ** 2, v, BETA2)
    t, rate = int(i["step"]), float(i["rate"])
    w = i["w" if c["masters"] else "p"].double()
    w = w - rate * (DECAY * w + (m / (1 - BETA1 ** t)) / (torch.sqrt(v / (1 - BETA2 ** t)) + EPS))
    out = {"p": w}
    if c["masters"]:
        out["w"] = w
    if c["bits"] == 32:
        return out | {"m": m, "v": v}
    # what a code becomes goes by a random number and by the last bit of what is rounded: it has no value in 64 bits
    return out | {"m": None, "v": None, "m_scales": m.abs().reshape(-1, BLOCK).amax(1) / 448,
                  "v_scales": v.sqrt().reshape(-1, BLOCK).amax(1) / 448}


def exact(case, seed):
    i = _inputs(case, seed)
    return {"attention": _exact_attention, "rotary": _exact_rotary, "adamw": _exact_adamw}[case["op"]](case, i)
