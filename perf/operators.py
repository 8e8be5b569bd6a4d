"""The transformer operators that a program calls by name, as cases that can be timed and compared.

A case is one program of one operator (for training: attention and its gradient, as a step runs them), compiled through
`Client.compile` and run through `LoadedExecutable.execute` on arguments that are resident on the GPU.  Where `own` is
false the same results are computed from their definition with elementary torch operations in 32 bits.
"""
from __future__ import annotations

import functools
import math

import torch

own = False

_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}


# ---- the cases ---------------------------------------------------------------------------------------------------------
#
# `rotary` and `rotary_gradient`: B sequences of S tokens with H query heads and G key heads of width D, of which the first
# R elements are rotated.  `attention` and `training`: Sq queries against Sk keys; with `cache` the queries are the last
# tokens of sequences of different lengths in a cache of Sk places.

def listed():
    return [
        # one new token for each of eight sequences, far into a context that was stretched by bands: nothing but the cost of a call
        _rotary("rotary_token", "rotary", 8, 1, 32, 8, 128, 128, "bf16", "bshd", False, True, True, 8.0, True),
        # a prompt of two sequences: queries and keys normalised and rotated on their way to attention
        _rotary("rotary_prompt", "rotary", 2, 4096, 32, 8, 128, 128, "bf16", "bshd", False, True, False, 1.0, False),
        # f32, an odd number of tokens, part of a narrow head, interleaved pairs, linearly scaled, heads in front of tokens
        _rotary("rotary_part_odd", "rotary", 3, 777, 5, 5, 80, 32, "f32", "bhsd", True, False, True, 4.0, False),
        # the backward pass of a training batch, with the gradients of both norms' weights
        _rotary("rotary_gradient_batch", "rotary_gradient", 4, 4096, 32, 8, 128, 128, "bf16", "bshd", False, True, False, 1.0, False),
        # the same in f16 with an odd number of tokens and equal head counts, as in a small model
        _rotary("rotary_gradient_odd", "rotary_gradient", 1, 1001, 12, 12, 64, 64, "f16", "bhsd", True, True, True, 1.0, False),
        # prompts through a layer with capped scores and grouped heads
        _attention("capped_prompt", "attention", 2, 4096, 4096, 16, 8, 128, "bf16", "bshd", causal=True, softcap=30.0),
        # an encoder with a bias by distance, sequences that end inside a tile, the narrower head
        _attention("distance_odd", "attention", 3, 1000, 1000, 12, 12, 64, "f16", "bhsd", distance=True),
        # documents packed into one long row
        _attention("documents_packed", "attention", 1, 8192, 8192, 16, 4, 128, "bf16", "bhsd", causal=True, documents=11),
        # serving: one token for each of many sequences of different lengths
        _attention("token_batch", "attention", 32, 1, 8192, 32, 8, 128, "bf16", "bshd", causal=True, cache=True, softcap=30.0),
        # serving: one sequence, where the call's own cost shows
        _attention("token_single", "attention", 1, 1, 2000, 8, 2, 64, "bf16", "bhsd", causal=True, cache=True, distance=True),
        # a training step's attention, forward and backward, with capped scores and grouped heads
        _attention("training_capped", "training", 2, 4096, 4096, 16, 4, 128, "bf16", "bshd", causal=True, softcap=50.0),
        # the same for a padded batch whose sequences begin with a prefix that every token sees; odd sizes, f16
        _attention("training_prefix_odd", "training", 3, 515, 515, 8, 8, 80, "f16", "bhsd", causal=True, prefix=True, padded=True),
    ]


def _rotary(name, kind, B, S, H, G, D, R, dtype, layout, interleaved, norm, positions, factor, bands):
    return {"name": name, "kind": kind, "B": B, "S": S, "H": H, "G": G, "D": D, "R": R, "dtype": dtype, "layout": layout, "interleaved": interleaved,
            "norm": norm, "positions": positions, "factor": factor, "bands": bands}


def _attention(name, kind, B, Sq, Sk, H, G, D, dtype, layout, causal=False, softcap=0.0, distance=False, documents=0, prefix=False, padded=False, cache=False):
    return {"name": name, "kind": kind, "B": B, "Sq": Sq, "Sk": Sk, "H": H, "G": G, "D": D, "dtype": dtype, "layout": layout, "causal": causal,
            "softcap": softcap, "distance": distance, "documents": documents, "prefix": prefix, "padded": padded, "cache": cache}


def _size(rng, low, high):
    """A size whose logarithm is spread evenly over [low, high]."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["rotary", "rotary_gradient", "attention", "attention", "token", "token", "training", "training"])
    layout = rng.choice(["bshd", "bhsd"])
    G = _size(rng, 1, 8)
    if kind in ("rotary", "rotary_gradient"):
        D = 8 * rng.randint(4, 16)
        H = G * rng.choice([1, 2, 4])
        B = _size(rng, 1, 8)
        c = _rotary("", kind, B, _size(rng, 1, 16384 // B), H, G, D, rng.choice([D, 2 * rng.randint(1, D // 2)]), rng.choice(["bf16", "f16", "f32"]), layout,
                    rng.choice([True, False]), rng.choice([True, False]), rng.choice([True, False]), rng.choice([1.0, 2.0, 8.0]), rng.choice([True, False]))
    else:
        dtype, D = rng.choice(["bf16", "f16"]), rng.choice([64, 128, 8 * rng.randint(4, 16)])
        causal = kind == "token" or rng.random() < 0.7
        mods = {"causal": causal, "softcap": rng.choice([0.0, 0.0, 30.0, 50.0, 80.0]), "distance": rng.random() < 0.3}
        if kind == "token":
            c = _attention("", "attention", _size(rng, 1, 32), rng.choice([1, 1, 1, 2, 5]), _size(rng, 16, 8192), G * rng.choice([1, 2, 4, 8]), G, D, dtype, layout, cache=True, **mods)
        else:
            S, B, H = _size(rng, 16, 4096), _size(rng, 1, 3), G * rng.choice([1, 2])
            mods["documents"] = _size(rng, 1, 12) if rng.random() < 0.4 and S > 64 else 0
            mods["prefix"] = causal and rng.random() < 0.3
            mods["padded"] = rng.random() < 0.3
            c = _attention("", kind, B, S, S, H, G, D, dtype, layout, **mods)
    del c["name"]
    return c


# ---- inputs --------------------------------------------------------------------------------------------------------------

def _shape(c, heads, tokens):
    return [c["B"], tokens, heads, c["D"]] if c["layout"] == "bshd" else [c["B"], heads, tokens, c["D"]]


def _scale(c):
    return c["D"] ** -0.5


def _lengths(c):
    """How many tokens each sequence of a padded batch or of a cache has: from full to short, evenly spread."""
    return [max(1, c["Sk"] * (i + 1) // c["B"]) for i in range(c["B"])]


def _prefixes(c):
    return [c["Sk"] * (i + 1) // (3 * c["B"]) for i in range(c["B"])]


def _document_sizes(c):
    """Documents of growing sizes that fill a row together."""
    n = c["documents"]
    cuts = [c["Sk"] * i * (i + 1) // (n * (n + 1)) for i in range(n + 1)]
    return [b - a for a, b in zip(cuts, cuts[1:])]


def _frequencies(c):
    """Radians per position of each rotated pair, in 64 bits."""
    out = []
    for i in range(c["R"] // 2):
        f = 10000.0 ** (-2.0 * i / c["R"])
        if c["bands"]:
            # wavelengths well below the original context stay, those well above it are stretched, those between are blended
            t = (8192.0 * f / (2 * math.pi) - 1.0) / (4.0 - 1.0)
            t = min(1.0, max(0.0, t))
            f = (1 - t) * f / c["factor"] + t * f
        else:
            f = f / c["factor"]
        out.append(f)
    return out


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    order = torch.Generator().manual_seed(seed)

    def normal(shape, scale=1.0, dtype=c["dtype"]):
        return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(_TORCH[dtype])

    if c["kind"].startswith("rotary"):
        t = [normal(_shape(c, c["H"], c["S"]), 2.0), normal(_shape(c, c["G"], c["S"]), 2.0)]
        if c["kind"] == "rotary_gradient":
            t = [normal(_shape(c, c["H"], c["S"]), 0.1), normal(_shape(c, c["G"], c["S"]), 0.1)] + (t if c["norm"] else [])
        if c["norm"]:
            t += [1.0 + normal([c["D"]], 0.2, "f32") for _ in range(2)]
        if c["positions"]:
            start = torch.randint(0, 131072 - c["S"], (c["B"], 1), generator=order, dtype=torch.int32)
            t.append((start + torch.arange(c["S"], dtype=torch.int32)).cuda().contiguous())
    else:
        t = [normal(_shape(c, c["H"], c["Sq"]), 2.0), normal(_shape(c, c["G"], c["Sk"])), normal(_shape(c, c["G"], c["Sk"]))]
        if c["kind"] == "training":
            t.append(normal(_shape(c, c["H"], c["Sq"]), 0.1))
        batch = torch.randperm(c["B"], generator=order)
        if c["distance"]:
            # the usual geometric series over heads
            t.append(torch.tensor([2.0 ** (-8.0 * (h + 1) / c["H"]) for h in range(c["H"])], dtype=torch.float32, device="cuda"))
        if c["documents"]:
            sizes = torch.tensor(_document_sizes(c))
            rows = [torch.repeat_interleave(torch.arange(len(sizes)), sizes[torch.randperm(len(sizes), generator=order)]) for _ in range(c["B"])]
            t.append(torch.stack(rows).to(torch.int32).cuda())
        if c["prefix"]:
            t.append(torch.tensor(_prefixes(c))[batch].to(torch.int32).cuda())
        if c["padded"] or c["cache"]:
            t.append(torch.tensor(_lengths(c))[batch].to(torch.int32).cuda())
    torch.cuda.current_stream().synchronize()
    return {"case": dict(c), "tensors": t}


def _named(c, t):
    """The tensors of an attention case by name."""
    t = list(t)
    n = {"q": t.pop(0), "k": t.pop(0), "v": t.pop(0)}
    for name, there in (("do", c["kind"] == "training"), ("slopes", c["distance"]), ("documents", c["documents"]), ("prefix", c["prefix"]),
                        ("lengths", c["padded"] or c["cache"])):
        n[name] = t.pop(0) if there else None
    return n


# ---- the framework's calls -------------------------------------------------------------------------------------------------

def _text(c):
    """The program of a case."""
    from ryft_b200.stablehlo import Builder

    b = Builder()
    if c["kind"].startswith("rotary"):
        q, k = _shape(c, c["H"], c["S"]), _shape(c, c["G"], c["S"])
        how = {"layout": c["layout"], "rotary_dims": c["R"], "interleaved": c["interleaved"], "factor": c["factor"]}
        if c["bands"]:
            how["bands"] = (1.0, 4.0, 8192)
        back = c["kind"] == "rotary_gradient"
        dy = [b.arg(q, c["dtype"]), b.arg(k, c["dtype"])] if back else None
        x = [b.arg(q, c["dtype"]), b.arg(k, c["dtype"])] if not back or c["norm"] else None
        if c["norm"]:
            how["weights"] = [b.arg([c["D"]], "f32"), b.arg([c["D"]], "f32")]
            how["epsilon"] = 1e-6
        if c["positions"]:
            how["positions"] = b.arg([c["B"], c["S"]], "i32")
        return b.build(*(b.rotary_gradient(dy, x, **how) if back else b.rotary(x, **how)))
    q, k, v = b.arg(_shape(c, c["H"], c["Sq"]), c["dtype"]), b.arg(_shape(c, c["G"], c["Sk"]), c["dtype"]), b.arg(_shape(c, c["G"], c["Sk"]), c["dtype"])
    do = b.arg(_shape(c, c["H"], c["Sq"]), c["dtype"]) if c["kind"] == "training" else None
    how = {"layout": c["layout"], "scale": _scale(c), "causal": c["causal"], "softcap": c["softcap"], "queries_at_end": c["cache"]}
    if c["distance"]:
        how["slopes"] = b.arg([c["H"]], "f32")
    if c["documents"]:
        how["documents"] = b.arg([c["B"], c["Sk"]], "i32")
    if c["prefix"]:
        how["prefix"] = b.arg([c["B"]], "i32")
    if c["padded"] or c["cache"]:
        how["lengths"] = b.arg([c["B"]], "i32")
    if do is None:
        return b.build(b.attention(q, k, v, **how))
    o, lse = b.attention(q, k, v, log_sum=True, **how)
    return b.build(o, lse, *b.attention_gradient(q, k, v, o, lse, do, **how))


@functools.lru_cache(maxsize=None)
def _client():
    from ryft_b200 import pjrt

    return pjrt.load_cuda_13_plugin().client({"visible_devices": [0]})


@functools.lru_cache(maxsize=None)
def _executable(text):
    from ryft_b200 import pjrt

    return _client().compile(pjrt.Program.mlir(text))


class _Result:
    """An output buffer as torch sees it: the memory stays the plugin's and lives as long as the tensor over it."""

    def __init__(self, buffer, shape, size):
        self.buffer = buffer
        self.__cuda_array_interface__ = {"shape": shape, "typestr": "<f4" if size == 4 else "<i2", "data": (buffer.device_pointer(), False), "version": 2}


def _loaded(state):
    """The compiled program, the arguments as buffers of the plugin and the results' shapes and types: a program keeps them from call to call."""
    from ryft_b200 import pjrt

    types = {torch.float32: pjrt.BufferType.F32, torch.bfloat16: pjrt.BufferType.BF16, torch.float16: pjrt.BufferType.F16, torch.int32: pjrt.BufferType.S32}
    back = {types[t]: t for t in types}
    executable = _executable(_text(state["case"]))
    buffers = [_client().view_of_device_buffer(t.data_ptr(), types[t.dtype], list(t.shape), keep=t) for t in state["tensors"]]
    of = executable.executable()
    results = [(tuple(shape), back[e]) for shape, e in zip(of.output_dimensions(), of.output_element_types())]
    return executable, [pjrt.ExecutionDeviceInputs(buffers)], results


def _run_own(state):
    if "loaded" not in state:
        state["loaded"] = _loaded(state)
    executable, arguments, results = state["loaded"]
    stream = torch.cuda.current_stream().cuda_stream
    tensors = []
    for buffer, (shape, dtype) in zip(executable.execute(arguments)[0].outputs, results):
        buffer.wait_until_ready_on_stream(stream)     # what torch does with the tensor comes after the program
        t = torch.as_tensor(_Result(buffer, shape, dtype.itemsize), device="cuda")
        tensors.append(t if dtype is torch.float32 else t.view(dtype))
    return tensors


# ---- the plain forms ---------------------------------------------------------------------------------------------------------

def _rotate(c, x, cos, sin):
    """The rotation of the first R elements of the last dimension."""
    R = c["R"]
    if c["interleaved"]:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., : R // 2], x[..., R // 2:R]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, x[..., R:]], dim=-1)


def _angles(c, positions, dtype):
    """cos and sin for every token and pair, laid out to multiply a tensor of the case's layout; angles in 64 bits."""
    p = positions if positions is not None else torch.arange(c["S"], device="cuda", dtype=torch.int32).expand(c["B"], c["S"])
    a = p.double()[..., None] * torch.tensor(_frequencies(c), dtype=torch.float64, device="cuda")
    a = a[:, :, None] if c["layout"] == "bshd" else a[:, None]
    return torch.cos(a).to(dtype), torch.sin(a).to(dtype)


def _norm_back(x, dn, w):
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    g = dn * w
    dx = r * (g - x * r * r * (g * x).mean(-1, keepdim=True))
    return dx, (dn * x * r).sum(dim=(0, 1, 2))


def _run_rotary(c, t):
    back = c["kind"] == "rotary_gradient"
    cos, sin = _angles(c, t[-1] if c["positions"] else None, torch.float32)
    first = [t[0].float(), t[1].float()]
    if not back:
        if c["norm"]:
            first = [x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w for x, w in zip(first, t[2:4])]
        return [_rotate(c, x, cos, sin).to(_TORCH[c["dtype"]]) for x in first]
    dn = [_rotate(c, dy, cos, -sin) for dy in first]
    if not c["norm"]:
        return [d.to(_TORCH[c["dtype"]]) for d in dn]
    (dq, wq), (dk, wk) = [_norm_back(x.float(), d, w) for x, d, w in zip(t[2:4], dn, t[4:6])]
    return [dq.to(_TORCH[c["dtype"]]), dk.to(_TORCH[c["dtype"]]), wq, wk]


def _allowed(c, n, rows=None):
    """[B, Sq, Sk]: which keys a query sees, and [B, Sq, Sk] how far they are."""
    B, Sq, Sk = c["B"], c["Sq"], c["Sk"]
    key = torch.arange(Sk, device="cuda")[None, None]
    at = torch.arange(Sq, device="cuda")[None, :, None].expand(B, Sq, 1)
    length = n["lengths"].long()[:, None, None] if n["lengths"] is not None else torch.full((B, 1, 1), Sk, device="cuda")
    if c["cache"]:
        at = at + length - Sq
    see = (key < length).expand(B, Sq, Sk)
    if c["causal"]:
        before = key <= at
        if n["prefix"] is not None:
            before = before | (key < n["prefix"].long()[:, None, None])
        see = see & before
    if n["documents"] is not None:
        see = see & (n["documents"][:, :, None] == n["documents"][:, None, :])
    return see, (at - key).abs()


def _heads_first(c, x):
    return x.transpose(1, 2) if c["layout"] == "bshd" else x


def _run_attention(c, t):
    n = _named(c, t)
    share = c["H"] // c["G"]
    see, far = _allowed(c, n)
    q = _heads_first(c, n["q"].float())
    k, v = (_heads_first(c, n[x].float()).repeat_interleave(share, dim=1) for x in ("k", "v"))
    s = q @ k.transpose(2, 3) * _scale(c)
    bend = None
    if c["softcap"]:
        bend = torch.tanh(s / c["softcap"])
        s = c["softcap"] * bend
    if c["distance"]:
        s = s - n["slopes"][None, :, None, None] * far[:, None].float()
    s = torch.where(see[:, None], s, float("-inf"))
    most = s.amax(-1, keepdim=True)
    most = torch.where(most == float("-inf"), 0.0, most)          # a query that sees nothing
    p = torch.exp(s - most)
    del s
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    o = _heads_first(c, p @ v).to(_TORCH[c["dtype"]]).contiguous()
    if c["kind"] != "training":
        return [o]
    do = _heads_first(c, n["do"].float())
    dv = p.transpose(2, 3) @ do
    dp = do @ v.transpose(2, 3)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * _scale(c)
    del dp, p
    if bend is not None:
        ds = ds * (1 - bend * bend)
    dq = ds @ k
    dk = ds.transpose(2, 3) @ q
    dk, dv = (x.unflatten(1, (c["G"], share)).sum(2) for x in (dk, dv))
    return [o, (most + torch.log(total)).squeeze(-1)] + [_heads_first(c, x).to(_TORCH[c["dtype"]]).contiguous() for x in (dq, dk, dv)]


def run(state):
    if own:
        return _run_own(state)
    c = state["case"]
    return _run_rotary(c, state["tensors"]) if c["kind"].startswith("rotary") else _run_attention(c, state["tensors"])


# ---- what a pass cannot do without, and what it has to yield ----------------------------------------------------------------

def _pairs(c):
    """Visible (query, key) pairs of one head over the batch."""
    total = 0
    lengths = _lengths(c) if c["padded"] or c["cache"] else [c["Sk"]] * c["B"]
    prefixes = _prefixes(c) if c["prefix"] else [0] * c["B"]
    if c["documents"] and not c["padded"] and not c["prefix"]:
        return c["B"] * sum(d * (d + 1) // 2 if c["causal"] else d * d for d in _document_sizes(c))
    for length, prefix in zip(lengths, prefixes):
        for i in range(c["Sq"]):
            at = length - c["Sq"] + i if c["cache"] else i
            total += max(0, min(length, max(at + 1, prefix)) if c["causal"] else length)
    if c["documents"]:
        # which documents the padding cuts is up to the seed: the share of pairs that lie in one document
        total = int(total * sum(d * d for d in _document_sizes(c)) / c["Sk"] ** 2)
    return total


def work(case):
    c = case
    es = _SIZE[c["dtype"]]
    if c["kind"].startswith("rotary"):
        x = c["B"] * c["S"] * (c["H"] + c["G"]) * c["D"] * es
        back = c["kind"] == "rotary_gradient" and c["norm"]
        n = x * (3 if back else 2) + (c["B"] * c["S"] * 4 if c["positions"] else 0) + (2 * c["D"] * 4 * (2 if back else 1) if c["norm"] else 0)
        return {"bytes": float(n), "flops": 0.0}
    q = c["B"] * c["Sq"] * c["H"] * c["D"] * es
    places = sum(_lengths(c)) if c["padded"] or c["cache"] else c["B"] * c["Sk"]
    k = places * c["G"] * c["D"] * es
    pairs = float(_pairs(c)) * c["H"] * c["D"]
    if c["kind"] == "training":
        # q, k, v, do in; o, its log sums, dq, dk, dv out; two products forward, five backward
        return {"bytes": float(4 * q + 2 * k + 2 * c["B"] * c["Sk"] * c["G"] * c["D"] * es + c["B"] * c["Sq"] * c["H"] * 4), "flops": 14.0 * pairs}
    return {"bytes": float(2 * q + 2 * k), "flops": 4.0 * pairs}


def _exact_rotary(c, t):
    back = c["kind"] == "rotary_gradient"
    token_axis = 1 if c["layout"] == "bshd" else 2
    p = t[-1].double() if c["positions"] else torch.arange(c["S"], device="cuda").double().repeat(c["B"], 1)
    turn = torch.exp(1j * p[..., None] * torch.tensor(_frequencies(c), dtype=torch.float64, device="cuda")).unsqueeze(3 - token_axis)
    if back:
        turn = turn.conj()
    half = c["R"] // 2

    def rotate(x):
        y = x.clone()
        i = torch.arange(half, device="cuda")
        first, second = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + half)
        z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
        y[..., first], y[..., second] = z.real, z.imag
        return y

    x = [a.double() for a in (t[2:4] if back and c["norm"] else t[0:2])]
    if not c["norm"]:
        return [rotate(a) for a in x]
    weights = [w.double() for w in (t[4:6] if back else t[2:4])]
    size = [(a.square().sum(-1, keepdim=True) / c["D"] + 1e-6).sqrt() for a in x]
    if not back:
        return [rotate(a / s * w) for a, s, w in zip(x, size, weights)]
    dx, dw = [], []
    for a, s, w, dy in zip(x, size, weights, t[0:2]):
        n, dn = a / s, rotate(dy.double())
        dw.append((dn * n).reshape(-1, c["D"]).sum(0))
        g = dn * w
        dx.append((g - n * (g * n).sum(-1, keepdim=True) / c["D"]) / s)
    return dx + dw


def _exact_attention(c, t):
    n = _named(c, t)
    training = c["kind"] == "training"
    see, far = _allowed(c, n)
    part = lambda x, i, h: _heads_first(c, x)[i, h].double()  # noqa: E731
    o = torch.empty(_shape(c, c["H"], c["Sq"]), dtype=torch.float64, device="cuda")
    out = [o]
    if training:
        lse = torch.empty(c["B"], c["H"], c["Sq"], dtype=torch.float64, device="cuda")
        dq = torch.empty_like(o)
        dk, dv = (torch.zeros(_shape(c, c["G"], c["Sk"]), dtype=torch.float64, device="cuda") for _ in range(2))
        out += [lse, dq, dk, dv]
    for i in range(c["B"]):
        for h in range(c["H"]):
            u = h * c["G"] // c["H"]
            q, k, v = part(n["q"], i, h), part(n["k"], i, u), part(n["v"], i, u)
            s = (q @ k.T).mul_(_scale(c))
            if c["softcap"]:
                s.div_(c["softcap"]).tanh_()
                slope = 1 - s.square() if training else None
                s.mul_(c["softcap"])
            if c["distance"]:
                s -= n["slopes"][h].double() * far[i]
            s.masked_fill_(~see[i], float("-inf"))
            sums = torch.logsumexp(s, dim=1)
            w = s.sub_(torch.where(sums.isinf(), 0.0, sums)[:, None]).exp_()
            result = w @ v
            _heads_first(c, o)[i, h] = result
            if not training:
                continue
            lse[i, h] = sums
            d = part(n["do"], i, h)
            _heads_first(c, dv)[i, u] += w.T @ d
            ds = w * (d @ v.T - (d * result).sum(1, keepdim=True)) * _scale(c)
            if c["softcap"]:
                ds *= slope
            _heads_first(c, dq)[i, h] = ds @ k
            _heads_first(c, dk)[i, u] += ds.T @ q
    return out


def exact(case, seed):
    t = prepare(case, seed)["tensors"]
    return _exact_rotary(case, t) if case["kind"].startswith("rotary") else _exact_attention(case, t)
