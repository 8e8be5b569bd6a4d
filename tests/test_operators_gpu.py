"""The named operators on the GPU, through Client.compile and execute, against 64-bit forms (operators_reference.py)."""
import numpy as np
import pytest
import torch

import operators_reference as ref
from ryft_b200 import pjrt
from ryft_b200.stablehlo import Builder

pytestmark = pytest.mark.gpu
BUFFER = {torch.bfloat16: pjrt.BufferType.BF16, torch.float16: pjrt.BufferType.F16, torch.float32: pjrt.BufferType.F32, torch.int32: pjrt.BufferType.S32}


@pytest.fixture(scope="module")
def client():
    c = pjrt.load_cuda_13_plugin().client({"visible_devices": [0]})
    yield c
    c.close()


def host(t):
    t = t.contiguous()
    return t.view(torch.int16).numpy() if t.dtype in (torch.bfloat16, torch.float16) else t.numpy()


def run(client, text, tensors):
    exe = client.compile(pjrt.Program.mlir(text))
    bufs = [client.buffer(host(t), BUFFER[t.dtype], list(t.shape)) for t in tensors]
    return collect(exe.execute([pjrt.ExecutionDeviceInputs(bufs)])[0])


def collect(result):
    result.done.await_()
    back = {int(b): t for t, b in BUFFER.items()}
    got = []
    for o in result.outputs:
        t = back[int(o.element_type())]
        shape = o.dimensions()
        raw = np.zeros(int(np.prod(shape)), np.float32 if t == torch.float32 else np.int16)
        if raw.size:
            o.copy_to_host(raw).await_()
        x = torch.from_numpy(raw)
        got.append((x if t == torch.float32 else x.view(t)).reshape(shape))
    return got


def within(got, want, bound, what):
    got = got.double()
    assert got.shape == want.shape, what
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), ~odd), f"{what}: {int((torch.isfinite(got) == odd).sum())} values are (not) finite"
    assert torch.equal(got[odd], want[odd]) or bool(torch.isnan(want[odd]).all() and torch.isnan(got[odd]).all()), what
    off = (got - want).abs()[~odd] / bound.expand_as(want)[~odd]
    assert off.numel() == 0 or off.max() <= 1.0, f"{what}: {float(off.max()):.3g} of the bound, {int((off > 1).sum())} of {off.numel()} values"


def normal(seed, *shapes, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=g) * scale for s in shapes]


# ---- rotary -----------------------------------------------------------------------------------------------------------------

def shape(layout, B, H, S, D):
    return [B, S, H, D] if layout == "bshd" else [B, H, S, D]


ROTARY = [
    # B, S, heads, D, R, dtype, layout, interleaved, norm, positions, how
    (2, 5, (4, 2), 128, 128, "bf16", "bshd", False, True, "far", {}),
    (1, 1, (32, 8), 128, 128, "bf16", "bshd", False, True, "far", {"factor": 8.0, "bands": (1.0, 4.0, 8192)}),
    (3, 7, (5,), 80, 32, "f32", "bhsd", True, False, None, {"factor": 4.0}),
    (1, 33, (3, 3), 64, 64, "f16", "bhsd", True, True, "far", {"base": 500000.0}),
    (2, 4, (3, 1), 72, 36, "bf16", "bshd", False, True, None, {}),          # half of 36 is no multiple of a piece
    (1, 3, (2, 1), 18, 10, "f16", "bshd", False, True, "negative", {}),      # rows that start anywhere
    (1, 3, (2, 1), 17, 6, "f32", "bhsd", True, True, None, {}),              # an odd width
    (1, 2, (1, 1), 256, 256, "f32", "bshd", False, True, "far", {}),
    (1, 2, (2, 1), 255, 250, "bf16", "bshd", True, True, None, {}),
    (2, 3, (2, 2), 96, 0, "bf16", "bhsd", False, True, None, {}),            # norms alone
    (1, 700, (9, 1), 40, 40, "bf16", "bshd", True, False, None, {}),
    (4, 301, (16, 4), 128, 64, "bf16", "bhsd", False, True, "far", {"factor": 2.0}),
    (1, 1, (1,), 2, 2, "f32", "bhsd", False, False, "far", {}),
]


def rotary_case(c, seed):
    B, S, heads, D, R, dtype, layout, interleaved, norm, positions, how = c
    t = ref.TORCH[dtype]
    x = [a.to(t) for a in normal(seed, *[shape(layout, B, h, S, D) for h in heads], scale=2.0)]
    dy = [a.to(t) for a in normal(seed + 1, *[shape(layout, B, h, S, D) for h in heads])]
    w = [1 + 0.3 * a for a in normal(seed + 2, *[[D] for _ in heads])] if norm else None
    g = torch.Generator().manual_seed(seed)
    pos = None
    if positions:
        pos = torch.randint(-(2 ** 31) if positions == "negative" else 0, 2 ** 31 - 1, (B, S), generator=g, dtype=torch.int64).to(torch.int32)
    return x, dy, w, pos


@pytest.mark.parametrize("case", ROTARY, ids=str)
def test_rotary_and_its_gradient(client, case):
    B, S, heads, D, R, dtype, layout, interleaved, norm, positions, how = case
    x, dy, w, pos = rotary_case(case, 3)
    at = pos if pos is not None else torch.arange(S, dtype=torch.int32).expand(B, S)
    b = Builder()
    xs = [b.arg(list(a.shape), dtype) for a in x]
    dys = [b.arg(list(a.shape), dtype) for a in dy]
    ws = [b.arg([D], "f32") for _ in heads] if norm else None
    ps = b.arg([B, S], "i32") if pos is not None else None
    opts = {"layout": layout, "rotary_dims": R, "interleaved": interleaved, "positions": ps, "weights": ws, "epsilon": 1e-5 if norm else None, **how}
    y, back = b.rotary(xs, **opts), b.rotary_gradient(dys, xs if norm else None, **opts)
    got = run(client, b.build(*y, *back), [*x, *dy, *(w or []), *([pos] if pos is not None else [])])
    n = len(heads)
    for i in range(n):
        args = (at, w[i] if norm else None, dtype, layout, R, interleaved, 1e-5)
        within(got[i], *ref.rotary(x[i], *args, **how), f"y{i}")
        dx, edx, dw, edw = ref.rotary_gradient(dy[i], x[i], *args, **how)
        within(got[n + i], dx, edx, f"dx{i}")
        if norm:
            within(got[2 * n + i], dw, edw, f"dw{i}")


def test_rotary_of_views_16_bit_weights_and_nothing(client):
    b = Builder()
    x = b.arg([2, 6, 3, 64], "bf16")                     # [B, S, H, D], read as [B, H, S, D] through a transpose
    w = b.arg([64], "bf16")
    t = b.transpose(x, [0, 2, 1, 3])
    none = b.arg([2, 0, 3, 64], "bf16")
    y = b.rotary([t], weights=[w], epsilon=1e-6)[0]
    dn = b.rotary_gradient([none], [none], weights=[w], layout="bshd", epsilon=1e-6)
    (xv,), (wv,) = [a.bfloat16() for a in normal(1, [2, 6, 3, 64])], [(1 + 0.1 * a).bfloat16() for a in normal(2, [64])]
    got = run(client, b.build(y, *dn), [xv, wv, torch.zeros(2, 0, 3, 64, dtype=torch.bfloat16)])
    within(got[0], *ref.rotary(xv.transpose(1, 2), torch.arange(6).expand(2, 6), wv, "bf16", "bhsd", 64, False, 1e-6), "y")
    assert got[1].numel() == 0 and torch.equal(got[2], torch.zeros(64))


def test_rotary_keeps_infinities_where_they_are(client):
    b = Builder()
    x = b.arg([1, 1, 2, 16], "f32")
    xv = torch.ones(1, 1, 2, 16)
    xv[0, 0, 0, 12] = float("inf")                       # behind the rotated part: its neighbours stay numbers
    xv[0, 0, 1, 3] = float("nan")
    got = run(client, b.build(*b.rotary([x], rotary_dims=8)), [xv])[0]
    assert torch.isinf(got[0, 0, 0, 12]) and torch.isfinite(got[0, 0, 0, [i for i in range(16) if i != 12]]).all()
    assert torch.isnan(got[0, 0, 1, [3, 7]]).all() and torch.isfinite(got[0, 0, 1, [i for i in range(16) if i not in (3, 7)]]).all()


# ---- attention -----------------------------------------------------------------------------------------------------------------

def attention_case(B, Sq, Sk, Hq, Hk, D, dtype, layout, seed, slopes=False, documents=None, prefix=None, lengths=None, **how):
    t = ref.TORCH[dtype]
    q, do = [a.to(t) for a in normal(seed, shape(layout, B, Hq, Sq, D), shape(layout, B, Hq, Sq, D))]
    k, v = [a.to(t) for a in normal(seed + 1, shape(layout, B, Hk, Sk, D), shape(layout, B, Hk, Sk, D))]
    q = (q.float() * 2).to(t)
    extra = {}
    if slopes:
        extra["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / Hq) for h in range(Hq)])
    if documents is not None:
        g = torch.Generator().manual_seed(seed)
        ids = torch.randint(0, documents, (B, Sk), generator=g, dtype=torch.int32)
        extra["documents"] = ids if how.pop("unsorted", False) else ids.sort(1).values.contiguous()
    if prefix is not None:
        extra["prefix"] = torch.tensor(prefix, dtype=torch.int32)
    if lengths is not None:
        extra["lengths"] = torch.tensor(lengths, dtype=torch.int32)
    return q, k, v, do, extra, how


def attention_run(client, q, k, v, do, extra, how, dtype, layout, gradient=True):
    b = Builder()
    args = [b.arg(list(a.shape), dtype) for a in ((q, k, v, do) if gradient else (q, k, v))]
    more = {n: b.arg(list(a.shape), "f32" if n == "slopes" else "i32") for n, a in extra.items()}
    o, lse = b.attention(*args[:3], layout=layout, log_sum=True, **more, **how)
    outs = [o, lse]
    if gradient:
        outs += b.attention_gradient(*args[:3], o, lse, args[3], layout=layout, **more, **how)
    return run(client, b.build(*outs), [q, k, v] + ([do] if gradient else []) + list(extra.values()))


def attention_check(client, B, Sq, Sk, Hq, Hk, D, dtype, layout, seed=7, gradient=True, **options):
    q, k, v, do, extra, how = attention_case(B, Sq, Sk, Hq, Hk, D, dtype, layout, seed, **options)
    got = attention_run(client, q, k, v, do, extra, how, dtype, layout, gradient)
    scale = how.pop("scale", D ** -0.5)
    want = ref.attention(q, k, v, dtype, layout, scale, do=do if gradient else None, **extra, **how)
    for name, x in zip(("o", "lse", "dq", "dk", "dv"), got):
        within(x, *want[name], name)


ATTENTION = [
    (dict(B=1, Sq=1, Sk=1, Hq=1, Hk=1, D=64, dtype="bf16", layout="bhsd"), dict()),
    (dict(B=2, Sq=128, Sk=128, Hq=2, Hk=1, D=128, dtype="bf16", layout="bshd"), dict(causal=True)),
    (dict(B=1, Sq=129, Sk=257, Hq=2, Hk=2, D=64, dtype="f16", layout="bhsd"), dict(softcap=20.0)),
    (dict(B=1, Sq=300, Sk=300, Hq=4, Hk=2, D=128, dtype="bf16", layout="bshd"), dict(causal=True, softcap=30.0)),
    (dict(B=1, Sq=300, Sk=300, Hq=2, Hk=2, D=72, dtype="bf16", layout="bhsd"), dict(causal=True, softcap=90.0)),
    (dict(B=2, Sq=200, Sk=333, Hq=6, Hk=2, D=80, dtype="f16", layout="bshd"), dict(slopes=True)),
    (dict(B=1, Sq=70, Sk=400, Hq=2, Hk=1, D=96, dtype="bf16", layout="bhsd"), dict(slopes=True, causal=True, query_offset=330)),
    (dict(B=2, Sq=390, Sk=390, Hq=2, Hk=1, D=128, dtype="bf16", layout="bhsd"), dict(causal=True, documents=4)),
    (dict(B=2, Sq=390, Sk=390, Hq=2, Hk=2, D=64, dtype="bf16", layout="bshd"), dict(documents=3)),
    (dict(B=1, Sq=200, Sk=200, Hq=2, Hk=2, D=64, dtype="f16", layout="bshd"), dict(documents=5, unsorted=True, causal=True, softcap=50.0, slopes=True)),
    (dict(B=1, Sq=300, Sk=900, Hq=1, Hk=1, D=64, dtype="bf16", layout="bhsd"), dict(documents=6, causal=True, query_offset=600)),
    (dict(B=3, Sq=270, Sk=270, Hq=2, Hk=2, D=40, dtype="f16", layout="bhsd"), dict(causal=True, prefix=[0, 100, 270])),
    (dict(B=4, Sq=260, Sk=260, Hq=2, Hk=1, D=128, dtype="bf16", layout="bshd"), dict(causal=True, prefix=[0, 30, 260, 140], lengths=[260, 0, 131, 128])),
    (dict(B=4, Sq=140, Sk=260, Hq=2, Hk=2, D=64, dtype="f16", layout="bhsd"), dict(lengths=[1, 0, 260, 129])),
    (dict(B=4, Sq=3, Sk=300, Hq=4, Hk=2, D=128, dtype="bf16", layout="bshd"), dict(causal=True, queries_at_end=True, lengths=[300, 2, 0, 129], softcap=30.0)),
    (dict(B=2, Sq=1, Sk=1500, Hq=8, Hk=1, D=64, dtype="f16", layout="bhsd"), dict(causal=True, queries_at_end=True, lengths=[1500, 700], slopes=True)),
    (dict(B=1, Sq=16, Sk=515, Hq=16, Hk=2, D=80, dtype="bf16", layout="bhsd"), dict(causal=True, query_offset=499)),
    (dict(B=2, Sq=2, Sk=900, Hq=2, Hk=2, D=128, dtype="bf16", layout="bshd"), dict(causal=True, queries_at_end=True, lengths=[900, 555], documents=3)),
    (dict(B=1, Sq=17, Sk=64, Hq=4, Hk=4, D=8, dtype="bf16", layout="bhsd"), dict(scale=0.5)),
    (dict(B=2, Sq=5, Sk=200, Hq=3, Hk=1, D=120, dtype="f16", layout="bshd"), dict(lengths=[3, 200], queries_at_end=True)),
    (dict(B=1, Sq=640, Sk=640, Hq=12, Hk=4, D=128, dtype="bf16", layout="bshd"), dict(causal=True)),
    (dict(B=1, Sq=1, Sk=37, Hq=40, Hk=1, D=8, dtype="bf16", layout="bhsd"), dict()),                                # rows of a key head over three tiles
    (dict(B=2, Sq=16, Sk=130, Hq=6, Hk=2, D=24, dtype="f16", layout="bshd"), dict(causal=True, query_offset=114, softcap=10.0, slopes=True)),
    (dict(B=3, Sq=40, Sk=300, Hq=2, Hk=1, D=64, dtype="bf16", layout="bhsd"), dict(causal=True, queries_at_end=True, lengths=[300, 20, 171], documents=4)),
    (dict(B=3, Sq=150, Sk=150, Hq=2, Hk=2, D=64, dtype="bf16", layout="bshd"), dict(causal=True, lengths=[-5, 10 ** 6, 150], prefix=[-7, 10 ** 6, 3])),
    (dict(B=3, Sq=2, Sk=150, Hq=2, Hk=2, D=64, dtype="bf16", layout="bshd"), dict(lengths=[-5, 10 ** 6, 150], queries_at_end=True, causal=True)),
    (dict(B=1, Sq=200, Sk=200, Hq=2, Hk=1, D=128, dtype="bf16", layout="bhsd"), dict(documents=3, causal=True, softcap=25.0)),
    (dict(B=1, Sq=140, Sk=140, Hq=2, Hk=1, D=64, dtype="bf16", layout="bhsd"), dict(scale=-0.2, causal=True)),
    (dict(B=1, Sq=140, Sk=140, Hq=2, Hk=1, D=64, dtype="f16", layout="bhsd"), dict(scale=-0.2, softcap=5.0)),
    (dict(B=1, Sq=130, Sk=60, Hq=1, Hk=1, D=64, dtype="bf16", layout="bhsd"), dict(scale=0.0)),
    (dict(B=1, Sq=150, Sk=260, Hq=2, Hk=2, D=64, dtype="bf16", layout="bhsd"), dict(scale=3.0, softcap=30.0, causal=True, query_offset=110)),   # scores far beyond the cap
]


@pytest.mark.parametrize("sizes,options", ATTENTION, ids=str)
def test_attention_and_its_gradient(client, sizes, options):
    attention_check(client, **sizes, **options)


def test_a_token_against_a_very_long_cache(client):
    attention_check(client, 1, 1, 200_001, 2, 1, 64, "bf16", "bhsd", gradient=False, causal=True, query_offset=200_000, softcap=30.0)


def test_operands_that_the_program_holds_itself(client):
    """Lengths, slopes and documents as constants and as results of other ops."""
    B, S, D = 2, 140, 64
    q, k, v, do, _, _ = attention_case(B, S, S, 2, 2, D, "bf16", "bhsd", 3)
    b = Builder()
    args = [b.arg([B, 2, S, D], "bf16") for _ in range(3)]
    position = b.iota(1, [B, S], "i32")
    documents = b._emit(position.type, f"stablehlo.divide {position}, {b.constant(50, [B, S], 'i32')} : {position.type}")
    o = b.attention(*args, causal=True, lengths=b.constant(100, [B], "i32"), slopes=b.constant_array([0.5, 0.25], "f32"), documents=documents)
    got = run(client, b.build(o), [q, k, v])[0]
    want = ref.attention(q, k, v, "bf16", "bhsd", D ** -0.5, slopes=torch.tensor([0.5, 0.25]), causal=True, lengths=torch.tensor([100, 100]),
                         documents=(torch.arange(S) // 50).expand(B, S).contiguous())
    within(got, *want["o"], "o")


def test_attention_of_nothing(client):
    attention_check(client, 2, 5, 0, 2, 1, 64, "bf16", "bhsd")
    attention_check(client, 2, 0, 5, 2, 1, 64, "bf16", "bshd")
    attention_check(client, 0, 5, 5, 2, 1, 64, "f16", "bhsd")


@pytest.mark.parametrize("Sq", [1, 140])
def test_what_lies_behind_the_length_does_not_show(client, Sq):
    B, Sk, D = 2, 300, 64
    q, k, v, do, extra, how = attention_case(B, Sq, Sk, 4, 2, D, "bf16", "bhsd", 11, causal=True, queries_at_end=True, lengths=[170, 299])
    clean = attention_run(client, q, k, v, do, extra, how, "bf16", "bhsd")
    for i, n in enumerate((170, 299)):
        k[i, :, n:], v[i, :, n:] = float("nan"), float("inf")
    dirty = attention_run(client, q, k, v, do, extra, how, "bf16", "bhsd")
    for a, c in zip(dirty, clean):
        assert torch.equal(a, c)


def test_nan_scores_make_their_own_rows_nan(client):
    q, k, v, do, extra, how = attention_case(1, 130, 130, 2, 2, 64, "bf16", "bhsd", 5, causal=True, softcap=30.0)
    q[0, 1, 77, 3] = float("nan")
    o, lse = attention_run(client, q, k, v, do, extra, how, "bf16", "bhsd", gradient=False)
    bad = torch.zeros(1, 2, 130, dtype=torch.bool)
    bad[0, 1, 77] = True
    assert torch.equal(torch.isnan(lse), bad) and torch.equal(torch.isnan(o).any(-1), bad)


# fewer tiles than SMs: the gradient's sums over queries or keys are cut into parts
PARTS = [
    (dict(B=1, Sq=1300, Sk=1300, Hq=2, Hk=1, D=128, dtype="bf16", layout="bshd"), dict(causal=True, softcap=30.0)),
    (dict(B=1, Sq=1100, Sk=2100, Hq=1, Hk=1, D=64, dtype="f16", layout="bhsd"), dict(lengths=[1500], slopes=True)),
    (dict(B=2, Sq=1060, Sk=1060, Hq=3, Hk=1, D=80, dtype="bf16", layout="bshd"), dict(causal=True, documents=5, prefix=[0, 700])),
    (dict(B=1, Sq=1100, Sk=1100, Hq=2, Hk=2, D=64, dtype="f16", layout="bhsd"), dict(documents=40, unsorted=True, causal=True)),
    (dict(B=1, Sq=200, Sk=200, Hq=12, Hk=1, D=128, dtype="f16", layout="bhsd"), dict(causal=True)),       # keys only: many query heads
    (dict(B=1, Sq=20, Sk=1200, Hq=2, Hk=2, D=40, dtype="bf16", layout="bshd"), dict(causal=True, query_offset=1180)),       # queries only
    (dict(B=2, Sq=1030, Sk=1030, Hq=1, Hk=1, D=128, dtype="bf16", layout="bhsd"), dict(causal=True, lengths=[0, 70])),      # parts without a unit
    (dict(B=1, Sq=64, Sk=64, Hq=40, Hk=1, D=8, dtype="f16", layout="bshd"), dict(scale=0.5, documents=3)),
]


@pytest.mark.parametrize("sizes,options", PARTS, ids=str)
def test_gradients_in_parts(client, sizes, options):
    attention_check(client, **sizes, **options)


# the same for the forward pass: parts of a walk over the keys, joined by their maxima
FORWARD_PARTS = [
    (dict(B=1, Sq=130, Sk=2500, Hq=2, Hk=1, D=128, dtype="bf16", layout="bhsd"), dict()),
    (dict(B=1, Sq=513, Sk=513, Hq=1, Hk=1, D=64, dtype="f16", layout="bshd"), dict(causal=True, softcap=20.0)),
    (dict(B=2, Sq=100, Sk=1537, Hq=2, Hk=2, D=72, dtype="bf16", layout="bshd"), dict(lengths=[1537, 3], softcap=50.0)),
    (dict(B=1, Sq=300, Sk=1700, Hq=3, Hk=1, D=128, dtype="f16", layout="bhsd"), dict(causal=True, query_offset=1400, slopes=True)),
    (dict(B=2, Sq=900, Sk=900, Hq=2, Hk=1, D=64, dtype="bf16", layout="bhsd"), dict(documents=7, softcap=30.0)),
    (dict(B=1, Sq=600, Sk=1200, Hq=2, Hk=2, D=128, dtype="bf16", layout="bshd"), dict(documents=30, causal=True, query_offset=600)),
    (dict(B=3, Sq=20, Sk=600, Hq=2, Hk=1, D=40, dtype="f16", layout="bhsd"), dict(causal=True, queries_at_end=True, lengths=[600, 0, 7])),
    (dict(B=1, Sq=140, Sk=700, Hq=1, Hk=1, D=64, dtype="bf16", layout="bhsd"), dict(scale=-0.2)),
]


@pytest.mark.parametrize("sizes,options", FORWARD_PARTS, ids=str)
def test_attention_in_parts(client, sizes, options):
    attention_check(client, gradient=False, **sizes, **options)


def test_nan_in_parts(client):
    """A NaN key poisons the queries that see it, whatever part it lies in; what lies behind the length does not show."""
    q, k, v, do, _, _ = attention_case(1, 200, 1200, 1, 1, 64, "bf16", "bhsd", 5)
    k[0, 0, 700] = float("nan")
    lengths = {"lengths": torch.tensor([1100], dtype=torch.int32)}
    k[0, 0, 1100:] = float("nan")
    v[0, 0, 1100:] = float("inf")
    o, lse = attention_run(client, q, k, v, do, lengths, dict(causal=True, query_offset=600), "bf16", "bhsd", gradient=False)
    sees = torch.arange(200) + 600 >= 700
    assert torch.equal(torch.isnan(lse.double().cpu())[0, 0], sees) and torch.equal(torch.isnan(o.float().cpu())[0, 0].all(-1), sees)
    assert torch.isfinite(o.float().cpu()[0, 0][~sees]).all()


def test_gradients_in_parts_do_not_differ_from_run_to_run(client):
    q, k, v, do, extra, how = attention_case(1, 1100, 1100, 4, 1, 128, "bf16", "bshd", 9, causal=True)
    first = attention_run(client, q, k, v, do, extra, how, "bf16", "bshd")
    for _ in range(3):
        for a, c in zip(attention_run(client, q, k, v, do, extra, how, "bf16", "bshd"), first):
            assert torch.equal(a, c)


def test_results_do_not_differ_from_run_to_run(client):
    q, k, v, do, extra, how = attention_case(2, 500, 500, 4, 2, 128, "bf16", "bshd", 9, causal=True, softcap=30.0)
    first = attention_run(client, q, k, v, do, extra, how, "bf16", "bshd")
    for _ in range(3):
        for a, c in zip(attention_run(client, q, k, v, do, extra, how, "bf16", "bshd"), first):
            assert torch.equal(a, c)


# ---- together -------------------------------------------------------------------------------------------------------------------

def test_a_layer_forward_and_backward(client):
    """Projection, norms and rotation, attention, and everything back to the projected queries, keys and their norms, as one program."""
    B, S, H, G, D, E, dtype = 2, 150, 4, 2, 64, 96, "bf16"
    b = Builder()
    x, wq, wk, wv = b.arg([B * S, E], dtype), b.arg([E, H * D], dtype), b.arg([E, G * D], dtype), b.arg([E, G * D], dtype)
    nq, nk, do = b.arg([D], "f32"), b.arg([D], "f32"), b.arg([B, S, H, D], dtype)
    heads = lambda w, h: b.reshape(b.convert(b.dot_general(x, w, ([], []), ([1], [0]), out_dtype="f32"), dtype), [B, S, h, D])  # noqa: E731
    q, k, v = heads(wq, H), heads(wk, G), heads(wv, G)
    rot = {"layout": "bshd", "weights": [nq, nk], "epsilon": 1e-6}
    at = {"layout": "bshd", "causal": True, "softcap": 30.0}
    qr, kr = b.rotary([q, k], **rot)
    o, lse = b.attention(qr, kr, v, log_sum=True, **at)
    dqr, dkr, dv = b.attention_gradient(qr, kr, v, o, lse, do, **at)
    dq, dk, dnq, dnk = b.rotary_gradient([dqr, dkr], [q, k], **rot)
    text = b.build(q, k, v, qr, kr, o, lse, dqr, dkr, dv, dq, dk, dnq, dnk)
    t = normal(21, [B * S, E], [E, H * D], [E, G * D], [E, G * D], [B, S, H, D])
    t = [(a * s).bfloat16() for a, s in zip(t, (1.0, E ** -0.5, E ** -0.5, E ** -0.5, 1.0))]
    w = [1 + 0.2 * a for a in normal(22, [D], [D])]
    q, k, v, qr, kr, o, lse, dqr, dkr, dv, dq, dk, dnq, dnk = run(client, text, [*t[:4], *w, t[4]])
    pos = torch.arange(S).expand(B, S)
    # each operator against its own operands, as the program passed them on
    for got, raw, weight in ((qr, q, w[0]), (kr, k, w[1])):
        within(got, *ref.rotary(raw, pos, weight, dtype, "bshd", D, False, 1e-6), "rotary")
    want = ref.attention(qr, kr, v, dtype, "bshd", D ** -0.5, do=t[4], causal=True, softcap=30.0)
    for name, got in (("o", o), ("lse", lse), ("dq", dqr), ("dk", dkr), ("dv", dv)):
        within(got, *want[name], name)
    for d, got, raw, weight, dw in ((dqr, dq, q, w[0], dnq), (dkr, dk, k, w[1], dnk)):
        dx, edx, dwx, edw = ref.rotary_gradient(d, raw, pos, weight, dtype, "bshd", D, False, 1e-6)
        within(got, dx, edx, "dx")
        within(dw, dwx, edw, "dw")


def test_a_prompt_and_its_next_token_agree(client):
    """The last query of a prompt and the same query alone against the cache see the same keys."""
    B, S, H, G, D = 2, 333, 8, 2, 128
    q, k, v, do, extra, how = attention_case(B, S, S, H, G, D, "bf16", "bshd", 4, causal=True, softcap=30.0)
    o, lse = attention_run(client, q, k, v, do, extra, how, "bf16", "bshd", gradient=False)
    extra = {"lengths": torch.tensor([S, S], dtype=torch.int32)}
    o1, lse1 = attention_run(client, q[:, -1:].contiguous(), k, v, do, extra, {**how, "queries_at_end": True}, "bf16", "bshd", gradient=False)
    want = ref.attention(q, k, v, "bf16", "bshd", D ** -0.5, **how)
    within(o1, want["o"][0][:, -1:], want["o"][1][:, -1:], "o")
    within(lse1, want["lse"][0][:, :, -1:], want["lse"][1][:, :, -1:], "lse")
    within(o, *want["o"], "prompt")
