"""The operators' kernel entry points on torch tensors: strides, offsets behind 32 bits, other streams, captured graphs, memory around
the results, refusals."""
import ctypes as C

import pytest
import torch

import operators_reference as ref
from ryft_b200 import kernels as K

pytestmark = pytest.mark.gpu
ELEM = {torch.bfloat16: K.EL_BF16, torch.float16: K.EL_F16, torch.float32: K.EL_F32}


@pytest.fixture(scope="module")
def lib():
    return K.load()


def strides(t, layout="bhsd"):
    a = t.stride()
    return K.HeadStrides(a[0], a[2], a[1]) if layout == "bshd" else K.HeadStrides(a[0], a[1], a[2])


def attention_args(lib, q, k, v, o, lse=None, gradient=None, **options):
    """Tensors as [B, H, S, D]; `gradient`: (do, dq, dk, dv)."""
    a = K.HeadAttentionArgs()
    a.elem = ELEM[q.dtype]
    a.B, a.Hq, a.Sq, a.D = q.shape
    a.Hk, a.Sk = k.shape[1], k.shape[2]
    a.scale = options.pop("scale", a.D ** -0.5)
    for n, t in (("q", q), ("k", k), ("v", v), ("o", o)):
        setattr(a, n, t.data_ptr())
        setattr(a, n + "s", strides(t))
    if lse is not None:
        a.lse = lse.data_ptr()
    if gradient is not None:
        for (n, s), t in zip((("dout", "dos"), ("dq", "dqs"), ("dk", "dks"), ("dv", "dvs")), gradient):
            setattr(a, n, t.data_ptr())
            setattr(a, s, strides(t))
    for n, x in options.items():
        setattr(a, n, x.data_ptr() if isinstance(x, torch.Tensor) else x)
    scratch = torch.empty(max(16, lib.b2x_head_attention_scratch_bytes(C.byref(a), int(gradient is not None))), dtype=torch.uint8, device="cuda")
    a.scratch = scratch.data_ptr()
    a.keep = (q, k, v, o, lse, gradient, scratch, [x for x in options.values()])
    return a


def launch(lib, a, gradient=False, stream=None):
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    torch.cuda.current_stream().synchronize()
    f = lib.b2x_launch_head_attention_gradient if gradient else lib.b2x_launch_head_attention
    rc = f(C.byref(a), status.data_ptr(), (stream or torch.cuda.current_stream()).cuda_stream)
    return rc, status


def make(seed, B, Hq, Hk, Sq, Sk, D, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)  # noqa: E731
    return n(B, Hq, Sq, D), n(B, Hk, Sk, D), n(B, Hk, Sk, D), n(B, Hq, Sq, D)


def close(got, want, bound, what):
    got, want, bound = got.double().cpu(), want, bound.expand_as(want)
    assert torch.isfinite(got).all() and ((got - want).abs() <= bound).all(), f"{what}: {float(((got - want).abs() / bound).max()):.3g} of the bound"


def inside(t, pad):
    """A copy of t inside a larger tensor of sevens, a view of every dimension but the last; and the larger tensor."""
    big = torch.full([s + 2 * pad for s in t.shape[:-1]] + [t.shape[-1] + 16], 7.0, dtype=t.dtype, device="cuda")
    view = big[pad:pad + t.shape[0], pad:pad + t.shape[1], pad:pad + t.shape[2], 8:8 + t.shape[3]]
    view.copy_(t)
    return view, big


def untouched(big, view):
    view.fill_(7.0)
    return bool((big == 7.0).all())


@pytest.mark.parametrize("Sq,Sk,D", [(200, 300, 80), (1, 300, 128), (3, 70, 64), (130, 130, 128)])
def test_views_into_larger_tensors_and_nothing_around_them(lib, Sq, Sk, D):
    q, k, v, do = make(1, 2, 4, 2, Sq, Sk, D)
    want = ref.attention(q.cpu(), k.cpu(), v.cpu(), "bf16", "bhsd", D ** -0.5, do=do.cpu(), causal=True, query_offset=Sk - Sq)
    (q, _), (k, _), (v, _), (do, _) = [inside(t, 1) for t in (q, k, v, do)]
    (o, bo), (dq, bq), (dk, bk), (dv, bv) = [inside(torch.zeros_like(t), 1) for t in (q, q, k, v)]
    lse = torch.zeros(2, 4, Sq, device="cuda")
    a = attention_args(lib, q, k, v, o, lse, (do, dq, dk, dv), causal=1, query_offset=Sk - Sq)
    f = attention_args(lib, q, k, v, o, lse, causal=1, query_offset=Sk - Sq)
    rc, s1 = launch(lib, f)
    assert rc == 0
    rc, s2 = launch(lib, a, True)
    assert rc == 0
    torch.cuda.synchronize()
    assert not s1.item() and not s2.item()
    for n, t in (("o", o), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
        close(t, *want[n], n)
    for big, view in ((bo, o), (bq, dq), (bk, dk), (bv, dv)):
        assert untouched(big, view)


@pytest.mark.parametrize("Sq", [1, 32])
def test_keys_behind_two_to_the_32_bytes(lib, Sq):
    """The last keys of a cache of 2.2 * 2^31 elements, of which a query sees only those (their scores stand out)."""
    Sk, D, H = 1 << 20, 128, 18
    k = torch.zeros(1, H, Sk, D, dtype=torch.bfloat16, device="cuda")
    assert k.numel() > 1 << 31
    v = torch.ones_like(k)
    q = torch.zeros(1, H, Sq, D, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = 64.0
    k[:, :, -3:, 0] = 32.0
    v[:, :, -3:] = 5.0
    v[0, -1, -3:] = 9.0
    o = torch.zeros_like(q)
    rc, status = launch(lib, attention_args(lib, q, k, v, o, scale=1.0))
    assert rc == 0
    torch.cuda.synchronize()
    want = torch.full_like(o, 5.0)
    want[0, -1] = 9.0
    assert not status.item() and torch.equal(o, want)


@pytest.mark.parametrize("Sq,softcap", [(300, 0.0), (300, 30.0), (2, 30.0)])
def test_captured_graphs_replayed_side_by_side(lib, Sq, softcap):
    """Two graphs of one stream (forward and, for many queries, backward), replayed on two others at once."""
    cases = []
    side = torch.cuda.Stream()
    for seed in (1, 2):
        q, k, v, do = make(seed, 2, 8, 4, Sq, 700, 64)
        o, lse = torch.empty_like(q), torch.empty(2, 8, Sq, device="cuda")
        grads = (do, torch.empty_like(q), torch.empty_like(k), torch.empty_like(v))
        options = dict(causal=1, query_offset=700 - Sq, softcap=softcap)
        f, b = attention_args(lib, q, k, v, o, lse, **options), attention_args(lib, q, k, v, o, lse, grads, **options)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")

        def both(stream):
            assert lib.b2x_launch_head_attention(C.byref(f), status.data_ptr(), stream.cuda_stream) == 0
            assert lib.b2x_launch_head_attention_gradient(C.byref(b), status.data_ptr(), stream.cuda_stream) == 0
        both(side)                                  # and once outside a capture
        side.synchronize()
        first = [t.clone() for t in (o, lse, *grads[1:])]
        for t in (o, lse, *grads[1:]):
            t.zero_()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            both(torch.cuda.current_stream())
        cases.append((graph, first, (o, lse, *grads[1:]), status, (f, b)))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for s, c in zip(streams, cases):
            with torch.cuda.stream(s):
                c[0].replay()
    torch.cuda.synchronize()
    for _, first, now, status, _ in cases:
        assert not status.item()
        for a, b in zip(first, now):
            assert torch.equal(a, b)


@pytest.mark.parametrize("S", [66_000, 132_000])
def test_documents_of_more_tokens_than_lists_cover(lib, S):
    """A row of documents of 500 tokens, each against the same document alone; behind 65536 (gradient) and 131072 (forward) tokens blocks
    are no longer listed but compared one by one."""
    D, n = 64, S // 500
    q, k, v, do = make(5, 1, 1, 1, S, S, D)
    documents = (torch.arange(S, device="cuda", dtype=torch.int32) // 500)[None].contiguous()
    o, lse = torch.empty_like(q), torch.empty(1, 1, S, device="cuda")
    grads = (do, torch.empty_like(q), torch.empty_like(k), torch.empty_like(v))
    for gradient in (False, True):
        rc, status = launch(lib, attention_args(lib, q, k, v, o, lse, grads if gradient else None, causal=1, documents=documents), gradient)
        torch.cuda.synchronize()
        assert rc == 0 and not status.item()
    alone = lambda t: t.cpu().reshape(n, 500, 1, D)  # noqa: E731
    pick = [0, 1, n // 2, n - 2, n - 1]
    want = ref.attention(*[alone(t)[pick] for t in (q, k, v)], "bf16", "bshd", D ** -0.5, do=alone(do)[pick], causal=True)
    for name, t in (("o", o), ("dq", grads[1]), ("dk", grads[2]), ("dv", grads[3])):
        close(alone(t)[pick], *want[name], name)
    close(lse.cpu().reshape(n, 1, 500)[pick], *want["lse"], "lse")


def test_what_cannot_be_addressed_is_refused(lib):
    q, k, v, do = make(3, 1, 2, 2, 40, 40, 64)
    o, lse = torch.zeros_like(q), torch.zeros(1, 2, 40, device="cuda")

    def refused(change, gradient=False):
        a = attention_args(lib, q, k, v, o, lse, (do, torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)) if gradient else None)
        change(a)
        before = lib.b2x_kernel_launch_count()
        assert launch(lib, a, gradient)[0] != 0 and lib.b2x_kernel_launch_count() == before
    refused(lambda a: setattr(a, "q", a.q + 2))                      # rows start on 16 bytes
    refused(lambda a: setattr(a.ks, "token", 65))
    refused(lambda a: setattr(a, "elem", K.EL_F32))
    refused(lambda a: setattr(a, "D", 60))
    refused(lambda a: setattr(a, "Hk", 3))
    refused(lambda a: setattr(a, "softcap", -1.0))
    refused(lambda a: setattr(a, "queries_at_end", 1))               # without lengths
    refused(lambda a: setattr(a, "lse", None), True)
    refused(lambda a: setattr(a, "scratch", None), True)
    refused(lambda a: setattr(a, "dv", a.dv + 8), True)
    torch.cuda.synchronize()


def rotary_args(lib, x, y, turns, gradient=False, dy=None, weight=None, dweight=None, positions=None, R=None, epsilon=1e-6):
    a = K.RotaryArgs()
    a.elem, a.weight_elem, a.n, a.norm = ELEM[y[0].dtype], K.EL_F32, len(y), int(weight is not None)
    a.B, _, a.S, a.D = y[0].shape
    a.R = a.D if R is None else R
    a.epsilon = epsilon
    for i in range(len(y)):
        a.heads[i] = y[i].shape[1]
        a.y[i], a.ys[i] = y[i].data_ptr(), strides(y[i])
        if x is not None:
            a.x[i], a.xs[i] = x[i].data_ptr(), strides(x[i])
        if dy is not None:
            a.dy[i], a.dys[i] = dy[i].data_ptr(), strides(dy[i])
        if weight is not None:
            a.weight[i] = weight[i].data_ptr()
        if dweight is not None:
            a.dweight[i] = dweight[i].data_ptr()
    a.turns = turns.data_ptr()
    if positions is not None:
        a.positions = positions.data_ptr()
    scratch = torch.empty(max(16, lib.b2x_rotary_scratch_bytes(C.byref(a))), dtype=torch.uint8, device="cuda")
    a.scratch = scratch.data_ptr()
    a.keep = (x, y, dy, weight, dweight, positions, turns, scratch)
    return a


def turns_of(R):
    f = ref.frequencies(R) / (2 * torch.pi)
    return torch.tensor([int(float(x) * 2 ** 53) * 2 ** 11 for x in f], dtype=torch.int64, device="cuda")


@pytest.mark.parametrize("start", [8, 1])       # rows that start on 16 bytes, and rows that do not
def test_rotary_on_views_and_another_stream(lib, start):
    B, H, S, D = 2, 3, 37, 64
    g = torch.Generator(device="cuda").manual_seed(0)
    big = [torch.randn(B, h, S, D + 16, generator=g, device="cuda").bfloat16() for h in (H, 1)]
    x = [t[..., start:start + D] for t in big]
    out = [torch.full_like(t, 7.0) for t in big]
    y = [t[..., start:start + D] for t in out]
    w = [1 + 0.1 * torch.randn(D, generator=g, device="cuda") for _ in big]
    pos = torch.randint(0, 1 << 20, (B, S), generator=g, device="cuda", dtype=torch.int32)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    assert lib.b2x_launch_rotary(C.byref(rotary_args(lib, x, y, turns_of(D), weight=w, positions=pos)), s.cuda_stream) == 0
    dx, dw = [torch.empty_like(t) for t in x], [torch.empty(D, device="cuda") for _ in x]
    assert lib.b2x_launch_rotary_gradient(C.byref(rotary_args(lib, x, dx, turns_of(D), dy=x, weight=w, dweight=dw, positions=pos)), s.cuda_stream) == 0
    s.synchronize()
    for i in range(2):
        args = (pos.cpu(), w[i].cpu(), "bf16", "bhsd", D, False, 1e-6)
        # the table above holds 53 bits of a turn: at a million positions 2^-33 of a turn, far below the bound
        close(y[i], *ref.rotary(x[i].cpu(), *args), "y")
        want, bound, wantw, boundw = ref.rotary_gradient(x[i].cpu(), x[i].cpu(), *args)
        close(dx[i], want, bound, "dx")
        close(dw[i], wantw, boundw, "dw")
        out[i][..., start:start + D] = 7.0
        assert (out[i] == 7.0).all()


def test_a_head_of_zeros_without_epsilon_spoils_its_own_gradient_only(lib):
    x = torch.ones(1, 3, 2, 16, device="cuda")
    dy = torch.ones_like(x)
    w, dw, dx = torch.ones(16, device="cuda"), torch.empty(16, device="cuda"), torch.empty_like(x)
    assert lib.b2x_launch_rotary_gradient(C.byref(rotary_args(lib, [x], [dx], turns_of(16), dy=[dy], weight=[w], dweight=[dw], epsilon=0.0)), None) == 0
    torch.cuda.synchronize()
    assert torch.isfinite(dw).all() and torch.isfinite(dx).all()
