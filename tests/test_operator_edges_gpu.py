"""The named operators at the edges of what they accept, on the GPU, against 64-bit forms (operators_reference.py)."""
import ctypes as C
import threading

import pytest
import torch

import operators_reference as ref
import test_operator_kernels_gpu as direct
import test_operators_gpu as program
from ryft_b200 import kernels as K
from ryft_b200 import pjrt

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def client():
    c = pjrt.load_cuda_13_plugin().client({"visible_devices": [0]})
    yield c
    c.close()


@pytest.fixture(scope="module")
def lib():
    return K.load()


# ---- no query heads -----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("documents", [False, True])
def test_key_heads_without_query_heads_have_gradients_of_zero(lib, documents):
    B, Hk, S, D = 2, 3, 200, 72
    q, k, v, do = direct.make(1, B, 0, Hk, S, S, D)
    o, lse = torch.empty_like(q), torch.empty(B, 0, S, device="cuda")
    grads = (do, torch.empty_like(q), torch.full_like(k, 7.0), torch.full_like(v, 7.0))
    options = {"documents": torch.zeros(B, S, dtype=torch.int32, device="cuda")} if documents else {}
    a = direct.attention_args(lib, q, k, v, o, lse, grads, causal=1, **options)
    before = lib.b2x_kernel_launch_count()
    rc, status = direct.launch(lib, a, True)
    torch.cuda.synchronize()
    assert rc == 0 and not status.item()
    assert lib.b2x_kernel_launch_count() - before == lib.b2x_head_attention_launches(C.byref(a), 1)
    assert not grads[2].any() and not grads[3].any()


# ---- caps over the whole accepted range ------------------------------------------------------------------------------------------

CAPS = [
    dict(B=2, Sq=1, Sk=300, Hq=4, Hk=2, D=64, dtype="f16", layout="bhsd"),
    dict(B=1, Sq=5, Sk=700, Hq=2, Hk=1, D=128, dtype="bf16", layout="bshd"),
    dict(B=1, Sq=150, Sk=150, Hq=2, Hk=1, D=128, dtype="f16", layout="bshd"),
]


@pytest.mark.parametrize("softcap", [1e-6, 1e-3, 1e3, 1e4, 1e5, 1e6])
@pytest.mark.parametrize("options", [dict(), dict(slopes=True), dict(scale=-0.2), dict(causal=True)], ids=str)
@pytest.mark.parametrize("sizes", CAPS, ids=str)
def test_caps_of_any_size(client, sizes, options, softcap):
    """A cap far above the scores changes hardly anything: its error must go with the score, not with the cap.

    Far below them the gradient is a matter of chance in 32 bits: an error of a product, 2^-24 of the sum of its terms' sizes (some 100
    here, times the scale: 1e-6), is 1e-3 of a cap of 1e-3 and 1 of a cap of 1e-6, and e^-2x changes by twice that.  There o and the log sums count."""
    how, sizes = dict(options), dict(sizes)
    dtype, layout = sizes["dtype"], sizes["layout"]
    gradient = softcap >= 1
    q, k, v, do, extra, how = program.attention_case(**sizes, seed=7, softcap=softcap, **how)
    got = program.attention_run(client, q, k, v, do, extra, how, dtype, layout, gradient)
    scale = how.pop("scale", sizes["D"] ** -0.5)
    # the bounds are for scales that are positive: the same scores from queries of the other sign
    sign = -1.0 if scale < 0 else 1.0
    want = ref.attention(sign * q, k, v, dtype, layout, abs(scale), do=do if gradient else None, **extra, **how)
    for name, x in zip(("o", "lse", "dq", "dk", "dv"), got):
        program.within(x, sign * want[name][0] if name == "dq" else want[name][0], want[name][1], name)


@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("Sq", [2, 150])
def test_one_large_score_leaves_the_others_as_they_are(client, Sq, slopes):
    """One query whose scores go beyond its cap of 1e5, next to queries whose scores are a few units."""
    q, k, v, do, extra, how = program.attention_case(1, Sq, 200, 2, 1, 64, "f16", "bhsd", 5, softcap=1e5, slopes=slopes)
    q[:, :, 1] = (q[:, :, 1].float() * 2000).half()
    how["scale"] = 8.0
    q[:, :, 0] = (q[:, :, 0].float() / 64).half()
    q[:, :, 2:] = (q[:, :, 2:].float() / 64).half()
    got = program.attention_run(client, q, k, v, do, extra, how, "f16", "bhsd")
    scale = how.pop("scale")
    want = ref.attention(q, k, v, "f16", "bhsd", scale, do=do, **extra, **how)
    others = [i for i in range(Sq) if i != 1]
    for name, x in (("o", got[0]), ("lse", got[1]), ("dq", got[2])):
        program.within(x[:, :, others], want[name][0][:, :, others], want[name][1].expand_as(want[name][0])[:, :, others], name)


@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_scores_far_beyond_the_cap_keep_the_slope_of_it(client, sign):
    """1 - tanh^2 of scores of 3 to 8 caps, on either side of zero: 2e-2 down to 5e-7, each as good as the score's own rounding."""
    B, H, S, D, cap = 1, 2, 70, 64, 2.0
    q, k, v, do, extra, how = program.attention_case(B, S, S, H, H, D, "f16", "bhsd", 3, softcap=cap)
    q, k = torch.zeros_like(q), torch.zeros_like(k)
    q[..., 0] = sign
    k[..., 0] = torch.linspace(6.0, 16.0, S)
    q[..., 1:9], k[..., 1:9] = torch.randn(B, H, S, 8).half() / 16, torch.randn(B, H, S, 8).half() / 16
    do = (do.float() * 4096).half()
    got = program.attention_run(client, q, k, v, do, extra, {**how, "scale": 1.0}, "f16", "bhsd")
    want = ref.attention(q, k, v, "f16", "bhsd", 1.0, do=do, **extra, **how)
    for name, x in zip(("o", "lse", "dq", "dk", "dv"), got):
        program.within(x, *want[name], name)


@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("Sq", [1, 40])
def test_products_beyond_f32_are_capped(client, Sq, slopes):
    """Products of -2e77 are infinite in f32 and -softcap as a score: every key weighs the same."""
    q = torch.full((1, 2, Sq, 64), 1e38).bfloat16()
    k = torch.full((1, 1, 150, 64), -1e38).bfloat16()
    v = program.normal(1, [1, 1, 150, 64])[0].bfloat16()
    extra = {"slopes": torch.zeros(2)} if slopes else {}
    o, lse = program.attention_run(client, q, k, v, None, extra, {"softcap": 300.0}, "bf16", "bhsd", gradient=False)
    want = ref.attention(q, k, v, "bf16", "bhsd", 0.125, softcap=300.0, **extra)
    program.within(o, *want["o"], "o")
    program.within(lse, *want["lse"], "lse")


# ---- rows that see nothing, far distances ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("Sk", [40, 700])
def test_a_query_that_sees_nothing_yields_0_whatever_others_see(client, Sk):
    """Queries in front of the first token see nothing; the value that the last query sees may be infinite or not a number."""
    q, k, v, do, _, _ = program.attention_case(1, 3, Sk, 2, 1, 64, "bf16", "bhsd", 2)
    v[0, 0, 0, :5], v[0, 0, 0, 5:9] = float("inf"), float("nan")
    extra = {"lengths": torch.tensor([1], dtype=torch.int32)}
    o, lse = program.attention_run(client, q, k, v, do, extra, dict(causal=True, queries_at_end=True), "bf16", "bhsd", gradient=False)
    assert not o[:, :, :2].any() and torch.equal(lse[:, :, :2], torch.full((1, 2, 2), -float("inf")))
    assert torch.isinf(o[:, :, 2, :5]).all() and torch.isnan(o[:, :, 2, 5:9]).all() and torch.isfinite(o[:, :, 2, 9:]).all()


@pytest.mark.parametrize("Sq", [1, 17])
def test_distances_of_positions_that_f32_does_not_hold(lib, Sq):
    """The end of a cache of more than 2^24 tokens: neighbouring keys' distances differ by one, as near its start."""
    Sk, D, near = (1 << 24) + 333, 8, 4096
    k, v = torch.zeros(1, 1, Sk, D, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, 1, Sk, D, dtype=torch.bfloat16, device="cuda")
    q, k[:, :, -near:], v[:, :, -near:], _ = direct.make(1, 1, 2, 1, Sq, near, D)
    slopes = torch.tensor([0.5, 0.03], device="cuda")      # at a distance of `near` the weights are below e^-122
    o, lse = torch.empty_like(q), torch.empty(1, 2, Sq, device="cuda")
    rc, status = direct.launch(lib, direct.attention_args(lib, q, k, v, o, lse, slopes=slopes, query_offset=Sk - Sq, causal=1))
    torch.cuda.synchronize()
    assert rc == 0 and not status.item()
    want = ref.attention(q.cpu(), k[:, :, -near:].cpu(), v[:, :, -near:].cpu(), "bf16", "bhsd", D ** -0.5, slopes=slopes.cpu(), query_offset=near - Sq, causal=True)
    direct.close(o, *want["o"], "o")
    direct.close(lse, *want["lse"], "lse")


# ---- threads and streams ----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("Sq", [1, 40])
@pytest.mark.parametrize("gradient", [False, True])
def test_the_first_call_of_a_thread(lib, gradient, Sq):
    """A thread that has not used CUDA yet has no current context."""
    q, k, v, do = direct.make(1, 1, 2, 1, Sq, 70, 64)
    o, lse = torch.empty_like(q), torch.empty(1, 2, Sq, device="cuda")
    grads = (do, torch.empty_like(q), torch.empty_like(k), torch.empty_like(v))
    assert direct.launch(lib, direct.attention_args(lib, q, k, v, o, lse))[0] == 0
    a = direct.attention_args(lib, q, k, v, o, lse, grads if gradient else None)
    status, codes = torch.zeros(1, dtype=torch.int32, device="cuda"), []
    torch.cuda.synchronize()
    f = lib.b2x_launch_head_attention_gradient if gradient else lib.b2x_launch_head_attention
    t = threading.Thread(target=lambda: codes.append(f(C.byref(a), status.data_ptr(), None)))
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert codes == [0] and not status.item()


def test_threads_on_their_own_default_streams(lib):
    """Every thread's own stream has the same handle; calls of two threads run side by side and each yields what it yields alone."""
    per_thread, cases = 2, []
    for seed in (1, 2):
        q, k, v, do = direct.make(seed, 2, 8, 4, 1500, 1500, 64)
        o, lse = torch.empty_like(q), torch.empty(2, 8, 1500, device="cuda")
        grads = (do, torch.empty_like(q), torch.empty_like(k), torch.empty_like(v))
        f, b = direct.attention_args(lib, q, k, v, o, lse, causal=1), direct.attention_args(lib, q, k, v, o, lse, grads, causal=1)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        for a, gradient in ((f, False), (b, True)):
            assert direct.launch(lib, a, gradient)[0] == 0
        torch.cuda.synchronize()
        cases.append((f, b, status, (o, lse, *grads[1:]), [t.clone() for t in (o, lse, *grads[1:])]))
        for t in cases[-1][3]:
            t.zero_()
    torch.cuda.synchronize()
    failures, start = [], threading.Barrier(2)

    def work(f, b, status):
        start.wait()
        for _ in range(10):
            for launch, a in ((lib.b2x_launch_head_attention, f), (lib.b2x_launch_head_attention_gradient, b)):
                if launch(C.byref(a), status.data_ptr(), per_thread) != 0:
                    failures.append("launch")
    threads = [threading.Thread(target=work, args=c[:3]) for c in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failures
    for _, _, status, now, alone in cases:
        assert not status.item()
        for x, y in zip(now, alone):
            assert torch.equal(x, y)


# ---- f16 gradients of any size that f16 holds --------------------------------------------------------------------------------------

@pytest.mark.parametrize("size", [2.0 ** -20, 2.0 ** -10, 1e4, 4e4])
@pytest.mark.parametrize("sizes,options", [
    (dict(B=2, Sq=130, Sk=130, Hq=4, Hk=2, D=128), dict(causal=True)),
    (dict(B=1, Sq=200, Sk=200, Hq=2, Hk=1, D=64), dict(causal=True, softcap=20.0)),
    (dict(B=1, Sq=1100, Sk=1100, Hq=2, Hk=1, D=80), dict(lengths=[700], slopes=True)),      # in parts
], ids=str)
def test_f16_gradients_over_the_range_of_f16(client, sizes, options, size):
    """P (dP - delta) passes f16's largest value where the gradients do not.  Values behind a length may be anything."""
    q, k, v, do, extra, how = program.attention_case(**sizes, dtype="f16", layout="bhsd", seed=3, **options)
    do = (do.float().clamp(-1.2, 1.2) * size).half()
    v, k, q = v.float().clamp(-2, 2).half(), (k.float() / 4).half(), (q.float() / 4).half()
    if "lengths" in options:
        v[:, :, options["lengths"][0]:] = float("inf")
    got = program.attention_run(client, q, k, v, do, extra, how, "f16", "bhsd")
    want = ref.attention(q, k, v, "f16", "bhsd", sizes["D"] ** -0.5, do=do, **extra, **how)
    assert want["dq"][0].abs().max() < 65000 and want["dk"][0].abs().max() < 65000, "the case is meant to fit"
    for name, x in zip(("o", "lse", "dq", "dk", "dv"), got):
        fits = want[name][0].abs() < 65000       # dv itself is larger in places
        program.within(torch.where(fits, x.double(), 0.0), torch.where(fits, want[name][0], 0.0), want[name][1], name)


@pytest.mark.parametrize("S,D", [(4000, 128), (1500, 40)])
def test_f16_gradients_of_many_small_shares_keep_their_figures(client, S, D):
    """Every key has a weight of 1 / S, and P (dP - delta) lies below f16's normal values: rounded there it would have a step of 2^-24.

    Three roundings of relative 2^-11 at most (P or dS, the result, O behind delta), each of root mean square 2^-11 / sqrt(3), and results
    that are sums of many independent ones: below 2^-10 of the norm."""
    q, k, v, do, extra, how = program.attention_case(1, S, S, 2, 1, D, "f16", "bshd", 5)
    q = (q.float() / 1024).half()
    k, v, do = (k.float() * 8).half(), (v.float() * 8).half(), (do.float() * 2.0 ** -12).half()
    do[:, ::2] = (do[:, ::2].float() * 2.0 ** -3).half()
    got = program.attention_run(client, q, k, v, do, extra, how, "f16", "bshd")
    want = ref.attention(q, k, v, "f16", "bshd", D ** -0.5, do=do, **extra, **how)
    dq, true = got[2].double(), want["dq"][0]
    normal = true.abs() >= 2.0 ** -14           # of the result, too, only what f16 holds to its full width
    assert normal[:, 1::2].double().mean() > 0.5
    off = torch.where(normal, dq - true, 0.0).norm() / torch.where(normal, true, 0.0).norm()
    assert off < 2.0 ** -10, float(off)


def test_f16_queries_do_not_lose_figures_to_larger_ones(client):
    """Neighbouring queries whose gradients differ by 2^18: dq goes by its own row."""
    S, D = 300, 64
    q, k, v, do, extra, how = program.attention_case(1, S, S, 2, 2, D, "f16", "bhsd", 5)
    do = do.float().clamp(-2, 2)
    do[:, :, ::2] *= 2.0 ** 12
    do[:, :, 1::2] *= 2.0 ** -6
    do, k = do.half(), (k.float() * 4).half()
    q = (q.float() / 4).half()
    got = program.attention_run(client, q, k, v, do, extra, how, "f16", "bhsd")[2].double()[:, :, 1::2]
    true = ref.attention(q, k, v, "f16", "bhsd", D ** -0.5, do=do, **extra, **how)["dq"][0][:, :, 1::2]
    assert (got - true).norm() / true.norm() < 2.0 ** -10


def test_f16_gradients_in_captured_graphs(lib):
    """The sizes of dO and V are found anew in every replay."""
    q, k, v, do = direct.make(1, 2, 4, 2, 300, 300, 64, torch.float16)
    o, lse = torch.empty_like(q), torch.empty(2, 4, 300, device="cuda")
    grads = (do, torch.empty_like(q), torch.empty_like(k), torch.empty_like(v))
    assert direct.launch(lib, direct.attention_args(lib, q, k, v, o, lse, causal=1))[0] == 0
    a = direct.attention_args(lib, q, k, v, o, lse, grads, causal=1)
    status, side = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.cuda.Stream()
    large = do.clone().clamp_(-1, 1) * 8192
    small = do * 2.0 ** -8
    alone = []
    for x in (large, small):
        do.copy_(x)
        assert direct.launch(lib, a, True)[0] == 0
        torch.cuda.synchronize()
        alone.append([t.clone() for t in grads[1:]])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        assert lib.b2x_launch_head_attention_gradient(C.byref(a), status.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
    for _ in range(2):
        for x, want in zip((large, small), alone):
            do.copy_(x)
            graph.replay()
            torch.cuda.synchronize()
            assert not status.item()
            for t, w in zip(grads[1:], want):
                assert torch.isfinite(t).all() and torch.equal(t, w)


# ---- a bias by distance far from every key --------------------------------------------------------------------------------------

@pytest.mark.parametrize("causal", [False, True])
def test_the_bias_far_from_every_key(client, causal):
    """Queries 3000 to 3200 positions behind the last key, with slopes up to 1/2: biases around -1600, where f32 has a step of 1.2e-4.

    The bias is rounded (half a step, in log2 units of 1.44 times the size: 1.2e-4), then once more with the score: 2.4e-4 log2 units of
    the score, 1.7e-4 of the log sum and of a weight, against a bound of 2e-5 + 2e-6 * 1600 = 3.2e-3 and the f16 bound of o (F = 2e-4 and
    a rounding); the log sum itself is compared at an eighth of that bound."""
    q, k, v, do, extra, how = program.attention_case(1, 200, 300, 4, 2, 64, "f16", "bhsd", 5, slopes=True, causal=causal, query_offset=3300)
    extra["slopes"] = torch.tensor([0.5, 0.25, 0.43, 0.06])
    o, lse = program.attention_run(client, q, k, v, do, extra, how, "f16", "bhsd", gradient=False)
    want = ref.attention(q, k, v, "f16", "bhsd", 0.125, **extra, **how)
    program.within(o, *want["o"], "o")
    program.within(lse, want["lse"][0], want["lse"][1] / 8, "lse")


# ---- norms of nothing ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("D", [16, 17, 128])
def test_a_head_of_zeros_without_epsilon_is_not_a_number_and_the_others_are(lib, D):
    """Its root is 0: its own result and gradient are NaN, and so is the gradient of the weights, which it is part of; no other head's."""
    g = torch.Generator(device="cuda").manual_seed(4)
    x, dy = (torch.randn(2, 5, 3, D, generator=g, device="cuda") for _ in range(2))
    x[1, 2, 1] = 0.0
    w, dw = 1 + 0.1 * torch.randn(D, generator=g, device="cuda"), torch.empty(D, device="cuda")
    y, dx, turns, R = torch.empty_like(x), torch.empty_like(x), direct.turns_of(D // 2 * 2), D // 2 * 2
    assert lib.b2x_launch_rotary(C.byref(direct.rotary_args(lib, [x], [y], turns, weight=[w], R=R, epsilon=0.0)), None) == 0
    a = direct.rotary_args(lib, [x], [dx], turns, dy=[dy], weight=[w], dweight=[dw], R=R, epsilon=0.0)
    assert lib.b2x_launch_rotary_gradient(C.byref(a), None) == 0
    torch.cuda.synchronize()
    how = (torch.arange(3).expand(2, 3), w.cpu(), "f32", "bhsd", R, False, 0.0)
    others = torch.ones(2, 5, 3, dtype=torch.bool)
    others[1, 2, 1] = False
    want, bound = ref.rotary(x.cpu(), *how)
    direct.close(y[others.cuda()], want[others], bound[others], "y")
    want, bound, _, _ = ref.rotary_gradient(dy.cpu(), x.cpu(), *how)
    direct.close(dx[others.cuda()], want[others], bound[others], "dx")
    assert torch.isnan(y[1, 2, 1]).all() and torch.isnan(dx[1, 2, 1]).all() and torch.isnan(dw).all()


# ---- memory that a program is handed ------------------------------------------------------------------------------------------------

def test_views_off_their_boundary_are_refused_and_the_program_goes_on(client):
    """Rows of attention start on 16 bytes, values on their own size; a view that does not is an error of its execution, not a fault."""
    from ryft_b200.stablehlo import Builder

    def program_of(make):
        b = Builder()
        return client.compile(pjrt.Program.mlir(b.build(*make(b))))
    T = [1, 2, 40, 64]
    attention = program_of(lambda b: [b.attention(*[b.arg(T, "bf16") for _ in range(3)])])
    rotary = program_of(lambda b: b.rotary([b.arg(T, "bf16")]))
    memory = torch.randn(3, 2 * 40 * 64 + 64, device="cuda").bfloat16()
    torch.cuda.synchronize()

    def run(exe, n, off):
        bufs = [client.view_of_device_buffer(memory[i].data_ptr() + off, pjrt.BufferType.BF16, T, keep=memory) for i in range(n)]
        return program.collect(exe.execute([pjrt.ExecutionDeviceInputs(bufs)])[0])
    whole = run(attention, 3, 0)[0]
    for off in (2, 8):
        with pytest.raises(pjrt.PjrtError):
            run(attention, 3, off)
    with pytest.raises(pjrt.PjrtError):
        run(rotary, 1, 1)
    turned = run(rotary, 1, 2)[0]
    x = memory[0, 1:1 + 2 * 40 * 64].cpu().reshape(T)
    program.within(turned, *ref.rotary(x, torch.arange(40).expand(1, 40), None, "bf16", "bhsd", 64, False, 0.0), "y")
    assert torch.equal(run(attention, 3, 0)[0], whole)
