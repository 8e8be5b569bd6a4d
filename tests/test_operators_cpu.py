"""The named operators without a GPU: how they are read, what is refused, and the 64-bit forms against differences."""
import ctypes

import pytest
import torch

import operators_reference as ref
import ryft_b200
from ryft_b200 import kernels, pjrt
from ryft_b200.stablehlo import Builder


def plan(make):
    b = Builder()
    return ryft_b200.plan_dump(b.build(*make(b)))


def refused(make, code, *needles):
    with pytest.raises(pjrt.PjrtError) as e:
        plan(make)
    assert e.value.code_name == code, e.value.message
    for n in needles:
        assert n in e.value.message, e.value.message


def heads(b, B=2, H=4, S=8, D=64, dtype="bf16"):
    return b.arg([B, H, S, D], dtype)


def test_a_call_is_one_step_and_its_operands_stay_where_they_are():
    dump = plan(lambda b: b.rotary([b.transpose(b.arg([2, 8, 4, 64], "bf16"), [0, 2, 1, 3])]))
    assert "1 steps" in dump and "call b2x.rotary" in dump and "(arg0) -> (out0)" in dump
    dump = plan(lambda b: [b.attention(heads(b), heads(b, H=2), heads(b, H=2), causal=True, softcap=30.0)])
    assert "1 steps" in dump and "call b2x.attention" in dump


def test_scratch_covers_what_the_operands_ask_for():
    # ranges of document numbers, 8 bytes per 128 keys; the gradient's delta, 4 bytes per query and head
    call = lambda b: dict(documents=b.arg([2, 300], "i32"), causal=True)  # noqa: E731
    dump = plan(lambda b: [b.attention(*[heads(b, S=300) for _ in range(3)], **call(b))])
    assert "scratch=48 B" in dump
    dump = plan(lambda b: [b.attention(*[heads(b, S=300) for _ in range(3)], causal=True)])
    assert "scratch=0 B" in dump


@pytest.mark.parametrize("B,Hq,Hk,Sq,Sk,D,causal,q_parts,k_parts", [
    (1, 2, 1, 1300, 1300, 128, 1, 2, 4),
    (1, 1, 1, 1100, 2100, 64, 0, 3, 2),
    (1, 12, 1, 200, 200, 128, 1, 1, 5),
    (1, 2, 2, 20, 1200, 40, 1, 2, 1),
    (1, 16, 4, 8192, 8192, 128, 1, 1, 1),
    (1, 1, 1, 40000, 100, 64, 0, 1, 16),
    (0, 2, 1, 100, 100, 64, 0, 1, 1),
    (1, 1, 1, 0, 100, 64, 0, 1, 1),
    (1, 0, 0, 100, 100, 64, 0, 1, 1),
])
def test_scratch_and_launches_of_gradients_in_parts(B, Hq, Hk, Sq, Sk, D, causal, q_parts, k_parts):
    lib = kernels.load()
    a = kernels.HeadAttentionArgs(elem=10, causal=causal, B=B, Hq=Hq, Hk=Hk, Sq=Sq, Sk=Sk, D=D)
    rows, keys, wide = -(-Sq // 128) * 128, -(-Sk // 128) * 128, 64 if D <= 64 else 128
    parts = max(q_parts * B * Hq * rows * wide * 4 if q_parts > 1 else 0, k_parts * 2 * B * Hk * keys * wide * 4 if k_parts > 1 else 0)
    assert lib.b2x_head_attention_scratch_bytes(ctypes.byref(a), 1) == B * Hq * rows * 8 + parts
    tiles = (2 + (q_parts > 1) if B * Hq * Sq else 0) + (1 + (k_parts > 1) if B * Hk * Sk else 0)
    assert lib.b2x_head_attention_launches(ctypes.byref(a), 1) == tiles



@pytest.mark.parametrize("B,Hq,Sq,Sk,D,causal,parts", [(1, 2, 1300, 1300, 128, 1, 2), (1, 1, 1100, 2100, 64, 0, 4), (1, 2, 130, 2500, 80, 0, 5), (1, 1, 17, 100000, 64, 0, 16),
                                                       (1, 16, 8192, 8192, 128, 1, 1), (1, 16, 2048, 2048, 128, 1, 1), (1, 8, 4096, 4096, 128, 1, 2), (3, 12, 1000, 1000, 64, 0, 1), (1, 1, 200, 500, 64, 0, 1), (0, 1, 200, 5000, 64, 0, 1), (1, 1, 200, 0, 64, 0, 1)])
def test_scratch_and_launches_of_attention_in_parts(B, Hq, Sq, Sk, D, causal, parts):
    lib = kernels.load()
    a = kernels.HeadAttentionArgs(elem=10, causal=causal, B=B, Hq=Hq, Hk=Hq, Sq=Sq, Sk=Sk, D=D)
    rows = B * Hq * -(-Sq // 128) * 128
    assert lib.b2x_head_attention_scratch_bytes(ctypes.byref(a), 0) == (parts * rows * ((64 if D <= 64 else 128) * 4 + 8) if parts > 1 else 0)
    assert lib.b2x_head_attention_launches(ctypes.byref(a), 0) == (0 if B == 0 else 1 + (parts > 1))


def test_rows_that_are_not_contiguous_are_copied():
    dump = plan(lambda b: b.rotary([b.transpose(b.arg([2, 4, 64, 8], "bf16"), [0, 1, 3, 2])]))
    assert "copy:call_operand" in dump and "2 steps" in dump


def test_both_printed_forms_are_read():
    body = {"pretty": 'stablehlo.custom_call @b2x.rotary(%arg0) {api_version = 4 : i32, backend_config = {base = 1.0e+04 : f64, rotary_dims = 32 : i64}}',
            "generic": '"stablehlo.custom_call"(%arg0) <{api_version = 4 : i32, backend_config = {base = 1.0e+04 : f64, rotary_dims = 32 : i64}, '
                       'call_target_name = "b2x.rotary", has_side_effect = false}>'}
    for name, op in body.items():
        text = ("module {\n  func.func @main(%arg0: tensor<2x4x8x64xbf16>) -> tensor<2x4x8x64xbf16> {\n"
                f"    %0 = {op} : (tensor<2x4x8x64xbf16>) -> tensor<2x4x8x64xbf16>\n    return %0 : tensor<2x4x8x64xbf16>\n  }}\n}}\n")
        assert "call b2x.rotary" in ryft_b200.plan_dump(text), name


@pytest.mark.parametrize("code,needle,make", [
    ("UNIMPLEMENTED", "element types", lambda b: b.rotary([heads(b, dtype="i32")])),
    ("UNIMPLEMENTED", "256", lambda b: b.rotary([heads(b, D=264)])),
    ("UNIMPLEMENTED", "one or two", lambda b: b.rotary([heads(b), heads(b), heads(b)])),
    ("INVALID_ARGUMENT", "rotary_dims", lambda b: b.rotary([heads(b)], rotary_dims=66)),
    ("INVALID_ARGUMENT", "rotary_dims", lambda b: b.rotary([heads(b)], rotary_dims=31)),
    ("INVALID_ARGUMENT", "operand 1", lambda b: b.rotary([heads(b), heads(b, S=9)])),
    ("INVALID_ARGUMENT", "positions", lambda b: b.rotary([heads(b)], positions=b.arg([2, 9], "i32"))),
    ("INVALID_ARGUMENT", "positions", lambda b: b.rotary([heads(b)], positions=b.arg([2, 8], "i64"))),
    ("INVALID_ARGUMENT", "weights", lambda b: b.rotary([heads(b)], weights=[b.arg([64], "f16")], epsilon=1e-6)),
    ("INVALID_ARGUMENT", "operand 1", lambda b: b.rotary([heads(b)], weights=[b.arg([32], "f32")], epsilon=1e-6)),
    ("INVALID_ARGUMENT", "factor", lambda b: b.rotary([heads(b)], factor=0.0)),
    ("INVALID_ARGUMENT", "base", lambda b: b.rotary([heads(b)], base=0.5)),
    ("INVALID_ARGUMENT", "bands", lambda b: b.rotary([heads(b)], bands=(4.0, 1.0, 8192))),
    ("INVALID_ARGUMENT", "epsilon", lambda b: b.rotary([heads(b)], weights=[b.arg([64], "f32")], epsilon=-1.0)),
    ("INVALID_ARGUMENT", "layout", lambda b: b.rotary([heads(b)], layout="sbhd")),
    ("INVALID_ARGUMENT", "four dimensions", lambda b: b.rotary([b.arg([8, 64], "bf16")])),
    ("UNIMPLEMENTED", "element types", lambda b: [b.attention(*[heads(b, dtype="f32") for _ in range(3)])]),
    ("UNIMPLEMENTED", "multiple of 8", lambda b: [b.attention(*[heads(b, D=60) for _ in range(3)])]),
    ("UNIMPLEMENTED", "multiple of 8", lambda b: [b.attention(*[heads(b, D=136) for _ in range(3)])]),
    ("INVALID_ARGUMENT", "multiple of the key heads", lambda b: [b.attention(heads(b), heads(b, H=3), heads(b, H=3))]),
    ("INVALID_ARGUMENT", "keys", lambda b: [b.attention(heads(b), heads(b, B=3), heads(b, B=3))]),
    ("INVALID_ARGUMENT", "values", lambda b: [b.attention(heads(b), heads(b), heads(b, S=9))]),
    ("INVALID_ARGUMENT", "prefix", lambda b: [b.attention(heads(b), heads(b), heads(b), prefix=b.arg([2], "i32"))]),
    ("INVALID_ARGUMENT", "lengths", lambda b: [b.attention(heads(b), heads(b), heads(b), queries_at_end=True)]),
    ("INVALID_ARGUMENT", "lengths", lambda b: [b.attention(heads(b), heads(b), heads(b), lengths=b.arg([3], "i32"))]),
    ("INVALID_ARGUMENT", "slopes", lambda b: [b.attention(heads(b), heads(b), heads(b), slopes=b.arg([3], "f32"))]),
    ("INVALID_ARGUMENT", "documents", lambda b: [b.attention(heads(b), heads(b), heads(b), documents=b.arg([2, 7], "i32"))]),
    ("INVALID_ARGUMENT", "place among the keys", lambda b: [b.attention(heads(b, S=9), heads(b), heads(b), documents=b.arg([2, 8], "i32"))]),
    ("INVALID_ARGUMENT", "softcap", lambda b: [b.attention(heads(b), heads(b), heads(b), softcap=-1.0)]),
    ("INVALID_ARGUMENT", "query_offset", lambda b: [b.attention(heads(b), heads(b), heads(b), query_offset=-1)]),
    ("INVALID_ARGUMENT", "exclude", lambda b: [b.attention(heads(b), heads(b), heads(b), query_offset=1, queries_at_end=True, lengths=b.arg([2], "i32"))]),
    ("INVALID_ARGUMENT", "log sums", lambda b: b.attention_gradient(heads(b), heads(b), heads(b), heads(b), b.arg([2, 4, 9], "f32"), heads(b))),
    ("INVALID_ARGUMENT", "gradient", lambda b: b.attention_gradient(heads(b), heads(b), heads(b), heads(b), b.arg([2, 4, 8], "f32"), heads(b, S=9))),
])
def test_refusals_name_what_is_wrong(code, needle, make):
    refused(make, code, "custom_call", needle)


@pytest.mark.parametrize("config,needle", [("{scale = 1.0 : f64, heads = 3 : i64}", "unknown attribute 'heads'"), ("{causal = 1 : i64}", "true or false"),
                                           ('{inputs = ["lengths"]}', "operands"), ('{inputs = ["mask"]}', "operands"), ('{scale = "big"}', "number")])
def test_attributes_are_checked(config, needle):
    t = "tensor<1x2x8x64xbf16>"
    text = (f"module {{\n  func.func @main(%arg0: {t}) -> {t} {{\n    %0 = stablehlo.custom_call @b2x.attention(%arg0, %arg0, %arg0) {{backend_config = {config}}} : "
            f"({t}, {t}, {t}) -> {t}\n    return %0 : {t}\n  }}\n}}\n")
    with pytest.raises(pjrt.PjrtError) as e:
        ryft_b200.plan_dump(text)
    assert e.value.code_name == "INVALID_ARGUMENT" and needle in e.value.message


# ---- the 64-bit gradients against differences ---------------------------------------------------------------------------------

def difference(f, x, d, h=1e-5):
    return (f(x + h * d) - f(x - h * d)) / (2 * h)


@pytest.mark.parametrize("mask", [dict(causal=True, softcap=3.0), dict(slopes=torch.tensor([0.5, 0.1])), dict(lengths=torch.tensor([4, 0]), softcap=2.0),
                                  dict(documents=torch.tensor([[0, 0, 1, 1, 1], [2, 1, 2, 1, 0]], dtype=torch.int32), causal=True)])
def test_attention_gradient_is_the_difference_quotient(mask):
    g = torch.Generator().manual_seed(0)
    rand = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)  # noqa: E731
    q, k, v, do = rand(2, 2, 5, 8), rand(2, 1, 5, 8), rand(2, 1, 5, 8), rand(2, 2, 5, 8)
    got = ref.attention(q, k, v, "bf16", "bhsd", 0.4, do=do, **mask)
    loss = lambda q, k, v: (ref.attention(q, k, v, "bf16", "bhsd", 0.4, **mask)["o"][0] * do).sum()  # noqa: E731
    for name, f, x in (("dq", lambda x: loss(x, k, v), q), ("dk", lambda x: loss(q, x, v), k), ("dv", lambda x: loss(q, k, x), v)):
        d = rand(*x.shape)
        assert abs(float(difference(f, x, d) - (got[name][0] * d).sum())) < 1e-7, name


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_gradient_is_the_difference_quotient(interleaved):
    g = torch.Generator().manual_seed(0)
    rand = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)  # noqa: E731
    x, dy, w, pos = rand(2, 3, 2, 10), rand(2, 3, 2, 10), rand(10), torch.tensor([[0, 5, 9], [7, 1, 100000]])
    args = ("f32", "bshd", 6, interleaved, 1e-3)
    dx, _, dw, _ = ref.rotary_gradient(dy, x, pos, w, *args)
    loss = lambda x, w: (ref.rotary(x, pos, w, *args)[0] * dy).sum()  # noqa: E731
    d, e = rand(*x.shape), rand(10)
    assert abs(float(difference(lambda a: loss(a, w), x, d) - (dx * d).sum())) < 1e-7
    assert abs(float(difference(lambda a: loss(x, a), w, e) - (dw * e).sum())) < 1e-7
