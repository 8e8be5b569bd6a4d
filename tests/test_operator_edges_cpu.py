"""The named operators at the edges of what is accepted, without a GPU: spellings of their options, and what the entry points refuse."""
import ctypes

import pytest

import ryft_b200
from ryft_b200 import kernels, pjrt

T = "tensor<1x2x8x64xbf16>"


def attention_text(dictionary, generic=False, target="b2x.attention"):
    op = (f'"stablehlo.custom_call"(%arg0, %arg0, %arg0) <{{call_target_name = "{target}"{", " if dictionary else ""}{dictionary}}}>' if generic
          else f"stablehlo.custom_call @{target}(%arg0, %arg0, %arg0) {{{dictionary}}}")
    return f"module {{\n  func.func @main(%arg0: {T}) -> {T} {{\n    %0 = {op} : ({T}, {T}, {T}) -> {T}\n    return %0 : {T}\n  }}\n}}\n"


def plan_refused(text, code, needle):
    with pytest.raises(pjrt.PjrtError) as e:
        ryft_b200.plan_dump(text)
    assert e.value.code_name == code and needle in e.value.message, e.value.message


# ---- spellings: an option is read or refused, never left out -------------------------------------------------------------------

@pytest.mark.parametrize("generic", [False, True])
@pytest.mark.parametrize("dictionary,needle", [
    ("backend_config = #foo.bar<causal>", "dictionary"),
    ("backend_config = #alias", "dictionary"),
    ("backend_config = @symbol", "dictionary"),
    ("backend_config = causal", "dictionary"),
    ('backend_config = "{causal = true}"', "dictionary"),
    ("mhlo.backend_config = #foo.bar<causal>", "dictionary"),
    ("causal = true", "causal"),
    ("dimensions = array<i64: 1>", "dimensions"),
    ("backend_configuration = {causal = true}", "backend_configuration"),
    ("backend_config = {causal = true}, mhlo.backend_config = {softcap = 3.0e+01 : f64}", "twice"),
    ("operand_layouts = [dense<[3, 1, 2, 0]> : tensor<4xi64>]", "operand_layouts"),
])
def test_options_that_are_not_read_are_refused(generic, dictionary, needle):
    plan_refused(attention_text(dictionary, generic), "UNIMPLEMENTED", needle)


@pytest.mark.parametrize("generic", [False, True])
def test_the_older_spelling_of_the_dictionary_is_read(generic):
    # under it, as under the other, options count: one that the operator does not have is refused
    assert "call b2x.attention" in ryft_b200.plan_dump(attention_text("mhlo.backend_config = {causal = true}", generic))
    plan_refused(attention_text("mhlo.backend_config = {heads = 3 : i64}", generic), "INVALID_ARGUMENT", "unknown attribute 'heads'")


@pytest.mark.parametrize("dictionary", ["", "api_version = 4 : i32, has_side_effect = false", 'backend_config = ""', "backend_config = {}",
                                        'mhlo.frontend_attributes = {key = "value"}, operand_layouts = [], result_layouts = [], called_computations = []'])
@pytest.mark.parametrize("generic", [False, True])
def test_attributes_that_change_nothing_are_accepted(generic, dictionary):
    assert "call b2x.attention" in ryft_b200.plan_dump(attention_text(dictionary, generic))


def test_a_name_given_twice_is_refused():
    plan_refused(attention_text("backend_config = {softcap = 3.0e+01 : f64, softcap = 5.0e+01 : f64}"), "INVALID_ARGUMENT", "twice")
    plan_refused(attention_text("api_version = 4 : i32, backend_config = {}, backend_config = {causal = true}"), "INVALID_ARGUMENT", "twice")


def test_numbers_written_as_their_bits_are_read_as_such():
    # MLIR prints infinities and NaN that way, and accepts it for every number
    assert "call b2x.attention" in ryft_b200.plan_dump(attention_text("backend_config = {softcap = 0x403E000000000000 : f64, scale = 0x3DCCCCCD : f32}"))
    plan_refused(attention_text("backend_config = {scale = 0x7FF0000000000000 : f64}"), "INVALID_ARGUMENT", "finite")
    plan_refused(attention_text("backend_config = {scale = 0x7FC00000 : f32}"), "INVALID_ARGUMENT", "finite")
    plan_refused(attention_text("backend_config = {softcap = 0xBFF0000000000000 : f64}"), "INVALID_ARGUMENT", "softcap")
    plan_refused(attention_text("backend_config = {scale = 0x3C00 : f16}"), "UNIMPLEMENTED", "f16")
    assert "call b2x.attention" in ryft_b200.plan_dump(attention_text("backend_config = {causal = true, query_offset = 0x10 : i64}"))


# ---- what the kernels' entry points refuse before they touch anything (cudaErrorInvalidValue, without a GPU) -----------------------

REFUSED = 1
SOMEWHERE = 1 << 12     # stands for memory: a call that is refused does not look at it


def attention_call(**change):
    a = kernels.HeadAttentionArgs(elem=kernels.EL_BF16, causal=1, B=2, Hq=4, Hk=2, Sq=32, Sk=48, D=64, scale=0.125)
    for n in ("q", "k", "v", "o", "dout", "dq", "dk", "dv", "lse", "scratch"):
        setattr(a, n, SOMEWHERE)
    for n, h, s in (("qs", 4, 32), ("os", 4, 32), ("dos", 4, 32), ("dqs", 4, 32), ("ks", 2, 48), ("vs", 2, 48), ("dks", 2, 48), ("dvs", 2, 48)):
        setattr(a, n, kernels.HeadStrides(h * s * 64, s * 64, 64))
    for n, x in change.items():
        setattr(a, n, x)
    return a


@pytest.mark.parametrize("gradient,change", [(g, c) for g in (False, True) for c in (
    dict(q=None), dict(k=None), dict(v=None), dict(o=None), dict(lse=SOMEWHERE + 2), dict(slopes=SOMEWHERE + 1), dict(documents=SOMEWHERE + 2),
    dict(prefix=SOMEWHERE + 3), dict(lengths=SOMEWHERE + 2), dict(B=-1), dict(Sq=-1), dict(Sk=-128), dict(Hq=-4), dict(Hk=-2), dict(Hq=0, Hk=-2),
    dict(B=1 << 40), dict(Hq=1 << 33, Hk=1), dict(scale=float("nan")), dict(softcap=float("nan")))
] + [(True, c) for c in (dict(dout=None), dict(dq=None), dict(dk=None), dict(dv=None), dict(lse=None))], ids=str)
@pytest.mark.parametrize("Sq", [1, 32])
def test_attention_without_its_memory_is_refused(gradient, change, Sq):
    lib = kernels.load()
    a = attention_call(**{"Sq": Sq, **change})
    before = lib.b2x_kernel_launch_count()
    f = lib.b2x_launch_head_attention_gradient if gradient else lib.b2x_launch_head_attention
    assert f(ctypes.byref(a), None, None) == REFUSED and lib.b2x_kernel_launch_count() == before


@pytest.mark.parametrize("change", [dict(B=0), dict(Hq=0, Hk=0), dict(B=0, q=None, k=None, v=None, o=None), dict(Sq=0, q=None, o=None)], ids=str)
def test_attention_of_nothing_needs_no_memory(change):
    lib = kernels.load()
    assert lib.b2x_launch_head_attention(ctypes.byref(attention_call(**change)), None, None) == 0


def rotary_call(elem, **change):
    a = kernels.RotaryArgs(elem=elem, weight_elem=kernels.EL_F32, n=2, norm=1, B=2, S=8, D=64, R=64, epsilon=1e-6)
    for i in range(2):
        a.heads[i] = 3
        for n in ("x", "y", "dy"):
            getattr(a, n)[i] = SOMEWHERE
            getattr(a, n + "s")[i] = kernels.HeadStrides(3 * 8 * 64, 8 * 64, 64)
        a.weight[i] = a.dweight[i] = SOMEWHERE
    a.turns = a.scratch = SOMEWHERE
    for n, x in change.items():
        if isinstance(x, tuple):
            getattr(a, n)[x[0]] = x[1]
        else:
            setattr(a, n, x)
    return a


@pytest.mark.parametrize("gradient,change", [(g, c) for g in (False, True) for c in (
    dict(x=(0, None)), dict(x=(1, SOMEWHERE + 1)), dict(y=(1, None)), dict(y=(0, SOMEWHERE + 1)), dict(weight=(1, None)), dict(weight=(0, SOMEWHERE + 2)),
    dict(turns=None), dict(turns=SOMEWHERE + 4), dict(positions=SOMEWHERE + 2), dict(B=-1), dict(S=-8), dict(B=1 << 40, S=1 << 40), dict(D=-64, R=0),
    dict(heads=(0, -1)), dict(heads=(1, 1 << 40)))
] + [(True, c) for c in (dict(dy=(1, None)), dict(dy=(0, SOMEWHERE + 1)), dict(dweight=(1, None)), dict(dweight=(0, SOMEWHERE + 2)), dict(scratch=None),
                         dict(scratch=SOMEWHERE + 2))], ids=str)
@pytest.mark.parametrize("elem", [kernels.EL_BF16, kernels.EL_F32])
def test_rotary_without_its_memory_is_refused(gradient, change, elem):
    lib = kernels.load()
    before = lib.b2x_kernel_launch_count()
    f = lib.b2x_launch_rotary_gradient if gradient else lib.b2x_launch_rotary
    assert f(ctypes.byref(rotary_call(elem, **change)), None) == REFUSED and lib.b2x_kernel_launch_count() == before


def test_rotary_of_nothing_needs_no_memory():
    lib = kernels.load()
    for change in (dict(D=0, R=0), dict(B=0, x=(0, None), turns=None), dict(S=0, weight=(1, None))):
        assert lib.b2x_launch_rotary(ctypes.byref(rotary_call(kernels.EL_BF16, **change)), None) == 0


# ---- scratch of f16 gradients -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("B,Hq,Hk,Sq,Sk,D,parts", [(4, 8, 4, 1500, 1500, 64, 0), (1, 2, 1, 1300, 1300, 128, 4 * 2 * 1 * 1408 * 128 * 4), (1, 0, 3, 200, 200, 64, 0), (1, 4, 2, 0, 200, 64, 0),
                                                   (0, 4, 2, 10, 10, 64, 0)])
def test_f16_gradients_have_room_for_the_sizes_of_their_rows(B, Hq, Hk, Sq, Sk, D, parts):
    """Beside the row constants (8 bytes a row) a squared length for each row and two for each key head; parts' sums start on 16 bytes."""
    lib = kernels.load()
    rows = -(-Sq // 128) * 128
    of = lambda elem: lib.b2x_head_attention_scratch_bytes(ctypes.byref(kernels.HeadAttentionArgs(  # noqa: E731
        elem=elem, causal=1, B=B, Hq=Hq, Hk=Hk, Sq=Sq, Sk=Sk, D=D)), 1)
    assert of(kernels.EL_BF16) == B * Hq * rows * 8 + parts
    head = B * Hq * rows * 12 + B * Hk * 8
    assert of(kernels.EL_F16) == (-(-head // 16) * 16 + parts if parts else head)
