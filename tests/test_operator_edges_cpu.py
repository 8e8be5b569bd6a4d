"""The named operators at the edges of what is accepted, without a GPU: spellings of their options, and what the entry points refuse."""
import pytest

import ryft_b200
from ryft_b200 import pjrt

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
