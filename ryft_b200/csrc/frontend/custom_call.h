// The operators a program names through stablehlo.custom_call: their attributes and operands, read from an op and checked.
//
//   @b2x.rotary              x.. [, weights..] [, positions]            -> y..
//   @b2x.rotary_gradient     dy.. [, x.., weights..] [, positions]      -> dx.. [, dweights..]
//   @b2x.attention           q, k, v [, slopes] [, documents] [, prefix] [, lengths]            -> o [, log_sum]
//   @b2x.attention_gradient  q, k, v, o, log_sum, do [, slopes] [, documents] [, prefix] [, lengths] -> dq, dk, dv
//
// Attributes are the entries of the op's `backend_config` dictionary.  Tensors of heads are [B, H, S, D] (`layout = "bhsd"`, the
// default) or [B, S, H, D] ("bshd").
#pragma once
#include "ir.h"

namespace b2x {

struct RotarySpec {
  bool gradient = false, norm = false, interleaved = false, bshd = false;
  int n = 1;                          // tensors: 1 or 2
  int64_t B = 0, S = 0, D = 0, R = 0;
  int64_t heads[2] = {0, 0};
  DType dtype = DType::BF16, weight_dtype = DType::F32;
  double base = 10000.0, factor = 1.0;
  bool bands = false;
  double low = 1.0, high = 4.0, original = 8192.0;
  double epsilon = 0.0;
  // operand numbers, -1 where absent: x[i] (or dy[i] of a gradient without norms), dy[i], weights[i], positions
  int x[2] = {-1, -1}, dy[2] = {-1, -1}, w[2] = {-1, -1}, positions = -1;
  // Turns per position of each rotated pair, as fractions of 2^64.
  std::vector<uint64_t> turns() const;
};

struct AttentionSpec {
  bool gradient = false, bshd = false, causal = false, queries_at_end = false, log_sum = false;
  int64_t B = 0, Hq = 0, Hk = 0, Sq = 0, Sk = 0, D = 0;
  DType dtype = DType::BF16;
  double scale = 1.0, softcap = 0.0;
  int64_t query_offset = 0;
  int slopes = -1, documents = -1, prefix = -1, lengths = -1;   // operand numbers, -1 where absent
};

enum class CallKind { ROTARY, ATTENTION };
struct CallSpec {
  CallKind kind = CallKind::ROTARY;
  RotarySpec rotary;
  AttentionSpec attention;
};

// Throws CompileError: UNIMPLEMENTED for a target this executor does not provide or a size it has no kernel for, INVALID_ARGUMENT
// for operands, results or attributes that contradict the operator.
CallSpec describe_call(const Op& op);

}  // namespace b2x
