// dg_attention_mfma.hpp -- the entry points of the matrix-unit attention (bfloat16, heads of up to
// 128 channels).
#pragma once
#include "dg_attention.hpp"

namespace dg {

constexpr int kMfmaDim = 128;

void forward_mfma(const AttnArgs& a, hipStream_t s);

// By target: dq and stats; where a.dtab is set also the table's partial sums, whose number is
// returned (at most kMfmaTableParts or the heads, whichever is more).
constexpr int kMfmaTableParts = 256 * 4;
int backward_q_mfma(const AttnArgs& a, hipStream_t s);

// By source: dk and dv.
void backward_kv_mfma(const AttnArgs& a, hipStream_t s);

}  // namespace dg
