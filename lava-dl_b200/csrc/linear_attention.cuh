// Shared by the translation units of the linear attention (api_linear_attention*.cu).
#pragma once

#include "api_util.cuh"

namespace sb {
namespace la {

constexpr int kMaxDim = 128;   // widest head

// One walk over time: o[t] = S[t]^T q[t].  The state's element (d, e) of a head lies at
// d * s_row + e * s_col, so that a walk on the transposed state reads and writes the caller's layout.
struct Walk {
  const float* q;
  const float* k;
  const float* v;
  float* o;
  const float* decay;
  const float* s_in;    // nullable: zero
  float* s_out;         // nullable
  int n_decay;          // 1 or heads per sample
  int64_t heads;
  int Dk, Dv;
  int64_t T;
  int64_t s_row, s_col;
  int reverse;          // from the last step to the first
  int after;            // the state decays before a step is added (1) or after it has been read (0)
  int64_t head0;        // the first head's place among all, for its decay
};

// Tensor-core walks (api_linear_attention_tc.cu): one launch for n <= 3 walks over the same heads and
// steps whose Dk lie on the same side of 64, with tc_scratch_floats() floats of scratch.
int64_t tc_scratch_floats(const Walk* walks, int n);
int tc_walks(const Walk* walks, int n, float* scratch, cudaStream_t s);

}  // namespace la
}  // namespace sb
