// Routing that is trained: what balance.hip and the C entry points share.
#pragma once
#include "common.hpp"

namespace gmlp {

struct BalanceArgs {
  const void* logits;          // [M, E]
  const unsigned char* mask;   // [M], nullable: 0 leaves the token out of counts and loss
  float* weights;              // [M, top_k]
  int64_t* experts;            // [M, top_k]
  int64_t* counts;             // [E]
  float* loss;                 // [1]
  float* slope;                // [E]: d loss / d (sum over the counted tokens of p_e)
  float* partial;              // [workgroups][balance_partial(E)]
  const float* d_weights;      // [M, top_k], nullable
  const float* d_loss;         // [1], nullable
  void* d_logits;              // [M, E]
  int64_t M;
  int E, top_k, normalize;
};
// What a workgroup of the first stage leaves: for each expert the sum of its probabilities and (as an int) its choices, and
// the number of tokens.
inline __host__ __device__ int balance_partial(int E) { return 2 * E + 1; }
int balance_workgroups(int64_t M, int E);

template <typename L>
hipError_t launch_balance_fwd(const BalanceArgs& a, hipStream_t s);
template <typename L>
hipError_t launch_balance_bwd(const BalanceArgs& a, hipStream_t s);

}  // namespace gmlp
