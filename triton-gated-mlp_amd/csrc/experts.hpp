// 4-bit weights and expert layers: what the kernels of experts.hip and the C entry points share.
#pragma once
#include "common.hpp"
#include "gmlp.h"

namespace gmlp {

constexpr int Q4_TILE = 16;          // weight rows of a tile
constexpr int Q4_BLOCK = 128;        // weight columns of a block
constexpr uint32_t EXPERTS_MAX_BYTES = 0x7fff0000u;  // a buffer descriptor of these kernels is shorter
constexpr int EXPERTS_MAX_M = 64;    // token rows of a call
constexpr int EXPERTS_MAX_E = 512;   // experts
constexpr int EXPERTS_MAX_K = 16;    // experts of a token

// One matrix of weights per expert: 16-bit [experts, rows, cols], or codes and scales of the 4-bit storage (gmlp.h).
struct ExpertWeights {
  const void* w;
  const void* scales;  // 4-bit weights only
};

// The routing of a call, which plan_kernel makes of the logits: device pointers into the caller's workspace.  An entry is an
// expert that is in use with some of its tokens, all of them up to the token tiles that the kernels take at once; one
// with more tokens has several.  Entries are in ascending order of expert and token.
struct ExpertPlan {
  int* active;      // [1 + entries]: how many, then their experts
  uint8_t* count;   // [entries]: tokens
  uint16_t* pairs;  // [entries][EXPERTS_MAX_M]: which, as token * top_k + the choice that the expert is
  int8_t* slot;     // [entries][EXPERTS_MAX_M], M <= 16: of a token, the choice that the expert is, -1: not chosen
  float* weight;    // [M * top_k]
};
inline int expert_entries(int M, int E, int top_k) {  // at most
  const int pairs = M * top_k, most = M > 16 ? E + pairs / 16 : E;
  return pairs < most ? pairs : most;
}

// Who runs through which expert: every token through the only one, with weight 1; as the plan says; or (gate/up), of one token,
// as the kernel finds from the logits itself, which then leaves the plan.
enum Routing : int { ROUTING_DENSE = 0, ROUTING_PLAN = 1, ROUTING_SOLO = 2 };

struct ExpertArgs {
  const void* x;      // [M, K]
  const void* bias[3];
  ExpertWeights gate, up, down;
  void* h;            // [M * top_k, N]; h_low: behind it another one, of what rounding to 16 bits left
  void* y;            // [M, K], of the activations' type or (y_f32, without partial) float
  float* partial;     // [parts][M, K], where the down projection's reduction is split
  int M, K, N, E, top_k, act;
  int y_f32, h_low;
  int routing;        // Routing
  int cus;            // compute units of the device
  const void* logits; // [M, E] of a GMLP_* type
  int logits_dtype, normalize;
  ExpertPlan plan;
};

// Whether the hidden states of M tokens come as two 16-bit values each, whether ROUTING_SOLO takes the call, and the bytes of `partial` that launch_experts_down asks for (it does with none).
inline int experts_h_low(int64_t M, int group) { return M <= (group ? GMLP_H_PAIR_ROWS_Q4 : GMLP_H_PAIR_ROWS_16BIT); }
bool experts_solo(int M, int E);
size_t experts_partial_bytes(const ExpertArgs& a, int group);

// Gate/up, then down, on 16-bit (group = 0) or 4-bit weights (group = 32, 64 or 128).
template <typename T>
hipError_t launch_experts_gateup(const ExpertArgs& a, int group, hipStream_t s);
// y[M, a.K] = sum over experts of weight * h[., a.N]·W_downᵀ (+ bias[2])
template <typename T>
hipError_t launch_experts_down(const ExpertArgs& a, int group, hipStream_t s);
template <typename L>
hipError_t launch_experts_plan(const L* logits, const ExpertArgs& a, hipStream_t s);
template <typename L>
hipError_t launch_route(const L* logits, float* weights, int64_t* experts, int64_t M, int E, int top_k, int normalize, hipStream_t s);

template <typename T>
hipError_t launch_q4_quantize(const T* w, uint8_t* codes, T* scales, int64_t count, int64_t rows, int64_t cols, int group, hipStream_t s);
template <typename T>
hipError_t launch_q4_dequantize(const uint8_t* codes, const T* scales, T* w, int64_t count, int64_t rows, int64_t cols, int group,
                                hipStream_t s);

}  // namespace gmlp
