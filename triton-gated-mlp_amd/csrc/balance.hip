// A router's training step: the choice of experts, how many tokens each gets, the balance loss, and the gradient of the logits.
//
//   p_t = softmax(l_t); the token's top_k choices and their weights as moe_route's
//   c_e = choices of expert e by the tokens that count, f_e = c_e / sum c, P_e = mean of p_te over the T tokens that count
//   loss = E sum_e f_e P_e          (f is a constant)
//   dl_te = d_loss E / T p_te (f_e - sum_j f_j p_tj)                              where t counts
//         + w_te (dw_te - sum_j w_tj dw_tj) for the chosen, or, not normalised,  p_te ([e chosen] dw_te - sum_j w_tj dw_tj)
//
// A token counts if the mask has it and at least one expert is available to it; a choice of an expert that is not (-inf) does
// not.  Four tokens to a wavefront, as in routing: a lane has the same VPL experts of every token it meets, so sums over
// tokens are registers, joined at the end in a fixed order (the results do not depend on timing).  The loss
// needs all tokens before the gradient of any: logits are read twice.
#include "balance.hpp"
#include "routing.hpp"

namespace gmlp {

constexpr int BAL_THREADS = 256, BAL_ROWS = BAL_THREADS / 16;  // tokens of a workgroup at a time

// Sums of all workgroups' parts -> counts, loss, slope.  1024 threads.
__device__ __forceinline__ void balance_finish(const BalanceArgs& a, int parts) {
  __shared__ double sum_p[1024];
  __shared__ long long sum_c[1024];
  __shared__ double in_loss[16];
  __shared__ long long all_c, all_t;
  const int tid = threadIdx.x, E = a.E, width = balance_partial(E);
  // thread g * E + e adds up parts g, g + groups, ...
  const int groups = 1024 / E, e = tid % E, g = tid / E;
  double p = 0.0;
  long long c = 0;
  if (g < groups)
    for (int i = g; i < parts; i += groups) {
      p += (double)a.partial[(size_t)i * width + e];
      c += __float_as_int(a.partial[(size_t)i * width + E + e]);
    }
  sum_p[tid] = p;
  sum_c[tid] = c;
  if (tid == 0) all_c = 0, all_t = 0;
  __syncthreads();
  if (tid < E) {
    for (int i = 1; i < groups; ++i) {
      p += sum_p[i * E + tid];
      c += sum_c[i * E + tid];
    }
    a.counts[tid] = c;
    if (c) atomicAdd((unsigned long long*)&all_c, (unsigned long long)c);
  }
  long long t = 0;
  for (int i = tid; i < parts; i += 1024) t += __float_as_int(a.partial[(size_t)i * width + 2 * E]);
  if (t) atomicAdd((unsigned long long*)&all_t, (unsigned long long)t);
  __syncthreads();
  // (no tokens: a loss of 0, and no slope)
  const double scale = all_c > 0 ? (double)E / ((double)all_c * (double)all_t) : 0.0;
  double part = 0.0;
  if (tid < E) {
    const double slope = scale * (double)c;
    a.slope[tid] = (float)slope;
    part = slope * p;
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) part += __shfl_xor(part, d);
  if ((tid & 63) == 0) in_loss[tid >> 6] = part;
  __syncthreads();
  if (tid == 0) {
    double loss = 0.0;
    for (int i = 0; i < 16; ++i) loss += in_loss[i];
    *a.loss = (float)loss;
  }
}
__global__ void __launch_bounds__(1024) balance_finish_kernel(BalanceArgs a, int parts) { balance_finish(a, parts); }

template <int VPL, typename L>
__global__ void __launch_bounds__(BAL_THREADS) balance_rows_kernel(BalanceArgs a) {
  extern __shared__ float wave_sums[];  // [wavefronts][balance_partial(E)]
  const int lane = threadIdx.x & 63, l = lane & 15, mine = threadIdx.x >> 4, E = a.E, top_k = a.top_k, width = balance_partial(E);
  const bool aligned = ((uintptr_t)a.logits & (sizeof(L) * VPL - 1)) == 0;
  float p[VPL];
  int chosen[VPL], tokens = 0;
#pragma unroll
  for (int v = 0; v < VPL; ++v) p[v] = 0.f, chosen[v] = 0;
  for (int64_t base = (int64_t)blockIdx.x * BAL_ROWS; base < a.M; base += (int64_t)gridDim.x * BAL_ROWS) {
    const int64_t token = base + mine, t = token < a.M ? token : a.M - 1;
    LogitRow<VPL, L> row;
    row.load((const L*)a.logits + t * E, aligned, E, l);
    const bool kept = a.mask == nullptr || a.mask[t] != 0;
    row.choose(E, top_k, l);
    const bool none = row.first == -__builtin_inff(), counts = token < a.M && kept && !none;
    float e[VPL], all = 0.f;
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      e[v] = l * VPL + v < E && !none ? expf(row.value[v] - row.first) : 0.f;
      all += e[v];
    }
    all = row_sum(all, lane);
    const float own = l < top_k && !none ? expf(row.own - row.first) : 0.f;
    const float over = a.normalize ? row_sum(own, lane) : all;
    if (token < a.M && l < top_k) {
      a.weights[t * top_k + l] = none ? 0.f : own / over;
      a.experts[t * top_k + l] = row.expert;
    }
    if (counts) {
      const float inv = 1.f / all;
#pragma unroll
      for (int v = 0; v < VPL; ++v) {
        p[v] += e[v] * inv;
        chosen[v] += (row.taken >> v & 1u) && row.value[v] != -__builtin_inff() ? 1 : 0;
      }
      tokens += 1;
    }
  }
  // the four rows of a wavefront, then the wavefronts
#pragma unroll
  for (int d = 16; d <= 32; d <<= 1) {
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      p[v] += __shfl_xor(p[v], d);
      chosen[v] += __shfl_xor(chosen[v], d);
    }
    tokens += __shfl_xor(tokens, d);
  }
  float* const own = wave_sums + (threadIdx.x >> 6) * width;
  if (lane < 16) {
#pragma unroll
    for (int v = 0; v < VPL; ++v)
      if (l * VPL + v < E) {
        own[l * VPL + v] = p[v];
        own[E + l * VPL + v] = __int_as_float(chosen[v]);
      }
    if (l == 0) own[2 * E] = __int_as_float(tokens);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < width; i += BAL_THREADS) {
    float sum = 0.f;
    int n = 0;
#pragma unroll
    for (int w = 0; w < BAL_THREADS / 64; ++w) {
      const float x = wave_sums[w * width + i];
      if (i < E) sum += x;
      else n += __float_as_int(x);
    }
    a.partial[(size_t)blockIdx.x * width + i] = i < E ? sum : __int_as_float(n);
  }
}

template <int VPL, typename L>
__global__ void __launch_bounds__(BAL_THREADS) balance_bwd_kernel(BalanceArgs a) {
  const int lane = threadIdx.x & 63, l = lane & 15, mine = threadIdx.x >> 4, E = a.E, top_k = a.top_k;
  const bool aligned = ((uintptr_t)a.logits & (sizeof(L) * VPL - 1)) == 0;
  const bool aligned_out = ((uintptr_t)a.d_logits & (sizeof(L) * VPL - 1)) == 0;
  const float d_loss = a.d_loss != nullptr ? *a.d_loss : 0.f;
  float slope[VPL];
#pragma unroll
  for (int v = 0; v < VPL; ++v) slope[v] = l * VPL + v < E && a.d_loss != nullptr ? a.slope[l * VPL + v] : 0.f;
  for (int64_t base = (int64_t)blockIdx.x * BAL_ROWS; base < a.M; base += (int64_t)gridDim.x * BAL_ROWS) {
    const int64_t token = base + mine, t = token < a.M ? token : a.M - 1;
    LogitRow<VPL, L> row;
    row.load((const L*)a.logits + t * E, aligned, E, l);
    const bool kept = a.d_loss != nullptr && (a.mask == nullptr || a.mask[t] != 0);
    float w = 0.f, dw = 0.f;
    int expert = -1;
    if (a.d_weights != nullptr && l < top_k) {
      w = a.weights[t * top_k + l];
      dw = a.d_weights[t * top_k + l];
      expert = (int)a.experts[t * top_k + l];
    }
    uint32_t best = 0u;
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      const uint32_t k = l * VPL + v < E ? logit_key(row.value[v]) : 0u;
      best = k > best ? k : best;
    }
    const float first = key_logit(across_row(best, [](uint32_t x, uint32_t y) { return x > y ? x : y; }));
    const bool none = first == -__builtin_inff();
    float p[VPL], all = 0.f, mean = 0.f;
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      p[v] = l * VPL + v < E && !none ? expf(row.value[v] - first) : 0.f;
      all += p[v];
    }
    all = row_sum(all, lane);
    const float inv = none ? 0.f : 1.f / all;
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      p[v] *= inv;
      mean += slope[v] * p[v];
    }
    mean = row_sum(mean, lane);
    const float mixed = a.d_weights != nullptr ? row_sum(w * dw, lane) : 0.f;
    float d[VPL];
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      d[v] = kept ? d_loss * (p[v] * (slope[v] - mean)) : 0.f;
      if (!a.normalize) d[v] -= p[v] * mixed;
    }
    if (a.d_weights != nullptr) {
      const float own = a.normalize ? w * (dw - mixed) : w * dw;
      for (int j = 0; j < top_k; ++j) {
        const int from = (lane & 48) + j, at = __shfl(expert, from) - l * VPL;
        const float x = __shfl(own, from);
#pragma unroll
        for (int v = 0; v < VPL; ++v)
          if (at == v) d[v] += x;
      }
    }
    if (token >= a.M) continue;
    L* const out = (L*)a.d_logits + t * E;
    typedef L vec __attribute__((ext_vector_type(VPL)));
    if (VPL > 1 && E % VPL == 0 && aligned_out) {
      if (l * VPL < E) {
        vec packed;
#pragma unroll
        for (int v = 0; v < VPL; ++v) packed[v] = (L)d[v];
        *(vec*)(out + l * VPL) = packed;
      }
    } else {
#pragma unroll
      for (int v = 0; v < VPL; ++v)
        if (l * VPL + v < E) out[l * VPL + v] = (L)d[v];
    }
  }
}

int balance_workgroups(int64_t M) {
  const int64_t n = (M + BAL_ROWS - 1) / BAL_ROWS;
  return (int)(n < 256 ? n : 256);
}

#define GMLP_BY_ROW(E, CALL)     \
  if ((E) <= 16) CALL(1);        \
  else if ((E) <= 64) CALL(4);   \
  else if ((E) <= 128) CALL(8);  \
  else if ((E) <= 256) CALL(16); \
  else CALL(32)

template <typename L>
hipError_t launch_balance_fwd(const BalanceArgs& a, hipStream_t s) {
  const int wgs = balance_workgroups(a.M);
  const size_t lds = (size_t)(BAL_THREADS / 64) * balance_partial(a.E) * sizeof(float);
#define CALL(V) hipLaunchKernelGGL((balance_rows_kernel<V, L>), dim3(wgs), dim3(BAL_THREADS), lds, s, a)
  GMLP_BY_ROW(a.E, CALL);
#undef CALL
  if (hipError_t e = hipGetLastError()) return e;
  hipLaunchKernelGGL(balance_finish_kernel, dim3(1), dim3(1024), 0, s, a, wgs);
  return hipGetLastError();
}
template <typename L>
hipError_t launch_balance_bwd(const BalanceArgs& a, hipStream_t s) {
  const int64_t n = (a.M + BAL_ROWS - 1) / BAL_ROWS;
  const int wgs = (int)(n < 2048 ? n : 2048);
#define CALL(V) hipLaunchKernelGGL((balance_bwd_kernel<V, L>), dim3(wgs), dim3(BAL_THREADS), 0, s, a)
  GMLP_BY_ROW(a.E, CALL);
#undef CALL
  return hipGetLastError();
}
#undef GMLP_BY_ROW

#define GMLP_INSTANTIATE(L)                                                  \
  template hipError_t launch_balance_fwd<L>(const BalanceArgs&, hipStream_t); \
  template hipError_t launch_balance_bwd<L>(const BalanceArgs&, hipStream_t);
GMLP_INSTANTIATE(f16)
GMLP_INSTANTIATE(bf16)
GMLP_INSTANTIATE(float)
#undef GMLP_INSTANTIATE

}  // namespace gmlp
