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

// Wavefronts of a workgroup in the first stage: sixteen, where their sums fit LDS.  (16384 tokens, 128 experts: one round of
// 256 workgroups.  Four wavefronts and four rounds 15.5 us, a wavefront on a SIMD.)
constexpr int bal_wavefronts(int vpl) { return vpl <= 16 ? 16 : 4; }
constexpr int BAL_BWD_THREADS = 256;
constexpr int64_t BAL_ALONE = 256;  // tokens that one workgroup takes, both stages in one launch

// Sums of all workgroups' parts -> counts, loss, slope.  1024 threads, and a chain of loads and barriers: eight loads of a thread are in
// flight together, sums join in trees (64-bit atomics in LDS on one word, one after the other, took 4 us for 128 experts).
__device__ __forceinline__ void balance_finish(const BalanceArgs& a, int parts) {
  __shared__ double sum_p[1024], sum_c[1024];  // (numbers of choices are exact up to 2^53)
  __shared__ double in_wave[3][16];
  const int tid = threadIdx.x, lane = tid & 63, E = a.E, width = balance_partial(E);
  // thread g * E + e adds up parts g, g + groups, ...
  const int groups = parts < 1024 / E ? parts : 1024 / E, g = tid / E, e = tid - g * E;
  double p = 0.0, c = 0.0, t = 0.0;
  if (g < groups)
#pragma unroll 8
    for (int i = g; i < parts; i += groups) {
      p += (double)a.partial[(size_t)i * width + e];
      c += (double)__float_as_int(a.partial[(size_t)i * width + E + e]);
    }
  for (int i = tid; i < parts; i += 1024) t += (double)__float_as_int(a.partial[(size_t)i * width + 2 * E]);
  int half = 1;
  while (half < groups) half *= 2;
  for (half /= 2; half > 0; half /= 2) {
    sum_p[tid] = p;
    sum_c[tid] = c;
    __syncthreads();
    if (g < half && g + half < groups) {
      p += sum_p[tid + half * E];
      c += sum_c[tid + half * E];
    }
    __syncthreads();
  }
  if (tid >= E) p = c = 0.0;
  double all[3] = {c, t, c * p};
#pragma unroll
  for (int d = 32; d > 0; d >>= 1)
#pragma unroll
    for (int k = 0; k < 3; ++k) all[k] += __shfl_xor(all[k], d);
  if (lane == 0)
#pragma unroll
    for (int k = 0; k < 3; ++k) in_wave[k][tid >> 6] = all[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 3; ++k) all[k] = in_wave[k][lane & 15];
#pragma unroll
  for (int d = 8; d > 0; d >>= 1)
#pragma unroll
    for (int k = 0; k < 3; ++k) all[k] += __shfl_xor(all[k], d);
  // (no tokens: a loss of 0, and no slope)
  const double scale = all[0] > 0.0 ? (double)E / (all[0] * all[1]) : 0.0;
  if (tid < E) {
    a.counts[tid] = (int64_t)c;
    a.slope[tid] = (float)(scale * c);
  }
  if (tid == 0) *a.loss = (float)(scale * all[2]);
}
__global__ void __launch_bounds__(1024) balance_finish_kernel(BalanceArgs a, int parts) { balance_finish(a, parts); }

template <int VPL, typename L>
__global__ void __launch_bounds__(bal_wavefronts(VPL) * 64) balance_rows_kernel(BalanceArgs a) {
  constexpr int THREADS = bal_wavefronts(VPL) * 64, ROWS = THREADS / 16;
  extern __shared__ float wave_sums[];  // [wavefronts][balance_partial(E)]
  const int lane = threadIdx.x & 63, l = lane & 15, mine = threadIdx.x >> 4, E = a.E, top_k = a.top_k, width = balance_partial(E);
  const bool aligned = ((uintptr_t)a.logits & (sizeof(L) * VPL - 1)) == 0;
  float p[VPL];
  int chosen[VPL], tokens = 0;
#pragma unroll
  for (int v = 0; v < VPL; ++v) p[v] = 0.f, chosen[v] = 0;
  for (int64_t base = (int64_t)blockIdx.x * ROWS; base < a.M; base += (int64_t)gridDim.x * ROWS) {
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
  for (int i = threadIdx.x; i < width; i += THREADS) {
    float sum = 0.f;
    int n = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
      const float x = wave_sums[w * width + i];
      if (i < E) sum += x;
      else n += __float_as_int(x);
    }
    a.partial[(size_t)blockIdx.x * width + i] = i < E ? sum : __int_as_float(n);
  }
  if constexpr (THREADS == 1024)
    if (gridDim.x == 1) {
      __threadfence_block();
      __syncthreads();
      balance_finish(a, 1);
    }
}

template <int VPL, typename L>
__global__ void __launch_bounds__(BAL_BWD_THREADS) balance_bwd_kernel(BalanceArgs a) {
  const int lane = threadIdx.x & 63, l = lane & 15, mine = threadIdx.x >> 4, E = a.E, top_k = a.top_k;
  const bool aligned = ((uintptr_t)a.logits & (sizeof(L) * VPL - 1)) == 0;
  const bool aligned_out = ((uintptr_t)a.d_logits & (sizeof(L) * VPL - 1)) == 0;
  const float d_loss = a.d_loss != nullptr ? *a.d_loss : 0.f;
  float slope[VPL];
#pragma unroll
  for (int v = 0; v < VPL; ++v) slope[v] = l * VPL + v < E && a.d_loss != nullptr ? a.slope[l * VPL + v] : 0.f;
  for (int64_t base = (int64_t)blockIdx.x * (BAL_BWD_THREADS / 16); base < a.M; base += (int64_t)gridDim.x * (BAL_BWD_THREADS / 16)) {
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
      // (nothing is taken off without gradients of the weights: p of a token left out may be NaN)
      if (!a.normalize && a.d_weights != nullptr) d[v] -= p[v] * mixed;
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

int balance_workgroups(int64_t M, int E) {
  const int64_t rows = E <= 256 ? 64 : 16, n = (M + rows - 1) / rows;
  return E <= 256 && M <= BAL_ALONE ? 1 : (int)(n < 256 ? n : 256);
}

#define GMLP_BY_ROW(E, CALL)     \
  if ((E) <= 16) CALL(1);        \
  else if ((E) <= 64) CALL(4);   \
  else if ((E) <= 128) CALL(8);  \
  else if ((E) <= 256) CALL(16); \
  else CALL(32)

template <typename L>
hipError_t launch_balance_fwd(const BalanceArgs& a, hipStream_t s) {
  const int wgs = balance_workgroups(a.M, a.E);
#define CALL(V)                                                                                                  \
  hipLaunchKernelGGL((balance_rows_kernel<V, L>), dim3(wgs), dim3(bal_wavefronts(V) * 64),                        \
                     (size_t)bal_wavefronts(V) * balance_partial(a.E) * sizeof(float), s, a)
  GMLP_BY_ROW(a.E, CALL);
#undef CALL
  if (hipError_t e = hipGetLastError()) return e;
  if (wgs == 1 && a.E <= 256) return hipSuccess;
  hipLaunchKernelGGL(balance_finish_kernel, dim3(1), dim3(1024), 0, s, a, wgs);
  return hipGetLastError();
}
template <typename L>
hipError_t launch_balance_bwd(const BalanceArgs& a, hipStream_t s) {
  const int64_t n = (a.M + BAL_BWD_THREADS / 16 - 1) / (BAL_BWD_THREADS / 16);
  const int wgs = (int)(n < 2048 ? n : 2048);
#define CALL(V) hipLaunchKernelGGL((balance_bwd_kernel<V, L>), dim3(wgs), dim3(BAL_BWD_THREADS), 0, s, a)
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
