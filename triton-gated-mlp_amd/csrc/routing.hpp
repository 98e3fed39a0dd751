// The choice of experts from a router's logits: what the kernels of experts.hip and balance.hip share.
#pragma once
#include "common.hpp"

namespace gmlp {

// A logit as an integer of the same order: NaN above everything, -0 equal to 0, and 0 below every logit.
__device__ __forceinline__ uint32_t logit_key(float v) {
  uint32_t u = __float_as_uint(v == 0.f ? 0.f : v);
  if (v != v) u = 0x7fffffffu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_logit(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
// Reductions over a wavefront in the vector units: along the rows of 16 lanes, then from row to row; lane 63 has them all.
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ uint32_t from_lane(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  auto take = [&](uint32_t o) { v = o > v ? o : v; };
  take(from_lane<0x111>(v));
  take(from_lane<0x112>(v));
  take(from_lane<0x114>(v));
  take(from_lane<0x118>(v));
  take(from_lane<0x142>(v));
  take(from_lane<0x143>(v));
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ float wave_sum(float v) {
  auto take = [&](uint32_t o) { v += __uint_as_float(o); };
  take(from_lane<0x111>(__float_as_uint(v)));
  take(from_lane<0x112>(__float_as_uint(v)));
  take(from_lane<0x114>(__float_as_uint(v)));
  take(from_lane<0x118>(__float_as_uint(v)));
  take(from_lane<0x142, 0xa>(__float_as_uint(v)));
  take(from_lane<0x143, 0xc>(__float_as_uint(v)));
  return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), 63));
}

// One wavefront, one token: lane j < top_k gets the token's j-th choice and its weight.  The experts lie in lane order
// (lane l: VPL l .. VPL l + VPL - 1), so among equal logits the lowest lane holds the lowest number.
// (-inf: not available, weight 0 and expert -1 - number.)
template <int VPL, typename F>
__device__ __forceinline__ void choose(F&& logit, int E, int top_k, bool normalize, int lane, int& expert, float& weight) {
  uint32_t key[VPL];
  float value[VPL];
#pragma unroll
  for (int v = 0; v < VPL; ++v) {
    const int e = lane * VPL + v;
    value[v] = e < E ? logit(e) : -__builtin_inff();
    key[v] = e < E ? logit_key(value[v]) : 0u;
  }
  uint32_t mine = 0, top = 0;
  expert = 0;
  for (int j = 0; j < top_k; ++j) {
    uint32_t best = key[0];
    int at = 0;
#pragma unroll
    for (int v = 1; v < VPL; ++v)
      if (key[v] > best) best = key[v], at = v;
    const uint32_t most = wave_max(best);
    const int owner = __builtin_ctzll(__ballot(best == most));
    const int e = __builtin_amdgcn_readlane(lane * VPL + at, owner);
#pragma unroll
    for (int v = 0; v < VPL; ++v)
      if (lane == owner && v == at) key[v] = 0u;
    if (j == 0) top = most;
    if (lane == j) mine = most, expert = e;
  }
  const float first = key_logit(top), own = key_logit(mine);
  const bool none = first == -__builtin_inff();
  const float e = lane < top_k && !none ? expf(own - first) : 0.f;
  float all = e;
  if (!normalize) {
    all = 0.f;
#pragma unroll
    for (int v = 0; v < VPL; ++v)
      if (lane * VPL + v < E && !none) all += expf(value[v] - first);
  }
  weight = none ? 0.f : e / wave_sum(all);
  if (own == -__builtin_inff()) expert = -1 - expert;
}

// Four tokens to a wavefront, a row of 16 lanes each; lane l of a row has VPL experts from VPL l on.
template <typename F>
__device__ __forceinline__ uint32_t across_row(uint32_t v, F&& f) {
  v = f(v, from_lane<0x121>(v));
  v = f(v, from_lane<0x122>(v));
  v = f(v, from_lane<0x124>(v));
  return f(v, from_lane<0x128>(v));
}
__device__ __forceinline__ float row_sum(float v, int lane) {
  const uint32_t s = across_row(__float_as_uint(v), [](uint32_t x, uint32_t y) { return __float_as_uint(__uint_as_float(x) + __uint_as_float(y)); });
  return __shfl(__uint_as_float(s), lane & 48);  // (the lanes' own sums are of other orders)
}

// A token's logits over such a row, and its top_k choices.
template <int VPL, typename L>
struct LogitRow {
  L raw[VPL] = {};
  float value[VPL];
  float first = 0.f, own = 0.f;  // the token's largest logit, and that of the lane's choice
  int expert = 0;                // lane l < top_k: the l-th choice
  uint32_t taken = 0;            // which of the lane's experts are chosen

  // A lane's logits in one load where they all exist and lie as the load wants them (VPL divides E: all or none exist).
  __device__ __forceinline__ void load(const L* row, bool aligned, int E, int l) {
    typedef L vec __attribute__((ext_vector_type(VPL)));
    if (VPL > 1 && E % VPL == 0 && aligned) {
      if (l * VPL < E) {
        const vec packed = *(const vec*)(row + l * VPL);
#pragma unroll
        for (int v = 0; v < VPL; ++v) raw[v] = packed[v];
      }
    } else {
#pragma unroll
      for (int v = 0; v < VPL; ++v)
        if (l * VPL + v < E) raw[v] = row[l * VPL + v];
    }
#pragma unroll
    for (int v = 0; v < VPL; ++v) value[v] = (float)raw[v];
  }
  __device__ __forceinline__ void choose(int E, int top_k, int l) {
    uint32_t key[VPL];
    if constexpr (sizeof(L) == 2) {
      // 16-bit logits leave room for the number in the key, the lower ones larger: one maximum finds both.
#pragma unroll
      for (int v = 0; v < VPL; ++v) {
        const int e = l * VPL + v;
        uint32_t u = __builtin_bit_cast(unsigned short, raw[v]);
        u = value[v] != value[v] ? 0x7fffu : value[v] == 0.f ? 0u : u;
        u = u & 0x8000u ? ~u & 0xffffu : u | 0x8000u;
        key[v] = e < E ? u << 16 | (uint32_t)(0xffff - e) : 0u;
      }
      for (int j = 0; j < top_k; ++j) {
        uint32_t best = key[0];
#pragma unroll
        for (int v = 1; v < VPL; ++v) best = key[v] > best ? key[v] : best;
        const uint32_t most = across_row(best, [](uint32_t x, uint32_t y) { return x > y ? x : y; });
#pragma unroll
        for (int v = 0; v < VPL; ++v)
          if (key[v] == most) key[v] = 0u, taken |= 1u << v;
        const uint32_t u = most >> 16, bits = u & 0x8000u ? u & 0x7fffu : ~u & 0xffffu;
        const float logit = (float)__builtin_bit_cast(L, (unsigned short)bits);
        if (j == 0) first = logit;
        if (l == j) own = logit, expert = (int)(0xffffu - (most & 0xffffu));
      }
    } else {
#pragma unroll
      for (int v = 0; v < VPL; ++v) key[v] = l * VPL + v < E ? logit_key(value[v]) : 0u;
      for (int j = 0; j < top_k; ++j) {
        uint32_t best = key[0];
        int at = 0;
#pragma unroll
        for (int v = 1; v < VPL; ++v)
          if (key[v] > best) best = key[v], at = v;
        const uint32_t most = across_row(best, [](uint32_t x, uint32_t y) { return x > y ? x : y; });
        const uint32_t e = across_row(best == most ? (uint32_t)(l * VPL + at) : ~0u, [](uint32_t x, uint32_t y) { return x < y ? x : y; });
        const int gone = (int)e - l * VPL;
#pragma unroll
        for (int v = 0; v < VPL; ++v)
          if (v == gone) key[v] = 0u, taken |= 1u << v;
        if (j == 0) first = key_logit(most);
        if (l == j) own = key_logit(most), expert = (int)e;
      }
    }
  }
};

}  // namespace gmlp
