// Expert layers and 4-bit weights for a few token rows (M <= 64).
//
//   route, plan    softmax of the router's logits, the top_k largest of each token; which experts are in use, by whom
//   gate/up        h[p] = act(W_gate_e x_t + b_gate) * (W_up_e x_t + b_up)   for every pair p = (token t, its choice e)
//   down           y[t] = sum_e w_te W_down_e h_te + b_down
//
// The products are bound by the weights' way from memory: each weight is read once per call and feeds one
// v_mfma_f32_16x16x32 column per token row.  A workgroup takes 16 weight rows (gate/up: 16 of each matrix); its wavefronts
// split the reduction and add up through LDS in a fixed order, so results do not depend on timing.  Every load is a
// buffer load with an exact descriptor: rows past the matrix, columns past its end, tokens that an expert does not have
// and the stages past the end of a wavefront's run all get an offset beyond it, which reads as zero and moves no data.
//
// 4-bit weights keep their integers for the matrix product (exact in 16 bits); a group's scale is applied to the
// product in fp32, so what is multiplied is scale·n itself, not its rounding.
#include "experts.hpp"

#include "gemm.hpp"

namespace gmlp {

typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));
typedef f16 f16x2 __attribute__((ext_vector_type(2)));

constexpr uint32_t EX_NOWHERE = 0x80000000u;  // byte offset beyond any descriptor (all are < 2 GiB)

typedef __amdgpu_buffer_rsrc_t ex_rsrc;
__device__ __forceinline__ ex_rsrc ex_make_rsrc(const void* p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, (int)bytes, 0x00020000);
}
constexpr int EX_STREAM = 2;  // cache policy: non-temporal, what is read once
template <int POLICY = 0>
__device__ __forceinline__ u32x4 ex_load16(ex_rsrc r, uint32_t off) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, POLICY));
}
template <int POLICY = 0>
__device__ __forceinline__ u32x2 ex_load8(ex_rsrc r, uint32_t off) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, (int)off, 0, POLICY));
}

// ------------------------------------------------------------------ 4-bit integers as 16-bit floats
// One 32-bit word holds columns 0, 2, 4, 6 of eight in its low half's nibbles and 1, 3, 5, 7 in its high half's, so
// one mask takes a pair of neighbours apart.  SCALE: what the products have to be multiplied by.
template <typename T>
struct Int4;
template <>
struct Int4<f16> {
  static constexpr float SCALE = 1.f;
  // 0x6400 | u is 1024 + u in fp16; u = n + 8
  static __device__ __forceinline__ f16x8 floats(uint32_t w) {
    u32x4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t v = ((w >> (4 * j)) & 0x000f000fu) | 0x64006400u;
      o[j] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, v) - f16x2{(f16)1032.f, (f16)1032.f});
    }
    return __builtin_bit_cast(f16x8, o);
  }
};
template <>
struct Int4<bf16> {
  static constexpr float SCALE = 16.f;
  // v_cvt_off_f32_i4 makes n / 16 of a signed nibble; a bf16 is the upper half of the fp32 number
  static __device__ __forceinline__ bf16x8 floats(uint32_t w) {
    const uint32_t even = w ^ 0x88888888u, odd = even >> 4;
    u32x4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t v = j % 2 ? odd : even;
      const float lo = __builtin_amdgcn_cvt_off_f32_i4((int)((v >> (8 * (j / 2))) & 0xffu));
      const float hi = __builtin_amdgcn_cvt_off_f32_i4((int)((v >> (8 * (j / 2) + 16)) & 0xffu));
      o[j] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, hi), __builtin_bit_cast(uint32_t, lo), 0x07060302u);
    }
    return __builtin_bit_cast(bf16x8, o);
  }
};

template <typename T>
__device__ __forceinline__ float bits_to_f32(uint32_t u) {
  return (float)__builtin_bit_cast(T, (unsigned short)u);
}

// ------------------------------------------------------------------ a block of the reduction
// 16 weight rows of NMAT matrices by 64 columns (16-bit weights) or 128 (4-bit ones), and MT tiles of 16 token
// rows by the same columns.  16-bit: a lane holds 32 consecutive bytes of its row in two loads, so a row's segment
// is one 128-byte line; 4-bit: 16 consecutive bytes, a wavefront one KiB.  (The products do not mind which columns share a
// step, so the token operands follow the weights.)
template <typename T, int G, int NMAT, int MT>
struct Block {
  typedef typename Traits<T>::vec8 vec8;
  static constexpr int COLS = G ? Q4_BLOCK : 64;
  static constexpr int STEPS = COLS / 32;
  static constexpr int GROUPS = G ? Q4_BLOCK / G : 1;
  static constexpr int WL = G ? 1 : 2;  // weight loads of a lane
  u32x4 w[NMAT][WL];
  u32x2 sc[NMAT][GROUPS];
  u32x4 x[MT][STEPS];

  static __device__ __forceinline__ uint32_t column(int kb, int s, int kg) {
    return (uint32_t)(kb * COLS + (G ? s * 32 + kg * 8 : kg * 16 + s * 8));
  }
  // of tile `tile` of a matrix of `rows` x `cols`
  static __device__ __forceinline__ ex_rsrc weights_of(const ExpertWeights& m, int expert, int tile, int rows, int cols) {
    const int tiles = (rows + Q4_TILE - 1) / Q4_TILE, blocks = (cols + Q4_BLOCK - 1) / Q4_BLOCK;
    if (G) return ex_make_rsrc((const char*)m.w + ((size_t)expert * tiles + tile) * blocks * 1024, (uint32_t)blocks * 1024u);
    const int first = tile * Q4_TILE, own = rows - first < Q4_TILE ? rows - first : Q4_TILE;
    return ex_make_rsrc((const T*)m.w + ((size_t)expert * rows + first) * cols, (uint32_t)own * (uint32_t)cols * 2u);
  }
  static __device__ __forceinline__ ex_rsrc scales_of(const ExpertWeights& m, int expert, int tile, int rows, int cols) {
    const int tiles = (rows + Q4_TILE - 1) / Q4_TILE, blocks = (cols + Q4_BLOCK - 1) / Q4_BLOCK;
    const uint32_t pitch = (uint32_t)blocks * (Q4_TILE * GROUPS * 2);
    return ex_make_rsrc((const char*)m.scales + ((size_t)expert * tiles + tile) * pitch, G ? pitch : 0u);
  }

  __device__ __forceinline__ void load_weights(int n, ex_rsrc rw, ex_rsrc rs, int kb, bool ok, int cols, int lane) {
    const int kg = lane >> 4, r16 = lane & 15;
    if (G) {
      w[n][0] = ex_load16<EX_STREAM>(rw, ok ? (uint32_t)kb * 1024u + (uint32_t)lane * 16u : EX_NOWHERE);
      const uint32_t at = ok ? (uint32_t)(kb * 4 + kg) * (GROUPS * 8u) : EX_NOWHERE;
      if constexpr (GROUPS == 1) {
        sc[n][0] = ex_load8<EX_STREAM>(rs, at);
      } else {
#pragma unroll
        for (int g = 0; g < GROUPS; g += 2) {
          const u32x4 v = ex_load16<EX_STREAM>(rs, at + (uint32_t)g * 8u);
          sc[n][g] = u32x2{v[0], v[1]};
          sc[n][g + 1] = u32x2{v[2], v[3]};
        }
      }
    } else {
#pragma unroll
      for (int s = 0; s < WL; ++s) {
        const uint32_t c = column(kb, s, kg);
        w[n][s] = ex_load16<EX_STREAM>(rw, ok && c < (uint32_t)cols ? ((uint32_t)r16 * (uint32_t)cols + c) * 2u : EX_NOWHERE);
      }
    }
  }
  // row[m]: byte offset of the lane's token row, or EX_NOWHERE
  __device__ __forceinline__ void load_tokens(ex_rsrc rx, const uint32_t (&row)[MT], int kb, bool ok, int cols, int lane) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const uint32_t c = column(kb, s, lane >> 4);
#pragma unroll
      for (int m = 0; m < MT; ++m) x[m][s] = ex_load16(rx, ok && c < (uint32_t)cols ? row[m] + c * 2u : EX_NOWHERE);
    }
  }
  __device__ __forceinline__ void multiply(f32x4 (&acc)[NMAT][MT]) const {
#pragma unroll
    for (int n = 0; n < NMAT; ++n) {
      if (G) {
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          f32x4 part[MT];
#pragma unroll
          for (int m = 0; m < MT; ++m) part[m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s = g * STEPS / GROUPS; s < (g + 1) * STEPS / GROUPS; ++s) {
            const vec8 a = Int4<T>::floats(w[n][0][s]);
#pragma unroll
            for (int m = 0; m < MT; ++m) part[m] = Traits<T>::mfma16(a, __builtin_bit_cast(vec8, x[m][s]), part[m]);
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float f = bits_to_f32<T>(sc[n][g][r / 2] >> (16 * (r % 2)) & 0xffffu) * Int4<T>::SCALE;
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[n][m][r] += f * part[m][r];
          }
        }
      } else {
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
          for (int m = 0; m < MT; ++m)
            acc[n][m] = Traits<T>::mfma16(__builtin_bit_cast(vec8, w[n][s]), __builtin_bit_cast(vec8, x[m][s]), acc[n][m]);
      }
    }
  }
};

// ------------------------------------------------------------------ gate/up
template <typename T, int G, int MT, int NW, int D>
__global__ void __launch_bounds__(NW * 64) experts_gateup_kernel(ExpertArgs a) {
  typedef Block<T, G, 2, MT> B;
  __shared__ f32x4 part[NW][2][MT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, kg = lane >> 4;
  const int tiles = (a.N + Q4_TILE - 1) / Q4_TILE;
  const int slot = (int)blockIdx.x / tiles, tile = (int)blockIdx.x - slot * tiles;
  int expert = 0, count = a.M;
  if (!a.dense) {
    if (slot >= a.plan.active[0]) return;
    expert = a.plan.active[1 + slot];
    count = a.plan.count[slot];
  }
  const ex_rsrc rx = ex_make_rsrc(a.x, (uint32_t)a.M * (uint32_t)a.K * 2u);
  const ExpertWeights* const mats[2] = {&a.gate, &a.up};
  ex_rsrc rw[2], rs[2];
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    rw[n] = B::weights_of(*mats[n], expert, tile, a.N, a.K);
    rs[n] = B::scales_of(*mats[n], expert, tile, a.N, a.K);
  }
  const int blocks = (a.K + B::COLS - 1) / B::COLS;
  const int b0 = blocks * wave / NW, run = blocks * (wave + 1) / NW - b0;

  for (int base = 0; base < count; base += 16 * MT) {
    uint32_t row[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int j = base + 16 * m + r16;
      const int t = j < count ? (a.dense ? j : a.plan.tokens[slot * EXPERTS_MAX_M + j]) : 0;
      row[m] = j < count ? (uint32_t)t * (uint32_t)a.K * 2u : EX_NOWHERE;
    }
    B st[D];
    auto load = [&](B& b, int i) {
#pragma unroll
      for (int n = 0; n < 2; ++n) b.load_weights(n, rw[n], rs[n], b0 + i, i < run, a.K, lane);
      b.load_tokens(rx, row, b0 + i, i < run, a.K, lane);
    };
    f32x4 acc[2][MT];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[n][m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < D; ++d) load(st[d], d);
    for (int i = 0; i < run; i += D)
#pragma unroll
      for (int d = 0; d < D; ++d) {
        st[d].multiply(acc);
        load(st[d], i + d + D);
      }
    if (base > 0) __syncthreads();
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int m = 0; m < MT; ++m) part[wave][n][m][lane] = acc[n][m];
    __syncthreads();
    if (wave < MT) {
      const int j = base + 16 * wave + r16, first = tile * Q4_TILE + 4 * kg;
      if (j < count && first < a.N) {
        float v[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          f32x4 sum = part[0][n][wave][lane];
#pragma unroll
          for (int w = 1; w < NW; ++w) sum += part[w][n][wave][lane];
#pragma unroll
          for (int r = 0; r < 4; ++r) v[n][r] = sum[r];
          if (a.bias[n]) add_w<T, 4>((const T*)a.bias[n] + first, v[n]);
        }
        float h[4];
        act_fwd_w<4>(a.act, v[0], h);
#pragma unroll
        for (int r = 0; r < 4; ++r) h[r] *= v[1][r];
        int p = j;
        if (!a.dense) {
          const int t = a.plan.tokens[slot * EXPERTS_MAX_M + j];
          p = t * a.top_k + a.plan.slot[slot * EXPERTS_MAX_M + t];
        }
        store_w<T, 4>((T*)a.h + (size_t)p * a.N + first, h);
      }
    }
  }
}

// ------------------------------------------------------------------ down
// The blocks of all experts in use, one expert behind the other, are shared out evenly over the wavefronts.  What an
// expert gives is added to a token's sum only where the token chose it (a weight that is not finite in one
// expert stays out of the others' tokens).
template <typename T, int G, int MT, int NW, int D>
__global__ void __launch_bounds__(NW * 64) experts_down_kernel(ExpertArgs a) {
  typedef Block<T, G, 1, MT> B;
  extern __shared__ __align__(16) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, kg = lane >> 4, tile = (int)blockIdx.x;
  const int pairs = a.M * a.top_k;
  // tables: the experts' numbers, the pairs' weights, the slots
  int in_use = 1;
  int* const numbers = (int*)smem;
  float* weight = nullptr;
  int8_t* slots = nullptr;
  if (!a.dense) {
    in_use = a.plan.active[0];
    weight = (float*)(numbers + in_use);
    slots = (int8_t*)(weight + pairs);
    for (int i = threadIdx.x; i < in_use; i += NW * 64) numbers[i] = a.plan.active[1 + i];
    for (int i = threadIdx.x; i < pairs; i += NW * 64) weight[i] = a.plan.weight[i];
    for (int i = threadIdx.x; i < in_use * (EXPERTS_MAX_M / 4); i += NW * 64)
      ((int*)slots)[i] = ((const int*)a.plan.slot)[i];
    __syncthreads();
  }
  const ex_rsrc rh = ex_make_rsrc(a.h, (uint32_t)pairs * (uint32_t)a.N * 2u);
  const int blocks = (a.N + B::COLS - 1) / B::COLS;
  const int total = in_use * blocks;
  const int b0 = (int)((int64_t)total * wave / NW), run = (int)((int64_t)total * (wave + 1) / NW) - b0;

  // choice of token row 16 m + r16 that expert e is, or -1
  auto slot_of = [&](int e, int m) -> int {
    const int t = 16 * m + r16;
    if (t >= a.M) return -1;
    return a.dense ? 0 : slots[e * EXPERTS_MAX_M + t];
  };
  // where loads go on: expert, block of it
  int le = b0 / blocks, lb = b0 - le * blocks;
  uint32_t row[MT];
  ex_rsrc rw, rs;
  auto enter = [&]() {
    const int e = le < in_use ? le : in_use - 1;
    const int number = a.dense ? 0 : __builtin_amdgcn_readfirstlane(numbers[e]);
    rw = B::weights_of(a.down, number, tile, a.K, a.N);
    rs = B::scales_of(a.down, number, tile, a.K, a.N);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int s = slot_of(e, m);
      row[m] = s < 0 ? EX_NOWHERE : (uint32_t)((16 * m + r16) * a.top_k + s) * (uint32_t)a.N * 2u;
    }
  };
  f32x4 acc[1][MT], sum[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) acc[0][m] = sum[m] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (run > 0) {
    enter();
    B st[D];
    auto load = [&](B& b, int i) {
      b.load_weights(0, rw, rs, lb, i < run, a.N, lane);
      b.load_tokens(rh, row, lb, i < run, a.N, lane);
      if (++lb == blocks) {
        lb = 0;
        ++le;
        enter();
      }
    };
    int me = le, mb = lb;  // where products are
    auto fold = [&]() {
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int s = slot_of(me, m);
        const float w = s < 0 ? 0.f : a.dense ? 1.f : weight[(16 * m + r16) * a.top_k + s];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (s >= 0) sum[m][r] += w * acc[0][m][r];
          acc[0][m][r] = 0.f;
        }
      }
    };
#pragma unroll
    for (int d = 0; d < D; ++d) load(st[d], d);
    for (int i = 0; i < run; i += D)
#pragma unroll
      for (int d = 0; d < D; ++d) {
        st[d].multiply(acc);
        load(st[d], i + d + D);
        if (++mb == blocks || i + d + 1 == run) {
          if (i + d < run) fold();
          mb = 0;
          ++me;
        }
      }
  }
  if (!a.dense) __syncthreads();  // the tables' last readers
  f32x4* const part = (f32x4*)smem;  // [NW][MT][64]
#pragma unroll
  for (int m = 0; m < MT; ++m) part[(wave * MT + m) * 64 + lane] = sum[m];
  __syncthreads();
  if (wave < MT) {
    const int t = 16 * wave + r16, first = tile * Q4_TILE + 4 * kg;
    if (t < a.M && first < a.K) {
      f32x4 v = part[wave * 64 + lane];
#pragma unroll
      for (int w = 1; w < NW; ++w) v += part[(w * MT + wave) * 64 + lane];
      float y[4] = {v[0], v[1], v[2], v[3]};
      if (a.bias[2]) add_w<T, 4>((const T*)a.bias[2] + first, y);
      store_w<T, 4>((T*)a.y + (size_t)t * a.K + first, y);
    }
  }
}

template <typename T, int G>
static hipError_t gateup_of(const ExpertArgs& a, hipStream_t s) {
  const int tiles = (a.N + Q4_TILE - 1) / Q4_TILE;
  const int experts = a.dense ? 1 : (a.E < a.M * a.top_k ? a.E : a.M * a.top_k);
  const dim3 grid((unsigned)(tiles * experts)), block(256);
  if (a.M <= 16) hipLaunchKernelGGL((experts_gateup_kernel<T, G, 1, 4, 2>), grid, block, 0, s, a);
  else if (a.M <= 32) hipLaunchKernelGGL((experts_gateup_kernel<T, G, 2, 4, 2>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((experts_gateup_kernel<T, G, 4, 4, 1>), grid, block, 0, s, a);
  return hipGetLastError();
}
template <typename T, int G>
static hipError_t down_of(const ExpertArgs& a, hipStream_t s) {
  constexpr int NW = 8;
  const dim3 grid((unsigned)((a.K + Q4_TILE - 1) / Q4_TILE)), block(NW * 64);
  const int experts = a.dense ? 0 : (a.E < a.M * a.top_k ? a.E : a.M * a.top_k);
  const size_t tables = (size_t)experts * (4 + EXPERTS_MAX_M) + (size_t)a.M * a.top_k * 4;
  auto lds = [&](int mt) { return (unsigned)(tables > (size_t)NW * mt * 1024 ? tables : (size_t)NW * mt * 1024); };
  if (a.M <= 16) hipLaunchKernelGGL((experts_down_kernel<T, G, 1, NW, 2>), grid, block, lds(1), s, a);
  else if (a.M <= 32) hipLaunchKernelGGL((experts_down_kernel<T, G, 2, NW, 2>), grid, block, lds(2), s, a);
  else hipLaunchKernelGGL((experts_down_kernel<T, G, 4, NW, 1>), grid, block, lds(4), s, a);
  return hipGetLastError();
}
template <typename T>
hipError_t launch_experts_gateup(const ExpertArgs& a, int group, hipStream_t s) {
  switch (group) {
    case 0: return gateup_of<T, 0>(a, s);
    case 32: return gateup_of<T, 32>(a, s);
    case 64: return gateup_of<T, 64>(a, s);
    default: return gateup_of<T, 128>(a, s);
  }
}
template <typename T>
hipError_t launch_experts_down(const ExpertArgs& a, int group, hipStream_t s) {
  switch (group) {
    case 0: return down_of<T, 0>(a, s);
    case 32: return down_of<T, 32>(a, s);
    case 64: return down_of<T, 64>(a, s);
    default: return down_of<T, 128>(a, s);
  }
}

// ------------------------------------------------------------------ routing
// A logit as an integer of the same order: NaN above everything, -0 equal to 0, and 0 below every logit.
__device__ __forceinline__ uint32_t logit_key(float v) {
  uint32_t u = __float_as_uint(v == 0.f ? 0.f : v);
  if (v != v) u = 0x7fffffffu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_logit(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) {
    const uint32_t o = (uint32_t)__shfl_xor((int)v, d);
    v = o > v ? o : v;
  }
  return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

// One wavefront, one token: lane j < top_k gets the token's j-th choice and its weight.  The experts lie in lane order
// (lane l: VPL l .. VPL l + VPL - 1), so among equal logits the lowest lane holds the lowest number.
// (-inf: not available, weight 0 and expert -1 - number.)
template <int VPL, typename L>
__device__ __forceinline__ void choose(const L* logits, int E, int top_k, bool normalize, int lane, int& expert, float& weight) {
  uint32_t key[VPL];
  float value[VPL];
#pragma unroll
  for (int v = 0; v < VPL; ++v) {
    const int e = lane * VPL + v;
    value[v] = e < E ? (float)logits[e] : -__builtin_inff();
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

template <int VPL, typename L>
__global__ void __launch_bounds__(256) route_kernel(const L* logits, float* weights, int64_t* experts, int64_t M, int E, int top_k,
                                                    int normalize) {
  const int lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= M) return;
  int e;
  float w;
  choose<VPL>(logits + t * E, E, top_k, normalize != 0, lane, e, w);
  if (lane < top_k) {
    weights[t * top_k + lane] = w;
    experts[t * top_k + lane] = e < 0 ? -1 - e : e;
  }
}

// The routing of at most 64 tokens, in one workgroup.
template <int VPL, typename L>
__global__ void __launch_bounds__(1024) plan_kernel(const L* logits, ExpertPlan p, int M, int E, int top_k, int normalize) {
  __shared__ uint32_t who[EXPERTS_MAX_E][2];  // tokens of an expert, a bit each
  __shared__ int index[EXPERTS_MAX_E];        // of an expert among those in use
  __shared__ short chosen[EXPERTS_MAX_M * EXPERTS_MAX_K];
  __shared__ int in_wave[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int i = tid; i < E * 2; i += 1024) (&who[0][0])[i] = 0u;
  __syncthreads();
  for (int t = wave; t < M; t += 16) {
    int e;
    float w;
    choose<VPL>(logits + (size_t)t * E, E, top_k, normalize != 0, lane, e, w);
    if (lane < top_k) {
      p.weight[t * top_k + lane] = w;
      chosen[t * top_k + lane] = (short)e;
      if (e >= 0) atomicOr(&who[e][t >> 5], 1u << (t & 31));
    }
  }
  __syncthreads();
  const bool used = tid < E && (who[tid][0] | who[tid][1]) != 0;
  const uint64_t ballot = __ballot(used);
  if (lane == 0) in_wave[wave] = __popcll(ballot);
  __syncthreads();
  int before = 0, total = 0;
  for (int w = 0; w < 16; ++w) {
    if (w < wave) before += in_wave[w];
    total += in_wave[w];
  }
  if (used) {
    const int i = before + __popcll(ballot & ((1ull << lane) - 1));
    index[tid] = i;
    p.active[1 + i] = tid;
    p.count[i] = (uint8_t)(__popc(who[tid][0]) + __popc(who[tid][1]));
  }
  if (tid == 0) p.active[0] = total;
  for (int i = tid; i < total * (EXPERTS_MAX_M / 4); i += 1024) ((int*)p.slot)[i] = -1;
  __syncthreads();
  for (int i = tid; i < M * top_k; i += 1024) {
    const int e = chosen[i], t = i / top_k;
    if (e < 0) continue;
    const uint64_t mask = (uint64_t)who[e][1] << 32 | who[e][0];
    const int at = index[e] * EXPERTS_MAX_M;
    p.tokens[at + __popcll(mask & ((1ull << t) - 1))] = (uint8_t)t;
    p.slot[at + t] = (int8_t)(i - t * top_k);
  }
}

#define GMLP_BY_EXPERTS(E, CALL)   \
  if ((E) <= 64) CALL(1);          \
  else if ((E) <= 128) CALL(2);    \
  else if ((E) <= 256) CALL(4);    \
  else CALL(8)

template <typename L>
hipError_t launch_route(const L* logits, float* weights, int64_t* experts, int64_t M, int E, int top_k, int normalize, hipStream_t s) {
#define CALL(V) \
  hipLaunchKernelGGL((route_kernel<V, L>), dim3((unsigned)((M + 3) / 4)), dim3(256), 0, s, logits, weights, experts, M, E, top_k, normalize)
  GMLP_BY_EXPERTS(E, CALL);
#undef CALL
  return hipGetLastError();
}
template <typename L>
hipError_t launch_experts_plan(const L* logits, const ExpertPlan& plan, int M, int E, int top_k, int normalize, hipStream_t s) {
#define CALL(V) hipLaunchKernelGGL((plan_kernel<V, L>), dim3(1), dim3(1024), 0, s, logits, plan, M, E, top_k, normalize)
  GMLP_BY_EXPERTS(E, CALL);
#undef CALL
  return hipGetLastError();
}

// ------------------------------------------------------------------ 4-bit storage
// One wavefront per tile and block; lane 16 q + r holds columns 32 s + 8 q + 0..7 of row r.
template <typename T, int G>
__global__ void __launch_bounds__(256) q4_quantize_kernel(const T* w, uint8_t* codes, T* scales, int64_t tiles, int blocks,
                                                          int64_t rows, int64_t cols, int tiles_each) {
  constexpr int GROUPS = Q4_BLOCK / G, PER = 4 / GROUPS;
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= tiles * blocks) return;
  const int64_t tile = unit / blocks, matrix = tile / tiles_each;
  const int block = (int)(unit - tile * blocks);
  const int64_t row = (tile - matrix * tiles_each) * Q4_TILE + r;
  const T* src = w + (matrix * rows + row) * cols;
  float v[4][8];
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int64_t c = (int64_t)block * Q4_BLOCK + s * 32 + q * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[s][i] = 0.f;
    if (row < rows && c < cols) {
      load_w<T, 4>(src + c, v[s]);
      load_w<T, 4>(src + c + 4, v[s] + 4);
    }
  }
  u32x4 out;
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    float most = 0.f;
#pragma unroll
    for (int s = g * PER; s < (g + 1) * PER; ++s)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float m = fabsf(v[s][i]);
        most = m > most || m != m ? m : most;  // (a NaN stays)
      }
#pragma unroll
    for (int d = 16; d <= 32; d <<= 1) {
      const float o = __shfl_xor(most, d);
      most = o > most || o != o ? o : most;
    }
    const T scale = Traits<T>::from_f32(most / 7.f);
    const float step = Traits<T>::to_f32(scale);
#pragma unroll
    for (int s = g * PER; s < (g + 1) * PER; ++s) {
      uint32_t word = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float n = step > 0.f ? rintf(v[s][i] / step) : 0.f;
        n = fminf(fmaxf(n, -8.f), 7.f);
        word |= (uint32_t)((int)n + 8) << (4 * (i / 2) + 16 * (i % 2));
      }
      out[s] = word;
    }
    if (q == 0) scales[((unit * 4 + r / 4) * GROUPS + g) * 4 + r % 4] = scale;
  }
  *(u32x4*)(codes + (unit * 64 + lane) * 16) = out;
}

template <typename T, int G>
__global__ void __launch_bounds__(256) q4_dequantize_kernel(const uint8_t* codes, const T* scales, T* w, int64_t tiles, int blocks,
                                                            int64_t rows, int64_t cols, int tiles_each) {
  constexpr int GROUPS = Q4_BLOCK / G, PER = 4 / GROUPS;
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= tiles * blocks) return;
  const int64_t tile = unit / blocks, matrix = tile / tiles_each;
  const int block = (int)(unit - tile * blocks);
  const int64_t row = (tile - matrix * tiles_each) * Q4_TILE + r;
  if (row >= rows) return;
  T* dst = w + (matrix * rows + row) * cols;
  const u32x4 in = *(const u32x4*)(codes + (unit * 64 + lane) * 16);
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int64_t c = (int64_t)block * Q4_BLOCK + s * 32 + q * 8;
    if (c >= cols) continue;
    const float scale = Traits<T>::to_f32(scales[((unit * 4 + r / 4) * GROUPS + s / PER) * 4 + r % 4]);
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = scale * (float)((int)(in[s] >> (4 * (i / 2) + 16 * (i % 2)) & 15u) - 8);
    store_w<T, 4>(dst + c, v);
    store_w<T, 4>(dst + c + 4, v + 4);
  }
}

#define GMLP_BY_GROUP(KERNEL, ...)                                                                                \
  const int tiles_each = (int)((rows + Q4_TILE - 1) / Q4_TILE), blocks = (int)((cols + Q4_BLOCK - 1) / Q4_BLOCK); \
  const int64_t tiles = count * tiles_each;                                                                       \
  const dim3 grid((unsigned)((tiles * blocks + 3) / 4));                                                          \
  if (group == 32) hipLaunchKernelGGL((KERNEL<T, 32>), grid, dim3(256), 0, s, __VA_ARGS__, tiles, blocks, rows, cols, tiles_each);      \
  else if (group == 64) hipLaunchKernelGGL((KERNEL<T, 64>), grid, dim3(256), 0, s, __VA_ARGS__, tiles, blocks, rows, cols, tiles_each); \
  else hipLaunchKernelGGL((KERNEL<T, 128>), grid, dim3(256), 0, s, __VA_ARGS__, tiles, blocks, rows, cols, tiles_each);                \
  return hipGetLastError()

template <typename T>
hipError_t launch_q4_quantize(const T* w, uint8_t* codes, T* scales, int64_t count, int64_t rows, int64_t cols, int group, hipStream_t s) {
  GMLP_BY_GROUP(q4_quantize_kernel, w, codes, scales);
}
template <typename T>
hipError_t launch_q4_dequantize(const uint8_t* codes, const T* scales, T* w, int64_t count, int64_t rows, int64_t cols, int group,
                                hipStream_t s) {
  GMLP_BY_GROUP(q4_dequantize_kernel, codes, scales, w);
}

#define GMLP_INSTANTIATE(T)                                                                                                    \
  template hipError_t launch_experts_gateup<T>(const ExpertArgs&, int, hipStream_t);                                          \
  template hipError_t launch_experts_down<T>(const ExpertArgs&, int, hipStream_t);                                            \
  template hipError_t launch_q4_quantize<T>(const T*, uint8_t*, T*, int64_t, int64_t, int64_t, int, hipStream_t);             \
  template hipError_t launch_q4_dequantize<T>(const uint8_t*, const T*, T*, int64_t, int64_t, int64_t, int, hipStream_t);     \
  template hipError_t launch_route<T>(const T*, float*, int64_t*, int64_t, int, int, int, hipStream_t);                       \
  template hipError_t launch_experts_plan<T>(const T*, const ExpertPlan&, int, int, int, int, hipStream_t);
GMLP_INSTANTIATE(f16)
GMLP_INSTANTIATE(bf16)
template hipError_t launch_route<float>(const float*, float*, int64_t*, int64_t, int, int, int, hipStream_t);
template hipError_t launch_experts_plan<float>(const float*, const ExpertPlan&, int, int, int, int, hipStream_t);

}  // namespace gmlp
