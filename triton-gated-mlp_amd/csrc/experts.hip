// Expert layers and 4-bit weights for a few token rows (M <= 64).
//
//   route, plan    softmax of the router's logits, the top_k largest of each token; which experts are in use, by whom
//   gate/up        h[p] = act(W_gate_e x_t + b_gate) * (W_up_e x_t + b_up)   for every pair p = (token t, its choice e)
//   down           y[t] = sum_e w_te W_down_e h_te + b_down
//
// The products are bound by the weights' way from memory: each weight is read once for the tokens of an entry (all of a
// dense call's, up to 16 or 32 of an expert's) and feeds one v_mfma_f32_16x16x32 column per token row.  A workgroup takes R
// tiles of 16 weight rows (gate/up: of each matrix), R = 1, 2 or 4; its wavefronts split the reduction and add up through LDS
// in a fixed order, so results do not depend on timing.  Every load is a buffer load with an exact descriptor: rows past
// the matrix, columns past its end, tokens that an expert does not have and the stages past the end of a wavefront's run all
// get an offset beyond it, which reads as zero and moves no data.
//
// 4-bit weights keep their integers for the matrix product (exact in 16 bits); a group's scale is applied to the
// product in fp32, so what is multiplied is scale·n itself, not its rounding.
#include "experts.hpp"

#include "launch.hpp"
#include "lds_dma.hpp"
#include "routing.hpp"

namespace gmlp {

typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));
typedef f16 f16x2 __attribute__((ext_vector_type(2)));

// Byte offsets beyond any descriptor (all are shorter than EX_PAST): of a lane that loads nothing, and of a stage that does
// not exist.  Their sum does not wrap.
constexpr uint32_t EX_NOWHERE = 0x80000000u, EX_PAST = EXPERTS_MAX_BYTES;

typedef __amdgpu_buffer_rsrc_t ex_rsrc;
__device__ __forceinline__ ex_rsrc ex_make_rsrc(const void* p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, (int)bytes, 0x00020000);
}
// Tokens for each expert on average up to which an entry has one token tile (token_tiles).
constexpr int ONE_TILE_TOKENS = 12;
// LDS of experts_down_kernel for the tables of the largest routing: without GATHER 16 tokens; with it one token tile an entry or,
// beyond ONE_TILE_TOKENS, two.
constexpr int ex_tables(int entries, bool gather, int token_tiles, int pairs) {
  return entries * (gather ? 4 + 1 + 16 * token_tiles * 2 : 4 + EXPERTS_MAX_M) + pairs * 4;
}
constexpr int ex_tables_at_most(bool gather, int token_tiles) {
  constexpr int pairs = EXPERTS_MAX_M * EXPERTS_MAX_K;
  return !gather ? ex_tables(16 * EXPERTS_MAX_K, false, 1, 16 * EXPERTS_MAX_K)
                 : ex_tables((token_tiles == 1 ? EXPERTS_MAX_E : pairs / ONE_TILE_TOKENS) + pairs / 16, true, token_tiles, pairs);
}
constexpr int EX_STREAM = 2;  // cache policy: non-temporal, what is read once
template <int POLICY = 0>
__device__ __forceinline__ u32x4 ex_load16(ex_rsrc r, uint32_t lane_off, uint32_t off) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)lane_off, (int)off, POLICY));
}
template <int POLICY = 0>
__device__ __forceinline__ u32x2 ex_load8(ex_rsrc r, uint32_t lane_off, uint32_t off) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, (int)lane_off, (int)off, POLICY));
}

// ------------------------------------------------------------------ 4-bit integers as 16-bit floats
// One 32-bit word holds columns 0, 2, 4, 6 of eight in its low half's nibbles and 1, 3, 5, 7 in its high half's, so
// one mask takes a pair of neighbours apart.  SCALE: what the products have to be multiplied by.
template <typename T>
struct Int4;
template <>
struct Int4<f16> {
  static constexpr float SCALE = 1.f;
  uint32_t magic;
  __device__ __forceinline__ Int4() : magic(0x64006400u) {
    asm("" : "+v"(magic));  // (in a register, so that the mask and it go into one instruction)
  }
  // 0x6400 | u is 1024 + u in fp16, 0x6400 | 16 u is 1024 + 16 u; u = n + 8
  __device__ __forceinline__ f16x8 floats(uint32_t w) const {
    const uint32_t v = w >> 8;
    const f16x2 low = {(f16)-1032.f, (f16)-1032.f}, high = {(f16)-72.f, (f16)-72.f}, part = {(f16)0.0625f, (f16)0.0625f};
    const f16x2 o[4] = {pair(w & 0x000f000fu | magic) + low, pair(w & 0x00f000f0u | magic) * part + high,
                        pair(v & 0x000f000fu | magic) + low, pair(v & 0x00f000f0u | magic) * part + high};
    return __builtin_bit_cast(f16x8, o);
  }
  static __device__ __forceinline__ f16x2 pair(uint32_t u) { return __builtin_bit_cast(f16x2, u); }
};
template <>
struct Int4<bf16> {
  static constexpr float SCALE = 16.f;
  // v_cvt_off_f32_i4 makes n / 16 of a signed nibble; a bf16 is the upper half of the fp32 number
  template <int BYTE>
  static __device__ __forceinline__ uint32_t sixteenth(uint32_t v) {
    float f;
    if constexpr (BYTE == 0) f = __builtin_amdgcn_cvt_off_f32_i4((int)v);
    else if constexpr (BYTE == 1) asm("v_cvt_off_f32_i4_sdwa %0, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1" : "=v"(f) : "v"(v));
    else if constexpr (BYTE == 2) asm("v_cvt_off_f32_i4_sdwa %0, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2" : "=v"(f) : "v"(v));
    else asm("v_cvt_off_f32_i4_sdwa %0, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3" : "=v"(f) : "v"(v));
    return __builtin_bit_cast(uint32_t, f);
  }
  __device__ __forceinline__ bf16x8 floats(uint32_t w) const {
    const uint32_t even = w ^ 0x88888888u, odd = even >> 4;
    const u32x4 o = {upper(sixteenth<2>(even), sixteenth<0>(even)), upper(sixteenth<2>(odd), sixteenth<0>(odd)),
                     upper(sixteenth<3>(even), sixteenth<1>(even)), upper(sixteenth<3>(odd), sixteenth<1>(odd))};
    return __builtin_bit_cast(bf16x8, o);
  }
  static __device__ __forceinline__ uint32_t upper(uint32_t hi, uint32_t lo) { return __builtin_amdgcn_perm(hi, lo, 0x07060302u); }
};

template <typename T>
__device__ __forceinline__ float bits_to_f32(uint32_t u) {
  return (float)__builtin_bit_cast(T, (unsigned short)u);
}

// ------------------------------------------------------------------ choice of experts
// The routing of the only token of a call: every wavefront of gate/up finds it from the logits, and one leaves the plan for
// down.  A launch less, and 1 us in the place of 4.
constexpr int SOLO_MAX_E = 256;
__device__ __forceinline__ void choose_solo(const ExpertArgs& a, int lane, int& expert, float& weight) {
  auto logit = [&](int i) -> float {
    if (a.logits_dtype == 0) return (float)((const f16*)a.logits)[i];
    if (a.logits_dtype == 1) return (float)((const bf16*)a.logits)[i];
    return ((const float*)a.logits)[i];
  };
  if (a.E <= 64) choose<1>(logit, a.E, a.top_k, a.normalize != 0, lane, expert, weight);
  else choose<SOLO_MAX_E / 64>(logit, a.E, a.top_k, a.normalize != 0, lane, expert, weight);
}

__device__ __forceinline__ void leave_plan(const ExpertArgs& a, int lane, int expert, float weight) {
  const uint64_t chosen = __ballot(lane < a.top_k && expert >= 0);
  if (lane == 0) a.plan.active[0] = __popcll(chosen);
  if (lane >= a.top_k) return;
  a.plan.weight[lane] = weight;
  if (expert >= 0) {
    const int i = __popcll(chosen & ((1ull << lane) - 1));
    a.plan.active[1 + i] = expert;
    a.plan.slot[i * EXPERTS_MAX_M] = (int8_t)lane;
  }
}

// ------------------------------------------------------------------ a block of the reduction
// 16 rows of NT weight tiles by 64 columns (16-bit weights) or 128 (4-bit ones), and MT tiles of 16 token rows by the
// same columns.  An MFMA wants neighbouring lanes on different rows; a load of that kind takes a cycle of the address unit per
// lane (16-bit down projections stood at 8 bytes a clock and CU, 5 TB/s, whatever the number of loads in flight).  So rows
// are loaded as they lie, 128 or 256 bytes of a row by neighbouring lanes, and change lanes through a piece of LDS of
// the wavefront's own (in order, so without a barrier).  4-bit weights are stored as the MFMA takes them.
// XR: loads per token tile; a load brings 8 (16-bit weights) or 4 token rows.
template <typename T, int G, int NT, int MT, int XR>
struct Block {
  typedef typename Traits<T>::vec8 vec8;
  static constexpr int COLS = G ? Q4_BLOCK : 64;
  static constexpr int STEPS = COLS / 32;
  static constexpr int GROUPS = G ? Q4_BLOCK / G : 1;
  static constexpr int PIECES = COLS / 8;       // 16-byte pieces of a row
  static constexpr int ROWS = 64 / PIECES;      // rows of a load
  static constexpr int WL = G ? 1 : 16 / ROWS;  // loads of a weight tile
  static constexpr int TILE = 16 * COLS * 2;    // bytes of a tile in LDS
  static constexpr int WB = G ? 0 : NT;         // weight tiles in LDS
  // 4-bit weights: token rows go to LDS without passing through registers (buffer_load ... lds), a slot for each stage; two
  // stages of the weights then fit where one of both did.  16-bit weights, and a single load of token rows, whose four
  // registers are no matter: one slot for what the wavefront multiplies.
  static constexpr bool DMA = G != 0 && MT * XR > 1;
  static constexpr int SLOT = (MT + WB) * TILE;
  static constexpr int lds_bytes(int depth) { return (DMA ? depth : 1) * SLOT; }  // of a wavefront
  static_assert(XR * ROWS <= 16, "a token tile has 16 rows");
  u32x4 w[NT][WL];
  u32x2 sc[NT][GROUPS];
  u32x4 x[DMA ? 1 : MT][DMA ? 1 : XR];

  // from tile `tile` of an expert's matrix on, of `rows` x `cols`: `tiles` of them
  static __device__ __forceinline__ ex_rsrc weights_of(const ExpertWeights& m, int expert, int tile, int tiles, int rows, int cols) {
    const int all = (rows + Q4_TILE - 1) / Q4_TILE, blocks = (cols + Q4_BLOCK - 1) / Q4_BLOCK;
    const int own = all - tile < tiles ? all - tile : tiles;
    if (G) return ex_make_rsrc((const char*)m.w + ((size_t)expert * all + tile) * blocks * 1024, (uint32_t)(own * blocks) * 1024u);
    const int first = tile * Q4_TILE, r = rows - first < tiles * Q4_TILE ? rows - first : tiles * Q4_TILE;
    return ex_make_rsrc((const T*)m.w + ((size_t)expert * rows + first) * cols, (uint32_t)r * (uint32_t)cols * 2u);
  }
  static __device__ __forceinline__ ex_rsrc scales_of(const ExpertWeights& m, int expert, int tile, int tiles, int rows, int cols) {
    const int all = (rows + Q4_TILE - 1) / Q4_TILE, blocks = (cols + Q4_BLOCK - 1) / Q4_BLOCK;
    const int own = all - tile < tiles ? all - tile : tiles;
    const uint32_t pitch = (uint32_t)blocks * (Q4_TILE * GROUPS * 2);
    return ex_make_rsrc((const char*)m.scales + ((size_t)expert * all + tile) * pitch, G ? (uint32_t)own * pitch : 0u);
  }
  // Row of a tile and byte in the row's segment that a lane loads.
  static __device__ __forceinline__ int load_row(int i, int lane) { return i * ROWS + lane / PIECES; }
  // (DMA fills LDS in the order of the lanes: the lane loads the piece that `at` has in its place)
  static __device__ __forceinline__ int load_piece(int i, int lane) { return DMA ? lane % PIECES ^ load_row(i, lane) : lane % PIECES; }
  static __device__ __forceinline__ uint32_t load_byte(int i, int lane) { return (uint32_t)load_piece(i, lane) * 16u; }
  // Byte in LDS of a row's piece.  256-byte rows reach all banks, 128-byte ones two by two.
  static __device__ __forceinline__ uint32_t at(int row, int piece) {
    return (uint32_t)(row * PIECES + (piece ^ (PIECES == 16 ? row : row >> 1))) * 16u;
  }

  // Tile n: tile r behind the descriptors' first one.  `ok`: the block exists; `tail`: it may reach past the last column.
  __device__ __forceinline__ void load_weights(int n, int r, ex_rsrc rw, ex_rsrc rs, int kb, bool ok, bool tail, int cols, int lane) {
    if (G) {
      const uint32_t unit = (uint32_t)(r * ((cols + Q4_BLOCK - 1) / Q4_BLOCK) + kb);
      w[n][0] = ex_load16<EX_STREAM>(rw, (uint32_t)lane * 16u, ok ? unit * 1024u : EX_PAST);
      const uint32_t from = ok ? unit * (GROUPS * 32u) : EX_PAST, own = (uint32_t)(lane >> 4) * (GROUPS * 8u);
      if constexpr (GROUPS == 1) {
        sc[n][0] = ex_load8(rs, own, from);
      } else {
#pragma unroll
        for (int g = 0; g < GROUPS; g += 2) {
          const u32x4 v = ex_load16(rs, own + (uint32_t)g * 8u, from);
          sc[n][g] = u32x2{v[0], v[1]};
          sc[n][g + 1] = u32x2{v[2], v[3]};
        }
      }
    } else {
      const uint32_t lane_off = tail && beyond(kb, cols, 0, lane) ? EX_NOWHERE : (uint32_t)load_row(0, lane) * (uint32_t)cols * 2u + load_byte(0, lane);
#pragma unroll
      for (int i = 0; i < WL; ++i)
        w[n][i] = ex_load16<EX_STREAM>(rw, lane_off, ok ? ((uint32_t)(r * Q4_TILE + i * ROWS) * (uint32_t)cols + (uint32_t)(kb * COLS)) * 2u : EX_PAST);
    }
  }
  // (What goes into scalar operands of inline assembly has to be known to be uniform.)
  static __device__ __forceinline__ uint32_t uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }
  static __device__ __forceinline__ buffer_rsrc uniform_rsrc(const void* p, uint32_t bytes) {
    buffer_rsrc r = make_rsrc(p, bytes);
#pragma unroll
    for (int i = 0; i < 3; ++i) r[i] = __builtin_amdgcn_readfirstlane(r[i]);
    return r;
  }
  static __device__ __forceinline__ bool beyond(int kb, int cols, int i, int lane) { return kb * COLS + load_piece(i, lane) * 8 >= cols; }
  // row[m][i]: byte offset of the lane's piece of its token row, or EX_NOWHERE; slot: LDS of the stage (DMA)
  __device__ __forceinline__ void load_tokens(const void* tokens, uint32_t bytes, const uint32_t (&row)[MT][XR], int kb, bool ok, bool tail,
                                              int cols, int lane, uint32_t slot) {
    const uint32_t from = ok ? (uint32_t)(kb * COLS) * 2u : EX_PAST;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < XR; ++i) {
        const uint32_t lane_off = tail && beyond(kb, cols, i, lane) ? EX_NOWHERE : row[m][i];
        if constexpr (DMA) load16_to_lds(uniform_rsrc(tokens, bytes), lane_off, uniform(from), uniform(slot + (uint32_t)(m * TILE + i * 1024)));
        else x[m][i] = ex_load16(ex_make_rsrc(tokens, bytes), lane_off, from);
      }
  }

  // Between a wavefront's writes to LDS and its other lanes' reads: the LDS takes them in order, the compiler has to leave them so.
  static __device__ __forceinline__ void turn() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
  }

  // Columns of a tile: step s takes 32 s + 8 (lane / 16) + 0..7.  (Token rows that XR leaves out are whatever LDS holds: their
  // columns of the product are not used.)
  static __device__ __forceinline__ vec8 operand(const char* tile, int s, int lane) {
    return *(const vec8*)(tile + at(lane & 15, s * 4 + (lane >> 4)));
  }
  template <int L>
  static __device__ __forceinline__ void to_lds(char* tile, const u32x4 (&v)[L], int lane) {
#pragma unroll
    for (int i = 0; i < L; ++i) *(u32x4*)(tile + at(load_row(i, lane), lane % PIECES)) = v[i];
  }
  __device__ __forceinline__ void multiply(const Int4<T>& int4, char* slot, int lane, f32x4 (&acc)[NT][MT]) {
    if constexpr (DMA) {
      // The token rows were asked for ahead of the weights and scales, and loads return in order: once the last scale is there
      // (the compiler waits for it here, it goes into the statement), they are in LDS.
      asm volatile("" : "+v"(sc[NT - 1][GROUPS - 1]) : : "memory");
    } else {
#pragma unroll
      for (int m = 0; m < MT; ++m) to_lds(slot + m * TILE, x[m], lane);
#pragma unroll
      for (int n = 0; n < WB; ++n) to_lds(slot + (MT + n) * TILE, w[n], lane);
      turn();
    }
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      constexpr int SG = STEPS / GROUPS;  // steps of a group
      vec8 xf[MT][SG];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int s = 0; s < SG; ++s) xf[m][s] = operand(slot + m * TILE, g * SG + s, lane);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if constexpr (G != 0) {
          f32x4 part[MT];
#pragma unroll
          for (int m = 0; m < MT; ++m) part[m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s = 0; s < SG; ++s) {
            const vec8 a = int4.floats(w[n][0][g * SG + s]);
#pragma unroll
            for (int m = 0; m < MT; ++m) part[m] = Traits<T>::mfma16(a, xf[m][s], part[m]);
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float f = bits_to_f32<T>(sc[n][g][r / 2] >> (16 * (r % 2)) & 0xffffu) * Int4<T>::SCALE;
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[n][m][r] += f * part[m][r];
          }
        } else {
          const char* const tile = slot + (MT + n) * TILE;
#pragma unroll
          for (int s = 0; s < SG; ++s) {
            const vec8 a = operand(tile, s, lane);
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[n][m] = Traits<T>::mfma16(a, xf[m][s], acc[n][m]);
          }
        }
      }
      // A group at a time: the scheduler would fetch the next one's token operands ahead, and pay in registers.
      if constexpr (MT > 1 && GROUPS > 1) __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (DMA) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the slot has been read
    else turn();
  }
};

// f(0), f(1), ... f(D - 1), each a constant
template <int D, int AT = 0, typename F>
__device__ __forceinline__ void each_stage(F&& f) {
  if constexpr (AT < D) {
    f(std::integral_constant<int, AT>{});
    each_stage<D, AT + 1>(f);
  }
}

// Adds up the wavefronts' sums, a few units of U vectors at a time through LDS, and calls done(unit, sums) for each in one
// wavefront.
template <int NW, int NU, int U>
constexpr int units_at_a_time() {
  return NW * NU * U <= 32 ? NU : 32 / (NW * U);  // 32 KiB
}
template <int NW, int NU, int U, typename F>
__device__ __forceinline__ void sum_wavefronts(const f32x4 (&acc)[NU][U], char* smem, int wave, int lane, F&& done) {
  constexpr int EACH = units_at_a_time<NW, NU, U>();
  static_assert(EACH > 0, "a unit of every wavefront fits");
  f32x4* const part = (f32x4*)smem;  // [NW][EACH][U][64]
#pragma unroll
  for (int first = 0; first < NU; first += EACH) {
    __syncthreads();  // the readers of what LDS held before
#pragma unroll
    for (int i = 0; i < EACH; ++i)
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (first + i < NU) part[((wave * EACH + i) * U + u) * 64 + lane] = acc[first + i][u];
    __syncthreads();
    for (int i = wave; i < EACH && first + i < NU; i += NW) {
      f32x4 sum[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        sum[u] = part[(i * U + u) * 64 + lane];
#pragma unroll
        for (int w = 1; w < NW; ++w) sum[u] += part[((w * EACH + i) * U + u) * 64 + lane];
      }
      done(first + i, sum);
    }
  }
}

// ------------------------------------------------------------------ gate/up
// A workgroup: 16 * R rows of each matrix of one expert.  What bounds it is the weights' stream: 16 bits, 8 experts of K=4096,
// N=14336, one token on two of them, 470 MB in 76 us (6.2 TB/s; a device copy moves 5.3); 4 bits, all 8 of them for
// 16 tokens, 480 MB in 80 us (6.0 TB/s).  One matrix of 4 bits is shorter than its start and end: K=2048, N=5632, one token, 12 MB
// in 6.5 us.  M=48, K=4096, N=11008, groups of 64, 48 MB in 25 us: there the grid (344 workgroups on two
// places a CU: 88 CUs hold two of them) and the conversions bound it.
template <typename T, int G, int MT, int XR, int R, int NW, int D>
constexpr int gateup_lds() {
  constexpr int ring = NW * Block<T, G, 2 * R, MT, XR>::lds_bytes(D), part = NW * units_at_a_time<NW, R * MT, 2>() * 2 * 1024;
  return ring > part ? ring : part;
}
// (Two or three token tiles: 256 registers, so that a CU holds two workgroups of four wavefronts.  M=48, K=4096, N=11008, groups of
// 64 36.7 -> 25.5 us.  Four tiles do not fit.)
template <typename T, int G, int MT, int XR, int R, int NW, int D>
__global__ void __launch_bounds__(NW * 64, MT > 1 && MT < 4 && R <= 2 ? 2 : 1) experts_gateup_kernel(ExpertArgs a) {
  typedef Block<T, G, 2 * R, MT, XR> B;
  extern __shared__ __align__(16) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, kg = lane >> 4;
  const int strips = (a.N + R * Q4_TILE - 1) / (R * Q4_TILE);
  const int slot = (int)blockIdx.x / strips, tile = ((int)blockIdx.x - slot * strips) * R;
  int expert = 0, count = a.M;
  if (a.routing == ROUTING_SOLO) {
    int e;
    float w;
    choose_solo(a, lane, e, w);
    expert = __builtin_amdgcn_readlane(e, slot);
    if (blockIdx.x == 0 && wave == 0) leave_plan(a, lane, e, w);
    if (expert < 0) return;
  } else if (a.routing == ROUTING_PLAN) {
    if (slot >= a.plan.active[0]) return;
    expert = a.plan.active[1 + slot];
    count = a.plan.count[slot];
  }
  const ex_rsrc rw[2] = {B::weights_of(a.gate, expert, tile, R, a.N, a.K), B::weights_of(a.up, expert, tile, R, a.N, a.K)};
  const ex_rsrc rs[2] = {B::scales_of(a.gate, expert, tile, R, a.N, a.K), B::scales_of(a.up, expert, tile, R, a.N, a.K)};
  const int blocks = (a.K + B::COLS - 1) / B::COLS;
  const int b0 = blocks * wave / NW, run = blocks * (wave + 1) / NW - b0;
  const int rot = run > 1 ? (int)blockIdx.x % run : 0;
  const bool ragged = a.K % B::COLS != 0;
  const Int4<T> int4;
  char* const lds = smem + wave * B::lds_bytes(D);
  const uint32_t lds_at = (uint32_t)(uintptr_t)(lds_void*)lds;

  uint32_t row[MT][XR];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < XR; ++i) {
      const int j = 16 * m + B::load_row(i, lane);
      const int t = j >= count ? 0 : a.routing == ROUTING_PLAN ? a.plan.pairs[slot * EXPERTS_MAX_M + j] / a.top_k : j;
      row[m][i] = j < count ? (uint32_t)t * (uint32_t)a.K * 2u + B::load_byte(i, lane) : EX_NOWHERE;
    }
  B st[D];
  auto load_block = [&](B& b, int kb, bool ok, bool tail, int d) {
    b.load_tokens(a.x, (uint32_t)a.M * (uint32_t)a.K * 2u, row, kb, ok, tail, a.K, lane, lds_at + (uint32_t)(d * B::SLOT));
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int n = 0; n < 2; ++n) b.load_weights(2 * r + n, r, rw[n], rs[n], kb, ok, tail, a.K, lane);
  };
  auto load = [&](B& b, int i, int d) {
    const int kb = b0 + (i + rot < run ? i + rot : i + rot - run);
    if (ragged && kb + 1 == blocks) load_block(b, kb, i < run, true, d);
    else load_block(b, kb, i < run, false, d);
  };
  f32x4 acc[2 * R][MT];
#pragma unroll
  for (int n = 0; n < 2 * R; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[n][m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int d = 0; d < D; ++d) load(st[d], d, d);
  int i = 0;
  for (; i + D < run; i += D)
#pragma unroll
    for (int d = 0; d < D; ++d) {
      st[d].multiply(int4, lds + (B::DMA ? d * B::SLOT : 0), lane, acc);
      load(st[d], i + d + D, d);
    }
  each_stage<D>([&](auto d) {
    if (i + d < run) st[d].multiply(int4, lds + (B::DMA ? d * B::SLOT : 0), lane, acc);
  });
  if constexpr (B::DMA) wait_vmem<0>();  // stages past the end bring nothing, but they write: not into the sums
  f32x4 both[R * MT][2];
#pragma unroll
  for (int i = 0; i < R * MT; ++i)
#pragma unroll
    for (int n = 0; n < 2; ++n) both[i][n] = acc[i / MT * 2 + n][i % MT];
  sum_wavefronts<NW>(both, smem, wave, lane, [&](int unit, const f32x4 (&sum)[2]) {
    const int r = unit / MT, j = 16 * (unit - r * MT) + r16, first = (tile + r) * Q4_TILE + 4 * kg;
    if (j >= count || first >= a.N) return;
    float v[2][4];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int q = 0; q < 4; ++q) v[n][q] = sum[n][q];
      if (a.bias[n]) add_w<T, 4>((const T*)a.bias[n] + first, v[n]);
    }
    float h[4];
    act_fwd_w<4>(a.act, v[0], h);
#pragma unroll
    for (int q = 0; q < 4; ++q) h[q] *= v[1][q];
    const int p = a.routing == ROUTING_SOLO ? slot : a.routing == ROUTING_PLAN ? a.plan.pairs[slot * EXPERTS_MAX_M + j] : j;
    store_w<T, 4>((T*)a.h + (size_t)p * a.N + first, h);
    if (a.h_low) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float kept = (float)(T)h[q];
        h[q] = __builtin_isfinite(kept) ? h[q] - kept : 0.f;
      }
      store_w<T, 4>((T*)a.h + (size_t)(a.M * a.top_k + p) * a.N + first, h);
    }
  });
}

// ------------------------------------------------------------------ down
// The blocks of all experts in use, one expert behind the other, are shared out evenly over the wavefronts.  What an
// expert gives is added to a token's sum only where the token chose it (a weight that is not finite in one
// expert stays out of the others' tokens).
// GATHER: token tiles are an entry's tokens, as many as its expert has, and its products are added to the tokens' sums in LDS;
// without, they are the call's tokens (M <= 16 * MT), whose sums are registers.  With more tokens than one tile holds and
// few of them for each expert, most columns would be empty: M=50, K=2816, N=5136, 32 experts, 4 bits, one of them a
// token, the whole layer 348 us without, 143 with.
// 16 bits, two experts of K=4096, N=14336 for a token, 235 MB in 40 us (5.9 TB/s); 4 bits, eight for 16 tokens, 240 MB in
// 45 us (5.3 TB/s) and 4.5 for the parts' sum; one matrix, K=8192, N=28672, 16 tokens, 121 MB in 25 us (4.8 TB/s); K=2048, N=5632,
// one token, 6 MB in 5.5 us, mostly its start and the join of the wavefronts.
// h_low: of as few tokens as half a load brings (2 with 4-bit weights, 4 with 16-bit ones) every hidden state comes as two 16-bit
// values, its rounding and what that left, in columns 2t and 2t + 1.  Rounding h to 16 bits alone costs as much as rounding
// y does; with more tokens it is rounded, as FusedGatedMLP's is: 6 tokens, K=4384, N=18032, 4 bits 54.9 us with both, 48.4 without.  bf16, 1 token,
// K=2048, N=5632, 4 bits: 11.9 -> 12.5 us, y off by 0.0017 of its norm instead of 0.0024.
template <typename T, int G, int MT, int XR, int R, int NW, int D>
constexpr int down_lds() {
  constexpr int ring = NW * Block<T, G, R, MT, XR>::lds_bytes(D), part = NW * units_at_a_time<NW, R * MT, 1>() * 1024;
  return ring > part ? ring : part;
}
template <typename T, int G, int MT, int XR, int R, int NW, int D, bool GATHER>
__global__ void __launch_bounds__(NW * 64) experts_down_kernel(ExpertArgs a) {
  typedef Block<T, G, R, MT, XR> B;
  extern __shared__ __align__(16) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, kg = lane >> 4, tile = (int)blockIdx.x * R;
  const int pairs = a.M * a.top_k, low = MT == 1 && !GATHER ? a.h_low : 0;
  // tables: the entries' experts, the pairs' weights, the slots or (GATHER) the pairs of each entry and their number
  int in_use = 1;
  char* at = smem + down_lds<T, G, MT, XR, R, NW, D>();
  float* const own = (float*)at + wave * (R * Q4_TILE) * a.M;  // GATHER: the wavefront's sums, [M][R * 16]
  if constexpr (GATHER) {
    for (int i = lane; i < a.M * R * Q4_TILE; i += 64) own[i] = 0.f;
    at += (size_t)NW * a.M * R * Q4_TILE * sizeof(float);
  }
  int* const numbers = (int*)at;
  float* weight = nullptr;
  int8_t* slots = nullptr;
  uint16_t* which = nullptr;
  uint8_t* counts = nullptr;
  if (a.routing == ROUTING_PLAN) {
    in_use = a.plan.active[0];
    const int rows = a.M == 1 ? pairs : in_use;  // (all there can be: their loads do not wait for the number)
    weight = (float*)(numbers + rows);
    for (int i = threadIdx.x; i < rows; i += NW * 64) numbers[i] = a.plan.active[1 + i];
    for (int i = threadIdx.x; i < pairs; i += NW * 64) weight[i] = a.plan.weight[i];
    if constexpr (GATHER) {
      which = (uint16_t*)(weight + pairs);
      counts = (uint8_t*)(which + rows * 16 * MT);
      for (int i = threadIdx.x; i < rows * 16 * MT; i += NW * 64)
        which[i] = a.plan.pairs[i / (16 * MT) * EXPERTS_MAX_M + i % (16 * MT)];
      for (int i = threadIdx.x; i < rows; i += NW * 64) counts[i] = a.plan.count[i];
    } else {
      slots = (int8_t*)(weight + pairs);
      for (int i = threadIdx.x; i < rows * (EXPERTS_MAX_M / 4); i += NW * 64)
        ((int*)slots)[i] = ((const int*)a.plan.slot)[i];
    }
    __syncthreads();
  }
  const int blocks = (a.N + B::COLS - 1) / B::COLS;
  const int total = in_use * blocks;
  const int parts = NW * (int)gridDim.y, me_part = (int)blockIdx.y * NW + wave;
  const int b0 = (int)((int64_t)total * me_part / parts), run = (int)((int64_t)total * (me_part + 1) / parts) - b0;
  const int rot = run > 1 ? (int)blockIdx.x % run : 0;
  const bool ragged = a.N % B::COLS != 0;
  const Int4<T> int4;
  char* const lds = smem + wave * B::lds_bytes(D);
  const uint32_t lds_at = (uint32_t)(uintptr_t)(lds_void*)lds;

  // row of h behind column j of entry e, or -1
  auto pair_of = [&](int e, int j) -> int {
    if constexpr (GATHER) return j < counts[e] ? which[e * (16 * MT) + j] : -1;
    if (j >= a.M || a.routing == ROUTING_DENSE) return j < a.M ? j : -1;
    const int s = slots[e * EXPERTS_MAX_M + j];
    return s < 0 ? -1 : j * a.top_k + s;
  };
  // where loads go on: expert, block of it
  const int first_e = b0 / blocks, first_b = b0 - first_e * blocks;
  int le = (b0 + rot) / blocks, lb = b0 + rot - le * blocks;
  uint32_t row[MT][XR];
  ex_rsrc rw, rs;
  auto enter = [&]() {
    const int e = le < in_use ? le : in_use - 1;
    const int number = a.routing == ROUTING_DENSE ? 0 : __builtin_amdgcn_readfirstlane(numbers[e]);
    rw = B::weights_of(a.down, number, tile, R, a.K, a.N);
    rs = B::scales_of(a.down, number, tile, R, a.K, a.N);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < XR; ++i) {
        const int j = 16 * m + B::load_row(i, lane), p = pair_of(e, j >> low);
        row[m][i] = p < 0 ? EX_NOWHERE : (uint32_t)(p + (j & low) * pairs) * (uint32_t)a.N * 2u + B::load_byte(i, lane);
      }
  };
  f32x4 acc[R][MT], sum[R * MT][1];
#pragma unroll
  for (int n = 0; n < R; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[n][m] = sum[n * MT + m][0] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (run > 0) {
    enter();
    B st[D];
    auto load_block = [&](B& b, bool ok, bool tail, int d) {
      b.load_tokens(a.h, (uint32_t)(pairs << low) * (uint32_t)a.N * 2u, row, lb, ok, tail, a.N, lane, lds_at + (uint32_t)(d * B::SLOT));
#pragma unroll
      for (int n = 0; n < R; ++n) b.load_weights(n, n, rw, rs, lb, ok, tail, a.N, lane);
    };
    auto load = [&](B& b, int i, int d) {
      if (ragged && lb + 1 == blocks) load_block(b, i < run, true, d);
      else load_block(b, i < run, false, d);
      const bool wrap = i + 1 == run - rot;
      if (++lb == blocks || wrap) {
        lb = wrap ? first_b : 0;
        le = wrap ? first_e : le + 1;
        enter();
      }
    };
    int me = le, mb = lb;  // where products are
    auto fold = [&]() {
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int p = pair_of(me, (16 * m + r16) >> low);
        const float w = p < 0 ? 0.f : a.routing == ROUTING_DENSE ? 1.f : weight[p];
#pragma unroll
        for (int n = 0; n < R; ++n) {
          if constexpr (GATHER) {
            if (p >= 0) {
              f32x4* const to = (f32x4*)(own + (p / a.top_k * R + n) * Q4_TILE + 4 * kg);
              f32x4 v = *to;
#pragma unroll
              for (int r = 0; r < 4; ++r) v[r] += w * acc[n][m][r];
              *to = v;
            }
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (p >= 0) sum[n * MT + m][0][r] += w * acc[n][m][r];
          }
          acc[n][m] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
      }
    };
#pragma unroll
    for (int d = 0; d < D; ++d) load(st[d], d, d);
    auto leave = [&](int i) {  // behind the products of block i
      const bool wrap = i + 1 == run - rot;
      if (++mb == blocks || wrap || i + 1 == run) {
        fold();
        mb = wrap ? first_b : 0;
        me = wrap ? first_e : me + 1;
      }
    };
    int i = 0;
    for (; i + D < run; i += D)
#pragma unroll
      for (int d = 0; d < D; ++d) {
        st[d].multiply(int4, lds + (B::DMA ? d * B::SLOT : 0), lane, acc);
        load(st[d], i + d + D, d);
        leave(i + d);
      }
    each_stage<D>([&](auto d) {
      if (i + d < run) {
        st[d].multiply(int4, lds + (B::DMA ? d * B::SLOT : 0), lane, acc);
        leave(i + d);
      }
    });
  }
  auto done = [&](int t, int first, f32x4 v) {
    if (t >= a.M || first >= a.K) return;
    if (gridDim.y > 1) {
      *(f32x4*)(a.partial + ((size_t)blockIdx.y * a.M + t) * a.K + first) = v;
      return;
    }
    if (a.y_f32) {  // (router logits: rows of whole fours)
      *(f32x4*)((float*)a.y + (size_t)t * a.K + first) = v;
      return;
    }
    float y[4] = {v[0], v[1], v[2], v[3]};
    if (a.bias[2]) add_w<T, 4>((const T*)a.bias[2] + first, y);
    store_w<T, 4>((T*)a.y + (size_t)t * a.K + first, y);
  };
  if constexpr (B::DMA) wait_vmem<0>();  // (as in gate/up)
  if constexpr (GATHER) {
    __syncthreads();
    const float* const all = own - wave * (R * Q4_TILE) * a.M;
    for (int i = threadIdx.x; i < a.M * R * 4; i += NW * 64) {
      f32x4 v = *(const f32x4*)(all + i * 4);
      for (int w = 1; w < NW; ++w) v += *(const f32x4*)(all + w * (R * Q4_TILE) * a.M + i * 4);
      done(i / (R * 4), tile * Q4_TILE + i % (R * 4) * 4, v);
    }
  } else {
    sum_wavefronts<NW>(sum, smem, wave, lane, [&](int unit, const f32x4 (&v)[1]) {
      const int n = unit / MT, j = 16 * (unit - n * MT) + r16;
      f32x4 y = v[0];
      if (low) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float rest = __shfl_xor(y[r], 1);
          y[r] += __builtin_isfinite(y[r]) ? rest : 0.f;  // (an infinite weight's product with a rest of 0)
        }
      }
      done(j & low ? a.M : j >> low, (tile + n) * Q4_TILE + 4 * kg, y);
    });
  }
}

// Second stage of a down projection whose reduction was split over workgroups: the parts' sums, in their order.
constexpr int DOWN_MAX_PARTS = 8;
template <typename T>
__global__ void __launch_bounds__(256) experts_join_kernel(ExpertArgs a, int parts) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4, all = (int64_t)a.M * a.K;
  if (i >= all) return;
  f32x4 v[DOWN_MAX_PARTS];
#pragma unroll
  for (int p = 0; p < DOWN_MAX_PARTS; ++p) v[p] = p < parts ? *(const f32x4*)(a.partial + p * all + i) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int p = 1; p < DOWN_MAX_PARTS; ++p) v[0] += v[p];
  float y[4] = {v[0][0], v[0][1], v[0][2], v[0][3]};
  if (a.bias[2]) add_w<T, 4>((const T*)a.bias[2] + i % a.K, y);
  store_w<T, 4>((T*)a.y + i, y);
}

// Experts that a call can use, and entries of its plan.
static int experts_at_most(const ExpertArgs& a) { return a.E < a.M * a.top_k ? a.E : a.M * a.top_k; }
static int entries_at_most(const ExpertArgs& a) { return a.routing == ROUTING_DENSE ? 1 : expert_entries(a.M, a.E, a.top_k); }
// Token tiles of an entry.  Experts of a plan: one, which nearly all of them fit in, up to 12 tokens for each on average,
// then two (weights of one with more tokens are read again).  us, plan, gate/up and down with one and two: 64 tokens, 32 experts of K=2048, N=1408,
// 8 tokens for each 105 106, 12 110 108, 14 122 110, 16 136 110; 4 bits 54 60, 57 62, 63 63, 70 64; 8 of K=N=4096, 16 bits, 48 tokens
// (12) 150 156, 56 tokens (14) 162 156; 4 bits 66 72, 72 73, 64 tokens (16) 79 73.
static int token_tiles(const ExpertArgs& a) {
  if (a.routing == ROUTING_DENSE || a.M <= 16) return (a.M + 15) / 16;
  return a.M * a.top_k <= ONE_TILE_TOKENS * a.E ? 1 : 2;
}
static double weight_bytes(const ExpertArgs& a, int group) {
  return (double)experts_at_most(a) * a.K * a.N * (group ? 0.5 + 2.0 / group : 2.0);
}

template <typename T, int G, int MT, int XR, int R, int NW, int D>
static hipError_t run_gateup(const ExpertArgs& a, hipStream_t s) {
  constexpr int LDS = gateup_lds<T, G, MT, XR, R, NW, D>();
  constexpr auto kern = experts_gateup_kernel<T, G, MT, XR, R, NW, D>;
  if constexpr (LDS > 64 * 1024)
    if (hipError_t e = allow_dynamic_lds(lds_kernel_of<kern, LDS>, s)) return e;
  const int strips = (a.N + R * Q4_TILE - 1) / (R * Q4_TILE);
  hipLaunchKernelGGL(kern, dim3((unsigned)(strips * entries_at_most(a))), dim3(NW * 64), LDS, s, a);
  return hipGetLastError();
}
template <typename T, int G, int MT, int XR, int R, int NW, int D, bool GATHER = false>
static hipError_t run_down(const ExpertArgs& a, int parts, hipStream_t s) {
  constexpr int LDS = down_lds<T, G, MT, XR, R, NW, D>(), SUMS = GATHER ? NW * R * Q4_TILE * 4 : 0,
                MOST = LDS + ex_tables_at_most(GATHER, MT) + SUMS * EXPERTS_MAX_M;
  static_assert(MOST <= 160 * 1024, "a workgroup has 160 KiB of LDS");
  const int lds = LDS + (a.routing == ROUTING_DENSE ? 0 : ex_tables(entries_at_most(a), GATHER, MT, a.M * a.top_k)) + SUMS * a.M;
  constexpr auto kern = experts_down_kernel<T, G, MT, XR, R, NW, D, GATHER>;
  if (lds > 64 * 1024)
    if (hipError_t e = allow_dynamic_lds(lds_kernel_of<kern, MOST>, s)) return e;
  const dim3 grid((unsigned)((a.K + R * Q4_TILE - 1) / (R * Q4_TILE)), (unsigned)parts);
  hipLaunchKernelGGL(kern, grid, dim3(NW * 64), (unsigned)lds, s, a);
  if (hipError_t e = hipGetLastError()) return e;
  if (parts > 1) hipLaunchKernelGGL(experts_join_kernel<T>, dim3((unsigned)(((int64_t)a.M * a.K / 4 + 255) / 256)), dim3(256), 0, s, a, parts);
  return hipGetLastError();
}

template <typename F>
static hipError_t by_token_tiles(int mt, F&& f) {
  if (mt == 2) return f(std::integral_constant<int, 2>{});
  if (mt == 3) return f(std::integral_constant<int, 3>{});
  return f(std::integral_constant<int, 4>{});
}

// Gate/up.
template <typename T, int G>
static hipError_t gateup_of(const ExpertArgs& a, hipStream_t s) {
  const int mt = token_tiles(a);
  const int tiles = (a.N + Q4_TILE - 1) / Q4_TILE * entries_at_most(a);
  const bool few = tiles <= 3 * a.cus;
  if constexpr (G == 0) {
    if (a.M <= 8) return run_gateup<T, 0, 1, 1, 1, 4, 2>(a, s);
    if (mt == 1) return run_gateup<T, 0, 1, 2, 1, 4, 2>(a, s);
    return run_gateup<T, 0, 2, 2, 2, 4, 1>(a, s);
  } else {
    // Eight wavefronts on a tile of each matrix, or four on two.  us, groups of 128, K=4096: one token, N=11008 (2.7 tiles a CU) 13.9
    // 16.1, 14336 (3.5) 16.9 16.5, 28672 (7) 29.2 27.4; 12 tokens 16.2 17.0, 20.2 17.6, 34.4 27.8; K=2048: 9.2 10.1, 10.7 10.3, 18.1 16.4;
    // 9.7 10.4, 12.0 10.6, 20.5 17.1.
    if (a.M <= 4) return few ? run_gateup<T, G, 1, 1, 1, 8, 2>(a, s) : run_gateup<T, G, 1, 1, 2, 4, 2>(a, s);
    if (mt == 1) return few ? run_gateup<T, G, 1, 4, 1, 8, 2>(a, s) : run_gateup<T, G, 1, 4, 2, 4, 1>(a, s);
    // More than one token tile.  Token rows are read again for every strip, so two tiles of each matrix, where the registers hold
    // them; but a tile for every CU first, and eight wavefronts where a CU gets one workgroup and each of them two blocks.  us,
    // groups of 128, as (tiles, wavefronts): 32 tokens, K=7168, N=2424 (1, 8) 12.8 (1, 4) 17.2 (2, 8) 17.4; K=1536, N=4096 5.7
    // 5.65 7.9; K=4096, N=7168 14.7 14.2 12.8; K=5280, N=13224 35 36 31 and (2, 4) 26.8; 64 tokens, that size, (1, 4) 53
    // (2, 8) 43 (2, 4) 36.  Two tiles in finer groups, 64 tokens, groups of 64 53.8 against 53.3, 48 tokens, groups of 32 93 against 49.
    const bool deep = a.K > 12 * Q4_BLOCK;
    return by_token_tiles(mt, [&](auto m) -> hipError_t {
      constexpr int MT = decltype(m)::value;
      constexpr bool wide = MT == 2 || (MT == 3 && G >= 64) || (MT == 4 && G == 128);
      if (tiles <= a.cus && deep) return run_gateup<T, G, MT, 4, 1, 8, 1>(a, s);
      if constexpr (wide) {
        if (tiles > a.cus && tiles <= 2 * a.cus && deep) return run_gateup<T, G, MT, 4, 2, 8, 1>(a, s);
        if (tiles > a.cus) return run_gateup<T, G, MT, 4, 2, 4, 1>(a, s);
      }
      return run_gateup<T, G, MT, 4, 1, 4, 1>(a, s);
    });
  }
}

// Down: tiles of a workgroup, and workgroups that share a strip of them.  The parts' sum is a launch more, 2 us behind others and
// more from an idle queue.  With more than one token tile it pays beyond 64 blocks (of all experts, times token tiles), even
// where the weights would not: M=48, 4 bits, 768 rows of 2048 columns 7.7 us whole, 8.4 in four parts; of 4096 10.8 and 8.7.
// Up to 16 tokens: large weights, which take as long anyway (us, 12 tokens, groups of 128, the tiles that smaller ones get, whole, and four
// split: 4096 rows of 14336 columns, 30 MB, 14.1 14.0, of 22528, 48 MB, 19.5 18.0; 8192 rows of 11008, 46 MB, 17.4 17.6, of 14336,
// 61 MB, 21.0 20.0; 16 bits whole and split, 2048 rows, 16 experts of 1024 columns, 67 MB, 18.2 14.7), and long reductions of all
// experts together in few rows, which would leave CUs idle: one token, groups of 128, 1024 rows of 64 blocks 7.1 7.1, of 160
// 11.35 8.9; 2048 rows of 96 8.8 9.0, of 160 12.0 10.9; 12 tokens, 2048 rows of 64 8.8 8.75, of 160 16.5 13.4; 1 of 32 experts of
// K=512, N=6144, 4 bits, the layer 51.8 us whole, 30.4 split.
struct DownPlan {
  int tiles, parts;
};
static DownPlan plan_down(const ExpertArgs& a, int group) {
  const bool large = weight_bytes(a, group) >= 48e6;
  const int tiles = (a.K + Q4_TILE - 1) / Q4_TILE;
  DownPlan p = {1, 1};
  const int cols = group ? 128 : 64, blocks = (a.N + cols - 1) / cols * experts_at_most(a);
  if (a.M > 16) {
    // A tile for every CU where the reduction is short (us, 48 tokens, groups of 128, one tile and two: 4096 rows of 4096 columns 10.1, 11.0,
    // 2048 of 2048 7.0, 7.6, but 4096 of 11008 20.7, 17.8), and of 64 tokens with the finest groups, where two would spill.
    const bool spill = a.M > 48 && group == 32, shallow = group && tiles <= a.cus && blocks <= 32;
    p.tiles = a.routing == ROUTING_DENSE && (spill || shallow) ? 1 : 2;
  } else if (group && a.M <= 4) p.tiles = tiles > a.cus ? 2 : 1;
  else if (group) p.tiles = large ? 4 : tiles <= a.cus ? 1 : tiles <= 2 * a.cus || blocks <= 8 ? 2 : 4;
  if (a.M > 16 ? blocks * token_tiles(a) > 64 : large || (2 * tiles <= a.cus && blocks > 128)) {
    p.parts = a.cus / ((tiles + p.tiles - 1) / p.tiles);
    p.parts = p.parts < 1 ? 1 : p.parts > DOWN_MAX_PARTS ? DOWN_MAX_PARTS : p.parts;
  }
  return p;
}
size_t experts_partial_bytes(const ExpertArgs& a, int group) {
  const int parts = plan_down(a, group).parts;
  return parts > 1 ? (size_t)parts * a.M * a.K * sizeof(float) : 0;
}
template <typename T, int G>
static hipError_t down_of(const ExpertArgs& a, hipStream_t s) {
  const DownPlan p = plan_down(a, G);
  const int parts = a.partial ? p.parts : 1;
  constexpr int FEW = G ? 4 : 8, ALL = 16 / FEW;
  const bool few = a.M << a.h_low <= FEW;
  if (a.M > 16 && a.routing == ROUTING_PLAN)
    return token_tiles(a) == 1 ? run_down<T, G, 1, ALL, 2, 8, 1, true>(a, parts, s) : run_down<T, G, 2, ALL, 2, 8, 1, true>(a, parts, s);
  if constexpr (G != 0) {
    const bool wide = G == 32 && a.K > Q4_TILE * a.cus;  // (more tiles than CUs: 8192 rows of 1024 columns 9.3 us, with eight wavefronts 12.9)
    if (a.M > 16 && p.tiles == 1 && !wide)
      return by_token_tiles(token_tiles(a), [&](auto m) { return run_down<T, G, decltype(m)::value, ALL, 1, 8, 1>(a, parts, s); });
  }
  if (a.M > 48) return run_down<T, G, 4, ALL, G == 32 ? 1 : 2, 4, 1>(a, parts, s);
  if (a.M > 32) return run_down<T, G, 3, ALL, 2, G == 32 ? 4 : 8, 1>(a, parts, s);
  if (a.M > 16) return run_down<T, G, 2, ALL, 2, 8, 1>(a, parts, s);
  if constexpr (G != 0)
    if (p.tiles == 4) return run_down<T, G, 1, ALL, 4, 8, 1>(a, parts, s);
  // One tile.  Enough wavefronts, and stages of them, for a share of the blocks that is in flight at once.
  constexpr int COLS = Block<T, G, 1, 1, 1>::COLS;
  const int blocks = (a.N + COLS - 1) / COLS * experts_at_most(a);
  // More than a tile for every CU: two each.  us, one token, groups of 128: 12312 rows of 7168 columns 13.5, one tile with stages
  // four deep 15.7 (groups of 32 17.1, 24.1), 21496 of 952 with four wavefronts 5.7, with eight 6.8, one tile 11.3 (groups of 32
  // 7.2, 7.4, 16.8).  16 tokens, groups of 128: 6144 of 6144 9.9 with two tiles, 12.1 with one, 13.5 with four; 12312 of 7168
  // 18.1 with two, 15.5 with four.
  if constexpr (G != 0)
    if (p.tiles == 2) {
      if (!few) return blocks <= 8 ? run_down<T, G, 1, ALL, 2, 4, 1>(a, parts, s) : run_down<T, G, 1, ALL, 2, 8, 1>(a, parts, s);
      return blocks <= 8 ? run_down<T, G, 1, 1, 2, 4, G == 32 ? 1 : 2>(a, parts, s) : run_down<T, G, 1, 1, 2, 8, G == 32 ? 1 : 2>(a, parts, s);
    }
  if constexpr (G != 0) {
    // us as (wavefronts, stages), one token, groups of 128, weights from memory: 2048 rows of 16 blocks (8, 2) 4.4 (8, 4) 4.6 (16, 2)
    // 5.0; 32 5.4 5.2 5.6; 44 6.3 6.45 6.6; 80 8.2 8.2 7.9; 4096 rows of 17 5.0 4.9 5.3; 32 5.55 5.4 5.7; 64 8.1 7.5 7.5; 80 9.4 8.8 8.1.
    if (few) {
      if (blocks <= 16) return run_down<T, G, 1, 1, 1, 8, 2>(a, parts, s);
      return blocks < 64 ? run_down<T, G, 1, 1, 1, 8, 4>(a, parts, s) : run_down<T, G, 1, 1, 1, 16, 2>(a, parts, s);
    }
  } else {
    if (few) return blocks < 32 ? run_down<T, 0, 1, 1, 1, 8, 1>(a, parts, s) : run_down<T, 0, 1, 1, 1, 16, 1>(a, parts, s);
  }
  // us with 8 and 16 wavefronts, 2048 rows: 12 tokens, groups of 128, 24 blocks 5.8 6.2, 32 6.6 6.4, 64 9.9 8.8; 16 bits, 2 tokens 5.2 5.35,
  // 5.9 5.5, 8.7 7.3; 12 tokens 5.4 5.6, 6.2 5.8, 9.3 8.6.
  return blocks < 32 ? run_down<T, G, 1, ALL, 1, 8, 1>(a, parts, s) : run_down<T, G, 1, ALL, 1, 16, 1>(a, parts, s);
}
bool experts_solo(int M, int E) { return M == 1 && E <= SOLO_MAX_E; }

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
// Four tokens to a wavefront, a row of 16 lanes each; lane l of a row has VPL experts from VPL l on.  What bounds routing many
// tokens is the instructions of its rounds, and a round of four tokens takes little more than one of one: 16384 tokens, 8 of
// 128 experts, bf16, 8.8 us with a token per wavefront, 7.0 with four, 6.4 with a lane's logits in one load,
// 5.5 with the number in the key.
template <int VPL, typename L>
__global__ void __launch_bounds__(256) route_rows_kernel(const L* logits, float* weights, int64_t* experts, int64_t M, int E, int top_k,
                                                         int normalize) {
  const int lane = threadIdx.x & 63, l = lane & 15;
  const int64_t token = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4), t = token < M ? token : M - 1;
  LogitRow<VPL, L> row;
  row.load(logits + t * E, ((uintptr_t)logits & (sizeof(L) * VPL - 1)) == 0, E, l);
  row.choose(E, top_k, l);
  const float first = row.first, own = row.own;
  const bool none = first == -__builtin_inff();
  const float e = l < top_k && !none ? expf(own - first) : 0.f;
  float all = e;
  if (!normalize) {
    all = 0.f;
#pragma unroll
    for (int v = 0; v < VPL; ++v)
      if (l * VPL + v < E && !none) all += expf(row.value[v] - first);
  }
  all = row_sum(all, lane);
  if (token < M && l < top_k) {
    weights[t * top_k + l] = none ? 0.f : e / all;
    experts[t * top_k + l] = row.expert;
  }
}

template <int VPL, typename L>
__global__ void __launch_bounds__(256) route_kernel(const L* logits, float* weights, int64_t* experts, int64_t M, int E, int top_k,
                                                    int normalize) {
  const int lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= M) return;
  int e;
  float w;
  choose<VPL>([&](int i) { return (float)logits[t * E + i]; }, E, top_k, normalize != 0, lane, e, w);
  if (lane < top_k) {
    weights[t * top_k + lane] = w;
    experts[t * top_k + lane] = e < 0 ? -1 - e : e;
  }
}

// The routing of at most 64 tokens, in one workgroup.  cap: tokens of an entry.
template <int VPL, typename L>
__global__ void __launch_bounds__(1024) plan_kernel(const L* logits, ExpertPlan p, int M, int E, int top_k, int normalize, int cap) {
  __shared__ uint32_t who[EXPERTS_MAX_E][2];  // tokens of an expert, a bit each
  __shared__ int index[EXPERTS_MAX_E];        // of an expert's first entry
  __shared__ short chosen[EXPERTS_MAX_M * EXPERTS_MAX_K];
  __shared__ int in_wave[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int i = tid; i < E * 2; i += 1024) (&who[0][0])[i] = 0u;
  __syncthreads();
  for (int t = wave; t < M; t += 16) {
    int e;
    float w;
    choose<VPL>([&](int i) { return (float)logits[(size_t)t * E + i]; }, E, top_k, normalize != 0, lane, e, w);
    if (lane < top_k) {
      p.weight[t * top_k + lane] = w;
      chosen[t * top_k + lane] = (short)e;
      if (e >= 0) atomicOr(&who[e][t >> 5], 1u << (t & 31));
    }
  }
  __syncthreads();
  // entries of the experts before this thread's
  const int tokens = tid < E ? __popc(who[tid][0]) + __popc(who[tid][1]) : 0;
  const int entries = (tokens + cap - 1) / cap;
  int upto = entries;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(upto, d);
    if (lane >= d) upto += o;
  }
  if (lane == 63) in_wave[wave] = upto;
  __syncthreads();
  int before = upto - entries, total = 0;
  for (int w = 0; w < 16; ++w) {
    if (w < wave) before += in_wave[w];
    total += in_wave[w];
  }
  if (tid < E) index[tid] = before;
  for (int q = 0; q < entries; ++q) {
    p.active[1 + before + q] = tid;
    p.count[before + q] = (uint8_t)(tokens - q * cap < cap ? tokens - q * cap : cap);
  }
  if (tid == 0) p.active[0] = total;
  if (M <= 16)
    for (int i = tid; i < total * (EXPERTS_MAX_M / 4); i += 1024) ((int*)p.slot)[i] = -1;
  __syncthreads();
  for (int i = tid; i < M * top_k; i += 1024) {
    const int e = chosen[i], t = i / top_k;
    if (e < 0) continue;
    const uint64_t mask = (uint64_t)who[e][1] << 32 | who[e][0];
    const int nth = __popcll(mask & ((1ull << t) - 1)), entry = index[e] + nth / cap;
    p.pairs[entry * EXPERTS_MAX_M + nth % cap] = (uint16_t)i;
    if (M <= 16) p.slot[entry * EXPERTS_MAX_M + t] = (int8_t)(i - t * top_k);
  }
}

#define GMLP_BY_EXPERTS(E, CALL)   \
  if ((E) <= 64) CALL(1);          \
  else if ((E) <= 128) CALL(2);    \
  else if ((E) <= 256) CALL(4);    \
  else CALL(8)

// Rows of a launch: it has fewer than 2^32 threads, 16 or 64 for a row.  (Past that the runtime starts fewer than asked for, and
// reports no error: 2^28 + 9 rows of two experts came back in part.)
constexpr int64_t ROUTE_ROWS = (int64_t)1 << 24;

template <typename L>
hipError_t launch_route(const L* logits, float* weights, int64_t* experts, int64_t M, int E, int top_k, int normalize, hipStream_t s) {
#define ROWS(V) \
  hipLaunchKernelGGL((route_rows_kernel<V, L>), dim3((unsigned)((m + 15) / 16)), dim3(256), 0, s, logits, weights, experts, m, E, top_k, normalize)
  for (int64_t m; M > 0; M -= m) {
    m = M < ROUTE_ROWS ? M : ROUTE_ROWS;
    if (E <= 16) ROWS(1);
    else if (E <= 64) ROWS(4);
    else if (E <= 128) ROWS(8);
    else if (E <= 256) ROWS(16);
    else
      hipLaunchKernelGGL((route_kernel<8, L>), dim3((unsigned)((m + 3) / 4)), dim3(256), 0, s, logits, weights, experts, m, E, top_k, normalize);
    if (hipError_t e = hipGetLastError()) return e;
    logits += m * E;
    weights += m * top_k;
    experts += m * top_k;
  }
#undef ROWS
  return hipSuccess;
}
template <typename L>
hipError_t launch_experts_plan(const L* logits, const ExpertArgs& a, hipStream_t s) {
#define CALL(V) \
  hipLaunchKernelGGL((plan_kernel<V, L>), dim3(1), dim3(1024), 0, s, logits, a.plan, a.M, a.E, a.top_k, a.normalize, 16 * token_tiles(a))
  GMLP_BY_EXPERTS(a.E, CALL);
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
  template hipError_t launch_experts_plan<T>(const T*, const ExpertArgs&, hipStream_t);
GMLP_INSTANTIATE(f16)
GMLP_INSTANTIATE(bf16)
template hipError_t launch_route<float>(const float*, float*, int64_t*, int64_t, int, int, int, hipStream_t);
template hipError_t launch_experts_plan<float>(const float*, const ExpertArgs&, hipStream_t);

}  // namespace gmlp
