// 8-bit integers: rows to integers, products for a few token rows, and the plan of routed choices (see q8.hpp).
#include "q8.hpp"

#include "launch.hpp"
#include "lds_dma.hpp"
#include "routing.hpp"

namespace gmlp {

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef __amdgpu_buffer_rsrc_t q8_rsrc;
__device__ __forceinline__ q8_rsrc q8_make_rsrc(const void* p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, (int)bytes, 0x00020000);
}
template <int POLICY>
__device__ __forceinline__ i32x4 q8_load16(q8_rsrc r, uint32_t lane_off, uint32_t off) {
  return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)lane_off, (int)off, POLICY));
}
constexpr int Q8_STREAM = 2;                 // cache policy: non-temporal, what is read once
constexpr uint32_t Q8_PAST = 0x7fff0000u;    // beyond any descriptor of these kernels: reads as zero and moves no data

// ------------------------------------------------------------------ rows to integers
// The largest magnitude of a row, as the bits of the 16-bit type without the sign: integers of the same order, in which
// infinity is above every number and NaN above infinity, so that neither is lost.
__device__ __forceinline__ uint32_t max_bits(uint32_t most, uint32_t two) {
  const u16x2 a = __builtin_bit_cast(u16x2, most), b = __builtin_bit_cast(u16x2, two & 0x7fff7fffu);
  return __builtin_bit_cast(uint32_t, (u16x2)__builtin_elementwise_max(a, b));
}
// n = 127 v / top rounded half to even: a product u of 127 v with fl(1 / top), one step of correction, and the addition of 1.5 2^23, whose
// result has n in its low bits.  With top = b and v = a 2^-k in units of top's last place, a and b of p bits (11 of fp16, 8 of bf16) and k
// the gap of the exponents, the quotient q = 127 a / (b 2^k) is below 2^(8-k) and, if it is no half, at least 1 / (2 b 2^k) > 2^-(12+k)
// from one: both shrink with the gap.  The first product is within 2^-23 q, so that its remainder, of 13 bits, is exact in the fused
// multiply-add; the correction is within 2^-47 q of what is missing, and the result off by its own rounding, 2^-24 q < 2^-(16+k): on the side
// of the half where q is.  A q that is a half is a number of fp32, which no rounding of what is within 2^-47 q of it misses.  From
// k = 9 on n is 0.  8 instructions a number in the place of the division's 15.
template <typename T>
struct RowScale {
  float top, pre, by, scale;
  bool finite;
  __device__ __forceinline__ explicit RowScale(uint32_t bits) {
    const float raw = Traits<T>::to_f32(__builtin_bit_cast(T, (unsigned short)bits));
    finite = raw < __builtin_inff();
    // powers of two, exact, that keep 127 v finite and its quotient out of the subnormals
    pre = raw > 0x1p64f ? 0x1p-64f : raw < 0x1p-64f ? 0x1p64f : 1.f;
    top = finite && raw > 0.f ? raw * pre : 1.f;
    by = 1.f / top;
    scale = finite ? raw / 127.f : __builtin_nanf("");
    if (!finite) pre = 0.f;
  }
  // the low byte is n
  __device__ __forceinline__ uint32_t of(float v) const {
    const float u = 127.f * (v * pre), first = u * by;
    const float n = __builtin_fmaf(__builtin_fmaf(-first, top, u), by, first);
    return __float_as_uint(n + 12582912.f);
  }
  // four of them
  __device__ __forceinline__ uint32_t four(const T* v) const {
    const uint32_t a = __builtin_amdgcn_perm(of(Traits<T>::to_f32(v[1])), of(Traits<T>::to_f32(v[0])), 0x0c0c0400u);
    const uint32_t b = __builtin_amdgcn_perm(of(Traits<T>::to_f32(v[3])), of(Traits<T>::to_f32(v[2])), 0x04000c0cu);
    return finite ? a | b : 0u;
  }
};
template <typename T>
__device__ __forceinline__ i32x4 q8_sixteen(const RowScale<T>& scale, const u32x4 (&v)[2]) {
  i32x4 out;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const u32x2 four = {v[i / 2][i % 2 * 2], v[i / 2][i % 2 * 2 + 1]};
    typedef typename Traits<T>::vec4 vec4;
    const vec4 x = __builtin_bit_cast(vec4, four);
    const T y[4] = {x[0], x[1], x[2], x[3]};
    out[i] = (int)scale.four(y);
  }
  return out;
}

// ROWS rows by NT threads.  A thread takes 16 numbers of a row at a time (32 bytes in, 16 out), PER times, and keeps them while the row's
// largest is found; PER = 0: rows of any length, read twice.  Neighbouring threads take the ROWS rows first.  src: this thread's row, of
// zeros if it is not `there`; put(c, integers of columns c..).  Returns the row's scale.
template <typename T, int NT, int ROWS, int PER, typename Put>
__device__ __forceinline__ float q8_some_rows(const T* src, bool there, int cols, int padded, Put&& put) {
  constexpr int LANES = NT / ROWS, NW = NT / 64;  // threads of a row
  __shared__ uint32_t part[NW][ROWS];
  const int r = threadIdx.x % ROWS, l = threadIdx.x / ROWS;
  auto read = [&](u32x4 (&v)[2], int c) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) v[h] = there && c + 8 * h < cols ? *(const u32x4*)(src + c + 8 * h) : u32x4{0, 0, 0, 0};
  };
  uint32_t most = 0;
  auto look = [&](const u32x4 (&v)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max_bits(most, v[i / 4][i % 4]);
  };
  u32x4 kept[PER > 0 ? PER : 1][2];
  if constexpr (PER > 0) {
#pragma unroll
    for (int i = 0; i < PER; ++i) read(kept[i], (l + i * LANES) * 16);
#pragma unroll
    for (int i = 0; i < PER; ++i) look(kept[i]);
  } else {
    for (int c = l * 16; c < cols; c += LANES * 16) {
      read(kept[0], c);
      look(kept[0]);
    }
  }
  most = max(most & 0xffffu, most >> 16);
#pragma unroll
  for (int d = ROWS; d < 64; d <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, d));
  if ((threadIdx.x & 63) < ROWS) part[threadIdx.x >> 6][r] = most;
  __syncthreads();
  most = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) most = max(most, part[w][r]);
  const RowScale<T> scale(most);
  if constexpr (PER > 0) {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if ((l + i * LANES) * 16 < padded) put((l + i * LANES) * 16, q8_sixteen<T>(scale, kept[i]));
  } else {
    for (int c = l * 16; c < padded; c += LANES * 16) {
      read(kept[0], c);
      put(c, q8_sixteen<T>(scale, kept[0]));
    }
  }
  return scale.scale;
}

// A workgroup: ROWS rows of a tile, which lie together in the result.
template <typename T, int NT, int ROWS, int PER>
__global__ void __launch_bounds__(NT) q8_rows_kernel(const T* x, int8_t* codes, float* scales, int64_t rows, int cols, int padded,
                                                     int tiles, const int* token_of, const int* rows_at) {
  constexpr int PARTS = 16 / ROWS;
  const int r = threadIdx.x % ROWS;
  // The workgroups of a tile are 8 apart: on the same die, whose cache joins what they write to a line.
  const int64_t b = blockIdx.x, whole = (int64_t)tiles / 8 * 8 * PARTS;
  const int64_t tile = b < whole ? b / (8 * PARTS) * 8 + b % 8 : b / PARTS, sub = b < whole ? b / 8 % PARTS : b % PARTS;
  const int64_t at = tile * 16 + sub * ROWS + r, matrix = blockIdx.y;
  int64_t from = at;
  bool there = at < rows;
  if (rows_at != nullptr && tile * 16 >= rows_at[0]) return;
  if (token_of != nullptr) {
    from = token_of[at];
    there = from >= 0;
  }
  int8_t* const dst = codes + ((matrix * tiles + tile) * (int64_t)padded) * 16 + (at % 16) * 16;
  const float scale = q8_some_rows<T, NT, ROWS, PER>(x + (matrix * rows + from) * cols, there, cols, padded,
                                                     [&](int c, i32x4 n) { *(i32x4*)(dst + (int64_t)(c / 16) * 256) = n; });
  if ((int)threadIdx.x < ROWS && at < rows) scales[matrix * rows + at] = there ? scale : 0.f;
}

// Four rows of `lines` by a workgroup of 1024, the `block`-th.
template <typename T>
__device__ __forceinline__ void q8_four_lines(const Q8Lines& a, int block) {
  const int64_t at = (int64_t)block * 4 + threadIdx.x % 4;
  const bool there = at < a.rows;
  const T* const src = (const T*)a.x + at * a.cols;
  int8_t* const dst = a.codes + at * a.padded;
  auto put = [&](int c, i32x4 n) __attribute__((always_inline)) {
    if (there) *(i32x4*)(dst + c) = n;
  };
  const float scale = a.padded <= 4096    ? q8_some_rows<T, 1024, 4, 1>(src, there, a.cols, a.padded, put)
                      : a.padded <= 16384 ? q8_some_rows<T, 1024, 4, 4>(src, there, a.cols, a.padded, put)
                                          : q8_some_rows<T, 1024, 4, 0>(src, there, a.cols, a.padded, put);
  if (threadIdx.x < 4 && there) a.scales[at] = scale;
}
__device__ __forceinline__ void q8_lines_of(const Q8Lines& a, int block) {
  if (a.dtype == 0) q8_four_lines<f16>(a, block);
  else q8_four_lines<bf16>(a, block);
}
unsigned q8_lines_workgroups(const Q8Lines* lines) { return lines != nullptr ? (unsigned)((lines->rows + 3) / 4) : 0u; }

template <typename T>
hipError_t launch_q8_rows(const T* x, int8_t* codes, float* scales, int64_t count, int64_t rows, int64_t cols, const int* token_of,
                          const int* rows_at, hipStream_t s) {
  const int64_t tiles = (rows + 15) / 16;
  const int padded = (int)q8_padded(cols);
#define CALL(NT, R, PER)                                                                                                  \
  hipLaunchKernelGGL((q8_rows_kernel<T, NT, R, PER>), dim3((unsigned)(tiles * (16 / R)), (unsigned)count), dim3(NT), 0, s, x, codes, scales, \
                     rows, (int)cols, padded, (int)tiles, token_of, rows_at)
  if (padded > 32768) CALL(1024, 4, 0);
  else if (tiles * count >= 64) {
    if (padded <= 4096) CALL(256, 4, 4);
    else if (padded <= 16384) CALL(1024, 4, 4);
    else CALL(1024, 4, 8);
  } else {
    if (padded <= 4096) CALL(256, 1, 1);
    else CALL(1024, 1, 2);
  }
#undef CALL
  return hipGetLastError();
}

template <typename T>
__global__ void __launch_bounds__(256) q8_dequantize_kernel(const int8_t* codes, const float* scales, T* w, int64_t rows, int cols,
                                                            int padded, int64_t tiles) {
  const int64_t unit = (int64_t)blockIdx.x * 256 + threadIdx.x, matrix = blockIdx.y;
  const int64_t row = unit / (padded / 8);
  const int c = (int)(unit % (padded / 8)) * 8;
  if (row >= rows || c >= cols) return;
  const u32x2 n = *(const u32x2*)(codes + (matrix * tiles + row / 16) * 16 * padded + (c / 16) * 256 + (row % 16) * 16 + c % 16);
  const float scale = scales[matrix * rows + row];
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = scale * (float)(int8_t)(n[i / 4] >> (8 * (i % 4)) & 0xffu);
  store_w<T, 8>(w + (matrix * rows + row) * cols + c, v);
}
template <typename T>
hipError_t launch_q8_dequantize(const int8_t* codes, const float* scales, T* w, int64_t count, int64_t rows, int64_t cols, hipStream_t s) {
  const int padded = (int)q8_padded(cols);
  const int64_t units = rows * (padded / 8);
  hipLaunchKernelGGL(q8_dequantize_kernel<T>, dim3((unsigned)((units + 255) / 256), (unsigned)count), dim3(256), 0, s, codes, scales, w,
                     rows, (int)cols, padded, (rows + 15) / 16);
  return hipGetLastError();
}

// ------------------------------------------------------------------ products for a few token rows
// A workgroup: R tiles of 16 weight rows (of each matrix) and the token rows of a tile, up to 16 * MT.  Its wavefronts split the
// reduction and add up through LDS (integers: in any order).  Bound by the weights' way from memory: a load is one KiB as it
// lies, D of each kind in flight for a wavefront; tokens come from the caches, and past the end a load moves nothing.
// Q: the token rows, 16 at most, come as they are and every workgroup makes integers of them for itself, in LDS, while its first
// weights are on their way: a launch less, and for one row no more time (one row of 4096 through two matrices of 14336 rows 20.3 us,
// of integers 20.9).
constexpr int Q8_OWN_ROWS = 16;
struct Q8Few {
  Q8Product p;
  const void* rows;  // Q: [rows][cols], those of a plan's tile in its order or (token_of) as tokens
  const int* token_of;
  int cols;
  int strips;        // workgroups side by side, R tiles of weight rows each
  Q8Solo solo;       // Q and solo.logits: the only token of an expert layer
};

// `count` rows [cols] as integers in LDS, [count][padded], by NT threads, 16 numbers of a row at a time; a thread's first AHEAD
// pieces are loaded by read_ahead, for the caller to have other loads behind them.  from (nullable): which of `rows` they are.
template <typename T, int NT, int AHEAD>
struct Q8RowsToLds {
  u32x4 ahead[AHEAD][2];
  __device__ __forceinline__ void read(u32x4 (&v)[2], const T* rows, int cols, int padded, int count, int i, const int* from) {
    const int pieces = padded / 16, row = i / pieces, c = (i - row * pieces) * 16;
    const int64_t at = from != nullptr && row < count ? from[row] : row;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      v[h] = row < count && c + 8 * h < cols ? *(const u32x4*)(rows + at * cols + c + 8 * h) : u32x4{0, 0, 0, 0};
  }
  __device__ __forceinline__ void read_ahead(const T* rows, int cols, int padded, int count, const int* from) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) read(ahead[i], rows, cols, padded, count, threadIdx.x + i * NT, from);
  }
  // most[count], zeros on entry and behind a barrier: the rows' largest magnitudes (max_bits); `to` is there behind the next barrier
  __device__ __forceinline__ void finish(const T* rows, int cols, int padded, int count, const int* from, uint32_t* most, char* to) {
    const int pieces = padded / 16, all = pieces * count;
    auto look = [&](const u32x4 (&v)[2], int i) __attribute__((always_inline)) {
      uint32_t m = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) m = max_bits(m, v[k / 4][k % 4]);
      m = max(m & 0xffffu, m >> 16);
      const int row = i < all ? i / pieces : 0;
      if (i >= all) m = 0;
      // (most wavefronts have one row)
      const int one = __builtin_amdgcn_readfirstlane(row);
      if (__all(row == one)) {
        m = wave_max(m);
        if ((threadIdx.x & 63) == 0) atomicMax(&most[one], m);
      } else {
        atomicMax(&most[row], m);
      }
    };
    u32x4 v[2];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if ((int)((threadIdx.x & ~63u) + i * NT) < all) look(ahead[i], threadIdx.x + i * NT);
    for (int i = threadIdx.x + AHEAD * NT; (int)((unsigned)i & ~63u) < all; i += NT) {
      read(v, rows, cols, padded, count, i, from);
      look(v, i);
    }
    __syncthreads();
    auto write = [&](const u32x4 (&v)[2], int i) __attribute__((always_inline)) {
      if (i < all) *(i32x4*)(to + (size_t)i * 16) = q8_sixteen<T>(RowScale<T>(most[i / pieces]), v);
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) write(ahead[i], threadIdx.x + i * NT);
    for (int i = threadIdx.x + AHEAD * NT; i < all; i += NT) {
      read(v, rows, cols, padded, count, i, from);
      write(v, i);
    }
  }
};

// The choices of a call's only token, every wavefront for itself: lane j < top_k has the j-th, expert < 0 where it is not run.
__device__ __forceinline__ void q8_choose_solo(const Q8Solo& solo, int lane, int& expert, float& weight) {
  auto logit = [&](int i) -> float {
    if (solo.logits_dtype == 0) return (float)((const f16*)solo.logits)[i];
    if (solo.logits_dtype == 1) return (float)((const bf16*)solo.logits)[i];
    return ((const float*)solo.logits)[i];
  };
  if (solo.E <= 64) choose<1>(logit, solo.E, solo.top_k, solo.normalize != 0, lane, expert, weight);
  else choose<Q8_SOLO_MAX_E / 64>(logit, solo.E, solo.top_k, solo.normalize != 0, lane, expert, weight);
  if (weight == 0.f && expert >= 0) expert = -1 - expert;
}

template <int SETS, int R, int MT, bool Q>
struct Q8Stage {
  i32x4 w[SETS][R], x[Q ? 1 : MT];
};
constexpr int q8_units_at_a_time(int NW, int units, int sets) { return NW * units * sets <= 32 ? units : 32 / (NW * sets); }

template <typename T, int SETS, int R, int MT, int NW, int D, bool F32, bool Q>
__global__ void __launch_bounds__(NW * 64) q8_few_kernel(Q8Few a) {
  const Q8Product& p = a.p;
  constexpr int UNITS = R * MT, EACH = q8_units_at_a_time(NW, UNITS, SETS);
  __shared__ i32x4 part[NW * EACH * SETS * 64];
  extern __shared__ __align__(16) char own_rows[];  // Q: [count][K]
  __shared__ uint32_t own_most[Q8_OWN_ROWS];
  static_assert(!Q || MT == 1, "a few rows are one tile");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int entry = (int)blockIdx.x / a.strips, first_tile = ((int)blockIdx.x - entry * a.strips) * R;
  int expert = 0, row = 0, count = p.M;
  if (Q && a.solo.logits != nullptr) {
    int e;
    float w;
    q8_choose_solo(a.solo, lane, e, w);
    if (blockIdx.x == 0 && wave == 0 && lane < a.solo.top_k) {
      a.solo.experts[lane] = e;
      a.solo.weights[lane] = w;
    }
    expert = __builtin_amdgcn_readlane(e, entry);
    if (expert < 0) return;
  } else if (p.tiles != nullptr) {
    if (entry >= p.total[0]) return;
    const Q8Tile t = p.tiles[entry];
    expert = __builtin_amdgcn_readfirstlane(t.expert);
    row = __builtin_amdgcn_readfirstlane(t.row);
    count = __builtin_amdgcn_readfirstlane(t.rows);
  }
  const int steps = p.K / 64, all_tiles = (p.N + 15) / 16;
  const uint32_t pitch = (uint32_t)p.K * 16u;  // bytes of a tile of rows
  const int own = all_tiles - first_tile < R ? all_tiles - first_tile : R;
  q8_rsrc rw[SETS];
#pragma unroll
  for (int b = 0; b < SETS; ++b)
    rw[b] = q8_make_rsrc(p.w[b] + ((int64_t)expert * all_tiles + first_tile) * pitch, (uint32_t)own * pitch);
  // GATHER: token rows that lie one behind the other are found by their numbers.  (Products of the columns beyond those that are there
  // repeat the first one, and are not used.)
  constexpr bool GATHER = SETS == 2 && !Q && MT <= 2;
  const bool gathered = GATHER && a.token_of != nullptr;
  const q8_rsrc rx = gathered ? q8_make_rsrc(p.x, (uint32_t)p.tokens * (uint32_t)p.K)
                              : q8_make_rsrc(p.x + (int64_t)(row / 16) * pitch, (uint32_t)((count + 15) / 16) * pitch);
  const int s0 = steps * wave / NW, run = steps * (wave + 1) / NW - s0;
  const uint32_t lane_off = (uint32_t)lane * 16u;
  uint32_t x_off[GATHER ? MT : 1];
  const uint32_t x_step = gathered ? 64u : 1024u;
  if constexpr (GATHER) {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int j = 16 * m + (lane & 15);
      x_off[m] = gathered ? (uint32_t)a.token_of[row + (j < count ? j : 0)] * (uint32_t)p.K + (uint32_t)(lane >> 4) * 16u
                          : lane_off + (uint32_t)m * pitch;
    }
  }
  Q8Stage<SETS, R, MT, Q> st[D];
  auto load = [&](Q8Stage<SETS, R, MT, Q>& t, int i) __attribute__((always_inline)) {
    const uint32_t at = (uint32_t)(s0 + i) * 1024u;
    if constexpr (GATHER)
#pragma unroll
      for (int m = 0; m < MT; ++m) t.x[m] = q8_load16<0>(rx, x_off[m], i < run ? (uint32_t)(s0 + i) * x_step : Q8_PAST);
    else if constexpr (!Q)
#pragma unroll
      for (int m = 0; m < MT; ++m) t.x[m] = q8_load16<0>(rx, lane_off, i < run ? at + (uint32_t)m * pitch : Q8_PAST);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int b = 0; b < SETS; ++b) t.w[b][r] = q8_load16<Q8_STREAM>(rw[b], lane_off, i < run ? at + (uint32_t)r * pitch : Q8_PAST);
  };
  i32x4 acc[UNITS][SETS] = {};
  const int r16 = lane & 15, kg = lane >> 4;
  // (Q: columns of the product beyond the rows there are repeat the first one, and are not used; past the end, where the weights
  // are zeros, the last integers are read again)
  const char* const integers = own_rows + (r16 < count ? r16 : 0) * p.K + kg * 16;
  auto multiply = [&](const Q8Stage<SETS, R, MT, Q>& t, int i) __attribute__((always_inline)) {
    i32x4 x[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
      if constexpr (Q) x[m] = *(const i32x4*)(integers + (i < run ? s0 + i : 0) * 64);
      else x[m] = t.x[m];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int b = 0; b < SETS; ++b)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[r * MT + m][b] = Traits<I8Pair>::mfma16(t.w[b][r], x[m], acc[r * MT + m][b]);
  };
  Q8RowsToLds<T, NW * 64, 2> rows;
  const T* const own_from = (const T*)a.rows + (a.token_of == nullptr ? (int64_t)row * a.cols : 0);
  const int* const own_tokens = a.token_of != nullptr ? a.token_of + row : nullptr;
  if constexpr (Q) {
    rows.read_ahead(own_from, a.cols, p.K, count, own_tokens);
    if (threadIdx.x < Q8_OWN_ROWS) own_most[threadIdx.x] = 0;
  }
#pragma unroll
  for (int d = 0; d < D; ++d) load(st[d], d);
  if constexpr (Q) {
    __syncthreads();
    rows.finish(own_from, a.cols, p.K, count, own_tokens, own_most, own_rows);
    __syncthreads();
  }
  for (int i = 0; i < run; i += D)
#pragma unroll
    for (int d = 0; d < D; ++d) {
      multiply(st[d], i + d);  // (zeros past the end)
      load(st[d], i + d + D);
    }
#pragma unroll
  for (int first = 0; first < UNITS; first += EACH) {
    if (first > 0) __syncthreads();
#pragma unroll
    for (int i = 0; i < EACH; ++i)
#pragma unroll
      for (int b = 0; b < SETS; ++b)
        if (first + i < UNITS) part[((wave * EACH + i) * SETS + b) * 64 + lane] = acc[first + i][b];
    __syncthreads();
    for (int i = wave; i < EACH && first + i < UNITS; i += NW) {
      i32x4 sum[SETS] = {};
#pragma unroll
      for (int w = 0; w < NW; ++w)
#pragma unroll
        for (int b = 0; b < SETS; ++b) sum[b] += part[((w * EACH + i) * SETS + b) * 64 + lane];
      // lane: four output columns of one token row
      const int r = (first + i) / MT, j = 16 * ((first + i) % MT) + r16, n = (first_tile + r) * 16 + 4 * kg;
      if (j >= count || n >= p.N) continue;
      const float sx = Q ? RowScale<T>(own_most[Q ? j : 0]).scale : p.sx[gathered ? a.token_of[row + j] : row + j];
      float v[SETS][4], o[4];
#pragma unroll
      for (int b = 0; b < SETS; ++b) {
        const f32x4 sw = *(const f32x4*)(p.sw[b] + (int64_t)expert * p.N + n);
#pragma unroll
        for (int q = 0; q < 4; ++q) v[b][q] = (float)sum[b][q] * (sx * sw[q]);
        if (!F32 && p.bias[b] != nullptr) add_w<T, 4>((const T*)p.bias[b] + n, v[b]);
      }
      if constexpr (SETS == 2) {
        act_fwd_w<4>(p.act, v[0], o);
#pragma unroll
        for (int q = 0; q < 4; ++q) o[q] *= v[1][q];
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) o[q] = v[0][q];
      }
      const size_t to = (size_t)((Q && a.solo.logits != nullptr ? entry : row) + j) * p.N + n;
      if constexpr (F32) *(f32x4*)((float*)p.out + to) = f32x4{o[0], o[1], o[2], o[3]};
      else store_w<T, 4>((T*)p.out + to, o);
    }
  }
}

template <typename T, int SETS, int R, int MT, int NW, int D, bool F32, bool Q>
hipError_t run_q8_few(const Q8Product& p, const void* rows, int cols, const Q8Solo* solo, hipStream_t s) {
  Q8Few a = {p, rows, p.token_of, cols, ((p.N + 15) / 16 + R - 1) / R, solo != nullptr ? *solo : Q8Solo{}};
  const dim3 grid((unsigned)(a.strips * (solo != nullptr ? solo->top_k : p.tiles != nullptr ? p.most_tiles : 1))), block(NW * 64);
  constexpr auto kern = q8_few_kernel<T, SETS, R, MT, NW, D, F32, Q>;
  const size_t lds = Q ? (size_t)p.most_rows * p.K : 0;
  hipLaunchKernelGGL(kern, grid, block, lds, s, a);
  return hipGetLastError();
}
// What the sizes choose.  us, weights from memory, as (tiles of weight rows a workgroup, wavefronts, stages).
// One token tile: two tiles of a single matrix where they are two for every CU and more, otherwise one.  Wavefronts: eight
// for reductions from 8192 on, or from 2048 on where workgroups are few; otherwise four, with stages two deep below 2048 and four
// deep beyond.  2048 x 2048, one row (1, 8, 4) 3.2, (1, 4, 4) 3.6, (2, 8, 4) 4.3; 16384 x 1024 (2, 4, 2) 5.1, (1, 4, 4) 5.8, (1, 8, 4) 7.3;
// 131072 x 1024, 16 rows (2, 4, 2) 24.9, (1, 8, 4) 45; 8192 x 28672, 16 rows (2, 8, 4) 37.2, (1, 8, 4) 41.1; gate and up of 14336 x 4096
// (1, 4, 4) 20.3, (1, 8, 4) 21.2; of 28672 x 8192, 16 rows (1, 8, 4) 72.0, (1, 4, 4) 74.5, (2, 4, 2) 90; of 65536 x 2048 (1, 4, 4) 43.6,
// (1, 8, 4) 47.3.
// More token tiles: every workgroup reads all of them from the caches, which is what bounds it unless it has several tiles of
// weights for them: four of a single matrix (two for two token tiles) where there are three for every CU, two from two for every CU
// on, two of gate and up.  128 rows, 14336 x 4096 (4, 4, 2) 21.5, (2, 4, 2) 25.0, (1, 4, 2) 40; gate and up of it (2, 4, 1) 34.7,
// (2, 4, 2) 38.7, (1, 4, 2) 48.7; 5632 x 2048 (2, 4, 2) 13.0, (2, 4, 1) 14.0, (1, 4, 1) 14.7; 4096 x 14336 (1, 4, 2) 32.7, (2, 4, 2) 38.1.
// 64 rows, 14336 x 4096 (4, 4, 2) 15.9, (1, 4, 1) 26.3; 4096 x 14336 (1, 4, 2) 21.9, (2, 8, 1) 25.9; 32 rows, 14336 x 4096 (2, 4, 2) 13.2,
// (1, 8, 2) 18.0; 4096 x 14336 (1, 8, 2) 15.3, (1, 4, 2) 18.7.
template <typename T, int SETS, int R, int MT, bool F32, bool Q>
hipError_t q8_few_depth(const Q8Product& p, const void* rows, int cols, const Q8Solo* solo, int entries, hipStream_t s) {
  const int steps = p.K / 64;
  const int64_t wgs = (int64_t)((p.N + 16 * R - 1) / (16 * R)) * entries;
  if constexpr (MT == 1) {
    if (steps >= 128 || (steps >= 32 && wgs <= 2 * p.cus)) return run_q8_few<T, SETS, R, MT, 8, 4, F32, Q>(p, rows, cols, solo, s);
    if constexpr (SETS == 2 || R == 2)  // (a single matrix has more workgroups than that of two tiles only)
      if (steps >= 32) return run_q8_few<T, SETS, R, MT, 4, 4, F32, Q>(p, rows, cols, solo, s);
  } else if constexpr (MT == 2 && R == 1) {
    if (steps >= 128) return run_q8_few<T, SETS, R, MT, 8, 2, F32, Q>(p, rows, cols, solo, s);
  } else if constexpr (MT == 8 && SETS == 2 && R == 2) {
    if (wgs > p.cus) return run_q8_few<T, SETS, R, MT, 4, 1, F32, Q>(p, rows, cols, solo, s);
  }
  return run_q8_few<T, SETS, R, MT, 4, 2, F32, Q>(p, rows, cols, solo, s);
}
template <typename T, int SETS, int MT, bool F32, bool Q>
hipError_t q8_few_tiles(const Q8Product& p, const void* rows, int cols, const Q8Solo* solo, hipStream_t s) {
  const int entries = solo != nullptr ? solo->top_k : p.tiles != nullptr ? p.most_tiles : 1;
  const int64_t tiles = (int64_t)((p.N + 15) / 16) * entries;
  if constexpr (SETS == 1 && MT >= 4)
    if (tiles >= 3 * p.cus) return q8_few_depth<T, SETS, 4, MT, F32, Q>(p, rows, cols, solo, entries, s);
  if constexpr (SETS == 1 || MT > 1)
    if (tiles >= (SETS == 2 ? 1 : 2) * p.cus) return q8_few_depth<T, SETS, 2, MT, F32, Q>(p, rows, cols, solo, entries, s);
  return q8_few_depth<T, SETS, 1, MT, F32, Q>(p, rows, cols, solo, entries, s);
}
template <typename T>
hipError_t launch_q8_few(const Q8Product& p, int sets, int token_tiles, hipStream_t s) {
#define CALL(SETS, F32)                                                                    \
  if (token_tiles == 1) return q8_few_tiles<T, SETS, 1, F32, false>(p, nullptr, 0, nullptr, s); \
  if (token_tiles == 2) return q8_few_tiles<T, SETS, 2, F32, false>(p, nullptr, 0, nullptr, s); \
  if (token_tiles == 4) return q8_few_tiles<T, SETS, 4, F32, false>(p, nullptr, 0, nullptr, s); \
  if constexpr (!F32) return q8_few_tiles<T, SETS, 8, F32, false>(p, nullptr, 0, nullptr, s); \
  else return hipErrorInvalidValue  // (an expert's down projection: up to 64 rows)
  if (sets == 2) { CALL(2, false); }
  if (p.out_f32) { CALL(1, true); }
  CALL(1, false);
#undef CALL
}
// Where every workgroup makes the integers itself.  A launch of their own takes 3 us; in every workgroup they take what it has rows
// for: us, in the workgroups and in a launch, 4096 x 4096 of 4096, 6 rows 7.8, 8.5, 8 rows 8.7, 8.5; 14336 rows of 4096 columns 4 rows 12.6,
// 15.0, 8 rows 15.4, 15.0; of 2048 columns 12 rows 11.6, 11.7, 16 rows 13.1, 11.8; 2048 of 2048, 16 rows 7.1, 8.6.
bool q8_own_rows(int64_t most_rows, int64_t padded, int64_t N, int cus) {
  if (most_rows == 1) return padded <= 32768;
  return most_rows <= Q8_OWN_ROWS && most_rows * padded <= (N <= 16 * cus ? 32768 : 24576);
}
template <typename T>
hipError_t launch_q8_few_rows(const Q8Product& p, const T* rows, int cols, int sets, const Q8Solo* solo, hipStream_t s) {
  if (sets == 2) return q8_few_tiles<T, 2, 1, false, true>(p, rows, cols, solo, s);
  if (p.out_f32) return q8_few_tiles<T, 1, 1, true, true>(p, rows, cols, solo, s);
  return q8_few_tiles<T, 1, 1, false, true>(p, rows, cols, solo, s);
}

// ------------------------------------------------------------------ the only token of an expert layer
// y = sum over the choices of weight * down_e(h): a workgroup has 16 output columns of all choices, whose hidden states it makes
// integers of for itself.  Its wavefronts are shared out over the choices; sums of a choice are added up as integers, then scaled
// and weighted, so nothing but the sum over the choices is in floats (in a fixed order).
struct Q8SoloDown {
  Q8Solo solo;
  const void* h;     // [top_k][cols]
  const int8_t* w;
  const float* sw;
  void* y;           // [N]
  int N, K, cols;
};
template <typename T, int NW, int D>
__global__ void __launch_bounds__(NW * 64) q8_solo_down_kernel(Q8SoloDown a) {
  __shared__ i32x4 part[NW * 64];
  __shared__ uint32_t most[16];
  extern __shared__ __align__(16) char integers[];  // [top_k][K]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), top_k = a.solo.top_k;
  const int r16 = lane & 15, kg = lane >> 4, tile = (int)blockIdx.x;
  Q8RowsToLds<T, NW * 64, 4> rows;
  rows.read_ahead((const T*)a.h, a.cols, a.K, top_k, nullptr);  // (rows of choices that are not run are whatever memory holds)
  if (threadIdx.x < 16) most[threadIdx.x] = 0;
  const int each = NW / top_k, choice = wave / each, me = wave - choice * each;  // NW >= top_k
  int expert = choice < top_k ? a.solo.experts[choice] : -1;
  expert = __builtin_amdgcn_readfirstlane(expert);
  const int steps = a.K / 64, all_tiles = (a.N + 15) / 16;
  const uint32_t pitch = (uint32_t)a.K * 16u;
  const int s0 = steps * me / each, run = expert >= 0 ? steps * (me + 1) / each - s0 : 0;
  const q8_rsrc rw = q8_make_rsrc(a.w + ((int64_t)(expert >= 0 ? expert : 0) * all_tiles + tile) * pitch, pitch);
  i32x4 st[D];
  auto load = [&](i32x4& t, int i) __attribute__((always_inline)) {
    t = q8_load16<Q8_STREAM>(rw, (uint32_t)lane * 16u, i < run ? (uint32_t)(s0 + i) * 1024u : Q8_PAST);
  };
#pragma unroll
  for (int d = 0; d < D; ++d) load(st[d], d);
  __syncthreads();
  rows.finish((const T*)a.h, a.cols, a.K, top_k, nullptr, most, integers);
  __syncthreads();
  i32x4 acc = {0, 0, 0, 0};
  const char* const mine = integers + (choice < top_k ? choice : 0) * a.K + kg * 16;
  for (int i = 0; i < run; i += D)
#pragma unroll
    for (int d = 0; d < D; ++d) {
      acc = Traits<I8Pair>::mfma16(st[d], *(const i32x4*)(mine + (i + d < run ? s0 + i + d : 0) * 64), acc);
      load(st[d], i + d + D);
    }
  part[threadIdx.x] = acc;
  __syncthreads();
  if (wave > 0) return;
  // lane (r16, kg): choice r16, columns 4 kg .. + 3 (every column of a product is the same row)
  const int n = tile * 16 + 4 * kg;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (r16 < top_k && n < a.N) {
    const int e = a.solo.experts[r16];
    if (e >= 0) {
      i32x4 sum = {0, 0, 0, 0};
      for (int w = 0; w < each; ++w) sum += part[(r16 * each + w) * 64 + lane];
      const f32x4 sw = *(const f32x4*)(a.sw + (int64_t)e * a.N + n);
      const float weight = a.solo.weights[r16], sx = RowScale<T>(most[r16]).scale;
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = weight * ((float)sum[q] * (sx * sw[q]));
    }
  }
#pragma unroll
  for (int d = 1; d < 16; d <<= 1)
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] += __shfl_xor(v[q], d);
  if (r16 == 0 && n < a.N) store_w<T, 4>((T*)a.y + n, v);
}
bool q8_solo(int64_t M, int64_t E, int64_t top_k, int64_t padded_k, int64_t padded_n) {
  return M == 1 && E <= Q8_SOLO_MAX_E && padded_k <= 32768 && top_k * padded_n <= 40960;
}
template <typename T>
hipError_t launch_q8_solo_down(const Q8Solo& solo, const T* h, const int8_t* w, const float* sw, T* y, int N, int cols, hipStream_t s) {
  const int padded = (int)q8_padded(cols);
  const Q8SoloDown a = {solo, h, w, sw, y, N, padded, cols};
  const dim3 grid((unsigned)((N + 15) / 16));
  const size_t lds = (size_t)solo.top_k * padded;
  if (solo.top_k <= 8) hipLaunchKernelGGL((q8_solo_down_kernel<T, 8, 4>), grid, dim3(512), lds, s, a);
  else hipLaunchKernelGGL((q8_solo_down_kernel<T, 16, 4>), grid, dim3(1024), lds, s, a);
  return hipGetLastError();
}

// ------------------------------------------------------------------ routed choices
// One workgroup: choices of each expert are counted, which gives each its place among its expert's, and experts laid out one behind
// the other from multiples of 16 rows on.  (Which place is up to the order of arrival; a row's results do not depend on it.)  Bound
// by the loads' latency, of which a thread has eight choices in flight, and by the additions in LDS: 16384 choices of 64 experts
// 26 us with a choice at a time and a second addition for its place.
struct Q8Choices {
  int* count;  // [1024], zeros; then where an expert's rows begin
  int (*in_wave)[16];
};
__device__ __forceinline__ void q8_lay_out(const Q8Choices& sh, const Q8Plan& plan, int E, int cap) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // rows and tiles (of each kind) of the experts before this thread's
  const int mine = tid < E ? sh.count[tid] : 0;
  const int per[3] = {(mine + 15) / 16 * 16, (mine + cap - 1) / cap, (mine + 255) / 256};
  int upto[3] = {per[0], per[1], per[2]};
#pragma unroll
  for (int d = 1; d < 64; d <<= 1)
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const int o = __shfl_up(upto[k], d);
      if (lane >= d) upto[k] += o;
    }
  if (lane == 63)
#pragma unroll
    for (int k = 0; k < 3; ++k) sh.in_wave[k][wave] = upto[k];
  __syncthreads();
  int before[3], total[3] = {0, 0, 0};
#pragma unroll
  for (int k = 0; k < 3; ++k) before[k] = upto[k] - per[k];
  for (int w = 0; w < 16; ++w)
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      if (w < wave) before[k] += sh.in_wave[k][w];
      total[k] += sh.in_wave[k][w];
    }
  sh.count[tid] = before[0];
  for (int q = 0; q < per[1]; ++q)
    plan.tiles[before[1] + q] = Q8Tile{tid, before[0] + q * cap, mine - q * cap < cap ? mine - q * cap : cap, 0};
  if (plan.large != nullptr)
    for (int q = 0; q < per[2]; ++q)
      plan.large[before[2] + q] = Q8Tile{tid, before[0] + q * 256, mine - q * 256 < 256 ? mine - q * 256 : 256, 0};
  if (tid == 0) plan.total[0] = total[1], plan.total[1] = total[0], plan.total[2] = total[2];
  __syncthreads();
}
__global__ void __launch_bounds__(1024) q8_plan_kernel(const int64_t* experts, const float* weights, Q8Plan plan, int pairs, int E, int top_k,
                                                       int cap, int most_rows, Q8Lines lines) {
  if (blockIdx.x > 0) return q8_lines_of(lines, (int)blockIdx.x - 1);
  __shared__ int count[1024], in_wave[3][16];
  constexpr int PER = 8;
  const int tid = threadIdx.x;
  const Q8Choices sh = {count, in_wave};
  count[tid] = 0;
  for (int i = tid; i < most_rows; i += 1024) plan.token_of[i] = -1;
  __syncthreads();
  int expert[PER], place[PER];
  // (a second pass over more choices than a thread keeps finds their places in row_of)
  auto pass = [&](int first, bool again) __attribute__((always_inline)) {
    float w[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int i = first + k * 1024 + tid;
      expert[k] = i < pairs ? (int)experts[i] : 0;
      if (again) place[k] = i < pairs ? plan.row_of[i] : -1;
      else w[k] = i < pairs ? weights[i] : 0.f;
    }
    if (!again)
#pragma unroll
      for (int k = 0; k < PER; ++k) place[k] = w[k] != 0.f ? atomicAdd(&count[expert[k]], 1) : -1;
  };
  for (int first = 0; first < pairs; first += PER * 1024) {
    pass(first, false);
    if (pairs > PER * 1024)
#pragma unroll
      for (int k = 0; k < PER; ++k)
        if (first + k * 1024 + tid < pairs) plan.row_of[first + k * 1024 + tid] = place[k];
  }
  __syncthreads();
  q8_lay_out(sh, plan, E, cap);
  for (int first = 0; first < pairs; first += PER * 1024) {
    if (pairs > PER * 1024) pass(first, true);
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int i = first + k * 1024 + tid;
      if (i >= pairs) continue;
      const int row = place[k] >= 0 ? count[expert[k]] + place[k] : -1;
      plan.row_of[i] = row;
      if (row >= 0) plan.token_of[row] = i / top_k;
    }
  }
}
// (rows that no choice has are marked for launch_q8_rows only)
static int q8_rows_to_mark(const Q8Lines* lines, int M, int E, int top_k) { return lines != nullptr ? 0 : (int)q8_plan_rows((int64_t)M * top_k, E); }
hipError_t launch_q8_plan(const int64_t* experts, const float* weights, const Q8Plan& plan, int M, int E, int top_k, int cap,
                          const Q8Lines* lines, hipStream_t s) {
  hipLaunchKernelGGL(q8_plan_kernel, dim3(1 + q8_lines_workgroups(lines)), dim3(1024), 0, s, experts, weights, plan, M * top_k, E, top_k, cap,
                     q8_rows_to_mark(lines, M, E, top_k), lines != nullptr ? *lines : Q8Lines{});
  return hipGetLastError();
}

// Routing and plan of a few tokens in one launch: 64 tokens at a time, four to a wavefront as in routing many.
template <int VPL, typename L>
__global__ void __launch_bounds__(1024) q8_route_plan_kernel(const L* logits, float* weights, Q8Plan plan, int M, int E, int top_k, int normalize,
                                                             int cap, int most_rows, Q8Lines lines) {
  if (blockIdx.x > 0) return q8_lines_of(lines, (int)blockIdx.x - 1);
  __shared__ int count[1024], in_wave[3][16];
  __shared__ short chosen[Q8_ROUTE_ROWS * 16];
  const int tid = threadIdx.x, lane = tid & 63, l = tid & 15;
  const Q8Choices sh = {count, in_wave};
  const bool aligned = ((uintptr_t)logits & (sizeof(L) * VPL - 1)) == 0;
  count[tid] = 0;
  for (int i = tid; i < most_rows; i += 1024) plan.token_of[i] = -1;
  __syncthreads();
  for (int base = 0; base < M; base += 64) {
    const int token = base + (tid >> 4), t = token < M ? token : M - 1;
    LogitRow<VPL, L> row;
    row.load(logits + (int64_t)t * E, aligned, E, l);
    row.choose(E, top_k, l);
    const bool none = row.first == -__builtin_inff();
    const float e = l < top_k && !none ? expf(row.own - row.first) : 0.f;
    float all = e;
    if (!normalize) {
      all = 0.f;
#pragma unroll
      for (int v = 0; v < VPL; ++v)
        if (l * VPL + v < E && !none) all += expf(row.value[v] - row.first);
    }
    all = row_sum(all, lane);
    if (token < M && l < top_k) {
      const float w = none ? 0.f : e / all;
      const bool run = w != 0.f && row.own != -__builtin_inff();
      weights[t * top_k + l] = w;
      chosen[t * top_k + l] = (short)(run ? row.expert : -1);
      if (run) atomicAdd(&count[row.expert], 1);
    }
  }
  __syncthreads();
  q8_lay_out(sh, plan, E, cap);
  for (int i = tid; i < M * top_k; i += 1024) {
    const int row = chosen[i] >= 0 ? atomicAdd(&count[chosen[i]], 1) : -1;
    plan.row_of[i] = row;
    if (row >= 0) plan.token_of[row] = i / top_k;
  }
}
template <typename L>
hipError_t launch_q8_route_plan(const L* logits, float* weights, const Q8Plan& plan, int M, int E, int top_k, int normalize, int cap,
                                const Q8Lines* lines, hipStream_t s) {
#define CALL(V)                                                                                                          \
  hipLaunchKernelGGL((q8_route_plan_kernel<V, L>), dim3(1 + q8_lines_workgroups(lines)), dim3(1024), 0, s, logits, weights, plan, M, E, top_k, \
                     normalize, cap, q8_rows_to_mark(lines, M, E, top_k), lines != nullptr ? *lines : Q8Lines{})
  if (E <= 16) CALL(1);
  else if (E <= 64) CALL(4);
  else if (E <= 128) CALL(8);
  else if (E <= 256) CALL(16);
  else CALL(32);
#undef CALL
  return hipGetLastError();
}

// Four columns a thread; four choices' parts are in flight together.
template <typename T>
__global__ void __launch_bounds__(256) q8_combine_kernel(const float* parts, const float* weights, const int* row_of, T* y, int64_t M,
                                                         int K, int top_k) {
  const int64_t unit = (int64_t)blockIdx.x * 256 + threadIdx.x, t = unit / (K / 4);
  if (t >= M) return;
  const int c = (int)(unit % (K / 4)) * 4;
  float v[4] = {};
  for (int first = 0; first < top_k; first += 4) {
    f32x4 part[4];
    float w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = first + j < top_k ? row_of[t * top_k + first + j] : -1;
      w[j] = row >= 0 ? weights[t * top_k + first + j] : 0.f;
      part[j] = row >= 0 ? __builtin_nontemporal_load((const f32x4*)(parts + (int64_t)row * K + c)) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += w[j] * part[j][i];
  }
  store_w<T, 4>(y + t * K + c, v);
}
template <typename T>
hipError_t launch_q8_combine(const float* parts, const float* weights, const int* row_of, T* y, int64_t M, int64_t K, int top_k,
                             hipStream_t s) {
  hipLaunchKernelGGL(q8_combine_kernel<T>, dim3((unsigned)((M * (K / 4) + 255) / 256)), dim3(256), 0, s, parts, weights, row_of, y, M, (int)K,
                     top_k);
  return hipGetLastError();
}

#define GMLP_INSTANTIATE(T)                                                                                                      \
  template hipError_t launch_q8_few<T>(const Q8Product&, int, int, hipStream_t);                                                 \
  template hipError_t launch_q8_few_rows<T>(const Q8Product&, const T*, int, int, const Q8Solo*, hipStream_t);                   \
  template hipError_t launch_q8_solo_down<T>(const Q8Solo&, const T*, const int8_t*, const float*, T*, int, int, hipStream_t);   \
  template hipError_t launch_q8_rows<T>(const T*, int8_t*, float*, int64_t, int64_t, int64_t, const int*, const int*, hipStream_t); \
  template hipError_t launch_q8_dequantize<T>(const int8_t*, const float*, T*, int64_t, int64_t, int64_t, hipStream_t);           \
  template hipError_t launch_q8_combine<T>(const float*, const float*, const int*, T*, int64_t, int64_t, int, hipStream_t);
GMLP_INSTANTIATE(f16)
GMLP_INSTANTIATE(bf16)
#undef GMLP_INSTANTIATE
template hipError_t launch_q8_route_plan<f16>(const f16*, float*, const Q8Plan&, int, int, int, int, int, const Q8Lines*, hipStream_t);
template hipError_t launch_q8_route_plan<bf16>(const bf16*, float*, const Q8Plan&, int, int, int, int, int, const Q8Lines*, hipStream_t);
template hipError_t launch_q8_route_plan<float>(const float*, float*, const Q8Plan&, int, int, int, int, int, const Q8Lines*, hipStream_t);

}  // namespace gmlp
