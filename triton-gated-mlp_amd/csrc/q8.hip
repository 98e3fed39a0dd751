// 8-bit integers: rows to integers, products for a few token rows, and the plan of routed choices (see q8.hpp).
#include "q8.hpp"

#include "launch.hpp"
#include "lds_dma.hpp"

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
// n = 127 v / top rounded half to even: a product of 127 v with fl(1 / top), one step of correction, and the addition of 1.5 2^23, whose
// result has n in its low bits.  127 v and top have few bits: a quotient that is no half is 1 / (2 top) from one at least, 2^-12 in
// units of n, far more than the two roundings; one that is a half is a number of fp32, and the corrected quotient is it (what
// the first product is off by is exact in the fused multiply-add).  8 instructions a number in the place of the division's 15.
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

// A workgroup of NT threads: ROWS rows of a tile.  A thread takes 16 numbers of a row at a time (32 bytes in, 16 out), PER times, and
// keeps them while the row's largest is found; PER = 0: rows of any length, read twice.  Neighbouring threads take the ROWS
// rows first, which lie together in the result.
template <typename T, int NT, int ROWS, int PER>
__global__ void __launch_bounds__(NT) q8_rows_kernel(const T* x, int8_t* codes, float* scales, int64_t rows, int cols, int padded,
                                                     int tiles, const int* token_of, const int* rows_at) {
  constexpr int LANES = NT / ROWS, NW = NT / 64, PARTS = 16 / ROWS;  // threads of a row
  __shared__ uint32_t part[NW][ROWS];
  const int r = threadIdx.x % ROWS, l = threadIdx.x / ROWS;
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
  const T* const src = x + (matrix * rows + from) * cols;
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
  if (l == 0 && at < rows) scales[matrix * rows + at] = there ? scale.scale : 0.f;
  int8_t* const dst = codes + ((matrix * tiles + tile) * (int64_t)padded) * 16 + (at % 16) * 16;
  auto write = [&](const u32x4 (&v)[2], int c) __attribute__((always_inline)) {
    if (c < padded) *(i32x4*)(dst + (int64_t)(c / 16) * 256) = q8_sixteen<T>(scale, v);
  };
  if constexpr (PER > 0) {
#pragma unroll
    for (int i = 0; i < PER; ++i) write(kept[i], (l + i * LANES) * 16);
  } else {
    for (int c = l * 16; c < padded; c += LANES * 16) {
      read(kept[0], c);
      write(kept[0], c);
    }
  }
}

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
struct Q8Few {
  Q8Product p;
  int strips;  // workgroups side by side, R tiles of weight rows each
};
template <int SETS, int R, int MT>
struct Q8Stage {
  i32x4 w[SETS][R], x[MT];
};
constexpr int q8_units_at_a_time(int NW, int units, int sets) { return NW * units * sets <= 32 ? units : 32 / (NW * sets); }

template <typename T, int SETS, int R, int MT, int NW, int D, bool F32>
__global__ void __launch_bounds__(NW * 64) q8_few_kernel(Q8Few a) {
  const Q8Product& p = a.p;
  constexpr int UNITS = R * MT, EACH = q8_units_at_a_time(NW, UNITS, SETS);
  __shared__ i32x4 part[NW * EACH * SETS * 64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int entry = (int)blockIdx.x / a.strips, first_tile = ((int)blockIdx.x - entry * a.strips) * R;
  int expert = 0, row = 0, count = p.M;
  if (p.tiles != nullptr) {
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
  const q8_rsrc rx = q8_make_rsrc(p.x + (int64_t)(row / 16) * pitch, (uint32_t)((count + 15) / 16) * pitch);
  const int s0 = steps * wave / NW, run = steps * (wave + 1) / NW - s0;
  const uint32_t lane_off = (uint32_t)lane * 16u;
  Q8Stage<SETS, R, MT> st[D];
  auto load = [&](Q8Stage<SETS, R, MT>& t, int i) __attribute__((always_inline)) {
    const uint32_t at = (uint32_t)(s0 + i) * 1024u;
#pragma unroll
    for (int m = 0; m < MT; ++m) t.x[m] = q8_load16<0>(rx, lane_off, i < run ? at + (uint32_t)m * pitch : Q8_PAST);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int b = 0; b < SETS; ++b) t.w[b][r] = q8_load16<Q8_STREAM>(rw[b], lane_off, i < run ? at + (uint32_t)r * pitch : Q8_PAST);
  };
  i32x4 acc[UNITS][SETS] = {};
  auto multiply = [&](const Q8Stage<SETS, R, MT>& t) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int b = 0; b < SETS; ++b)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[r * MT + m][b] = Traits<I8Pair>::mfma16(t.w[b][r], t.x[m], acc[r * MT + m][b]);
  };
#pragma unroll
  for (int d = 0; d < D; ++d) load(st[d], d);
  for (int i = 0; i < run; i += D)
#pragma unroll
    for (int d = 0; d < D; ++d) {
      multiply(st[d]);  // (zeros past the end)
      load(st[d], i + d + D);
    }
  const int r16 = lane & 15, kg = lane >> 4;
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
      const float sx = p.sx[row + j];
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
      const size_t to = (size_t)(row + j) * p.N + n;
      if constexpr (F32) *(f32x4*)((float*)p.out + to) = f32x4{o[0], o[1], o[2], o[3]};
      else store_w<T, 4>((T*)p.out + to, o);
    }
  }
}

template <typename T, int SETS, int R, int MT, int NW, int D>
hipError_t run_q8_few(const Q8Product& p, hipStream_t s) {
  Q8Few a = {p, 0};
  a.strips = ((p.N + 15) / 16 + R - 1) / R;
  const dim3 grid((unsigned)(a.strips * (p.tiles != nullptr ? p.most_tiles : 1))), block(NW * 64);
  if constexpr (SETS == 1)
    if (p.out_f32) {
      hipLaunchKernelGGL((q8_few_kernel<T, SETS, R, MT, NW, D, true>), grid, block, 0, s, a);
      return hipGetLastError();
    }
  hipLaunchKernelGGL((q8_few_kernel<T, SETS, R, MT, NW, D, false>), grid, block, 0, s, a);
  return hipGetLastError();
}
template <typename T>
hipError_t launch_q8_few(const Q8Product& p, int sets, int token_tiles, hipStream_t s) {
  if (sets == 2) {
    if (token_tiles == 1) return run_q8_few<T, 2, 1, 1, 8, 4>(p, s);
    if (token_tiles == 2) return run_q8_few<T, 2, 1, 2, 8, 4>(p, s);
    return run_q8_few<T, 2, 1, 4, 8, 4>(p, s);
  }
  if (token_tiles == 1) return run_q8_few<T, 1, 1, 1, 8, 4>(p, s);
  if (token_tiles == 2) return run_q8_few<T, 1, 1, 2, 8, 4>(p, s);
  return run_q8_few<T, 1, 1, 4, 8, 4>(p, s);
}

// ------------------------------------------------------------------ routed choices
// One workgroup: choices of each expert are counted, experts laid out one behind the other from multiples of 16 rows on, and
// every choice takes the next row of its expert.  (Which of an expert's rows it gets is up to the order of arrival; a row's
// results do not depend on its place.)
__global__ void __launch_bounds__(1024) q8_plan_kernel(const int64_t* experts, const float* weights, Q8Plan plan, int pairs, int E, int top_k,
                                                       int cap, int most_rows) {
  __shared__ int count[1024], next[1024], in_wave[2][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  count[tid] = 0;
  for (int i = tid; i < most_rows; i += 1024) plan.token_of[i] = -1;
  __syncthreads();
  for (int i = tid; i < pairs; i += 1024)
    if (weights[i] != 0.f) atomicAdd(&count[(int)experts[i]], 1);
  __syncthreads();
  // rows and tiles of the experts before this thread's
  const int mine = tid < E ? count[tid] : 0;
  const int rows = (mine + 15) / 16 * 16, tiles = (mine + cap - 1) / cap;
  int upto[2] = {rows, tiles};
#pragma unroll
  for (int d = 1; d < 64; d <<= 1)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int o = __shfl_up(upto[k], d);
      if (lane >= d) upto[k] += o;
    }
  if (lane == 63) in_wave[0][wave] = upto[0], in_wave[1][wave] = upto[1];
  __syncthreads();
  int before[2] = {upto[0] - rows, upto[1] - tiles}, total[2] = {0, 0};
  for (int w = 0; w < 16; ++w)
    for (int k = 0; k < 2; ++k) {
      if (w < wave) before[k] += in_wave[k][w];
      total[k] += in_wave[k][w];
    }
  next[tid] = before[0];
  for (int q = 0; q < tiles; ++q)
    plan.tiles[before[1] + q] = Q8Tile{tid, before[0] + q * cap, mine - q * cap < cap ? mine - q * cap : cap, 0};
  if (tid == 0) plan.total[0] = total[1], plan.total[1] = total[0];
  __syncthreads();
  for (int i = tid; i < pairs; i += 1024) {
    int row = -1;
    if (weights[i] != 0.f) {
      row = atomicAdd(&next[(int)experts[i]], 1);
      plan.token_of[row] = i / top_k;
    }
    plan.row_of[i] = row;
  }
}
hipError_t launch_q8_plan(const int64_t* experts, const float* weights, const Q8Plan& plan, int M, int E, int top_k, int cap, hipStream_t s) {
  hipLaunchKernelGGL(q8_plan_kernel, dim3(1), dim3(1024), 0, s, experts, weights, plan, M * top_k, E, top_k, cap,
                     (int)q8_plan_rows((int64_t)M * top_k, E));
  return hipGetLastError();
}

template <typename T>
__global__ void __launch_bounds__(256) q8_combine_kernel(const float* parts, const float* weights, const int* row_of, T* y, int64_t M,
                                                         int K, int top_k) {
  const int64_t unit = (int64_t)blockIdx.x * 256 + threadIdx.x, t = unit / (K / 8);
  if (t >= M) return;
  const int c = (int)(unit % (K / 8)) * 8;
  float v[8] = {};
  for (int j = 0; j < top_k; ++j) {
    const int row = row_of[t * top_k + j];
    if (row < 0) continue;
    const float w = weights[t * top_k + j];
    float part[8];
    load_w<float, 4>(parts + (int64_t)row * K + c, part);
    load_w<float, 4>(parts + (int64_t)row * K + c + 4, part + 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += w * part[i];
  }
  store_w<T, 8>(y + t * K + c, v);
}
template <typename T>
hipError_t launch_q8_combine(const float* parts, const float* weights, const int* row_of, T* y, int64_t M, int64_t K, int top_k,
                             hipStream_t s) {
  hipLaunchKernelGGL(q8_combine_kernel<T>, dim3((unsigned)((M * (K / 8) + 255) / 256)), dim3(256), 0, s, parts, weights, row_of, y, M, (int)K,
                     top_k);
  return hipGetLastError();
}

#define GMLP_INSTANTIATE(T)                                                                                                      \
  template hipError_t launch_q8_few<T>(const Q8Product&, int, int, hipStream_t);                                                 \
  template hipError_t launch_q8_rows<T>(const T*, int8_t*, float*, int64_t, int64_t, int64_t, const int*, const int*, hipStream_t); \
  template hipError_t launch_q8_dequantize<T>(const int8_t*, const float*, T*, int64_t, int64_t, int64_t, hipStream_t);           \
  template hipError_t launch_q8_combine<T>(const float*, const float*, const int*, T*, int64_t, int64_t, int, hipStream_t);
GMLP_INSTANTIATE(f16)
GMLP_INSTANTIATE(bf16)
#undef GMLP_INSTANTIATE

}  // namespace gmlp
