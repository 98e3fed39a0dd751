// The pipelined GEMM (gemm_pipelined.hpp) on 8-bit integers, dense and over the experts of a plan: compiled with
// -DGMLP_DT=<0|1> (output type) -DGMLP_KIND=<0|1> (gate/up or one product).  Bound by the matrix cores, whose 8-bit
// instructions take 16-bit operands' bytes and time for twice the products.
//
// A workgroup hands gemm_pipelined_body one output tile as a problem of its own: its pointers then say which expert it
// belongs to, 32-bit offsets reach into the tile only (operands of any size), and a tile of the expert's last rows
// has only those.
#include "gemm_pipelined.hpp"
#include "launch.hpp"
#include "q8.hpp"

namespace gmlp {

#if GMLP_DT == 0
typedef f16 DT;
#else
typedef bf16 DT;
#endif

__device__ __forceinline__ float q8_sum(float bits) { return (float)__builtin_bit_cast(int, bits); }
template <typename T>
__device__ __forceinline__ u32x2 q8_pack(const T (&v)[4]) {
  typename Traits<T>::vec4 o = {v[0], v[1], v[2], v[3]};
  return __builtin_bit_cast(u32x2, o);
}

// What the epilogues below share: nothing worth fetching ahead.
struct EpiQ8Base {
  static constexpr int PREFETCH_DEPTH = 0;
  static constexpr bool SPLIT = false;
  template <int W>
  struct Prefetch {};
  template <int W, typename A>
  static __device__ __forceinline__ void prefetch(const A&, int, int, Prefetch<W>&) {}
  static constexpr int PLANES = 1;
  template <typename A>
  static __device__ __forceinline__ int planes_on(const A&) { return 1; }
};

template <typename T>
struct EpiQ8Store : EpiQ8Base {
  struct Args {
    T* out;
    const float *sx, *sw;
    const T* bias;  // nullable
    int ldc, M;
  };
  static constexpr bool HAS_ACT = false, PACKED = true, STREAM_OUT = true;
  static constexpr int NBIAS = 2;
  static __device__ __forceinline__ T* plane(const Args& a, int) { return a.out; }
  static __device__ __forceinline__ void bias4(const Args& a, int n, float (&b)[NBIAS][4]) {
    load_w<float, 4>(a.sw + n, b[0]);
#pragma unroll
    for (int r = 0; r < 4; ++r) b[1][r] = 0.f;
    if (a.bias) load_w<T, 4>(a.bias + n, b[1]);
  }
  static __device__ __forceinline__ void pack4(const Args& a, int m, int, const float (&b)[NBIAS][4], const float* v, const float*,
                                               u32x2 (&o)[1]) {
    const float sx = a.sx[min(m, a.M - 1)];
    T y[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) y[r] = Traits<T>::from_f32(q8_sum(v[r]) * (sx * b[0][r]) + b[1][r]);
    o[0] = q8_pack(y);
  }
  template <int W, int ACT>
  static __device__ __forceinline__ void apply(const Args& a, int m, int n, float* v, float*, const Prefetch<W>&) {
    const float sx = a.sx[m];
    float sw[W];
    load_w<float, W>(a.sw + n, sw);
#pragma unroll
    for (int r = 0; r < W; ++r) v[r] = q8_sum(v[r]) * (sx * sw[r]);
    if (a.bias) add_w<T, W>(a.bias + n, v);
    store_w<T, W, true>(a.out + (size_t)m * a.ldc + n, v);
  }
  static __device__ __forceinline__ void to_tile(Args& a, int64_t row, int col, int rows, int64_t expert, int N) {
    a.out += row * a.ldc + col;
    a.sx += row;
    a.sw += expert * N + col;
    if (a.bias) a.bias += col;
    a.M = rows;
  }
};

// An expert's products, which are added up over a token's experts in fp32.
struct EpiQ8Float : EpiQ8Base {
  struct Args {
    float* out;
    const float *sx, *sw;
    int ldc;
  };
  static constexpr bool HAS_ACT = false, PACKED = false;
  template <int W, int ACT>
  static __device__ __forceinline__ void apply(const Args& a, int m, int n, float* v, float*, const Prefetch<W>&) {
    const float sx = a.sx[m];
    float sw[W];
    load_w<float, W>(a.sw + n, sw);
#pragma unroll
    for (int q = 0; q < W / 4; ++q) {
      f32x4 o;
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r] = q8_sum(v[4 * q + r]) * (sx * sw[4 * q + r]);
      __builtin_nontemporal_store(o, (f32x4*)(a.out + (size_t)m * a.ldc + n + 4 * q));
    }
  }
  static __device__ __forceinline__ void to_tile(Args& a, int64_t row, int col, int, int64_t expert, int N) {
    a.out += row * a.ldc + col;
    a.sx += row;
    a.sw += expert * N + col;
  }
};

template <typename T>
struct EpiQ8GateUp : EpiQ8Base {
  struct Args {
    T* h;
    const float *sx, *s_gate, *s_up;
    const T *b_gate, *b_up;  // nullable
    int ldc, M, act;
  };
  static constexpr bool HAS_ACT = true, PACKED = false;
  template <int W, int ACT>
  static __device__ __forceinline__ void apply(const Args& a, int m, int n, float* g, float* u, const Prefetch<W>&) {
    const float sx = a.sx[m];
    float sg[W], su[W], h[W];
    load_w<float, W>(a.s_gate + n, sg);
    load_w<float, W>(a.s_up + n, su);
#pragma unroll
    for (int r = 0; r < W; ++r) {
      g[r] = q8_sum(g[r]) * (sx * sg[r]);
      u[r] = q8_sum(u[r]) * (sx * su[r]);
    }
    if (a.b_gate) add_w<T, W>(a.b_gate + n, g);
    if (a.b_up) add_w<T, W>(a.b_up + n, u);
    act_fwd_w<W, ACT>(a.act, g, h);
#pragma unroll
    for (int r = 0; r < W; ++r) h[r] *= u[r];
    store_w<T, W>(a.h + (size_t)m * a.ldc + n, h);
  }
  static __device__ __forceinline__ void to_tile(Args& a, int64_t row, int col, int rows, int64_t expert, int N) {
    a.h += row * a.ldc + col;
    a.sx += row;
    a.s_gate += expert * N + col;
    a.s_up += expert * N + col;
    if (a.b_gate) a.b_gate += col;
    if (a.b_up) a.b_up += col;
    a.M = rows;
  }
};
// SiLU in the accumulator layout, as EpiGateUpPacked.
template <typename T>
struct EpiQ8GateUpPacked : EpiQ8GateUp<T> {
  typedef typename EpiQ8GateUp<T>::Args Args;
  static constexpr bool PACKED = true, STREAM_OUT = false;
  static constexpr int NBIAS = 4;
  static __device__ __forceinline__ T* plane(const Args& a, int) { return a.h; }
  static __device__ __forceinline__ void bias4(const Args& a, int n, float (&b)[NBIAS][4]) {
    load_w<float, 4>(a.s_gate + n, b[0]);
    load_w<float, 4>(a.s_up + n, b[1]);
#pragma unroll
    for (int r = 0; r < 4; ++r) b[2][r] = b[3][r] = 0.f;
    if (a.b_gate) load_w<T, 4>(a.b_gate + n, b[2]);
    if (a.b_up) load_w<T, 4>(a.b_up + n, b[3]);
  }
  static __device__ __forceinline__ void pack4(const Args& a, int m, int, const float (&b)[NBIAS][4], const float* gacc,
                                               const float* uacc, u32x2 (&o)[1]) {
    const float sx = a.sx[min(m, a.M - 1)];
    float g[4], u[4], h[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      g[r] = q8_sum(gacc[r]) * (sx * b[0][r]) + b[2][r];
      u[r] = q8_sum(uacc[r]) * (sx * b[1][r]) + b[3][r];
    }
    act_fwd_w<4, ACT_SILU>(ACT_SILU, g, h);
    T y[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) y[r] = Traits<T>::from_f32(h[r] * u[r]);
    o[0] = q8_pack(y);
  }
};

// A split reduction's sums, as integers in the floats' place.
struct EpiQ8Partial : EpiPartial<I8Pair> {
  static __device__ __forceinline__ void to_tile(Args& a, int64_t row, int col, int, int64_t, int) { a.ws += row * a.ldc + col; }
};

template <int BM, int BN, int WGN, int NB, typename Epi>
__global__ void __launch_bounds__(2 * WGN * 64) gemm_q8_kernel_pipelined(Q8Product p, typename Epi::Args ea) {
  const int tiles_n = (p.cols + BN - 1) / BN;
  const int tiles_m = p.tiles != nullptr ? p.total[0] : (p.M + BM - 1) / BM;
  const int each = tiles_m * tiles_n, all = each * (Epi::SPLIT ? p.splits : 1);
  if ((int)blockIdx.x >= all) return;
  const int u = xcd_contiguous((int)blockIdx.x, all, p.nxcd), split = Epi::SPLIT ? u / each : 0;
  int tm, tn;
  tile_of_grouped(u - split * each, tiles_m, tiles_n, p.group_m, tm, tn);
  tm = __builtin_amdgcn_readfirstlane(tm);
  tn = __builtin_amdgcn_readfirstlane(tn);
  int64_t expert = 0, row = (int64_t)tm * BM;
  int rows = min(BM, p.M - tm * BM);
  if (p.tiles != nullptr) {
    const Q8Tile t = p.tiles[tm];
    expert = __builtin_amdgcn_readfirstlane(t.expert);
    row = __builtin_amdgcn_readfirstlane(t.row);
    rows = __builtin_amdgcn_readfirstlane(t.rows);
  }
  const int col = p.first_col + tn * BN;
  const int64_t from = (expert * ((p.N + 15) / 16 * 16) + col) * p.K;
  GemmArgs ga = {};
  ga.A[0] = ga.A[1] = p.x + row * p.K;
  ga.B[0] = p.w[0] + from;
  ga.B[1] = NB == 2 ? p.w[1] + from : ga.B[0];
  ga.M = rows;
  ga.N = min(BN, p.first_col + p.cols - col);
  ga.K = ga.lda = ga.ldb = p.K / 2;
  ga.nseg = 1;
  ga.group_m = 1;
  ga.splits = p.splits;
  ga.rotate = p.rotate ? 1 + tn : 0;
  Epi::to_tile(ea, row, col, rows, expert, p.N);
  gemm_pipelined_body<I8Pair, BM, BN, 16, 2, WGN, false, false, NB, Epi>(ga, ea, split, Epi::SPLIT ? p.splits : 1);
}

template <int BM, int BN, int WGN, int NB, typename Epi>
hipError_t launch_q8_class(const Q8Product& p, const typename Epi::Args& ea, hipStream_t s) {
  typedef PipeConfig<I8Pair, BM, BN, 16, 2, WGN, false, false, NB, true> Cfg;
  constexpr auto kern = gemm_q8_kernel_pipelined<BM, BN, WGN, NB, Epi>;
  if (hipError_t e = allow_dynamic_lds(lds_kernel_of<kern, Cfg::LDS_BYTES>, s)) return e;
  const int tiles_m = p.tiles != nullptr ? p.most_tiles : (p.M + BM - 1) / BM, tiles_n = (p.cols + BN - 1) / BN;
  hipLaunchKernelGGL(kern, dim3((unsigned)(tiles_m * tiles_n * (Epi::SPLIT ? p.splits : 1))), dim3(Cfg::NW * 64), Cfg::LDS_BYTES, s, p, ea);
  return hipGetLastError();
}

// Adds up a split reduction's integers and runs the epilogue.
template <int SETS, typename Epi>
__global__ void __launch_bounds__(256) q8_reduce_kernel(const float* ws, int splits, size_t set, typename Epi::Args ea, int N) {
  for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < set / 8; i += (size_t)gridDim.x * blockDim.x) {
    i32x4 sum[SETS][2] = {};
    for (int k = 0; k < splits; ++k)
#pragma unroll
      for (int b = 0; b < SETS; ++b) {
        const i32x4* const from = (const i32x4*)(ws + ((size_t)k * SETS + b) * set + i * 8);
        sum[b][0] += from[0];
        sum[b][1] += from[1];
      }
    alignas(16) float v[2][8] = {};
#pragma unroll
    for (int b = 0; b < SETS; ++b)
#pragma unroll
      for (int r = 0; r < 8; ++r) v[b][r] = __int_as_float(sum[b][r / 4][r % 4]);
    const int m = (int)(i * 8 / (size_t)N), n = (int)(i * 8 % (size_t)N);
    Epi::template apply<8, ACT_RUNTIME>(ea, m, n, v[0], v[1], typename Epi::template Prefetch<8>{});
  }
}
template <int SETS, typename Epi>
hipError_t launch_q8_split(const Q8Product& p, const typename Epi::Args& ea, hipStream_t s) {
  const size_t set = (size_t)p.M * p.N;
  EpiQ8Partial::Args pa = {p.partial, SETS * set, SETS == 2 ? set : 0, p.N};
  hipError_t e = p.tile_class == TILE_WIDE ? launch_q8_class<128, 256 / SETS, 2, SETS, EpiQ8Partial>(p, pa, s)
                                           : launch_q8_class<128, 128 / SETS, 2, SETS, EpiQ8Partial>(p, pa, s);
  if (e) return e;
  const size_t blocks = (set / 8 + 255) / 256;
  hipLaunchKernelGGL((q8_reduce_kernel<SETS, Epi>), dim3((unsigned)(blocks < 2048 ? blocks : 2048)), dim3(256), 0, s, p.partial, p.splits,
                     set, ea, p.N);
  return hipGetLastError();
}

#if GMLP_KIND == 0
template <typename T>
hipError_t launch_q8_gateup(const Q8Product& p, hipStream_t s);
template <>
hipError_t launch_q8_gateup<DT>(const Q8Product& p, hipStream_t s) {
  EpiQ8GateUp<DT>::Args ea = {(DT*)p.out, p.sx, p.sw[0], p.sw[1], (const DT*)p.bias[0], (const DT*)p.bias[1], p.N, p.M, p.act};
  if (p.splits > 1) return launch_q8_split<2, EpiQ8GateUp<DT>>(p, ea, s);
#define CLASSES(EPI)                                                                             \
  if (p.tile_class == TILE_LARGE) return launch_q8_class<256, 128, 2, 2, EPI>(p, ea, s);         \
  if (p.tile_class == TILE_WIDE) return launch_q8_class<128, 128, 4, 2, EPI>(p, ea, s);          \
  return launch_q8_class<128, 64, 2, 2, EPI>(p, ea, s)
  if (p.act == ACT_SILU) { CLASSES(EpiQ8GateUpPacked<DT>); }
  CLASSES(EpiQ8GateUp<DT>);
#undef CLASSES
}
#else
template <typename T>
hipError_t launch_q8_single(const Q8Product& p, hipStream_t s);
template <>
hipError_t launch_q8_single<DT>(const Q8Product& p, hipStream_t s) {
#define CLASSES(EPI)                                                                             \
  if (p.tile_class == TILE_LARGE) return launch_q8_class<256, 256, 2, 1, EPI>(p, ea, s);         \
  if (p.tile_class == TILE_WIDE) return launch_q8_class<128, 256, 2, 1, EPI>(p, ea, s);          \
  return launch_q8_class<128, 128, 2, 1, EPI>(p, ea, s)
#if GMLP_DT == 0  // (of no type: once is enough)
  if (p.out_f32) {
    EpiQ8Float::Args ea = {(float*)p.out, p.sx, p.sw[0], p.N};
    CLASSES(EpiQ8Float);
  }
#endif
  EpiQ8Store<DT>::Args ea = {(DT*)p.out, p.sx, p.sw[0], (const DT*)p.bias[0], p.N, p.M};
  if (p.splits > 1) return launch_q8_split<1, EpiQ8Store<DT>>(p, ea, s);
  CLASSES(EpiQ8Store<DT>);
#undef CLASSES
}
#endif

}  // namespace gmlp
