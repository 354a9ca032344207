// GatedGemm, QGemm and QGatedGemm for any sizes, alignments and either weight
// layout: the form for inner dimensions that the TMA kernels do not take
// (rows that are no multiple of 16 bytes, [K, N] weights that are not
// constants).
//
//   GatedGemm   y = act(x . Wg) (x . Wu)                     FP32 sums
//   QGemm       y = (q . W) (s[m] ws[n]) + bias[n]           32-bit integer sums
//   QGatedGemm  y = act((q . Wg) (s[m] gs[n])) ((q . Wu) (s[m] us[n]))
//
// 64 x 64 tiles, 256 threads of 4 x 4 outputs, K in chunks of 32 through
// shared memory; 8-bit operands lie there four k to a word (dp4a). FP32 and
// integer units bound it, far below the tensor cores' rate; every access is
// one element, so nothing has to be aligned. The blocks of one column of tiles
// are neighbours in a grid of one dimension (the second one ends at 65535).

#include "product.cuh"

namespace {

using namespace ctb;

constexpr int kTile = 64;
constexpr int kChunk = 32;
constexpr int kThreads = 256;

struct Half {
  using Element = __half;
  using Word = float;  // one k
  using Sum = float;
  static constexpr int kPerWord = 1;
  static __device__ __forceinline__ Word pack(const Element* e) { return __half2float(e[0]); }
  static __device__ __forceinline__ Sum mad(Word a, Word b, Sum c) { return fmaf(a, b, c); }
};
struct Int8 {
  using Element = signed char;
  using Word = int;  // four k
  using Sum = int;
  static constexpr int kPerWord = 4;
  static __device__ __forceinline__ Word pack(const Element* e) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= static_cast<uint32_t>(static_cast<unsigned char>(e[i])) << (8 * i);
    return static_cast<int>(w);
  }
  static __device__ __forceinline__ Sum mad(Word a, Word b, Sum c) { return __dp4a(a, b, c); }
};

// Tile rows r of [rows, K] (row stride `row_step`, k stride `k_step`) into
// words[k word][row].
template <typename T>
__device__ __forceinline__ void stage(typename T::Word (&words)[kChunk / T::kPerWord][kTile + 1],
                                      const typename T::Element* __restrict__ src, long long row0, int rows,
                                      long long row_step, int k0, int k, long long k_step) {
  constexpr int kWords = kChunk / T::kPerWord;
  for (int i = threadIdx.x; i < kTile * kWords; i += kThreads) {
    // Neighbouring threads take neighbouring addresses of either layout.
    const int row = k_step == 1 ? i / kWords : i % kTile;
    const int word = k_step == 1 ? i % kWords : i / kTile;
    typename T::Element e[T::kPerWord];
#pragma unroll
    for (int j = 0; j < T::kPerWord; ++j) {
      const int kk = k0 + word * T::kPerWord + j;
      const bool inside = row0 + row < rows && kk < k;
      e[j] = inside ? src[(row0 + row) * row_step + kk * k_step] : typename T::Element(0);
    }
    words[word][row] = T::pack(e);
  }
}

// First row and column of this block's tile.
__device__ __forceinline__ void tile_origin(int m, long long* m0, long long* n0) {
  const unsigned m_tiles = (static_cast<unsigned>(m) + kTile - 1) / kTile;
  *m0 = static_cast<long long>(blockIdx.x % m_tiles) * kTile;
  *n0 = static_cast<long long>(blockIdx.x / m_tiles) * kTile;
}

template <typename T, int kOperands>
__device__ __forceinline__ void tile_sums(typename T::Sum (&sum)[kOperands][4][4],
                                          const typename T::Element* x, const typename T::Element* const (&w)[kOperands],
                                          int m, int n, int k, int trans_b) {
  constexpr int kWords = kChunk / T::kPerWord;
  __shared__ typename T::Word xs[kWords][kTile + 1];
  __shared__ typename T::Word ws[kOperands][kWords][kTile + 1];
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  long long m0, n0;
  tile_origin(m, &m0, &n0);
#pragma unroll
  for (int o = 0; o < kOperands; ++o)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[o][i][j] = 0;
  for (int k0 = 0; k0 < k; k0 += kChunk) {
    stage<T>(xs, x, m0, m, k, k0, k, 1);
#pragma unroll
    for (int o = 0; o < kOperands; ++o) stage<T>(ws[o], w[o], n0, n, trans_b ? k : 1, k0, k, trans_b ? 1 : n);
    __syncthreads();
#pragma unroll
    for (int kw = 0; kw < kWords; ++kw) {
      typename T::Word a[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = xs[kw][ty + 16 * i];
#pragma unroll
      for (int o = 0; o < kOperands; ++o)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const typename T::Word b = ws[o][kw][tx + 16 * j];
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[o][i][j] = T::mad(a[i], b, sum[o][i][j]);
        }
    }
    __syncthreads();
  }
}

// Calls store(row, column, i, j) for this thread's outputs inside the matrix.
template <typename F>
__device__ __forceinline__ void each_output(int m, int n, F store) {
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  long long m0, n0;
  tile_origin(m, &m0, &n0);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const long long row = m0 + ty + 16 * i, column = n0 + tx + 16 * j;
      if (row < m && column < n) store(row, column, i, j);
    }
}

}  // namespace

extern "C" __global__ void __launch_bounds__(kThreads)
ctb_gated_gemm_f16_any(const __half* x, const __half* w_gate, const __half* w_up, __half* output, int m, int n, int k,
                       int activation, int trans_b, CTB_RESERVED_PARAMS) {
  CTB_UNUSED_RESERVED();
  CTB_GRID_DEPENDENCY_SYNC();
  float sum[2][4][4];
  tile_sums<Half, 2>(sum, x, {w_gate, w_up}, m, n, k, trans_b);
  each_output(m, n, [&](long long row, long long column, int i, int j) {
    output[row * n + column] = __float2half_rn(gated(sum[0][i][j], sum[1][i][j], activation));
  });
}

extern "C" __global__ void __launch_bounds__(kThreads)
ctb_qgemm_i8_any(const signed char* x, const float* x_scale, const signed char* w, const float* w_scale,
                 const __half* bias, __half* output, int m, int n, int k, int trans_b, CTB_RESERVED_PARAMS) {
  CTB_UNUSED_RESERVED();
  CTB_GRID_DEPENDENCY_SYNC();
  int sum[1][4][4];
  tile_sums<Int8, 1>(sum, x, {w}, m, n, k, trans_b);
  each_output(m, n, [&](long long row, long long column, int i, int j) {
    const float b = bias != nullptr ? __half2float(bias[column]) : 0.0f;
    output[row * n + column] = __float2half_rn(dequantized(sum[0][i][j], x_scale[row], w_scale[column], b));
  });
}

extern "C" __global__ void __launch_bounds__(kThreads)
ctb_qgated_gemm_i8_any(const signed char* x, const float* x_scale, const signed char* w_gate, const float* gate_scale,
                       const signed char* w_up, const float* up_scale, __half* output, int m, int n, int k,
                       int activation, int trans_b, CTB_RESERVED_PARAMS) {
  CTB_UNUSED_RESERVED();
  CTB_GRID_DEPENDENCY_SYNC();
  int sum[2][4][4];
  tile_sums<Int8, 2>(sum, x, {w_gate, w_up}, m, n, k, trans_b);
  each_output(m, n, [&](long long row, long long column, int i, int j) {
    const float gate = dequantized(sum[0][i][j], x_scale[row], gate_scale[column], 0.0f);
    const float up = dequantized(sum[1][i][j], x_scale[row], up_scale[column], 0.0f);
    output[row * n + column] = __float2half_rn(gated(gate, up, activation));
  });
}
