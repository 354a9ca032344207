// QuantizeRows: FP16 rows to 8-bit integers with one scale a row.
//
//   s[m] = fl32(max_k |x[m, k]| / 127),  q[m, k] = round_half_even(x[m, k] / s[m])
//
// exactly, i.e. as if the quotient were not rounded before it is rounded to
// an integer. A row of zeros has s = 0 and q = 0. A row that holds an infinity
// or a NaN has s = inf or NaN and q = 0, so that a product with it is NaN.
//
// One pass over HBM (3 bytes an element): a row is read into registers, its
// maximum found, and the integers written from the registers; only rows above
// kCached vectors a thread read their tail again (from L2). Element i of x
// and of q have the same flat index, so a vector of 8 elements that starts at
// a multiple of 8 is 16-byte aligned in x and 8-byte aligned in q whatever
// the row length: rows of odd length move by whole vectors too, and the one
// or two vectors that a row shares with its neighbours element by element.
// Rows of at most 1024 elements take a warp each (eight a block), longer
// ones a block: a block's two barriers cost more than a short row's transfer.

#include "common.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kCached = 4;             // vectors of 8 elements a thread holds: 8192 elements a block
constexpr int kWarpRow = 1024;         // longest row of the warp form (4 vectors a lane)
constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23: adding it rounds to an integer, half to even

// Eight consecutive elements as bits; those outside [begin, end) read as 0.
__device__ __forceinline__ uint4 load_vector(const unsigned short* __restrict__ x, long long at, long long begin,
                                             long long end, bool aligned) {
  if (aligned && at >= begin && at + 8 <= end) return __ldg(reinterpret_cast<const uint4*>(x + at));
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t bits = at + e >= begin && at + e < end ? x[at + e] : 0u;
    w[e / 2] |= bits << (16 * (e & 1));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Largest |x| of each 16-bit half as its bits: magnitudes order like
// integers, infinity above every number and NaN above infinity.
__device__ __forceinline__ uint32_t largest(uint4 v, uint32_t m) {
  m = __vmaxu2(m, v.x & 0x7FFF7FFFu);
  m = __vmaxu2(m, v.y & 0x7FFF7FFFu);
  m = __vmaxu2(m, v.z & 0x7FFF7FFFu);
  return __vmaxu2(m, v.w & 0x7FFF7FFFu);
}

// round_half_even(x / s) from the approximate quotient's rounding q, off by
// at most one. r = x - q s is exact: x and s are multiples of s's last place
// (|x| >= s / 2 here and x has 11 bits to s's 24) and |r| < s.
__device__ __noinline__ float settle(float x, float s, float q) {
  const float r = fmaf(-q, s, x);
  const float twice = 2.0f * fabsf(r);
  const bool odd = fmodf(q, 2.0f) != 0.0f;
  return twice > s || (twice == s && odd) ? q + copysignf(1.0f, r) : q;
}

// Eight integers of one vector, a byte each.
__device__ __forceinline__ uint2 quantize(uint4 v, float s, float inv) {
  const __half2* h = reinterpret_cast<const __half2*>(&v);
  float x[8], t[8];
  float border = 0.0f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 f = __half22float2(h[e]);
    x[2 * e] = f.x;
    x[2 * e + 1] = f.y;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    t[e] = fmaf(x[e], inv, kMagic);
    border = fmaxf(border, fabsf(fmaf(x[e], inv, kMagic - t[e])));
  }
  // inv is off by 2^-24 relative and |x inv| <= 127, so a quotient whose
  // distance to its integer is below 0.5 - 2^-15 is rounded rightly.
  if (border > 0.49996f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = kMagic + settle(x[e], s, t[e] - kMagic);
  }
  // The low byte of t's bits is the integer in two's complement.
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t lo = __byte_perm(__float_as_uint(t[4 * i]), __float_as_uint(t[4 * i + 1]), 0x0040);
    const uint32_t hi = __byte_perm(__float_as_uint(t[4 * i + 2]), __float_as_uint(t[4 * i + 3]), 0x0040);
    w[i] = __byte_perm(lo, hi, 0x5410);
  }
  return make_uint2(w[0], w[1]);
}

__device__ __forceinline__ void store_vector(signed char* __restrict__ q, long long at, long long begin, long long end,
                                             bool aligned, uint2 w) {
  if (aligned && at >= begin && at + 8 <= end) {
    *reinterpret_cast<uint2*>(q + at) = w;
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (at + e >= begin && at + e < end) q[at + e] = static_cast<signed char>((e < 4 ? w.x : w.y) >> (8 * (e & 3)));
  }
}

// One row by `kLanes` threads (a warp or the block), `lane` of them this one.
template <int kLanes>
__device__ __forceinline__ void quantize_row(const unsigned short* __restrict__ x, signed char* __restrict__ q,
                                             float* __restrict__ scale, long long row, int columns, int lane,
                                             bool aligned, uint32_t* shared) {
  const long long begin = row * columns, end = begin + columns;
  const long long first = begin & ~7ll;
  const int vectors = static_cast<int>((end - first + 7) >> 3);
  uint4 v[kCached];
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < kCached; ++j) {
    const int i = j * kLanes + lane;
    v[j] = i < vectors ? load_vector(x, first + 8ll * i, begin, end, aligned) : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int j = 0; j < kCached; ++j) m = largest(v[j], m);
  for (int i = kCached * kLanes + lane; i < vectors; i += kLanes) {
    m = largest(load_vector(x, first + 8ll * i, begin, end, aligned), m);
  }
  m = max(m & 0xFFFFu, m >> 16);
  m = __reduce_max_sync(0xFFFFFFFFu, m);
  if (kLanes > 32) {
    __syncthreads();  // the previous row's readers are done with `shared`
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x / 32] = m;
    __syncthreads();
    m = __reduce_max_sync(0xFFFFFFFFu, shared[threadIdx.x & (kWarps - 1)]);
  }
  const float amax = __half2float(__ushort_as_half(static_cast<unsigned short>(m)));
  const float s = __fdiv_rn(amax, 127.0f);
  if (lane == 0) scale[row] = s;
  const bool regular = m != 0 && m < 0x7C00u;
  const float inv = regular ? __fdiv_rn(1.0f, s) : 0.0f;
#pragma unroll
  for (int j = 0; j < kCached; ++j) {
    const int i = j * kLanes + lane;
    if (i < vectors) {
      store_vector(q, first + 8ll * i, begin, end, aligned, regular ? quantize(v[j], s, inv) : make_uint2(0, 0));
    }
  }
  for (int i = kCached * kLanes + lane; i < vectors; i += kLanes) {
    const uint4 again = load_vector(x, first + 8ll * i, begin, end, aligned);
    store_vector(q, first + 8ll * i, begin, end, aligned, regular ? quantize(again, s, inv) : make_uint2(0, 0));
  }
}

}  // namespace

extern "C" __global__ void __launch_bounds__(kThreads)
ctb_quantize_rows_f16(const unsigned short* x, signed char* q, float* scale, int rows, int columns,
                      CTB_RESERVED_PARAMS) {
  CTB_UNUSED_RESERVED();
  CTB_GRID_DEPENDENCY_SYNC();
  __shared__ uint32_t shared[kWarps];
  const bool aligned = ctb::aligned16(x) && (reinterpret_cast<uintptr_t>(q) & 7u) == 0;
  if (columns <= kWarpRow) {
    const int stride = gridDim.x * kWarps;
    for (int row = blockIdx.x * kWarps + threadIdx.x / 32; row < rows; row += stride) {
      quantize_row<32>(x, q, scale, row, columns, threadIdx.x & 31, aligned, shared);
    }
    return;
  }
  for (int row = blockIdx.x; row < rows; row += gridDim.x) {
    quantize_row<kThreads>(x, q, scale, row, columns, threadIdx.x, aligned, shared);
  }
}
